"""The operators that train a network's matrices and its head over discretised actions: what is measured of them.

* ``orthogonalize``: a quintic Newton-Schulz iteration that moves a matrix's singular values towards one;
* ``muon_step``: momentum, orthogonalisation and update of a list of weight matrices;
* ``linear_cross_entropy``: softmax cross entropy of ``hidden @ weight.T + bias`` with its gradients, without the logits.

Each has a plain form in elementary torch operations here, in 32 bits, beside the call a user's program makes."""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1
IGNORE = -100
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

#: the weight matrices of the [512, 256, 128] residual network of the offline-RL configurations (17 state and 6 action
#: dimensions, 32 time features)
NET = ("32x17,128x64,128x128,512x6,512x128,512x512,512x6,256x512,256x128,256x256,256x512,128x256,128x128,128x128,"
       "128x256,128x128,128x128,128x128,256x256,256x128,256x256,512x512,512x128,512x512,6x1024")


def _blocks(layers, width):
    """The matrices of `layers` blocks of four width x width products and a four times wider pair."""
    return ",".join(["%dx%d" % (width, width)] * 4 * layers + ["%dx%d" % (4 * width, width), "%dx%d" % (width, 4 * width)] * layers)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def listed():
    return [
        # the gradient of one narrow layer: the smallest call there is, all latency
        {"name": "orth 128x64 fp32", "op": "orth", "batch": 1, "rows": 128, "cols": 64, "dtype": "fp32"},
        # a wide layer whose gradient comes in half precision
        {"name": "orth 1024x1024 bf16", "op": "orth", "batch": 1, "rows": 1024, "cols": 1024, "dtype": "bf16"},
        # three gradients of one odd shape, more rows than columns
        {"name": "orth 3x1000x777 fp32", "op": "orth", "batch": 3, "rows": 1000, "cols": 777, "dtype": "fp32"},
        # one matrix of a large network
        {"name": "orth 2048x4096 fp32", "op": "orth", "batch": 1, "rows": 2048, "cols": 4096, "dtype": "fp32"},
        # the optimiser step of the framework's own benchmark network: many small matrices
        {"name": "muon 25 small", "op": "muon", "shapes": NET},
        # the optimiser step of four wide blocks
        {"name": "muon 24 wide", "op": "muon", "shapes": _blocks(4, 1024)},
        # the log-probability of one token: serving, bound by reading the weight once
        {"name": "token bf16", "op": "ce", "rows": 1, "hidden": 1024, "vocab": 32000, "dtype": "bf16", "train": False, "bias": False, "ignored": 0.0},
        # a scored batch, odd vocabulary, no gradient
        {"name": "score bf16 odd", "op": "ce", "rows": 2000, "hidden": 1024, "vocab": 50257, "dtype": "bf16", "train": False, "bias": False, "ignored": 0.1},
        # the batch of the reference configurations on a discretised action head with invalid actions masked
        {"name": "train fp32 small", "op": "ce", "rows": 4096, "hidden": 128, "vocab": 1024, "dtype": "fp32", "train": True, "bias": True, "ignored": 0.0},
        {"name": "train fp32 odd", "op": "ce", "rows": 1500, "hidden": 1000, "vocab": 32001, "dtype": "fp32", "train": True, "bias": False, "ignored": 0.25},
        # a padded batch, a third of the rows ignored
        {"name": "train bf16 padded", "op": "ce", "rows": 4096, "hidden": 512, "vocab": 16384, "dtype": "bf16", "train": True, "bias": True, "ignored": 0.33},
        # the largest
        {"name": "train bf16 large", "op": "ce", "rows": 8192, "hidden": 2048, "vocab": 65536, "dtype": "bf16", "train": True, "bias": False, "ignored": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("orth", "orth", "muon", "ce", "ce", "ce"))
    if kind == "orth":
        batch, rows, cols = rng.choice((1, 1, 2, 4)), _log(rng, 2, 4096), _log(rng, 2, 4096)
        while batch * min(rows, cols) ** 2 * max(rows, cols) > 2048 * 2048 * 4096:
            rows, cols = max(1, rows // 2), max(1, cols // 2)
        return {"op": "orth", "batch": batch, "rows": rows, "cols": cols, "dtype": rng.choice(("fp32", "bf16", "fp16"))}
    if kind == "muon":
        width, count = _log(rng, 16, 1024), rng.randint(2, 24)
        sides = [max(1, width // 4), width // 2 + 1, width, width]
        return {"op": "muon", "shapes": ",".join("%dx%d" % (rng.choice(sides), rng.choice(sides)) for _ in range(count))}
    train = rng.random() < 0.7
    rows, hidden, vocab = _log(rng, 1, 8192), _log(rng, 32, 2048), _log(rng, 100, 131072)
    while rows * hidden * vocab > 8192 * 2048 * 65536 or rows * vocab > 8192 * 65536:
        rows, vocab = max(1, rows // 2), max(100, vocab * 3 // 4)
    return {"op": "ce", "rows": rows, "hidden": hidden, "vocab": vocab, "dtype": rng.choice(("fp32", "bf16", "bf16", "fp16")),
            "train": train, "bias": rng.random() < 0.4, "ignored": rng.choice((0.0, 0.1, 0.5))}


def _gradient(gen, dev, rows, cols):
    """What the gradient of a linear layer looks like: a product over a batch with a decaying spectrum, and noise."""
    rank = max(1, min(rows, cols, 512) // 2)
    left = torch.randn(rows, rank, generator=gen, device=dev) * torch.logspace(0, -1, rank, device=dev)
    g = left @ torch.randn(rank, cols, generator=gen, device=dev) / math.sqrt(rank)
    return (g + 0.1 * torch.randn(rows, cols, generator=gen, device=dev)) * 1e-3


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case}
    if case["op"] == "orth":
        g = torch.stack([_gradient(gen, dev, case["rows"], case["cols"]) for _ in range(case["batch"])])
        state["matrices"] = g.to(DTYPES[case["dtype"]])
    elif case["op"] == "muon":
        shapes = _shapes(case)
        total = sum(r * c for r, c in shapes)
        flat = [torch.zeros(total, device=dev) for _ in range(3)]      # one buffer of parameters, gradients, momentum
        views, at = [[], [], []], 0
        for r, c in shapes:
            values = (torch.randn(r, c, generator=gen, device=dev) / math.sqrt(c), _gradient(gen, dev, r, c),
                      0.3 * _gradient(gen, dev, r, c))
            for f, v, x in zip(flat, views, values):
                v.append(f[at:at + r * c].view(r, c))
                v[-1].copy_(x)
            at += r * c
        state.update(flat=flat, params=views[0], grads=views[1], buffers=views[2])
    else:
        n, h, v, dtype = case["rows"], case["hidden"], case["vocab"], DTYPES[case["dtype"]]
        hidden = torch.randn(n, h, generator=gen, device=dev).to(dtype)
        weight = (torch.randn(v, h, generator=gen, device=dev) * (2.0 / math.sqrt(h))).to(dtype)
        target = torch.randint(0, v, (n,), generator=gen, device=dev)
        row_weight = torch.rand(n, generator=gen, device=dev) * 2.0    # exp(advantage / temperature) in use
        bias = None
        if case["bias"]:                                               # a tenth of the actions is not allowed
            bias = 0.5 * torch.randn(v, generator=gen, device=dev)
            bias[torch.rand(v, generator=gen, device=dev) < 0.1] = -math.inf
            bias[target] = 0.0
            bias = bias.to(dtype)
        target[torch.rand(n, generator=gen, device=dev) < case["ignored"]] = IGNORE
        if case["train"]:
            hidden.requires_grad_()
            weight.requires_grad_()
            if bias is not None:
                bias.requires_grad_()
        state.update(hidden=hidden, weight=weight, target=target, bias=bias, row_weight=row_weight)
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        return {"orth": _own_orth, "muon": _own_muon, "ce": _own_ce}[op](state)
    return {"orth": _plain_orth, "muon": _plain_muon, "ce": _plain_ce}[op](state)


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own_orth(state):
    from generativerl_preview_amd.optim import orthogonalize
    return orthogonalize(state["matrices"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)


def _own_muon(state):
    from generativerl_preview_amd.optim import muon_step
    muon_step(state["params"], state["grads"], state["buffers"], lr=LR, momentum=MOMENTUM, nesterov=True,
              weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, adjust_lr="original")
    return state["flat"][0], state["flat"][2]


def _own_ce(state):
    from generativerl_preview_amd.generative_models.model_functions import linear_cross_entropy
    args = state["hidden"], state["weight"], state["target"]
    if not state["case"]["train"]:
        return linear_cross_entropy(*args, bias=state["bias"], ignore_index=IGNORE, reduction="none")
    loss = linear_cross_entropy(*args, bias=state["bias"], row_weight=state["row_weight"], ignore_index=IGNORE, reduction="mean")
    leaves = [t for t in (state["hidden"], state["weight"], state["bias"]) if t is not None]
    return [loss.detach(), *torch.autograd.grad(loss, leaves)]


# ----------------------------------------------------------------------------------------------------- the plain forms
def _newton_schulz(g):
    """(..., m, n) in 32 bits; the norm, a long sum on which every later product depends, in 64."""
    a, b, c = COEFFICIENTS
    wide = g.shape[-2] <= g.shape[-1]
    x = g if wide else g.transpose(-1, -2)
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp(min=EPS)
    x = (x / norm.float()).contiguous()
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x if wide else x.transpose(-1, -2)


def _plain_orth(state):
    g = state["matrices"]
    return _newton_schulz(g.float()).to(g.dtype).contiguous()


def _plain_muon(state):
    for p, g, buf in zip(state["params"], state["grads"], state["buffers"]):
        buf.mul_(MOMENTUM).add_(g, alpha=1.0 - MOMENTUM)
        update = _newton_schulz((1.0 - MOMENTUM) * g + MOMENTUM * buf)
        p.mul_(1.0 - LR * DECAY).add_(update, alpha=-LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1])))
    return state["flat"][0], state["flat"][2]


@torch.no_grad()
def _plain_ce(state):
    hidden, weight, target = state["hidden"], state["weight"], state["target"]
    h, w = hidden.float(), weight.float()
    z = h @ w.t()
    if state["bias"] is not None:
        z += state["bias"].float()
    kept = target != IGNORE
    at = target.clamp(min=0).unsqueeze(1)
    picked = z.gather(1, at).squeeze(1)
    top = z.max(1, keepdim=True).values
    z.sub_(top).exp_()
    total = z.sum(1, keepdim=True)
    loss = torch.where(kept, total.log().squeeze(1) + top.squeeze(1) - picked, 0.0)
    if not state["case"]["train"]:
        return loss
    scale = torch.where(kept, state["row_weight"], 0.0) / kept.sum().clamp(min=1)
    z.div_(total)
    z.scatter_add_(1, at, torch.full_like(z[:, :1], -1.0))
    z.mul_(scale.unsqueeze(1))
    out = [(loss * scale).sum(), (z @ w).to(hidden.dtype), (z.t() @ h).to(weight.dtype)]
    if state["bias"] is not None:
        out.append(z.sum(0).to(state["bias"].dtype))
    return out


# ------------------------------------------------------------------------------------------------------ what it costs
def _orth_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3 * m * m * n + m ** 3)          # two symmetric products (half of each is enough) and one full one


def work(case):
    if case["op"] == "orth":
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": 2 * size * case["batch"] * case["rows"] * case["cols"],
                "flops": case["batch"] * _orth_flops(case["rows"], case["cols"])}
    if case["op"] == "muon":
        shapes = _shapes(case)
        return {"bytes": 20 * sum(r * c for r, c in shapes), "flops": sum(_orth_flops(r, c) for r, c in shapes)}
    n, h, v, size = case["rows"], case["hidden"], case["vocab"], DTYPES[case["dtype"]].itemsize
    touched = n * h + v * h + (v if case["bias"] else 0)
    return {"bytes": size * touched * (2 if case["train"] else 1) + 12 * n, "flops": (6 if case["train"] else 2) * n * h * v}


# ------------------------------------------------------------------------------------------------- the same in 64 bits
def _polar(g):
    """The iteration by its definition, on rows x columns as they are, in 64 bits."""
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / max(float(torch.linalg.vector_norm(x)), EPS)
    for _ in range(STEPS):
        s = torch.mm(x, x.t())
        x = COEFFICIENTS[0] * x + COEFFICIENTS[1] * torch.mm(s, x) + COEFFICIENTS[2] * torch.mm(s, torch.mm(s, x))
    return x.t() if tall else x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orth":
        return torch.stack([_polar(g) for g in state["matrices"]])
    if case["op"] == "muon":
        new, kept = [], []
        for p, g, buf in zip(state["params"], state["grads"], state["buffers"]):
            g, buf = g.double(), buf.double()
            buf = MOMENTUM * buf + (1.0 - MOMENTUM) * g
            rate = LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            new.append((p.double() * (1.0 - LR * DECAY) - rate * _polar((1.0 - MOMENTUM) * g + MOMENTUM * buf)).reshape(-1))
            kept.append(buf.reshape(-1))
        return torch.cat(new), torch.cat(kept)
    with torch.no_grad():
        w, target = state["weight"].double(), state["target"]
        bias = None if state["bias"] is None else state["bias"].double()
        count = max(1, int((target != IGNORE).sum()))
        loss = torch.zeros(case["rows"], dtype=torch.float64, device=w.device)
        dh, dw = [], torch.zeros_like(w)
        db = torch.zeros(case["vocab"], dtype=torch.float64, device=w.device)
        for lo in range(0, case["rows"], 2048):
            h, t = state["hidden"][lo:lo + 2048].double(), target[lo:lo + 2048]
            here = torch.nonzero(t != IGNORE).squeeze(1)
            z = torch.mm(h, w.t())
            z = z if bias is None else z + bias
            logp = torch.log_softmax(z, 1)
            loss[lo + here] = -logp[here, t[here]]
            if case["train"]:
                d = torch.exp(logp)
                d[here, t[here]] -= 1.0
                scale = torch.zeros(len(t), dtype=torch.float64, device=w.device)
                scale[here] = state["row_weight"][lo + here].double() / count
                d *= scale.unsqueeze(1)
                dh.append(torch.mm(d, w))
                dw += torch.mm(d.t(), h)
                db += d.sum(0)
        if not case["train"]:
            return loss
        total = (loss * state["row_weight"].double()).sum() / count
        return [total, torch.cat(dh), dw] + ([db] if bias is not None else [])
