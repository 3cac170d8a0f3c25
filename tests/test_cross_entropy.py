"""linear_cross_entropy (grlhip_linear_ce_forward / _backward) against the formulas in 64 bits.

Tolerances, entry by entry, from the arithmetic (K features, N rows, u the half step of a type: finfo.eps / 2):
  z:  16-bit operands are multiplied exactly, fp32 ones as two fp16 pieces (2^-21 of |h| |w|); the matrix core adds blocks of
      16 products in fp32: (K / 16 + 16) 2^-24 of sum_k |h| |w|.
  loss: the largest error of z in the row twice (logsumexp and the target), 2^-21 of the magnitudes for exp, log and sums.
  D = softmax - onehot: twice the error of z and exp's own |z - lse| 2^-22 relative to the softmax, then the rounding of D
      (bf16 operands: u of fp16; others: 2^-21 for two pieces; 2^-38 absolute for fp16's smallest numbers).
  dh, dW: these times |W|, |h|; the fp32 sum over V or N; the result's own rounding (u, and fp16's smallest number)."""
import ctypes
import math

import pytest
import torch

from generativerl_preview_amd import _lib as L
from generativerl_preview_amd.generative_models.model_functions import linear_cross_entropy

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def inputs(n, k, v, dtype, seed=0, bias=True, weights=True, ignored=0.2):
    gen = torch.Generator().manual_seed(seed)
    h = torch.randn(n, k, generator=gen).to(dtype).to(DEV)
    w = (torch.randn(v, k, generator=gen) * 2 / math.sqrt(k)).to(dtype).to(DEV)
    t = torch.randint(0, v, (n,), generator=gen)
    b = None
    if bias:
        b = 0.5 * torch.randn(v, generator=gen)
        b[torch.rand(v, generator=gen) < 0.2] = -math.inf
        b[t] = 0.25
        b = b.to(DEV)
    t[torch.rand(n, generator=gen) < ignored] = -100
    rw = None
    if weights:
        rw = torch.rand(n, generator=gen) * 3
        rw[torch.rand(n, generator=gen) < 0.1] = 0.0
        rw = rw.to(DEV)
    return h, w, t.to(DEV), b, rw


def oracle(h, w, t, b, rw, reduction, upstream=None):
    """Everything in 64 bits, and the entrywise tolerances: {name: (value, tolerance)}."""
    n, k = h.shape
    kind = h.dtype
    H, W = h.detach().double(), w.detach().double()
    kept = (t != -100) & (torch.ones_like(t, dtype=torch.bool) if rw is None else rw != 0)
    H = torch.where(kept.unsqueeze(1), H, 0.0)
    z = H @ W.t()
    reach = H.abs() @ W.abs().t()
    if b is not None:
        z = z + b.detach().double()
    lse = torch.logsumexp(z, 1)
    at = t.clamp(min=0).unsqueeze(1)
    picked = z.gather(1, at).squeeze(1)
    weight = torch.where(kept, torch.ones(n, dtype=torch.float64, device=h.device) if rw is None else rw.double(), 0.0)
    losses = torch.where(kept, (lse - picked) * weight, 0.0)
    finite = torch.where(z.isfinite(), z, 0.0).abs()
    ez = ((k / 16 + 16) * 2.0 ** -24 + (2.0 ** -21 if kind == F32 else 0.0)) * reach + 2.0 ** -23 * finite
    e_row = ez.max(1).values
    e_loss = torch.where(kept, weight * (2 * e_row + 2.0 ** -21 * (1 + lse.abs() + picked.abs())), 0.0)
    count = max(1, int((t != -100).sum()))
    out = {"losses": (losses, e_loss)}
    total = losses.sum() / (count if reduction == "mean" else 1)
    out["total"] = (total, e_loss.sum() / (count if reduction == "mean" else 1) + 2.0 ** -23 * total.abs())
    g = weight * (torch.ones(n, dtype=torch.float64, device=h.device) if upstream is None else upstream.double())
    if reduction == "mean":
        g = g / count
    p = torch.exp(z - lse.unsqueeze(1))
    ep = p * (2 * e_row.unsqueeze(1) + (torch.where(z.isfinite(), (z - lse.unsqueeze(1)).abs(), 0.0) + 2) * 2.0 ** -22)
    d = p.clone()
    d.scatter_add_(1, at, torch.full_like(d[:, :1], -1.0))
    u = torch.finfo(F16).eps / 2 if kind == BF16 else 2.0 ** -21
    ed = ep + u * d.abs() + 2.0 ** -38
    d, ed = torch.where(kept.unsqueeze(1), d, 0.0), torch.where(kept.unsqueeze(1), ed, 0.0)
    g = torch.where(kept, g, 0.0)
    uo = torch.finfo(kind).eps / 2
    least = 2.0 ** -25 if kind == F16 else 0.0
    v = w.shape[0]
    dh = (d @ W) * g.unsqueeze(1)
    edh = (ed + (v / 16 + 16 + 64) * 2.0 ** -24 * d.abs()) @ W.abs() * g.abs().unsqueeze(1)
    gd, egd = d * g.unsqueeze(1), (ed + (n / 16 + 16 + 64) * 2.0 ** -24 * d.abs()) * g.abs().max()
    egd = torch.where(kept.unsqueeze(1), (ep + u * d.abs() + (n / 16 + 80) * 2.0 ** -24 * d.abs()) * g.abs().unsqueeze(1)
                      + 2.0 ** -37 * g.abs().max(), 0.0)
    dw = gd.t() @ H
    edw = egd.t() @ H.abs()
    out["dh"] = (dh, edh + uo * (dh.abs() + edh) + 2.0 ** -21 * dh.abs() + least)
    out["dw"] = (dw, edw + uo * (dw.abs() + edw) + 2.0 ** -21 * dw.abs() + least)
    db = gd.sum(0)
    out["db"] = (db, ((ep + d.abs() * (n * 2.0 ** -24 + 2.0 ** -21)) * g.abs().unsqueeze(1)).sum(0))
    return out


def near(got, name, out):
    want, tol = out[name]
    gap = (got.double() - want).abs()
    assert got.shape == want.shape and bool(got.isfinite().all()), name
    worst = float((gap - tol).max()) if gap.numel() else 0.0
    assert worst <= 0.0, "%s: off by up to %.3g beyond the tolerance (largest gap %.3g)" % (name, worst, float(gap.max()))


SIZES = [(1, 1, 1), (1, 64, 100), (2, 3, 2), (3, 5, 7), (64, 64, 64), (65, 63, 129), (128, 128, 1000), (200, 100, 333), (257, 192, 1030),
         (33, 512, 3001), (500, 40, 257), (1, 1000, 5000), (17, 256, 4099)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_gpu_loss_and_gradients_match_64_bits(size, dtype):
    h, w, t, b, rw = inputs(*size, dtype)
    leaves = [h.requires_grad_(), w.requires_grad_(), b.requires_grad_()]
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw, reduction=reduction)
        up = None
        if reduction == "none":
            up = torch.linspace(-1, 2, size[0], device=DEV)
        out = oracle(h, w, t, b, rw, reduction, up)
        assert loss.dtype == F32
        near(loss.detach(), "losses" if reduction == "none" else "total", out)
        dh, dw, db = torch.autograd.grad(loss, leaves, grad_outputs=up)
        assert (dh.dtype, dw.dtype, db.dtype) == (dtype, dtype, F32)
        near(dh, "dh", out)
        near(dw, "dw", out)
        near(db, "db", out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_forward_without_a_gradient_is_the_same_loss(dtype):
    h, w, t, b, rw = inputs(77, 128, 2049, dtype, seed=3)
    a = linear_cross_entropy(h, w, t, bias=b, row_weight=rw, reduction="none")
    assert not a.requires_grad
    near(a, "losses", oracle(h, w, t, b, rw, "none"))
    plain = linear_cross_entropy(h, w, t, ignore_index=-100, reduction="none")
    near(plain, "losses", oracle(h, w, t, None, None, "none"))
    # a batch of any shape
    c = linear_cross_entropy(h.view(7, 11, 128), w, t.view(7, 11), bias=b, row_weight=rw.view(7, 11), reduction="none")
    assert c.shape == (7, 11) and torch.equal(c.view(-1), a)
    one = linear_cross_entropy(h[0], w, t[0].clamp(min=0), bias=b, reduction="none")
    assert one.shape == ()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_each_gradient_alone(dtype):
    """What is not asked for is not computed; the rest is the same, bit for bit."""
    for size in ((150, 72, 333), (40, 128, 5000)):
        h, w, t, b, rw = inputs(*size, dtype, seed=41)
        leaves = [h.requires_grad_(), w.requires_grad_(), b.requires_grad_()]
        want = torch.autograd.grad(linear_cross_entropy(*leaves[:2], t, bias=b, row_weight=rw), leaves)
        for chosen in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
            some = [x.detach().requires_grad_(k in chosen) for k, x in enumerate(leaves)]
            loss = linear_cross_entropy(*some[:2], t, bias=some[2], row_weight=rw)
            for g, k in zip(torch.autograd.grad(loss, [some[k] for k in chosen]), chosen):
                assert torch.equal(g, want[k]), (size, chosen, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_pieces_of_the_vocabulary(dtype):
    """More rows than one piece of the vocabulary holds entries for: the gradients are added up over the pieces."""
    n, k, v = 50000, 64, 5000
    h, w, t, b, rw = inputs(n, k, v, dtype, seed=5)
    leaves = [h.requires_grad_(), w.requires_grad_(), b.requires_grad_()]
    loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw)
    grads = torch.autograd.grad(loss, leaves)
    out = oracle(h, w, t, b, rw, "mean")
    near(loss.detach(), "total", out)
    for g, name in zip(grads, ("dh", "dw", "db")):
        near(g, name, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_a_vocabulary_that_is_packed_in_pieces(dtype):
    """A weight that has to be laid out anew (its rows are no whole K blocks), larger than one piece of it, few rows."""
    h, w, t, b, rw = inputs(3, 2001, 70000, dtype, seed=6, ignored=0.0)
    h.requires_grad_(), w.requires_grad_()
    t[2] = 69999
    b[69999] = 0.0
    loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw, reduction="sum")
    out = oracle(h, w, t, b, rw, "sum")
    near(loss.detach(), "total", out)
    for g, name in zip(torch.autograd.grad(loss, [h, w]), ("dh", "dw")):
        near(g, name, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_padding_may_hold_anything(dtype):
    """Infinities and NaN in ignored rows, and in rows of weight 0, reach nothing."""
    h, w, t, b, rw = inputs(130, 64, 300, dtype, seed=6)
    t[5], t[77], t[9] = -100, -100, 3
    rw[9] = 0.0
    clean = [x.clone() for x in (h, w)]
    want = linear_cross_entropy(clean[0].requires_grad_(), clean[1].requires_grad_(), t, bias=b, row_weight=rw)
    want_g = torch.autograd.grad(want, clean)
    h[5], h[77], h[9] = math.nan, math.inf, -math.inf
    got = linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), t, bias=b, row_weight=rw)
    got_g = torch.autograd.grad(got, [h, w])
    assert torch.equal(got, want)
    assert torch.equal(got_g[1], want_g[1])
    assert torch.equal(got_g[0], want_g[0]) and not got_g[0][[5, 77, 9]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("features", [64, 7, 3])
def test_gpu_large_numbers_in_padding_cost_the_others_nothing(features, dtype):
    """Finite ones, in ignored rows, rows of weight 0 and masked rows of the vocabulary: they must not set the operands' scale."""
    h, w, t, b, rw = inputs(130, features, 301, dtype, seed=16)
    t[5], t[77], t[9] = -100, -100, 3
    rw[9] = 0.0
    b[[4, 300]] = -math.inf
    t[(t == 4) | (t == 300)] = 3
    b[3] = 0.0
    gone = (b == -math.inf).nonzero()[0, 0].item(), 300
    huge = 6e4 if dtype == F16 else 1e30
    first = [x.clone() for x in (h, w)]
    second = [x.clone() for x in (h, w)]
    second[0][[5, 77, 9]] = huge
    second[1][[gone[0], gone[1]]] = torch.where(torch.arange(features, device=DEV) % 2 == 0, huge, -huge).to(dtype)
    for layout in (lambda x: x, lambda x: x.t().contiguous().t()):
        results = []
        for hh, ww in (first, second):
            leaves = [layout(hh).requires_grad_(), layout(ww).requires_grad_()]
            loss = linear_cross_entropy(*leaves, t, bias=b, row_weight=rw)
            results.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
        for got, want in zip(results[1], results[0]):
            assert torch.equal(got, want)
        near(results[1][0], "total", oracle(h, w, t, b, rw, "mean"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("features", [64, 128, 65])
def test_gpu_masked_entries_may_hold_anything(features, dtype):
    """The type's largest numbers, whose products leave fp32's range, infinities and NaN in masked rows of the weight reach nothing, whether
    the weight is read where it lies (16-bit rows of whole K blocks) or laid out anew."""
    h, w, t, b, rw = inputs(100, features, 300, dtype, seed=33)
    b[[4, 299]] = -math.inf
    t[(t == 4) | (t == 299)] = 3
    b[3] = 0.0
    signs = torch.where(torch.arange(features, device=DEV) % 2 == 0, 1.0, -1.0)
    results = []
    for fill in (0.0, torch.finfo(dtype).max, math.inf, math.nan):
        x, y, bias = h.clone().requires_grad_(), w.clone(), b.clone().requires_grad_()
        y[[4, 299]] = (signs * fill if math.isfinite(fill) else signs + fill).to(dtype)
        y.requires_grad_()
        loss = linear_cross_entropy(x, y, t, bias=bias, row_weight=rw)
        results.append([loss.detach(), *torch.autograd.grad(loss, [x, y, bias])])
    for got in results:
        assert all(bool(g.isfinite().all()) for g in got)
        assert all(torch.equal(g, want) for g, want in zip(got, results[0]))
    near(results[0][0], "total", oracle(h, w, t, b, rw, "mean"))


@pytest.mark.gpu
def test_gpu_all_rows_ignored_and_no_rows():
    h, w, t, b, rw = inputs(40, 64, 90, BF16)
    t.fill_(-100)
    loss = linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), t, bias=b.requires_grad_())
    grads = torch.autograd.grad(loss, [h, w, b])
    assert float(loss.detach()) == 0.0 and not any(g.any() for g in grads)
    e = h[:0].detach().requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(e, w, t[:0], bias=b, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ())
        gw, gb = torch.autograd.grad(loss.sum(), [w, b])
        assert not gw.any() and not gb.any()
    assert linear_cross_entropy(h[:0].detach(), w.detach(), t[:0], reduction="none").shape == (0,)


@pytest.mark.gpu
def test_gpu_masks_and_bad_targets():
    h, w, t, _, _ = inputs(70, 64, 200, F32, bias=False, weights=False, ignored=0.0)
    low = torch.zeros(200, device=DEV)
    low[::2] = torch.finfo(F32).min          # masked by the type's lowest value: the same as -inf
    t = (t // 2 * 2 + 1) % 200
    inf = torch.where(low < 0, -math.inf, low)
    a, b = (linear_cross_entropy(h, w, t, bias=x, reduction="none") for x in (low, inf))
    assert torch.equal(a, b)
    near(a, "losses", oracle(h, w, t, inf, None, "none"))
    # a masked target: an infinite loss, and still a finite gradient
    w.requires_grad_()
    t2 = t.clone()
    t2[3] = 0
    loss = linear_cross_entropy(h, w, t2, bias=inf, reduction="none")
    assert float(loss[3].detach()) == math.inf and bool(loss[torch.arange(70, device=DEV) != 3].isfinite().all())
    (g,) = torch.autograd.grad(loss, [w], grad_outputs=torch.ones_like(loss))
    assert bool(g.isfinite().all())
    # everything masked: NaN, in the loss and in the gradient
    assert bool(linear_cross_entropy(h, w.detach(), t, bias=torch.full_like(low, -math.inf), reduction="none").isnan().all())
    # targets outside the vocabulary that are not ignore_index: NaN in their rows only; the weight's gradient says it too
    for bad in (200, -1, 1 << 40):
        t3 = t.clone()
        t3[11] = bad
        loss = linear_cross_entropy(h, w, t3, reduction="none")
        assert bool(loss[11].isnan()) and int(loss.isnan().sum()) == 1
        (g,) = torch.autograd.grad(loss.sum(), [w])
        assert bool(g.isnan().any())
        assert bool(linear_cross_entropy(h, w, t3, ignore_index=bad, reduction="none").isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_strides_and_alignment(dtype):
    """Transposed, sliced, misaligned and broadcast operands give what their dense copies give."""
    h, w, t, b, rw = inputs(90, 128, 210, dtype, seed=8)
    wide = torch.randn(90, 300, device=DEV).to(dtype)
    cases = [(h.t().contiguous().t(), w), (h, w.t().contiguous().t()), (wide[:, 7:135], w), (wide[:, ::2][:, :128], w),
             (h[:1].expand(90, 128), w), (h, w[:1].expand(210, 128)), (h, torch.cat([w, w], 1)[:, 128:]), (h, w.repeat(2, 1)[::2])]
    for x, y in cases:
        dense = x.contiguous().detach().requires_grad_(), y.contiguous().detach().requires_grad_()
        want = linear_cross_entropy(*dense, t, bias=b, row_weight=rw)
        wg = torch.autograd.grad(want, dense)
        odd = x.detach().requires_grad_(), y.detach().requires_grad_()
        got = linear_cross_entropy(*odd, t, bias=b, row_weight=rw)
        gg = torch.autograd.grad(got, odd)
        assert torch.equal(got, want) and all(torch.equal(p, q) for p, q in zip(gg, wg))
    # target and weights of other types and strides
    a = linear_cross_entropy(h, w, t, bias=b, row_weight=rw)
    t2 = torch.stack([t, t], 1)[:, 0]
    r2 = torch.stack([rw, rw], 1)[:, 1].double()
    b2 = torch.stack([b, b], 1)[:, 0].double()
    assert torch.equal(linear_cross_entropy(h, w, t2.int(), bias=b2, row_weight=r2), a)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-20, 1e15])
def test_gpu_fp32_operands_of_any_magnitude(scale):
    """The two-piece products follow the operands' magnitudes: small and large factors that cancel change little."""
    h, w, t, b, rw = inputs(64, 96, 150, F32, seed=9)
    h, w = (h * scale).requires_grad_(), (w / scale).requires_grad_()
    loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw)
    out = oracle(h, w, t, b, rw, "mean")
    near(loss.detach(), "total", out)
    for g, name in zip(torch.autograd.grad(loss, [h, w]), ("dh", "dw")):
        near(g, name, out)


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [1e6, 1e9])
def test_gpu_rows_of_very_different_magnitudes(ratio):
    """One row of hidden and one of the weight that count and are `ratio` times the others: in fp32 their size is their own matter.  The logits'
    error is the products' (2^-21 and the sums', entry by entry) and the pieces' ends, 2^-38 of the largest entry of the ROW; softmax of
    logits that are off by at most e lies between those of z_v + e_v against z_u - e_u and the reverse.  The gradients' operands end at
    2^-25 of their scaled values, half of the rows' exponents taken by D."""
    h, w, t, b, rw = inputs(130, 256, 300, F32, seed=21, ignored=0.1)
    n, k, v = 130, 256, 300
    t[7], rw[7], b[11], b[12] = 12, 1.5, 0.25, 0.25
    h[7] *= ratio
    w[11] *= ratio
    leaves = [h.requires_grad_(), w.requires_grad_()]
    loss = linear_cross_entropy(*leaves, t, bias=b, row_weight=rw, reduction="none")
    total = linear_cross_entropy(*leaves, t, bias=b, row_weight=rw, reduction="sum")
    dh, dw = torch.autograd.grad(total, leaves)
    H, W, B = h.detach().double(), w.detach().double(), b.double()
    kept = (t != -100) & (rw != 0)
    z = H @ W.t() + B
    open_ = z > -math.inf
    hm, wm = H.abs().max(1, keepdim=True).values, W.abs().max(1, keepdim=True).values
    ez = ((k / 16 + 16) * 2.0 ** -24 + 2.0 ** -21) * (H.abs() @ W.abs().t()) + 2.0 ** -23 * torch.where(open_, z.abs(), 0.0)
    ez = ez + 2.0 ** -38 * (hm * W.abs().sum(1) + H.abs().sum(1, keepdim=True) * wm.t())
    lse = torch.logsumexp(z, 1)
    e_lse = torch.maximum(torch.logsumexp(z + ez, 1) - lse, lse - torch.logsumexp(z - ez, 1))
    at = t.clamp(min=0).unsqueeze(1)
    picked, e_picked = z.gather(1, at).squeeze(1), ez.gather(1, at).squeeze(1)
    g = torch.where(kept, rw.double(), 0.0)
    near(loss.detach(), "losses", {"losses": (torch.where(kept, (lse - picked) * g, 0.0),
                                              torch.where(kept, g * (e_lse + e_picked + 2.0 ** -21 * (1 + lse.abs() + picked.abs())), 0.0))})
    # log of what the others' exponentials come to, without entry u: [n][v]
    others = lambda x: torch.logsumexp(x.unsqueeze(1).expand(n, v, v).masked_fill(torch.eye(v, dtype=torch.bool, device=DEV), -math.inf), 2)  # noqa: E731
    p = torch.softmax(z, 1)
    hi, lo = torch.sigmoid(z + ez - others(z - ez)), torch.sigmoid(z - ez - others(z + ez))
    ep = torch.maximum(hi - p, p - lo) + p * (torch.where(open_, (z - lse.unsqueeze(1)).abs(), 0.0) + 2) * 2.0 ** -22
    d = p.scatter_add(1, at, torch.full_like(p[:, :1], -1.0))
    d, ep = torch.where(kept.unsqueeze(1), d, 0.0), torch.where(kept.unsqueeze(1), ep, 0.0)
    masked = (b == -math.inf).unsqueeze(1)
    W, wm = W.masked_fill(masked, 0.0), wm.masked_fill(masked, 0.0)
    H, hm = H.masked_fill(~kept.unsqueeze(1), 0.0), hm.masked_fill(~kept.unsqueeze(1), 0.0)
    # the pieces' ends: of a row's entries 2^-38 of sqrt(its largest x the tensor's), of D 2^-39 of the square root of their ratio (2: odd exponents)
    wend, dend = 2.0 ** -38 * 2 * (wm * wm.max()).sqrt(), 2.0 ** -39 * 2 * (wm.max() / wm.clamp(min=1e-30)).sqrt()
    hend, gend = 2.0 ** -38 * 2 * (hm * hm.max()).sqrt(), 2.0 ** -39 * 2 * (hm.max() / hm.clamp(min=1e-30)).sqrt() * g.max()
    want = (d @ W) * g.unsqueeze(1)
    e = (ep + 2.0 ** -20 * d.abs() + (v / 16 + 80) * 2.0 ** -24 * d.abs() + dend.t() * kept.unsqueeze(1)) @ W.abs() + d.abs() @ wend.expand(v, k)
    near(dh, "dh", {"dh": (want, e * g.unsqueeze(1) + 2.0 ** -21 * want.abs())})
    gd = d * g.unsqueeze(1)
    want = gd.t() @ H
    e = ((ep + 2.0 ** -20 * d.abs() + (n / 16 + 80) * 2.0 ** -24 * d.abs()) * g.unsqueeze(1) + gend).t() @ H.abs() + gd.abs().t() @ hend.expand(n, k)
    near(dw, "dw", {"dw": (want, e + 2.0 ** -21 * want.abs())})


@pytest.mark.gpu
def test_gpu_large_logits_of_operands_at_the_ends_of_the_range():
    """Logits of 5e4 from hidden of 1e35: what the operands were multiplied by is undone at once, not one factor after the other."""
    h, w, t, b, rw = inputs(64, 96, 150, F32, seed=9)
    h, w = (h * 1e35).requires_grad_(), (w * 1e-31).requires_grad_()
    loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw, reduction="none")
    near(loss.detach(), "losses", oracle(h, w, t, b, rw, "none"))
    assert all(bool(g.isfinite().all()) for g in torch.autograd.grad(loss.sum() / 64, [h, w]))


@pytest.mark.gpu
def test_gpu_sums_over_many_rows_of_large_numbers():
    """40 000 rows of 1e35: their sum before the mean's factor passes fp32's range, the gradient does not."""
    n, k, v = 40000, 8, 8
    h = torch.full((n, k), 1e35, device=DEV)
    w = torch.linspace(-1, 1, v, device=DEV).unsqueeze(1).expand(v, k).contiguous() * 1e-35
    t = torch.zeros(n, dtype=torch.int64, device=DEV)
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, t)
    out = oracle(h, w, t, None, None, "mean")
    near(loss.detach(), "total", out)
    (g,) = torch.autograd.grad(loss, [w])
    near(g, "dw", out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_tiny_gradients_of_the_rows(dtype):
    """Row weights or an upstream gradient far below 2^-114: the gradients are the same ones, smaller by that power of two, down
    to where the type's own numbers end (half its smallest one, scaled back)."""
    h, w, t, b, rw = inputs(90, 64, 200, dtype, seed=31, weights=True)
    leaves = [h.requires_grad_(), w.requires_grad_(), b.requires_grad_()]
    out = oracle(h, w, t, b, rw, "sum")
    tiny = 2.0 ** -118
    end = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}
    for case in range(3):
        if case == 0:
            loss, up = linear_cross_entropy(h, w, t, bias=b, row_weight=rw * tiny, reduction="sum"), None
            near(loss.detach().double() / tiny, "total", out)
        else:
            loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw, reduction="sum" if case == 1 else "none")
            up = torch.full_like(loss, tiny)
        for g, name, kind in zip(torch.autograd.grad(loss, leaves, grad_outputs=up), ("dh", "dw", "db"), (dtype, dtype, F32)):
            want, tol = out[name]
            near(g.double() / tiny, name, {name: (want, tol + end[kind] / tiny)})


# by the rules of the tiles alone, the forward pass would take wide tiles here and the backward pass, whose epilogue is longer, 64-wide ones,
# which add up K in two parts: fp32 and fp16, bf16 and fp16
SATURATED = [(300, 200, 9000), (174, 70, 34497)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SATURATED)
def test_gpu_a_saturated_row_has_no_gradient(size, dtype):
    """Logits of 1e5 whose target wins by far: softmax - onehot is 0, as long as the logits of the backward pass are the bits of
    the forward pass'; one half step of 1e5 in fp32 is 2^-8, and exp of that is no 1 any more."""
    n, k, v = size
    gen = torch.Generator().manual_seed(51)
    h = torch.randn(n, k, generator=gen).to(dtype).to(DEV)
    w = (torch.randn(v, k, generator=gen) * 3e4 / math.sqrt(k)).to(dtype).to(DEV)
    z = h.double() @ w.double().t()
    two = z.topk(2, dim=1)
    t = two.indices[:, 0].contiguous()
    t[two.values[:, 0] - two.values[:, 1] < 100.0] = -100       # the error of a logit of 1e5 is 1e5 (k / 16 + 16) 2^-24 < 1
    assert int((t != -100).sum()) > n // 2
    leaves = [h.requires_grad_(), w.requires_grad_()]
    loss = linear_cross_entropy(*leaves, t)
    assert float(loss.detach()) == 0.0
    for g in torch.autograd.grad(loss, leaves):
        assert not g.any()


@pytest.mark.gpu
def test_gpu_gradient_matches_differences():
    """Central differences of the loss along a direction: (f(x + s d) - f(x - s d)) / 2 s is off by s^2 f''' / 6 and by the
    loss' own rounding over s; at s = 2^-6, |f'''| <= 1 and a loss of about 7 to 2^-21 that is 4e-5 + 2e-4."""
    h, w, t, b, rw = inputs(50, 64, 400, F32, seed=10, bias=False)
    h.requires_grad_(), w.requires_grad_()
    gh, gw = torch.autograd.grad(linear_cross_entropy(h, w, t, row_weight=rw), [h, w])
    gen = torch.Generator().manual_seed(1)
    for x, g in ((h, gh), (w, gw)):
        d = torch.randn(x.shape, generator=gen).to(DEV)
        d /= d.norm()
        s = 2.0 ** -6
        with torch.no_grad():
            f = [float(linear_cross_entropy(*((x + k * s * d, w) if x is h else (h, x + k * s * d)), t, row_weight=rw)) for k in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * s) - float((g * d).sum())) <= 3e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_results_repeat_and_follow_the_stream(dtype):
    h, w, t, b, rw = inputs(300, 192, 1500, dtype, seed=11)
    h.requires_grad_(), w.requires_grad_(), b.requires_grad_()

    def both():
        loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw)
        return [loss.detach(), *torch.autograd.grad(loss, [h, w, b])]

    want = both()
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        a = both()
    c = both()              # two calls at once: each has its own workspace
    torch.cuda.synchronize()
    for got in (a, c, both()):
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
def test_gpu_captured_step_replays():
    """Loss and gradients captured once and replayed between eager calls, on changing inputs."""
    h, w, t, b, rw = inputs(200, 128, 900, BF16, seed=12)
    h.requires_grad_(), w.requires_grad_(), b.requires_grad_()

    def both():
        loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw)
        return [loss.detach(), *torch.autograd.grad(loss, [h, w, b])]

    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    gen = torch.Generator().manual_seed(2)
    for _ in range(3):
        with torch.no_grad():
            h.copy_(torch.randn(h.shape, generator=gen))
            t.copy_(torch.randint(0, 900, t.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        assert all(torch.equal(x, y) for x, y in zip(got, both()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
def test_gpu_captured_step_of_other_types_replays(dtype):
    """What the forward call leaves for the backward call (fp32: the scales of the rows) follows the inputs of each replay."""
    h, w, t, b, rw = inputs(190, 130, 700, dtype, seed=13)
    h.requires_grad_(), w.requires_grad_()

    def both():
        loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw)
        return [loss.detach(), *torch.autograd.grad(loss, [h, w])]

    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    gen = torch.Generator().manual_seed(3)
    for k in range(3):
        with torch.no_grad():
            h.copy_(torch.randn(h.shape, generator=gen) * 4.0 ** k)
            w.mul_(0.25)
            rw.copy_(torch.rand(rw.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        assert all(torch.equal(x, y) for x, y in zip(got, both()))


@pytest.mark.gpu
def test_gpu_capture_beside_a_live_eager_loss_is_refused(monkeypatch):
    """autograd would add up the leaves' gradients on the default stream, which cannot be captured."""
    h, w, t, _, _ = inputs(20, 64, 50, F32)
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, t)
    other = w.detach().clone().requires_grad_()
    side = torch.cuda.Stream(device=DEV)
    with torch.cuda.stream(side):
        elsewhere = linear_cross_entropy(h, other, t)
    with monkeypatch.context() as m:      # as it looks from inside a capture; nothing is captured here
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(L.GrlHipError, match="still alive"):
            linear_cross_entropy(h, w, t)
        linear_cross_entropy(h, other, t).backward()       # the live loss of another stream
        linear_cross_entropy(h, w.detach(), t)             # no gradient, no graph
        for again in (lambda: linear_cross_entropy(h, w * 1.0, t), lambda: linear_cross_entropy(h * w[:1], w.detach(), t)):
            with pytest.raises(L.GrlHipError, match="still alive"):
                again()                                    # the leaf stands behind other operations
        loss.backward()
        del loss
        linear_cross_entropy(h, w, t).backward()
    torch.cuda.synchronize()
    assert elsewhere.requires_grad


@pytest.mark.gpu
def test_gpu_capture_beside_a_live_loss_of_a_batch_of_sequences_is_refused(monkeypatch):
    """hidden of three dimensions is a leaf behind a view."""
    h, w, t, _, _ = inputs(20, 64, 50, F32)
    cube = h.view(4, 5, 64).requires_grad_()
    loss = linear_cross_entropy(cube, w, t.view(4, 5), reduction="sum")
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(L.GrlHipError, match="still alive"):
            linear_cross_entropy(cube, w, t.view(4, 5), reduction="sum")
        del loss
        linear_cross_entropy(cube, w, t.view(4, 5), reduction="sum").backward()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_gpu_a_head_over_a_network_trains_with_flat_muon():
    """The operators together: features of a HIP network, the head's loss over discretised actions with advantage weights,
    gradients through both, a FlatMuon step of the network and a muon_step of the head."""
    from generativerl_preview_amd.optim import FlatMuon, muon_step
    from generativerl_preview_amd.generative_models.intrinsic_model import IntrinsicModel
    torch.manual_seed(3)
    net = IntrinsicModel(dict(t_encoder=dict(type="GaussianFourierProjectionTimeEncoder", args=dict(embed_dim=32, scale=1.0)),
                              backbone=dict(type="TemporalSpatialResidualNet",
                                            args=dict(hidden_sizes=[128, 64], input_dim=11, output_dim=80, t_dim=32)))).to(DEV)
    head = torch.nn.Parameter(torch.randn(700, 80, device=DEV) / 9)
    time, state, t = torch.rand(256, device=DEV), torch.randn(256, 11, device=DEV), torch.randint(0, 700, (256,), device=DEV)
    weight = torch.rand(256, device=DEV) + 0.5
    opt = FlatMuon(net, lr=0.02)
    buf = torch.zeros_like(head)
    for _ in range(3):
        opt.zero_grad()
        head.grad = None
        features = net(time, state)
        loss = linear_cross_entropy(features, head, t, row_weight=weight)
        loss.backward()
        # the network's gradients are those of the plain head, through the same network
        plain = ((torch.nn.functional.cross_entropy(net(time, state) @ head.detach().t(), t, reduction="none")) * weight).mean()
        names = [p for p in net.parameters() if p.requires_grad]
        for p, g in zip(names, torch.autograd.grad(plain, names)):
            assert float((p.grad - g).abs().max()) <= 2e-5 * float(g.abs().max()) + 1e-9
        before = [p.detach().clone() for p in names]
        opt.step()
        muon_step([head.data], [head.grad], [buf], lr=0.02)
        assert all(not torch.equal(p, q) and bool(p.isfinite().all()) for p, q in zip(names, before))
        assert bool(head.isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_c_calls_write_the_magnitudes_as_the_header_says(dtype):
    """`largest`: by the forward call, for fp32 only."""
    h, w, t, _, _ = inputs(70, 100, 130, dtype, seed=17, bias=False, weights=False, ignored=0.1)
    lib, elem = L.lib(), {F32: L.ELEM_F32, BF16: L.ELEM_BF16, F16: L.ELEM_F16}[dtype]
    f = lambda n: torch.full((n,), -7.0, device=DEV)  # noqa: E731
    losses, lse, total, count, largest, gh = f(70), f(70), f(1), f(1), f(4), torch.empty_like(h)
    one = torch.ones((), device=DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream(DEV).cuda_stream)
    spaces = []
    for back in (0, 1):
        need = lib.grlhip_linear_ce_workspace_bytes(h.data_ptr(), None, w.data_ptr(), None, 70, 100, 130, elem, back)
        spaces.append(torch.full((need,), 0x3f, dtype=torch.uint8, device=DEV))
    args = (h.data_ptr(), None, w.data_ptr(), None, None, t.data_ptr(), -100, None, 70, 100, 130, elem, L.REDUCE_MEAN)
    L.check(lib.grlhip_linear_ce_forward(*args, losses.data_ptr(), lse.data_ptr(), total.data_ptr(), count.data_ptr(), largest.data_ptr(),
                                         spaces[0].data_ptr(), spaces[0].numel(), stream))
    want = torch.tensor([float(h[t != -100].abs().max()), float(w.abs().max()), -7.0, -7.0]) if dtype == F32 else torch.full((4,), -7.0)
    assert torch.equal(largest.cpu(), want)
    L.check(lib.grlhip_linear_ce_backward(*args, lse.data_ptr(), count.data_ptr(), largest.data_ptr(), one.data_ptr(), 0, gh.data_ptr(), None, None,
                                          spaces[1].data_ptr(), spaces[1].numel(), stream))
    assert torch.equal(largest.cpu(), want)
    out = oracle(h, w, t, None, None, "mean")
    near(total[0], "total", out)
    near(gh, "dh", out)


@pytest.mark.gpu
def test_gpu_c_calls_take_the_scales_that_the_forward_call_left():
    """GRLHIP_ELEM_SCALES: the gradients are those of a backward call that reads the operands itself, bit for bit."""
    n, k, v = 70, 100, 130
    h, w, t, b, rw = inputs(n, k, v, F32, seed=18)
    lib, stream = L.lib(), ctypes.c_void_p(torch.cuda.current_stream(DEV).cuda_stream)
    f = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    losses, lse, count, total, one = f(n), f(n), f(1), f(1), torch.ones((), device=DEV)
    scales = torch.empty(lib.grlhip_linear_ce_scales_bytes(n, v), dtype=torch.uint8, device=DEV)
    ws = [torch.empty(lib.grlhip_linear_ce_workspace_bytes(h.data_ptr(), None, w.data_ptr(), None, n, k, v, L.ELEM_F32, back), dtype=torch.uint8, device=DEV)
          for back in (0, 1)]
    head = (h.data_ptr(), None, w.data_ptr(), None, b.data_ptr(), t.data_ptr(), -100, rw.data_ptr(), n, k, v)
    L.check(lib.grlhip_linear_ce_forward(*head, L.ELEM_F32 | L.ELEM_SCALES, L.REDUCE_MEAN, losses.data_ptr(), lse.data_ptr(), total.data_ptr(),
                                         count.data_ptr(), scales.data_ptr(), ws[0].data_ptr(), ws[0].numel(), stream))
    results = []
    for elem, given in ((L.ELEM_F32 | L.ELEM_SCALES, scales.data_ptr()), (L.ELEM_F32, None), (L.ELEM_F32 | L.ELEM_SCALES, None)):
        grads = f(n, k), f(v, k), f(v)
        ws[1].fill_(0x3f)
        L.check(lib.grlhip_linear_ce_backward(*head, elem, L.REDUCE_MEAN, lse.data_ptr(), count.data_ptr(), given, one.data_ptr(), 0,
                                              *(g.data_ptr() for g in grads), ws[1].data_ptr(), ws[1].numel(), stream))
        results.append(grads)
    out = oracle(h, w, t, b, rw, "mean")
    near(total[0], "total", out)
    for k, name in enumerate(("dh", "dw", "db")):
        near(results[0][k], name, out)
        assert torch.equal(results[0][k], results[1][k]) and torch.equal(results[0][k], results[2][k])


# sizes that between them take every kind of tile for the logits, forward and backward, and for the gradients, with rests and more K blocks
# than a tile's ring has stages
KINDS = [(53, 213, 51), (66, 237, 17081), (131, 201, 41215), (133, 205, 51755), (2421, 691, 67), (7323, 685, 131), (8275, 663, 391)]


def test_the_sizes_below_take_every_kind_of_tile():
    lib, kinds = L.lib(), (ctypes.c_int32 * 3)()
    for elem in (L.ELEM_F32, L.ELEM_BF16, L.ELEM_F16):
        seen = [set(), set(), set()]
        for n, k, v in KINDS:
            assert lib.grlhip_linear_ce_tiles(n, k, v, elem, kinds) == 0
            assert (kinds[0] == 0) == (kinds[1] == 0)      # the same sums of the logits in both passes
            for s in range(3):
                seen[s].add(kinds[s])
        assert seen == [{0, 1, 2}] * 3, (elem, seen)
    for n, k, v in ((1, 1, 1), (300, 200, 9000), (174, 70, 34497), (1000, 100, 2600), (1 << 20, 64, 5000), (7, 65536, 100000)):
        for elem in (L.ELEM_F32, L.ELEM_BF16, L.ELEM_F16):
            assert lib.grlhip_linear_ce_tiles(n, k, v, elem, kinds) == 0 and (kinds[0] == 0) == (kinds[1] == 0)
    assert lib.grlhip_linear_ce_tiles(4, 8, 0, L.ELEM_F32, kinds) == -1 and lib.grlhip_linear_ce_tiles(4, 8, 9, 7, kinds) == -1
    assert lib.grlhip_linear_ce_tiles(4, 8, 9, L.ELEM_F32, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", KINDS)
def test_gpu_every_kind_of_tile(size, dtype):
    h, w, t, b, rw = inputs(*size, dtype, seed=61)
    leaves = [h.requires_grad_(), w.requires_grad_(), b.requires_grad_()]
    loss = linear_cross_entropy(h, w, t, bias=b, row_weight=rw)
    out = oracle(h, w, t, b, rw, "mean")
    near(loss.detach(), "total", out)
    for g, name in zip(torch.autograd.grad(loss, leaves), ("dh", "dw", "db")):
        near(g, name, out)


# ------------------------------------------------------------------------------------------------- refusals, on the CPU
def test_refusals_of_the_python_call():
    h, w, t = torch.randn(4, 8), torch.randn(10, 8), torch.zeros(4, dtype=torch.int64)
    call = linear_cross_entropy
    with pytest.raises(L.GrlHipError, match="HIP device"):
        call(h, w, t)
    for bad in (lambda: call(h, w, t, reduction="max"), lambda: call(h, w[:, :7], t), lambda: call(h, w[0], t), lambda: call(h, w, t[:3]),
                lambda: call(h, w[:0], t), lambda: call(h[:, :0], w[:, :0], t), lambda: call(h, w, t, bias=torch.zeros(9)),
                lambda: call(h, w, t, row_weight=torch.ones(3)), lambda: call(h, w, t, row_weight=torch.ones(4, requires_grad=True))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: call(h.double(), w.double(), t), lambda: call(h.half(), w, t), lambda: call(h, w, t.float()),
                lambda: call(h, w, t, bias=torch.zeros(10, dtype=torch.int64))):
        with pytest.raises(TypeError):
            bad()


def test_forward_mode_derivatives_are_refused():
    """A dual tensor requires no gradient; a result without a tangent would be a derivative of zero."""
    import torch.autograd.forward_ad as fad
    h, w, t, b, r = torch.randn(4, 8), torch.randn(10, 8), torch.zeros(4, dtype=torch.int64), torch.randn(10), torch.rand(4)
    with fad.dual_level():
        dual = lambda x: fad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for args, kw in (((dual(h), w, t), {}), ((h, dual(w), t), {}), ((h, w, t), dict(bias=dual(b))), ((h, w, t), dict(row_weight=dual(r)))):
            with pytest.raises(NotImplementedError, match="forward"):
                linear_cross_entropy(*args, **kw)
        with pytest.raises(L.GrlHipError, match="HIP device"):
            linear_cross_entropy(h, w, t, bias=b, row_weight=r)


def test_watching_live_losses_from_several_threads(monkeypatch):
    """Losses that come and go on other threads while one thread looks through the live ones, as it does under capture."""
    import sys
    import threading
    import types
    from generativerl_preview_amd.generative_models.model_functions import cross_entropy as ce
    me = threading.get_ident()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: threading.get_ident() == me)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
    leaves = [torch.zeros(1, requires_grad=True) for _ in range(4)]
    stop, failed = threading.Event(), []

    def work(leaf):
        kept = []
        try:
            while not stop.is_set():
                kept.append(types.SimpleNamespace())
                ce._watch(kept[-1], leaf)
                if len(kept) > 40:
                    del kept[::2]
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(x,)) for x in leaves]
    interval = sys.getswitchinterval()
    try:
        sys.setswitchinterval(1e-6)
        for th in threads:
            th.start()
        for _ in range(300):
            ce._watch(types.SimpleNamespace(), torch.zeros(1, requires_grad=True))
    finally:
        sys.setswitchinterval(interval)
        stop.set()
        for th in threads:
            th.join()
    assert not failed


def test_c_entry_points_check_their_arguments_without_a_gpu():
    lib = L.lib()
    size = lambda n=4, k=8, v=10, elem=L.ELEM_F32, back=0: lib.grlhip_linear_ce_workspace_bytes(None, None, None, None, n, k, v, elem, back)  # noqa: E731
    assert size() > 0 and size(back=1) > size()
    assert size(n=0) == size(k=0) == size(v=0) == size(elem=3) == size(n=(1 << 20) + 1) == size(k=1 << 17) == size(v=1 << 22) == 0
    assert b"linear_ce" in lib.grlhip_last_error()
    # 16-bit rows that are whole K blocks are read where they are
    assert size(v=100000, k=64, elem=L.ELEM_BF16) < size(v=100000, k=65, elem=L.ELEM_BF16)
    buf = (ctypes.c_char * 512)()
    p = ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256)

    def fwd(h=p, w=p, t=p, n=4, k=8, v=10, elem=L.ELEM_F32, red=L.REDUCE_MEAN, losses=p, lse=p, total=p, count=p, ws=p, bytes_=1):
        return lib.grlhip_linear_ce_forward(h, None, w, None, None, t, -100, None, n, k, v, elem, red, losses, lse, total, count, None, ws, bytes_, None)

    def bwd(h=p, w=p, t=p, n=4, red=L.REDUCE_MEAN, lse=p, count=p, grad=p, gh=p, ws=p, bytes_=1):
        return lib.grlhip_linear_ce_backward(h, None, w, None, None, t, -100, None, n, 8, 10, L.ELEM_F32, red, lse, count, None, grad, 0, gh, None, None, ws, bytes_, None)

    assert fwd() == -4 and bwd() == -4 and b"workspace" in lib.grlhip_last_error()
    assert fwd(total=None, count=None) == -1 and fwd(total=None, count=None, red=L.REDUCE_NONE) == -4
    assert fwd(lse=None) == -4
    for bad in ("h", "w", "t", "losses", "total", "count"):
        assert fwd(**{bad: None}) == -1, bad
    for bad in ("h", "w", "t", "lse", "count", "grad"):
        assert bwd(**{bad: None}) == -1, bad
    assert fwd(n=0) == -1 and fwd(elem=9) == -1 and fwd(red=3) == -1 and fwd(n=1 << 21) == -2 and fwd(ws=ctypes.c_void_p(p.value + 8)) == -1
    assert bwd(gh=None) == 0      # nothing is asked for


def test_c_scales_check_their_arguments_without_a_gpu():
    lib = L.lib()
    size = lib.grlhip_linear_ce_scales_bytes
    assert size(5, 7) >= 4 * 12 and size(5, 7) % 256 == 0 and size(1 << 20, 1 << 21) >= 4 * 3 * (1 << 20)
    assert size(0, 7) == size(5, 0) == size((1 << 20) + 1, 7) == size(5, (1 << 21) + 1) == 0
    buf = (ctypes.c_char * 512)()
    p = ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256)
    odd = ctypes.c_void_p(p.value + 64)
    fwd = lambda elem, scales: lib.grlhip_linear_ce_forward(p, None, p, None, None, p, -100, None, 4, 8, 10, elem, L.REDUCE_MEAN, p, p, p, p, scales, p, 1, None)  # noqa: E731
    bwd = lambda elem, scales: lib.grlhip_linear_ce_backward(p, None, p, None, None, p, -100, None, 4, 8, 10, elem, L.REDUCE_MEAN, p, p, scales, p, 0, p, None, None, p, 1, None)  # noqa: E731
    for call in (fwd, bwd):
        assert call(L.ELEM_F32 | L.ELEM_SCALES, p) == -4                 # the workspace is too small; the rest is fine
        assert call(L.ELEM_F32 | L.ELEM_SCALES, odd) == -1 and call(L.ELEM_F32, odd) == -4
        assert call(L.ELEM_BF16 | L.ELEM_SCALES, p) == call(L.ELEM_F16 | L.ELEM_SCALES, p) == call(L.ELEM_SCALES << 1, p) == -1
