"""orthogonalize / muon_step / FlatMuon (grlhip_orthogonalize, grlhip_muon_step) against the formulas in 64 bits.

Tolerances, relative 2-norm.  A product of two-piece values is off by 2^-22 of the norms multiplied (dropped low x low and
the pieces' own 2^-23 each), the fp32 sums by less; what a step leaves in the direction of a small singular value grows by
a = 3.4445 in each of at most 4 further steps.  5 steps: 5 a^4 2^-22 = 1.7e-4, which single fp16 pieces (2^-11 in the place of
2^-22) pass 1000 times.  A result in a 16-bit type is rounded once more, by half a step: eps / 2."""
import copy
import ctypes
import math

import pytest
import torch

import util_models as um
from generativerl_preview_amd import _lib as L
from generativerl_preview_amd import optim

DEV = "cuda:0"
ABC = (3.4445, -4.7750, 2.0315)
TOL = 5 * 3.4445 ** 4 * 2.0 ** -22


def polar(g, steps=5, abc=ABC, eps=1e-7):
    x = g.detach().double().cpu()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / max(float(torch.linalg.vector_norm(x)), eps)
    for _ in range(steps):
        s = x @ x.t()
        x = abc[0] * x + abc[1] * (s @ x) + abc[2] * (s @ (s @ x))
    return x.t() if tall else x


def off(got, want):
    want = want.double().cpu()
    return float(torch.linalg.vector_norm(got.double().cpu() - want)) / max(float(torch.linalg.vector_norm(want)), 1e-300)


def tol(dtype):
    return TOL + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def grad_like(rows, cols, seed=0, dtype=torch.float32, scale=1e-3):
    gen = torch.Generator().manual_seed(seed)
    rank = max(1, min(rows, cols) // 2)
    g = torch.randn(rows, rank, generator=gen) @ torch.randn(rank, cols, generator=gen) / math.sqrt(rank)
    return ((g + 0.1 * torch.randn(rows, cols, generator=gen)) * scale).to(dtype).to(DEV)


SHAPES = [(1, 1), (1, 9), (7, 1), (2, 2), (17, 32), (63, 65), (64, 64), (6, 1024), (512, 6), (128, 64), (129, 300), (257, 100),
          (520, 400)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gpu_orthogonalize_matches_the_iteration_in_64_bits(shape, dtype):
    g = grad_like(*shape, dtype=dtype)
    before = g.clone()
    got = optim.orthogonalize(g)
    assert got.shape == g.shape and got.dtype == dtype and got.device == g.device
    assert torch.equal(g, before)
    assert off(got, polar(g)) <= tol(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1000, 777), (1024, 1024), (300, 2500), (1300, 1300)])
def test_gpu_orthogonalize_of_larger_matrices(shape):
    g = grad_like(*shape, seed=3)
    assert off(optim.orthogonalize(g), polar(g)) <= TOL


@pytest.mark.gpu
def test_gpu_orthogonalize_moves_singular_values_towards_one():
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(200, 300, generator=gen).to(DEV)
    s = torch.linalg.svdvals(optim.orthogonalize(g).double().cpu())
    assert 0.5 < float(s.min()) and float(s.max()) < 1.2


@pytest.mark.gpu
@pytest.mark.parametrize("steps,abc", [(0, ABC), (1, ABC), (2, ABC), (8, (1.5, -0.5, 0.0)), (6, (1.875, -1.25, 0.375))])
def test_gpu_orthogonalize_with_other_steps_and_coefficients(steps, abc):
    g = grad_like(70, 90, seed=1)
    assert off(optim.orthogonalize(g, steps=steps, coefficients=abc), polar(g, steps, abc)) <= TOL


@pytest.mark.gpu
def test_gpu_orthogonalize_takes_strides_batches_and_lists():
    big = grad_like(300, 400, seed=2)
    for view in (big.t(), big[10:75, 3:200], big[::2, ::3], big[:, 5:6].expand(300, 4), big.view(3, 100, 400)[1].t()[7:100]):
        got = optim.orthogonalize(view)
        assert got.shape == view.shape and off(got, polar(view)) <= TOL
    batch = torch.stack([grad_like(40, 30, seed=k) for k in range(6)]).view(2, 3, 40, 30)
    for b in (batch, batch.transpose(0, 1), batch.transpose(-1, -2)):
        got = optim.orthogonalize(b)
        assert got.shape == b.shape
        for i in range(b.shape[0]):
            for k in range(b.shape[1]):
                assert off(got[i, k], polar(b[i, k])) <= TOL
    # more small matrices than one launch describes (a workgroup each), with every side of the padding
    few = [grad_like(1 + 3 * k % 64, 190 - 5 * k, seed=k) for k in range(37)] + [grad_like(64, 192), grad_like(192, 33), grad_like(65, 4)[:64]]
    for g, m in zip(optim.orthogonalize(few), few):
        assert off(g, polar(m)) <= TOL
    # more matrices than one launch describes, of all shapes; empty ones among them
    many = [grad_like(5 + 7 * k, 90 - 3 * k, seed=k) for k in range(29)] + [torch.empty(0, 5, device=DEV), torch.empty(2, 0, 3, device=DEV),
                                                                            torch.empty(0, 4, 4, device=DEV)]
    got = optim.orthogonalize(many)
    assert [g.shape for g in got] == [m.shape for m in many]
    for g, m in zip(got[:29], many):
        assert off(g, polar(m)) <= TOL
    assert optim.orthogonalize([]) == []
    # more descriptions than one launch carries, too large for one workgroup each; the longest sums are not the first ones
    long_list = [grad_like(70 + k, 75 + 9 * ((k * 7) % 40), seed=k) for k in range(41)]
    for g, m in zip(optim.orthogonalize(long_list), long_list):
        assert off(g, polar(m)) <= TOL


@pytest.mark.gpu
def test_gpu_orthogonalize_at_the_ends_of_the_range():
    """Tiny and huge matrices (their squares leave fp32's range), zeros, infinities and NaN -- each on its own."""
    base = grad_like(50, 60, seed=4)
    ms = [base * 1e-30, base * 1e30, torch.zeros(50, 60, device=DEV), base.clone(), base.clone(), base]
    ms[3][7, 9] = math.inf
    ms[4][0, 0] = math.nan
    got = optim.orthogonalize(ms, eps=1e-38)
    assert off(got[0], polar(ms[0], eps=1e-38)) <= TOL
    assert off(got[1], polar(ms[1])) <= TOL
    assert not got[2].any()
    assert got[3].isnan().any() and got[4].isnan().all()
    assert off(got[5], polar(base)) <= TOL
    # below eps the matrix is divided by eps: it stays small
    assert off(optim.orthogonalize(base * 1e-9), polar(base * 1e-9)) <= TOL
    # one entry that dominates, and a rank of one
    spike = torch.zeros(90, 90, device=DEV)
    spike[3, 4] = 2.0
    assert off(optim.orthogonalize(spike), polar(spike)) <= TOL


@pytest.mark.gpu
def test_gpu_orthogonalize_repeats_its_bits_and_follows_the_stream():
    g = grad_like(333, 222, seed=6)
    want = optim.orthogonalize(g)
    assert torch.equal(optim.orthogonalize(g), want)
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        a = optim.orthogonalize(g)
    b = optim.orthogonalize(g)          # two calls at once: each has its own workspace
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def reference_step(p, g, buf, lr, momentum, nesterov, decay, adjust):
    p, g, buf = (t.detach().double().cpu() for t in (p, g, buf))
    buf = momentum * buf + (1 - momentum) * g
    u = (1 - momentum) * g + momentum * buf if nesterov else buf
    r, c = p.shape
    rate = lr * (math.sqrt(max(1.0, r / c)) if adjust == "original" else 0.2 * math.sqrt(max(r, c)))
    return p, (1 - lr * decay) * p - rate * polar(u), buf


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,decay,adjust", [(True, 0.1, "original"), (False, 0.0, "match_rms_adamw")])
def test_gpu_muon_step_matches_the_formula_in_64_bits(nesterov, decay, adjust):
    shapes = [(40, 70), (200, 30), (64, 64), (1, 5), (130, 257)]
    gen = torch.Generator().manual_seed(8)
    ps = [torch.randn(*s, generator=gen).to(DEV) for s in shapes]
    ps[1] = torch.randn(30, 200, generator=gen).to(DEV).t()           # stored by columns
    gs = [grad_like(*s, seed=k) for k, s in enumerate(shapes)]
    gs[2] = torch.randn(64, 128, generator=gen).to(DEV)[:, ::2]
    bs = [0.1 * grad_like(*s, seed=9 + k) for k, s in enumerate(shapes)]
    want = [reference_step(p, g, b, 0.05, 0.9, nesterov, decay, adjust) for p, g, b in zip(ps, gs, bs)]
    kept = [g.clone() for g in gs]
    optim.muon_step(ps, gs, bs, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=decay, adjust_lr=adjust)
    for p, g, b, k, (old, new, buf) in zip(ps, gs, bs, kept, want):
        assert torch.equal(g, k)
        # the momentum: three fp32 roundings; the change of the parameter: the iteration's error, and the rounding of p
        assert off(b, buf) <= 3 * 2.0 ** -24
        change = float(torch.linalg.vector_norm(new - old))
        slip = float(torch.linalg.vector_norm(p.double().cpu() - new))
        assert slip <= TOL * change + 2.0 ** -23 * float(torch.linalg.vector_norm(old))


@pytest.mark.gpu
def test_gpu_flat_muon_steps_a_network_in_training():
    """FlatMuon on a policy network trained through its fused loss: every matrix moves by the formula, everything else as
    torch.optim.Adam moves it, frozen parameters not at all; the state survives a round trip."""
    name = "small_icfm"
    kind, cfg, m = um.build(name, DEV)
    opt = optim.FlatMuon(m.model, lr=0.02, weight_decay=0.1, adam_lr=3e-3, adam_betas=(0.8, 0.95), adam_eps=1e-7)
    names = [n for n, _ in m.model.plan.params]
    assert len(opt.matrix_names) > 5 and all(n.endswith(".weight") for n in opt.matrix_names)
    frozen = m.model.model["t_encoder"].W.detach().clone()
    slices = dict(zip(names, opt.fg.slices))
    rest = {n: p for n, (p, _, _) in slices.items() if n not in opt.matrix_names and p.requires_grad}
    twins = {n: p.detach().clone().requires_grad_() for n, p in rest.items()}
    adam = torch.optim.Adam(list(twins.values()), lr=3e-3, betas=(0.8, 0.95), eps=1e-7)
    gen = torch.Generator().manual_seed(4)
    B = 300
    for step in range(3):
        x0, x1 = torch.randn(B, 6, generator=gen).to(DEV), torch.rand(B, 6, generator=gen).to(DEV)
        cond, t, eps = torch.randn(B, 17, generator=gen).to(DEV), torch.rand(B, generator=gen).to(DEV), torch.randn(B, 6, generator=gen).to(DEV)
        opt.zero_grad()
        m.flow_matching_loss(x0, x1, cond, t=t, noise=eps).backward()
        want = {}
        for n in opt.matrix_names:
            p, at, cnt = slices[n]
            want[n] = reference_step(p, p.grad, opt.exp_avg[at:at + cnt].view(p.shape), 0.02, 0.95, True, 0.1, "original")
        for n, p in rest.items():
            twins[n].grad = p.grad.detach().clone()
        opt.step()
        adam.step()
        for n, (old, new, buf) in want.items():
            p, at, cnt = slices[n]
            change = float(torch.linalg.vector_norm(new - old))
            assert float(torch.linalg.vector_norm(p.detach().double().cpu() - new)) <= TOL * change + 2.0 ** -23 * float(torch.linalg.vector_norm(old)), (step, n)
        for n, p in rest.items():
            assert float((p - twins[n]).detach().abs().max()) <= 2e-5 * (float(p.detach().abs().max()) + 1e-12), (step, n)
    assert torch.equal(m.model.model["t_encoder"].W.detach(), frozen)
    sd = copy.deepcopy(opt.state_dict())
    assert sd["step"] == 3 and len(sd["param_groups"]) == 2
    opt.exp_avg.zero_()
    opt.param_groups[1]["lr"] = 1.0
    opt.load_state_dict(sd)
    assert float(opt.exp_avg.abs().max()) > 0 and opt.param_groups[1]["lr"] == 0.02 and opt.step_count == 3
    sd["matrices"] = []
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)


@pytest.mark.gpu
def test_gpu_flat_muon_replays_from_a_captured_graph():
    """A training step with FlatMuon(capturable=True), captured once and replayed between eager work, takes the eager steps."""
    name = "small_icfm"
    kind, cfg, a = um.build(name, DEV)
    kind, cfg, b = um.build(name, DEV)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    oa, ob = (optim.FlatMuon(m.model, lr=0.01, capturable=True) for m in (a, b))
    gen = torch.Generator().manual_seed(9)
    B = 500
    x0, x1 = torch.randn(B, 6, generator=gen).to(DEV), torch.rand(B, 6, generator=gen).to(DEV)
    cond, t, eps = torch.randn(B, 17, generator=gen).to(DEV), torch.rand(B, generator=gen).to(DEV), torch.randn(B, 6, generator=gen).to(DEV)

    def step(m, o):
        o.zero_grad()
        loss = m.flow_matching_loss(x0, x1, cond, t=t, noise=eps)
        loss.backward()
        o.step()
        return loss.detach()

    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step(b, ob)
    torch.cuda.current_stream(DEV).wait_stream(side)
    step(a, oa)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, ob)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        step(a, oa)
        for (k, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
            assert torch.equal(p, q), k
    assert oa.step_count == ob.step_count == 5


def _residual_net():
    from generativerl_preview_amd.generative_models.intrinsic_model import IntrinsicModel
    return IntrinsicModel(dict(t_encoder=dict(type="GaussianFourierProjectionTimeEncoder", args=dict(embed_dim=32, scale=1.0)),
                               backbone=dict(type="TemporalSpatialResidualNet",
                                             args=dict(hidden_sizes=[64, 32], input_dim=11, output_dim=9, t_dim=32)))).to(DEV)


def _value_net():
    from generativerl_preview_amd.rl_modules.value_network.value_network import VNetwork
    return VNetwork(dict(backbone=dict(type="MultiLayerPerceptron", args=dict(hidden_sizes=[17, 64, 64], output_size=1, activation="relu")))).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("make,inputs", [(_residual_net, ((50,), (50, 11))), (_value_net, ((50, 17),))])
def test_gpu_muon_step_of_a_networks_matrices_is_seen_by_its_next_forward_pass(make, inputs):
    """The networks keep a packed image of their weights, which follows the parameters' version counters."""
    torch.manual_seed(11)
    net, fresh = make(), make()
    x = [torch.rand(s, device=DEV) for s in inputs]
    with torch.no_grad():
        first = net(*x).clone()
        matrices = [p for p in net.parameters() if p.dim() == 2 and p.requires_grad]
        grads, bufs = [grad_like(*p.shape, seed=k) for k, p in enumerate(matrices)], [torch.zeros_like(p) for p in matrices]
        versions = [t._version for t in (*matrices, *bufs)]
        optim.muon_step(matrices, grads, bufs, lr=0.1)
        assert all(t._version > v for t, v in zip((*matrices, *bufs), versions))
        fresh.load_state_dict(net.state_dict())
        second = net(*x)
        assert torch.equal(second, fresh(*x)) and not torch.equal(second, first)


@pytest.mark.gpu
def test_gpu_a_weight_stepped_between_forward_and_backward_is_noticed():
    from generativerl_preview_amd.generative_models.model_functions import linear_cross_entropy
    w, h = torch.nn.Parameter(torch.randn(40, 16, device=DEV)), torch.randn(8, 16, device=DEV)
    loss = linear_cross_entropy(h, w, torch.arange(8, device=DEV))
    optim.muon_step([w], [grad_like(40, 16)], [torch.zeros(40, 16, device=DEV)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("make", [optim.FlatMuon, optim.FlatAdam])
@pytest.mark.parametrize("before,between", [(True, False), (False, True), (True, True)])
def test_gpu_captured_steps_and_eager_passes_see_each_others_weights(make, before, between):
    """Forward passes before the capture, and between the replays: the captured loss follows the weights, and so do the passes."""
    kind, cfg, a = um.build("small_icfm", DEV)
    kind, cfg, b = um.build("small_icfm", DEV)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    oa, ob = (make(m.model, lr=0.01, capturable=True) for m in (a, b))
    gen = torch.Generator().manual_seed(9)
    B = 300
    x0, x1 = torch.randn(B, 6, generator=gen).to(DEV), torch.rand(B, 6, generator=gen).to(DEV)
    cond, t, eps = torch.randn(B, 17, generator=gen).to(DEV), torch.rand(B, generator=gen).to(DEV), torch.randn(B, 6, generator=gen).to(DEV)

    def step(m, o):
        o.zero_grad()
        loss = m.flow_matching_loss(x0, x1, cond, t=t, noise=eps)
        loss.backward()
        o.step()
        return loss.detach()

    def look(m):
        with torch.no_grad():
            return m.model(t, x0, cond).clone()

    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step(b, ob)
    torch.cuda.current_stream(DEV).wait_stream(side)
    step(a, oa)
    if before:
        assert torch.equal(look(a), look(b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(b, ob)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, step(a, oa)), k
        if between:
            assert torch.equal(look(a), look(b)), k
    assert torch.equal(look(a), look(b))


def _q_net():
    from generativerl_preview_amd.rl_modules.value_network.q_network import QNetwork
    net = QNetwork(dict(backbone=dict(type="ConcatenateMLP", args=dict(hidden_sizes=[17, 64, 64], output_size=1, activation="relu")))).to(DEV)
    net.set_io_dims(6, 11)
    return net


@pytest.mark.gpu
@pytest.mark.parametrize("make,inputs", [(_residual_net, ((50,), (50, 11))), (_value_net, ((50, 17),)), (_q_net, ((50, 6), (50, 11)))])
def test_gpu_a_captured_forward_pass_follows_the_weights(make, inputs):
    torch.manual_seed(12)
    net, fresh = make(), make()
    x = [torch.rand(s, device=DEV) for s in inputs]
    with torch.no_grad():
        net(*x)                                  # what is packed already must not be what the graph reads
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = net(*x)
        for k in range(3):
            for p in net.parameters():
                p.mul_(0.5 + k)
            fresh.load_state_dict(net.state_dict())
            want = fresh(*x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want) and torch.equal(net(*x), want)
    twin = copy.deepcopy(net)
    assert not twin._in_graph and torch.equal(twin(*x), want)


@pytest.mark.gpu
def test_gpu_a_capture_packs_once_and_for_itself(monkeypatch):
    """The calls of one capture share a packed image; another capture does not read it, and eager calls do not either."""
    torch.manual_seed(13)
    net, x = _value_net(), torch.rand(50, 17, device=DEV)
    packs, pack = [], type(net.plan).pack
    monkeypatch.setattr(type(net.plan), "pack", lambda *a: packs.append(1) or pack(*a))
    with torch.no_grad():
        net(x), net(x)
        assert len(packs) == 1
        graphs, held = [], []
        for k in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                held.append((net(x), net(x)))
            assert len(packs) == 2 + k
        graphs[1].replay()             # the second graph alone: nothing of the first one's
        torch.cuda.synchronize()
        want = net(x)
        assert len(packs) == 4 and all(torch.equal(y, want) for y in held[1])
        for p in net.parameters():
            p.mul_(1.5)
        want = net(x)
        for g, ys in zip(graphs, held):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(y, want) for y in ys)
    assert L.lib().grlhip_capture_id(ctypes.c_void_p(torch.cuda.current_stream(DEV).cuda_stream)) == 0


# groups that between them take every kind of tile in every product, with rests in all of them
GROUPS = [(1, (65, 65)), (6, (660, 540)), (1, (193, 2)), (1, (2, 225)), (1, (226, 225)), (24, (195, 198)), (24, (225, 266)), (24, (292, 308)),
          (12, (518, 523)), (24, (454, 464)), (24, (587, 594)), (12, (356, 370)), (24, (169, 161)), (24, (676, 33)), (8, (98, 3085)), (24, (1696, 97)),
          (24, (193, 1411)), (8, (1432, 1411))]


def test_the_groups_below_take_every_kind_of_tile():
    lib, kinds, seen = L.lib(), (ctypes.c_int32 * 3)(), [set(), set(), set()]
    for count, shape in GROUPS:
        assert lib.grlhip_orthogonalize_tiles((ctypes.c_int64 * (2 * count))(*(shape * count)), count, kinds) == 0
        for s in range(3):
            seen[s].add(kinds[s])
    assert seen == [set(range(9))] * 3, seen
    assert lib.grlhip_orthogonalize_tiles((ctypes.c_int64 * 2)(64, 192), 1, kinds) == 0 and list(kinds) == [-1] * 3
    assert lib.grlhip_orthogonalize_tiles((ctypes.c_int64 * 2)(64, 192), 1, None) == -1
    assert lib.grlhip_orthogonalize_tiles((ctypes.c_int64 * 2)(-1, 192), 1, kinds) == -2


def polar_on_the_gpu(g):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / float(torch.linalg.vector_norm(x))
    for _ in range(5):
        s = x @ x.t().contiguous()
        x = ABC[0] * x + ABC[1] * (s @ x) + ABC[2] * (s @ (s @ x))
    return x.t() if tall else x


@pytest.mark.gpu
@pytest.mark.parametrize("group", range(len(GROUPS)))
def test_gpu_every_kind_of_tile(group):
    """Each type, and the optimiser step, of the first, a middle and the last matrix of each group."""
    count, shape = GROUPS[group]
    some = sorted({0, count // 2, count - 1})
    gs = [grad_like(*shape, seed=100 * group + k) if k in some else 1e-3 * torch.randn(shape, device=DEV) for k in range(count)]
    want = {k: polar_on_the_gpu(gs[k]) for k in some}
    got = optim.orthogonalize(gs)
    for k in some:
        assert off(got[k], want[k]) <= TOL, k
    for dtype in (torch.bfloat16, torch.float16):
        half = [g.to(dtype) for g in gs]
        got = optim.orthogonalize(half)
        for k in some:
            assert off(got[k], polar_on_the_gpu(half[k])) <= tol(dtype), (dtype, k)
    ps, bufs = [torch.randn(shape, device=DEV) for _ in gs], [torch.zeros_like(g) for g in gs]
    old = [p.double() for p in ps]
    optim.muon_step(ps, gs, bufs, lr=0.05, momentum=0.9, nesterov=False, weight_decay=0.1)
    rate = 0.05 * math.sqrt(max(1.0, shape[0] / shape[1]))
    for k in some:      # the momentum is 0.1 of the gradient: the same direction
        slip = float(torch.linalg.vector_norm(ps[k].double() - ((1 - 0.005) * old[k] - rate * want[k])))
        change = float(torch.linalg.vector_norm(rate * want[k] + 0.005 * old[k]))
        assert slip <= TOL * change + 2.0 ** -23 * float(torch.linalg.vector_norm(old[k])), k


# ------------------------------------------------------------------------------------------------- refusals, on the CPU
def test_refusals_of_the_python_calls():
    m = torch.randn(4, 5)
    with pytest.raises(L.GrlHipError, match="HIP device"):
        optim.orthogonalize(m)
    with pytest.raises(ValueError, match="rows, cols"):
        optim.orthogonalize(torch.randn(4))
    with pytest.raises(TypeError):
        optim.orthogonalize(m.double())
    with pytest.raises(L.GrlHipError, match="HIP device"):
        optim.muon_step([m], [m.clone()], [m.clone()], lr=0.1)
    with pytest.raises(ValueError, match="gradients"):
        optim.muon_step([m], [], [m], lr=0.1)
    for bad in (dict(lr=-1.0), dict(lr=0.1, momentum=1.0), dict(lr=0.1, weight_decay=-1.0), dict(lr=0.1, eps=-1.0),
                dict(lr=0.1, adjust_lr="no")):
        with pytest.raises(ValueError):
            optim.muon_step([m], [m], [m], **bad)
    assert optim.muon_step([], [], [], lr=0.1) is None


@pytest.mark.gpu
def test_gpu_refusals_that_need_device_tensors():
    m, g, b = (torch.randn(4, 5, device=DEV) for _ in range(3))
    step = lambda *a: optim.muon_step(*a, lr=0.1)  # noqa: E731
    for bad in (([m, m], [g, g], [b, b.clone()]), ([m], [m], [b]), ([m], [g], [g]), ([m], [g], [m]), ([m], [g.t()], [b]),
                ([m[:1].expand(4, 5)], [g], [b]), ([m.view(-1)], [g], [b])):
        with pytest.raises(ValueError):
            step(*bad)
    for bad in (([m], [g.half()], [b]), ([m], [g], [b.bfloat16()])):
        with pytest.raises(TypeError):
            step(*bad)
    with pytest.raises(ValueError):
        optim.orthogonalize([m, m.half()])
    for abc in ((30.0, 0.0, 0.0), (math.nan, 0.0, 0.0), (1.0, -9.0, 13.9)):
        with pytest.raises(L.GrlHipError):
            optim.orthogonalize(m, coefficients=abc)
    # |b s^2 + c s^4| <= 2.25 and |x| <= 1 for s <= 1: in range
    assert off(optim.orthogonalize(m, coefficients=(1.0, -9.0, 9.0)), polar(m, abc=(1.0, -9.0, 9.0))) <= TOL
    with pytest.raises(L.GrlHipError):
        optim.orthogonalize(m, steps=-1)


def test_shared_memory_is_found_exactly():
    """Against the sets of places, for slices, transposes and strange strides of one buffer."""
    buf = torch.zeros(400)
    views = [buf.as_strided(size, stride, at) for size in ((3, 4), (1, 5), (4, 1), (2, 2), (5, 6), (1, 1), (0, 3)) for stride in ((10, 1), (1, 10), (6, 2), (2, 3), (5, 5), (0, 1))
             for at in (0, 1, 4, 7, 13)]
    places = lambda t: [t.storage_offset() + i * t.stride(0) + j * t.stride(1) for i in range(t.shape[0]) for j in range(t.shape[1])]  # noqa: E731
    sets = [set(places(t)) for t in views]
    plain = []
    for t, s in zip(views, sets):
        assert optim._meets_itself(t) == (len(s) < t.numel()), (t.shape, t.stride())
        if len(s) == t.numel() > 0:
            plain.append((t, s))
    for t, s in plain:
        for u, r in plain:
            assert optim._share(t, u) == bool(s & r), (t.shape, t.stride(), t.storage_offset(), u.shape, u.stride(), u.storage_offset())


def test_matrices_that_share_memory_are_refused():
    def check(p, g, b):
        lists = tuple([x] if torch.is_tensor(x) else x for x in (p, g, b))
        optim._check_memory(lists, [[t.data_ptr() if t.numel() else 0 for t in ts] for ts in lists], [all(t.is_contiguous() for t in ts) for ts in lists])

    big, other, third = torch.zeros(12, 10), torch.zeros(12, 10), torch.zeros(24, 10)
    for bad in (([big[:6], big[5:11]], [other[:6], other[6:]], [third[:6], third[6:12]]),       # parameters that overlap
                (big[:6], big[3:9], third[:6]),                                                 # a gradient inside of a parameter
                (big[:6], other[:6], other[4:10]),                                              # a buffer over a gradient
                (big[:, :6], other[:, :6], big[:, 5:]),                                         # one column in common
                (big[::2], other[::2], big[2:8]),                                                    # rows 2, 4 and 6 of both
                (big.as_strided((3, 3), (2, 2)), other[:3, :3], third[:3, :3])):                # a parameter that meets itself
        with pytest.raises(ValueError, match="share memory"):
            check(*bad)
    # one buffer, no place in common: halves of its columns, every other row, rows beside each other; gradients may share
    check([big[:, :5], big[:, 5:]], [other[:, :5], other[:, :5]], [third[:12, :5], third[12:, 5:]])
    check(big[::2], big[1::2], other[::2])
    check([big[:6], big[6:]], [other[:6], other[2:8]], [third[:6], third[6:12]])
    check([big[:, :1].t(), big[:0]], [other[:, :1].t(), other[:0]], [big[:, 1:2].t(), other[:0]])


@pytest.mark.gpu
def test_gpu_muon_step_refuses_matrices_that_overlap_and_takes_those_that_do_not():
    big, g = torch.randn(20, 30, device=DEV), [grad_like(10, 30), grad_like(10, 30, seed=1)]
    with pytest.raises(ValueError, match="share memory"):
        optim.muon_step([big[:10], big[9:19]], g, [torch.zeros(10, 30, device=DEV) for _ in range(2)], lr=0.1)
    # interleaved rows and buffers in one tensor: the same step as of copies
    store = torch.zeros(20, 60, device=DEV)
    want_p, want_b = [big[::2].clone(), big[1::2].clone()], [torch.zeros(10, 30, device=DEV) for _ in range(2)]
    optim.muon_step(want_p, g, want_b, lr=0.1)
    bufs = [store[:10, :30], store[:10, 30:]]
    optim.muon_step([big[::2], big[1::2]], g, bufs, lr=0.1)
    for got, want in zip((big[::2], big[1::2], *bufs), (*want_p, *want_b)):
        assert torch.equal(got, want)
    assert not store[10:].any()


def test_c_entry_points_check_their_arguments_without_a_gpu():
    lib = L.lib()
    shapes = (ctypes.c_int64 * 2)(8, 8)
    need = lib.grlhip_orthogonalize_workspace_bytes(shapes, 1)
    # at least two X and X^T of 32 x 32 four-byte values each, A and B; more matrices need more
    assert need >= 6 * 32 * 32 * 4
    assert lib.grlhip_orthogonalize_workspace_bytes((ctypes.c_int64 * 4)(8, 8, 8, 8), 2) >= 2 * 6 * 32 * 32 * 4
    buf = (ctypes.c_char * (need + 256))()
    ws = ctypes.c_void_p((ctypes.addressof(buf) + 255) // 256 * 256)
    one = (ctypes.c_void_p * 1)(ws.value)
    null = (ctypes.c_void_p * 1)(None)
    orth = lambda src=one, dst=one, sh=shapes, n=1, elem=L.ELEM_F32, steps=5, abc=ABC, eps=1e-7, w=ws, size=need: lib.grlhip_orthogonalize(  # noqa: E731
        src, dst, sh, None, n, elem, steps, *abc, eps, w, size, None)
    assert orth(n=0) == 0
    assert orth(n=-1) != 0 and orth(sh=None) != 0 and orth(src=null) != 0 and orth(dst=null) != 0
    assert orth(elem=7) != 0 and orth(steps=-1) != 0 and orth(steps=33) != 0 and orth(eps=-1.0) != 0 and orth(eps=0.0) != 0 and orth(eps=math.nan) != 0
    assert orth(abc=(9.0, 0.0, 0.0)) == -2 and b"1.9" in lib.grlhip_last_error()
    assert orth(size=need - 1) == -4 and orth(w=None) == -4
    assert orth(w=ctypes.c_void_p(ws.value + 8)) == -1
    assert orth(sh=(ctypes.c_int64 * 2)(8, 1 << 17)) == -2
    rates = (ctypes.c_float * 1)(0.1)
    muon = lambda p=one, g=one, b=one, r=rates, mom=0.9: lib.grlhip_muon_step(p, g, b, shapes, None, r, 1, mom, 1, 1.0, 5, *ABC, 1e-7, ws, 0, None)  # noqa: E731
    assert muon() == -4
    for bad in (dict(p=null), dict(g=null), dict(b=null), dict(r=None), dict(mom=1.0), dict(mom=math.nan)):
        assert muon(**bad) == -1, bad
    assert lib.grlhip_orthogonalize_workspace_bytes((ctypes.c_int64 * 2)(-1, 2), 1) == 0


def test_c_entry_point_refuses_dense_matrices_that_overlap():
    """Each of these calls is refused before anything is launched: the memory is the host's."""
    lib = L.lib()
    shapes = (ctypes.c_int64 * 4)(8, 8, 4, 4)
    need = lib.grlhip_orthogonalize_workspace_bytes(shapes, 2)
    buf = (ctypes.c_char * (need + 8192))()
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    at = base + (need + 255) // 256 * 256
    rates = (ctypes.c_float * 2)(0.1, 0.1)
    ptrs = lambda *offsets: (ctypes.c_void_p * 2)(*(at + o for o in offsets))  # noqa: E731
    step = lambda p, g, b: lib.grlhip_muon_step(ptrs(*p), ptrs(*g), ptrs(*b), shapes, None, rates, 2, 0.9, 1, 1.0, 5, *ABC, 1e-7, base, need, None)  # noqa: E731
    ok = ((0, 256), (512, 1024), (2048, 2304))         # 256 and 64 bytes each
    for bad in (((0, 252), *ok[1:]), ((0, 0), *ok[1:]), (ok[0], (0, 1024), ok[2]), (ok[0], (512, 316), ok[2]), (ok[0], ok[1], (764, 2304)), (ok[0], ok[1], (2048, 2048))):
        assert step(*bad) == -1 and b"share memory" in lib.grlhip_last_error(), bad
