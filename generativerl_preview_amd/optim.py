"""Adam over ONE flat parameter buffer (grlhip_adam_step): the optimizer of the reference's training loops
(``torch.optim.Adam`` over one network's parameters, grl/algorithms/qgpo.py:554,637,642, gmpo.py:788,942,946,1061) as a
single launch instead of the per-tensor kernels of the foreach implementation.

``FlatAdam(owner)`` takes an IntrinsicModel-like owner (``plan``, ``_named()``; what ``attach_flat_grads`` takes).  The
parameters are moved into ONE flat fp32 buffer in the library's gradient layout (their ``.data`` become views of it, so
``state_dict()``, ``named_parameters()`` and the weight packing see ordinary tensors) and their ``.grad`` are the views
of the FlatGrads buffer the fused losses accumulate into.  ``step()`` is one kernel over the trainable range(s);
``zero_grad()`` one memset.  Same update rule and defaults as ``torch.optim.Adam`` (amsgrad / maximize off).

``capturable=True`` keeps the step count on the device (grlhip_adam_step_counted), as ``torch.optim.Adam(capturable=True)``
does: a whole training step -- loss forward + backward, gradient all-reduce, ``step()`` -- can then be captured once with
``torch.cuda.graph`` and replayed (``tests/test_optim.py``).

``orthogonalize`` / ``muon_step`` / ``FlatMuon`` are the matrix-aware step beside it (grlhip_orthogonalize,
grlhip_muon_step): the momentum of every weight matrix is orthogonalised by a Newton-Schulz iteration before it is applied,
all matrices of a network in the same chain of launches; biases and other vectors keep Adam."""
import ctypes
import math

import torch

from . import _lib as L
from .distributed import attach_flat_grads
from .engine import _on, _ptr, _stream

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)   # a, b, c: 5 steps bring singular values from 0.002 on into [0.68, 1.21]
_ELEM = {torch.float32: L.ELEM_F32, torch.bfloat16: L.ELEM_BF16, torch.float16: L.ELEM_F16}


class FlatAdam:
    def __init__(self, owner, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, capturable=False):
        if lr < 0.0 or eps < 0.0 or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or weight_decay < 0.0:
            raise ValueError("invalid Adam hyper-parameters")
        self.owner = owner
        self.fg = attach_flat_grads(owner)
        self.defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay)
        self.param_groups = [dict(self.defaults, params=[p for p, _, _ in self.fg.slices if p.requires_grad])]
        self._steps = 0
        self.capturable = bool(capturable)
        dev = self.fg.flat.device
        # capturable: {int64 step; float step_size; float bc2_sqrt} on the device, advanced by the library
        self.step_record = torch.zeros(2, dtype=torch.int64, device=dev) if capturable else None
        n = self.fg.n
        self.flat_params = torch.zeros(n, dtype=torch.float32, device=dev)
        with torch.no_grad():
            for p, off, cnt in self.fg.slices:
                view = self.flat_params[off:off + cnt].view(p.shape)
                view.copy_(p.data)
                p.data = view                      # the module's parameter now lives in the flat buffer
        self.exp_avg = torch.zeros(n, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(n, dtype=torch.float32, device=dev)
        # contiguous ranges of trainable elements (frozen parameters, e.g. the Fourier frequencies, are skipped)
        self.ranges = []
        for p, off, cnt in sorted(self.fg.slices, key=lambda s: s[1]):
            if not p.requires_grad:
                continue
            if self.ranges and self.ranges[-1][1] == off:
                self.ranges[-1][1] = off + cnt
            else:
                self.ranges.append([off, off + cnt])

    def _check_views(self):
        base = self.flat_params.data_ptr()
        for p, off, cnt in self.fg.slices:
            if p.data_ptr() != base + 4 * off:
                raise RuntimeError("a parameter no longer lives in FlatAdam's buffer (module moved or re-assigned): "
                                   "build a new FlatAdam")

    @property
    def step_count(self):
        return int(self.step_record[0].item()) if self.capturable else self._steps

    @step_count.setter
    def step_count(self, value):
        if self.capturable:
            self.step_record.zero_()
            self.step_record[0] = int(value)
        else:
            self._steps = int(value)

    def zero_grad(self, set_to_none=False):
        self.fg.ensure()
        self.fg.zero()

    @torch.no_grad()
    def step(self):
        self._check_views()
        self.fg.ensure()
        g = self.param_groups[0]
        dev = self.flat_params.device
        if not self.capturable:
            self._steps += 1
        with torch.cuda.device(dev):
            stream = torch.cuda.current_stream(dev).cuda_stream
            for i, (lo, hi) in enumerate(self.ranges):
                ptrs = (self.flat_params.data_ptr() + 4 * lo, self.fg.flat.data_ptr() + 4 * lo,
                        self.exp_avg.data_ptr() + 4 * lo, self.exp_avg_sq.data_ptr() + 4 * lo, hi - lo,
                        g["lr"], g["betas"][0], g["betas"][1], g["eps"], g["weight_decay"])
                if self.capturable:   # the step count lives on the device: nothing per-step is frozen into a captured graph
                    L.check(L.lib().grlhip_adam_step_counted(*ptrs, self.step_record.data_ptr(), int(i == 0), stream))
                else:
                    L.check(L.lib().grlhip_adam_step(*ptrs, self._steps, stream))
        # the library wrote the parameters behind torch's back: their version counters did not move, and the owner's
        # packed-image cache (IntrinsicModel.packed) is keyed on them -- drop it explicitly
        if hasattr(self.owner, "_packed"):
            self.owner._packed = {} if isinstance(self.owner._packed, dict) else None
            if torch.cuda.is_current_stream_capturing():   # every replay writes them
                self.owner._in_graph = True

    def state_dict(self):
        return {"step": self.step_count, "exp_avg": self.exp_avg.clone(), "exp_avg_sq": self.exp_avg_sq.clone(),
                "param_groups": [{k: v for k, v in self.param_groups[0].items() if k != "params"}]}

    def load_state_dict(self, sd):
        self.step_count = int(sd["step"])
        self.exp_avg.copy_(sd["exp_avg"])
        self.exp_avg_sq.copy_(sd["exp_avg_sq"])
        self.param_groups[0].update(sd["param_groups"][0])


def _matrices(tensors, name, like=None):
    """Checks a list of matrices on one HIP device (that of `like`, with its shapes); returns their addresses and whether all
    are dense."""
    first = tensors[0] if like is None else like[0]
    dev, dtype, dense = first.device, tensors[0].dtype, True
    if dev.type != "cuda":
        raise L.GrlHipError("%s must live on a HIP device (got %s): there is no CPU fallback" % (name, dev))
    for i, t in enumerate(tensors):
        if t.device != dev or t.dtype != dtype:
            raise ValueError("%s[%d]: all matrices must be on one device and of one type (%s %s, got %s %s)" %
                             (name, i, dev, dtype, t.device, t.dtype))
        if t.dim() != 2 or (like is not None and t.shape != like[i].shape):
            raise ValueError("%s[%d]: expected %s, got shape %s" %
                             (name, i, "a matrix" if like is None else "shape %s" % (tuple(like[i].shape),), tuple(t.shape)))
        dense = dense and t.is_contiguous()
    return [t.data_ptr() if t.numel() else 0 for t in tensors], dense


def _meets_itself(t):
    """Whether two entries of a matrix lie at one place: i s0 = j s1 for some i, j inside of it."""
    (rows, cols), (s0, s1) = t.shape, t.stride()
    if rows < 2 or cols < 2:
        return max(rows, cols) > 1 and min(rows, cols) > 0 and (s0 if rows > 1 else s1) == 0
    g = math.gcd(s0, s1)
    return g == 0 or (s1 // g < rows and s0 // g < cols)


def _share(a, b):
    """Whether two matrices of 4-byte entries, none of which meets itself, have a place in common."""
    away, part = divmod(b.data_ptr() - a.data_ptr(), 4)
    if part:
        return True
    # axes of one entry have any stride: the other matrix' one; the larger stride first
    strides = [(x if n > 1 else y, y if m > 1 else x) for x, y, n, m in zip(a.stride(), b.stride(), a.shape, b.shape)]
    if strides[0][0] == strides[0][1] and strides[1][0] == strides[1][1]:
        # slices of one buffer: i s + j t = away for some i, j between -(sizes of b) and the sizes of a
        (s, n, m), (t, p, q) = sorted(((x, n, m) for (x, _), n, m in zip(strides, a.shape, b.shape)), reverse=True)
        return any((away - j * t) % s == 0 and -m < (away - j * t) // s < n for j in range(1 - q, p)) if s else away == 0
    if a.numel() + b.numel() > 1 << 24:
        return True
    places = lambda x, at: (at + torch.arange(x.shape[0])[:, None] * x.stride(0) + torch.arange(x.shape[1]) * x.stride(1)).view(-1)  # noqa: E731
    return bool(torch.isin(places(a, 0), places(b, away)).any())


def _check_memory(lists, pointers, dense):
    """``lists``: parameters, gradients, momentum buffers.  What is written, all but the gradients, shares no memory with itself or with
    anything else.  Ranges of addresses first; the matrices behind them are looked at where these meet."""
    if not all(dense) and any(_meets_itself(t) for k in (0, 2) for t in lists[k]):
        raise ValueError("muon_step: a matrix that is written to must not share memory with itself")
    spans = sorted((at, at + 4 * (t.numel() if d else 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))), k, i)
                   for k, (ts, ats, d) in enumerate(zip(lists, pointers, dense)) for i, (t, at) in enumerate(zip(ts, ats)) if at)
    written = read = 0      # where those so far end
    meet = False
    for at, end, k, _ in spans:
        meet = meet or at < written or (k != 1 and at < read)
        if k == 1:
            read = max(read, end)
        else:
            written = max(written, end)
    if not meet:
        return
    for n, (at, end, k, i) in enumerate(spans):
        for at2, end2, k2, i2 in spans[n + 1:]:
            if at2 >= end:
                break
            if not k == k2 == 1 and _share(lists[k][i], lists[k2][i2]):
                raise ValueError("muon_step: parameters, gradients and momentum buffers must not share memory")


def _pointers(addresses):
    return (ctypes.c_void_p * len(addresses))(*addresses)


def _shape_array(tensors):
    return (ctypes.c_int64 * (2 * len(tensors)))(*[n for t in tensors for n in t.shape])


def _stride_array(*lists):
    """[count][6] element strides of up to three lists of matrices."""
    lists = lists + (lists[0],) * (3 - len(lists))
    return (ctypes.c_int64 * (6 * len(lists[0])))(*[v for ts in zip(*lists) for t in ts for v in t.stride()])


def _newton_schulz_workspace(shapes, count, device):
    need = L.lib().grlhip_orthogonalize_workspace_bytes(shapes, count)
    if need == 0:
        raise L.GrlHipError(L.lib().grlhip_last_error().decode())
    # one per call: calls on different streams and captured graphs must not share it
    return torch.empty(need, dtype=torch.uint8, device=device)


@torch.no_grad()
def orthogonalize(matrices, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7):
    """Newton-Schulz orthogonalisation: ``steps`` times ``X <- a X + (b A + c A A) X`` with ``A = X X^T``, from
    ``X = G / max(|G|_F, eps)`` (grlhip_orthogonalize).  ``matrices``: a tensor ``(..., rows, cols)`` -- every matrix of it on
    its own -- or a list of such tensors, fp32, bf16 or fp16, any strides; all of them go through one chain of launches.
    Returns new tensors of the same shapes and type.  Products are fp32 (two fp16 pieces per value), rounded to the type once at the end;
    the order of their sums depends on all matrices of the call, so that beside others a matrix' result may differ by roundings.
    No gradient is recorded.  A matrix that holds an infinity or NaN comes back as NaN, a zero matrix as zeros."""
    single = torch.is_tensor(matrices)
    tensors = [matrices] if single else list(matrices)
    if not tensors:
        return []
    for i, t in enumerate(tensors):
        if t.dim() < 2:
            raise ValueError("matrices[%d]: expected (..., rows, cols), got shape %s" % (i, tuple(t.shape)))
        if t.dtype not in _ELEM:
            raise TypeError("matrices[%d]: expected float32, bfloat16 or float16, got %s" % (i, t.dtype))
    # batches as lists of matrices; a view where the strides allow one
    flat = [t if t.dim() == 2 else t.reshape(-1, *t.shape[-2:]) if t.numel() else t.new_empty(0, *t.shape[-2:]) for t in tensors]
    out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in flat]
    src = [m for t in flat for m in (t.unbind(0) if t.dim() == 3 else (t,))]
    dst = [m for t in out for m in (t.unbind(0) if t.dim() == 3 else (t,))]
    if src:
        pointers, dense = _matrices(src, "matrices")
        shapes = _shape_array(src)
        dev = src[0].device
        a, b, c = coefficients
        ws = _newton_schulz_workspace(shapes, len(src), dev)
        with _on(dev):
            L.check(L.lib().grlhip_orthogonalize(_pointers(pointers), _pointers([t.data_ptr() for t in dst]), shapes,
                                                 None if dense else _stride_array(src, dst), len(src), _ELEM[src[0].dtype],
                                                 int(steps), a, b, c, eps, _ptr(ws), ws.numel(), _stream(dev)))
    out = [o.view(t.shape) for o, t in zip(out, tensors)]
    return out[0] if single else out


@torch.no_grad()
def muon_step(params, grads, momentum_buffers, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
              coefficients=NEWTON_SCHULZ, eps=1e-7, adjust_lr="original"):
    """One step, in place, of lists of fp32 matrices (grlhip_muon_step):
        buf = momentum buf + (1 - momentum) grad;   u = (1 - momentum) grad + momentum buf if nesterov else buf
        param = (1 - lr weight_decay) param - lr' orthogonalize(u)
    with lr' = lr sqrt(max(1, rows / cols)) for ``adjust_lr="original"`` and 0.2 lr sqrt(max(rows, cols)) for
    ``"match_rms_adamw"`` (updates of the size of Adam's).  Any strides; the three lists must not share memory.  ``lr`` and the
    other numbers are read on the host: a captured graph keeps the ones it was captured with.  The call counts as an in-place
    operation on the parameters and buffers (their version counters move; a replay of a captured graph moves none, and a
    network of this framework that was not captured with the step does not see it)."""
    params, grads, bufs = list(params), list(grads), list(momentum_buffers)
    if not len(params) == len(grads) == len(bufs):
        raise ValueError("muon_step: %d parameters, %d gradients, %d momentum buffers" % (len(params), len(grads), len(bufs)))
    if lr < 0.0 or not 0.0 <= momentum < 1.0 or weight_decay < 0.0 or not eps > 0.0:
        raise ValueError("invalid Muon hyper-parameters")
    if adjust_lr not in ("original", "match_rms_adamw"):
        raise ValueError("adjust_lr: expected 'original' or 'match_rms_adamw', got %r" % (adjust_lr,))
    if not params:
        return
    (pp, pd), (gp, gd), (bp, bd) = _matrices(params, "params"), _matrices(grads, "grads", params), _matrices(bufs, "momentum_buffers", params)
    for name, ts in (("params", params), ("grads", grads), ("momentum_buffers", bufs)):
        if ts[0].dtype != torch.float32:
            raise TypeError("%s: expected float32, got %s" % (name, ts[0].dtype))
    check = lambda: _check_memory((params, grads, bufs), (pp, gp, bp), (pd, gd, bd))  # noqa: E731
    dense = pd and gd and bd      # then the library looks, in a tenth of the time
    if not dense:
        check()
    sides = [t.shape for t in params]
    rates = (ctypes.c_float * len(params))(*(
        [lr * math.sqrt(max(1.0, r / max(c, 1))) for r, c in sides] if adjust_lr == "original" else
        [lr * 0.2 * math.sqrt(max(r, c)) for r, c in sides]))
    shapes, dev = _shape_array(params), params[0].device
    a, b, c = coefficients
    ws = _newton_schulz_workspace(shapes, len(params), dev)
    with _on(dev):
        rc = L.lib().grlhip_muon_step(_pointers(pp), _pointers(gp), _pointers(bp), shapes, None if dense else _stride_array(grads, params, bufs),
                                      rates, len(params), momentum, int(nesterov), 1.0 - lr * weight_decay, int(steps), a, b, c, eps, _ptr(ws),
                                      ws.numel(), _stream(dev))
    if rc:
        check()
        L.check(rc)
    # the library wrote behind torch's back: packed weight images are keyed on these counters, and autograd checks them for
    # what it saved
    torch.autograd.graph.increment_version(params + bufs)


class FlatMuon(FlatAdam):
    """Muon over the weight matrices of ``owner`` and Adam over everything else, on FlatAdam's flat buffers (the momentum of
    a matrix takes the place of Adam's first moment there).  ``matrices(name, parameter)`` says which parameters are stepped
    as matrices; by default every trainable one with at least two rows and columns (input and output layers may be better
    off with Adam: name them there).  ``param_groups[1]`` holds Muon's numbers, ``param_groups[0]`` Adam's (``adam_*``)."""

    def __init__(self, owner, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NEWTON_SCHULZ,
                 eps=1e-7, adjust_lr="original", matrices=None, adam_lr=1e-3, adam_betas=(0.9, 0.999), adam_eps=1e-8,
                 adam_weight_decay=0.0, capturable=False):
        if lr < 0.0 or not 0.0 <= momentum < 1.0 or weight_decay < 0.0 or not eps > 0.0:
            raise ValueError("invalid Muon hyper-parameters")
        super().__init__(owner, lr=adam_lr, betas=adam_betas, eps=adam_eps, weight_decay=adam_weight_decay, capturable=capturable)
        names = [name for name, _ in owner.plan.params]
        if matrices is None:
            matrices = lambda name, p: p.dim() == 2 and min(p.shape) > 1  # noqa: E731
        self.matrix_names, chosen = [], []
        for name, (p, off, cnt) in zip(names, self.fg.slices):
            if p.requires_grad and matrices(name, p):
                if p.dim() != 2:
                    raise ValueError("FlatMuon: %s is no matrix (shape %s)" % (name, tuple(p.shape)))
                self.matrix_names.append(name)
                chosen.append((p, off, cnt))
        views = lambda flat: [flat[off:off + cnt].view(p.shape) for p, off, cnt in chosen]  # noqa: E731
        self._matrices = [p for p, _, _ in chosen], views(self.fg.flat), views(self.exp_avg)
        taken = {off for _, off, _ in chosen}
        self.ranges = []
        for p, off, cnt in sorted(self.fg.slices, key=lambda s: s[1]):
            if not p.requires_grad or off in taken:
                continue
            if self.ranges and self.ranges[-1][1] == off:
                self.ranges[-1][1] = off + cnt
            else:
                self.ranges.append([off, off + cnt])
        picked = {id(p) for p, _, _ in chosen}
        self.param_groups[0]["params"] = [p for p in self.param_groups[0]["params"] if id(p) not in picked]
        self.param_groups.append(dict(lr=lr, momentum=momentum, nesterov=bool(nesterov), weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps, adjust_lr=adjust_lr,
                                      params=[p for p, _, _ in chosen]))

    @torch.no_grad()
    def step(self):
        self._check_views()
        self.fg.ensure()
        muon_step(*self._matrices, **{k: v for k, v in self.param_groups[1].items() if k != "params"})
        super().step()

    def state_dict(self):
        sd = super().state_dict()
        sd["param_groups"].append({k: v for k, v in self.param_groups[1].items() if k != "params"})
        sd["matrices"] = list(self.matrix_names)
        return sd

    def load_state_dict(self, sd):
        if sd.get("matrices") != self.matrix_names:
            raise ValueError("the state was saved for other matrices")
        super().load_state_dict(sd)
        self.param_groups[1].update(sd["param_groups"][1])
