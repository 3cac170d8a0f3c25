"""Softmax cross entropy of a linear head over a large vocabulary, without storing the logits: the loss of a policy over
discretised actions (behaviour cloning, or advantage-weighted with ``row_weight``), beside the fused losses of the continuous
models.  ``grlhip_linear_ce_forward`` / ``grlhip_linear_ce_backward``."""
import ctypes
import threading
import weakref

import torch
from torch.autograd import forward_ad

from ... import _lib as L
from ...engine import _on

_ELEM = {torch.float32: L.ELEM_F32, torch.bfloat16: L.ELEM_BF16, torch.float16: L.ELEM_F16}
_REDUCE = {"none": L.REDUCE_NONE, "mean": L.REDUCE_MEAN, "sum": L.REDUCE_SUM}


def _address(t):
    return None if t is None else t.data_ptr()


def _strides(t):
    return None if t.is_contiguous() else (ctypes.c_int64 * 2)(*t.stride())


def _has_tangent(*tensors):
    if getattr(forward_ad, "_current_level", 0) < 0:   # no dual level, no dual tensor: the question costs 1 us a tensor
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _Head:
    """The arguments that the forward and the backward call share."""

    def __init__(self, hidden, weight, bias, target, row_weight, ignore_index, reduction):
        self.device, self.dtype, self.reduction = hidden.device, hidden.dtype, reduction
        bias = None if bias is None else bias.float().contiguous()
        self.kept = hidden, weight, bias, target, row_weight     # alive until the launches are queued
        (rows, features), vocab = hidden.shape, weight.shape[0]
        self.shape = rows, features, vocab
        self.operands = hidden.data_ptr(), _strides(hidden), weight.data_ptr(), _strides(weight)
        self.sizes = rows, features, vocab, _ELEM[hidden.dtype]
        self.arguments = (*self.operands, _address(bias), target.data_ptr(), ignore_index, _address(row_weight), rows, features, vocab)

    def call(self, name, backward, scales, *rest):
        lib = L.lib()
        need = lib.grlhip_linear_ce_workspace_bytes(*self.operands, *self.sizes, backward)
        if need == 0:
            raise L.GrlHipError(lib.grlhip_last_error().decode())
        # one workspace per call: calls on different streams and captured graphs must not share it
        with _on(self.device):
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            stream = torch.cuda.current_stream(self.device).cuda_stream
            L.check(getattr(lib, name)(*self.arguments, self.sizes[3] if scales is None else self.sizes[3] | L.ELEM_SCALES, self.reduction, *rest,
                                       ws.data_ptr(), need, stream))

    def forward(self, train=False):
        """(losses, reduced loss, what the backward pass needs: number of rows that are not ignored, scales of fp32 operands, logsumexp)"""
        (rows, _, vocab), dev = self.shape, self.device
        losses = torch.empty(rows, dtype=torch.float32, device=dev)
        total = kept = scales = lse = count = None
        if train:
            # one buffer: the count, from the 64th number on the scales (aligned to 256 bytes), the logsumexps last
            room = L.lib().grlhip_linear_ce_scales_bytes(rows, vocab) // 4 if self.dtype == torch.float32 else 0
            kept = torch.empty(64 + room + rows, dtype=torch.float32, device=dev)
            scales, lse = kept.data_ptr() + 256 if room else None, kept.data_ptr() + 4 * (64 + room)
        if self.reduction != L.REDUCE_NONE:
            total = torch.empty((), dtype=torch.float32, device=dev)
            kept = torch.empty(1, dtype=torch.float32, device=dev) if kept is None else kept
            count = kept.data_ptr()
        self.call("grlhip_linear_ce_forward", 0, scales, losses.data_ptr(), lse, _address(total), count, scales)
        return losses, total, kept

    def backward(self, kept, grad, need_hidden, need_weight, need_bias):
        rows, features, vocab = self.shape
        dev, at = self.device, kept.data_ptr()
        scales, lse = at + 256 if self.dtype == torch.float32 else None, at + 4 * (kept.numel() - rows)
        gh = torch.empty(rows, features, dtype=self.dtype, device=dev) if need_hidden else None
        gw = torch.empty(vocab, features, dtype=self.dtype, device=dev) if need_weight else None
        gb = torch.empty(vocab, dtype=torch.float32, device=dev) if need_bias else None
        self.call("grlhip_linear_ce_backward", 1, scales, lse, at, scales, grad.data_ptr(),
                  0 if grad.dim() == 0 else grad.stride(0), _address(gh), _address(gw), _address(gb))
        return gh, gw, gb


class _Graph:
    """Lives as long as the autograd graph of one eager loss; `roots`: where that graph goes on, leaves or the nodes of others."""
    __slots__ = ("roots", "__weakref__")

    def __init__(self, roots):
        self.roots = roots


_ON_DEFAULT_STREAM = weakref.WeakSet()   # of all threads and devices
_WATCH = threading.RLock()               # one thread's capture looks through it while others add to it


def _leaves(roots):
    """{id: leaf} of the tensors that the graphs of `roots` end in."""
    found, seen, queue = {}, set(), []
    for r in roots:
        if torch.is_tensor(r):
            found[id(r)] = r
        else:
            queue.append(r)
    while queue:
        node = queue.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        leaf = getattr(node, "variable", None)
        if torch.is_tensor(leaf):
            found[id(leaf)] = leaf
        queue.extend(n for n, _ in node.next_functions)
    return found


def _watch(ctx, *tensors):
    """autograd adds up a leaf's gradient on the stream where the leaf first entered a live graph.  If that is the default
    stream, a backward pass under capture reaches for a stream that cannot be captured, and the process ends: such a
    call is refused while it is still a call.  The graphs are walked under capture only."""
    roots = [t if t.is_leaf else t.grad_fn for t in tensors if t is not None and t.requires_grad]
    if not roots:
        return
    if torch.cuda.is_current_stream_capturing():
        with _WATCH:
            graphs = list(_ON_DEFAULT_STREAM)
        live = [r for graph in graphs for r in graph.roots]
        if live and _leaves(roots).keys() & _leaves(live).keys():
            raise L.GrlHipError("linear_cross_entropy under graph capture: an eager loss of the same leaves, computed on the "
                                "default stream, is still alive; drop it (del loss) before the capture")
    elif torch.cuda.current_stream(tensors[0].device).cuda_stream == 0:
        ctx.graph = _Graph(roots)
        with _WATCH:
            _ON_DEFAULT_STREAM.add(ctx.graph)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, target, row_weight, ignore_index, reduction):
        _watch(ctx, hidden, weight, bias)
        head = _Head(hidden, weight, bias, target, row_weight, ignore_index, reduction)
        losses, total, kept = head.forward(train=True)
        ctx.save_for_backward(hidden, weight, bias, target, row_weight, kept)
        ctx.numbers = ignore_index, reduction
        return losses if reduction == L.REDUCE_NONE else total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, bias, target, row_weight, kept = ctx.saved_tensors
        head = _Head(hidden, weight, bias, target, row_weight, *ctx.numbers)
        gh, gw, gb = head.backward(kept, grad.float(), *ctx.needs_input_grad[:3])
        return gh, gw, None if gb is None else gb.to(bias.dtype), None, None, None, None


def linear_cross_entropy(hidden, weight, target, bias=None, row_weight=None, ignore_index=-100, reduction="mean"):
    """Cross entropy of ``softmax(hidden @ weight.T + bias)`` at ``target``.

    ``hidden`` (..., features) and ``weight`` (vocabulary, features): fp32, bf16 or fp16, of one type, any strides;
    ``target`` (...): int64 (or int32); ``bias`` (vocabulary,): any floating type, -inf masks an action, whatever its row of the
    weight holds; ``row_weight`` (...): a factor of every row's loss (an advantage weight), no gradient is taken to it.  Rows whose
    target is ``ignore_index`` or whose weight is 0 (padding) contribute nothing, whatever their hidden row holds; any other target
    outside the vocabulary gives NaN.
    ``reduction``: ``"none"`` (losses of target's shape), ``"sum"``, or ``"mean"`` -- the weighted sum over the number of rows
    that are not ignored (0 when there are none).  The loss is fp32.

    Differentiable (once, in reverse mode) with respect to hidden, weight and bias; the gradients have the operands' types.  Logits are never stored:
    the forward pass keeps one logsumexp per row, the backward pass recomputes them in pieces of the vocabulary.  With
    ``reduction="none"`` and no gradient this is the negative log-probability of single tokens (serving).  While a HIP graph is
    captured, no eager loss over the same leaves from the default stream may be alive: such a call is refused, also where no gradient of it
    would be taken (under ``torch.no_grad()`` it is not), and graphs that other operations keep alive are not seen: PyTorch's own
    rule for them holds.

    Precision.  Logits: 16-bit operands are multiplied as they are; fp32 ones lose 2^-23 of themselves or 2^-38 of the largest entry of
    their own row.  Gradients: bf16 operands hold their bits down to 2^-28 of their tensor's largest entry, and ``softmax - onehot``
    beside them loses 2^-11 of itself or 2^-39; beside fp16 operands 2^-22 of itself or 2^-39; fp32 operands, and it beside them, lose
    2^-22 of themselves or, in a row 2^d smaller than the largest one, 2^(d/2 - 38) of the row's largest entry and of 1.  In the weight's
    gradient that is: of the largest row gradient."""
    if reduction not in _REDUCE:
        raise ValueError("reduction: expected 'none', 'mean' or 'sum', got %r" % (reduction,))
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("expected hidden (..., features) and weight (vocabulary, features), got %s and %s" %
                         (tuple(hidden.shape), tuple(weight.shape)))
    if hidden.dtype not in _ELEM or weight.dtype != hidden.dtype:
        raise TypeError("hidden and weight must both be float32, bfloat16 or float16, got %s and %s" % (hidden.dtype, weight.dtype))
    if target.shape != hidden.shape[:-1]:
        raise ValueError("target: expected shape %s, got %s" % (tuple(hidden.shape[:-1]), tuple(target.shape)))
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError("target: expected int64 or int32, got %s" % target.dtype)
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("the vocabulary and the features must not be empty, got weight %s" % (tuple(weight.shape),))
    if bias is not None:
        if tuple(bias.shape) != (weight.shape[0],):
            raise ValueError("bias: expected shape %s, got %s" % ((weight.shape[0],), tuple(bias.shape)))
        if not bias.dtype.is_floating_point:
            raise TypeError("bias: expected a floating type, got %s" % bias.dtype)
    if row_weight is not None:
        if row_weight.shape != target.shape:
            raise ValueError("row_weight: expected shape %s, got %s" % (tuple(target.shape), tuple(row_weight.shape)))
        if row_weight.requires_grad:
            raise ValueError("row_weight: no gradient is taken to the weights of rows; detach them")
    if _has_tangent(hidden, weight, bias, row_weight):
        raise NotImplementedError("linear_cross_entropy has no forward-mode derivative")
    dev = hidden.device
    if dev.type != "cuda":
        raise L.GrlHipError("hidden must live on a HIP device (got %s): there is no CPU fallback" % dev)
    for name, t in (("weight", weight), ("target", target), ("bias", bias), ("row_weight", row_weight)):
        if t is not None and t.device != dev:
            raise ValueError("%s is on %s, hidden on %s" % (name, t.device, dev))
    rows = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    flat = target.reshape(-1).long().contiguous()
    if row_weight is not None:
        row_weight = row_weight.reshape(-1).float().contiguous()
    if rows.shape[0] == 0:   # nothing to launch; the result still has a (zero) gradient
        empty = (rows.float().sum() + weight[:0].float().sum()) + (0.0 if bias is None else bias[:0].float().sum())
        return empty if reduction != "none" else empty + torch.zeros(target.shape, device=hidden.device)
    if torch.is_grad_enabled() and (rows.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        loss = _LinearCrossEntropy.apply(rows, weight, bias, flat, row_weight, int(ignore_index), _REDUCE[reduction])
    else:
        losses, total, _ = _Head(rows, weight, bias, flat, row_weight, int(ignore_index), _REDUCE[reduction]).forward()
        loss = losses if reduction == "none" else total
    return loss.view(target.shape) if reduction == "none" else loss
