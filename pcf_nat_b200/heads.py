"""Losses of a classification head that never stores its (rows, classes) logits.

``model.AAMSoftmax`` computes the extractor's loss as PyTorch does: fp32 cosines of every row and class, their softmax, both kept for the
backward pass. With many rows (a label for every frame), many classes, or a vocabulary, these tensors are the largest of the
whole step. Here the products run tile by tile on the tensor cores and leave a maximum and a sum per row and 64 classes (rows x classes / 8 bytes
of workspace); the backward pass forms them again, a piece of the classes at a time, as 16-bit gradients that the products with weight and rows read next.

* ``linear_cross_entropy``   softmax cross entropy of ``scale * x @ weight.T``
* ``angular_cross_entropy``  of scaled cosines with an additive angular margin (AAM-softmax)
* ``linear_distillation``    Kullback-Leibler divergence from a teacher's top logits

``x`` is bfloat16 or float16 (or, under autocast, float32, rounded to autocast's type), ``weight`` of the same type or float32 (then
rounded to that type, as autocast does with a projection's; its gradient is float32). Rows may have any stride; there may be up to
2^22 of them, of up to 2^14 channels, and 2^24 classes. Losses are float32.
"""
import ctypes

import torch

from . import _lib, ops
from ._lib import check

_L = _lib.lib()
_CODE = {torch.bfloat16: _lib.NA1D_BF16, torch.float16: _lib.NA1D_FP16, torch.float32: _lib.NA1D_FP32}
_REDUCTION = {"mean": 0, "sum": 1, "none": 2}


def _bytes(status, where):
    if status < 0:
        check(status, where)
    return status


def _buffer(n, device):
    return torch.empty(max(int(n), 1), dtype=torch.uint8, device=device)


def _head(cfg, x, weight, labels, teacher_logits, teacher_index):
    code, ignore_index, scale, margin, temperature, normalize, reduction = cfg
    return _lib.Head(rows=x.shape[0], dim=x.shape[1], classes=weight.shape[0], top=0 if teacher_index is None else teacher_index.shape[1], x=x.data_ptr(),
                     x_stride=x.stride(0), weight=weight.data_ptr(), weight_stride=weight.stride(0), labels=None if labels is None else labels.data_ptr(),
                     teacher_logits=None if teacher_logits is None else teacher_logits.data_ptr(),
                     teacher_index=None if teacher_index is None else teacher_index.data_ptr(), ignore_index=ignore_index, scale=scale, margin=margin,
                     temperature=temperature, normalize=int(normalize), reduction=reduction, dtype=code, x_type=_CODE[x.dtype],
                     weight_type=_CODE[weight.dtype])


def _forward(cfg, x, weight, labels, teacher_logits, teacher_index):
    head = _head(cfg, x, weight, labels, teacher_logits, teacher_index)
    ref = ctypes.byref(head)
    with ops._on_device(x.device):
        saved = _buffer(_bytes(_L.na1d_head_saved_bytes(ref), "na1d_head_saved_bytes"), x.device)
        scratch = _buffer(_bytes(_L.na1d_head_forward_scratch(ref), "na1d_head_forward_scratch"), x.device)
        loss = torch.empty((x.shape[0],) if cfg[-1] == 2 else (), dtype=torch.float32, device=x.device)
        check(_L.na1d_head_forward(ref, loss.data_ptr(), saved.data_ptr(), scratch.data_ptr(), ops._stream(x)), "na1d_head_forward")
    return loss, saved, head


def _in_place(head, weight):
    """Makes `weight` the head's: whether the kernels read it there (`saved` has no copy of it)."""
    head.weight, head.weight_stride = weight.data_ptr(), weight.stride(0)
    return bool(_bytes(_L.na1d_head_weight_in_place(ctypes.byref(head)), "na1d_head_weight_in_place"))


class _HeadFunction(torch.autograd.Function):
    """The route of calls that the C++ node (csrc/torch_nodes.cpp) leaves to Python."""

    @staticmethod
    def forward(ctx, x, weight, labels, teacher_logits, teacher_index, cfg):
        loss, saved, head = _forward(cfg, x, weight, labels, teacher_logits, teacher_index)
        # the weight is read again where it is, unless the forward pass made a copy of its own (then the copy is in `saved`)
        ctx.in_place = _in_place(head, weight)
        ctx.save_for_backward(saved, weight if ctx.in_place else None)
        ctx.head, ctx.x_dtype, ctx.w_dtype = head, x.dtype, weight.dtype
        ctx.set_materialize_grads(False)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss):
        if d_loss is None:
            return (None,) * 6
        saved, weight = ctx.saved_tensors
        head, want_x, want_w = _lib.Head.from_buffer_copy(ctx.head), ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        dev = saved.device
        with ops._on_device(dev):
            saved = saved.contiguous()                  # (saved tensors come back from wherever a hook has put them, in any stride)
            if saved.data_ptr() % 256:
                saved = saved.clone()
            head.x = head.labels = head.teacher_logits = head.teacher_index = saved.data_ptr()   # not read any more
            if ctx.in_place:
                if weight.stride(1) != 1 or not _in_place(head, weight):
                    weight = weight.clone(memory_format=torch.contiguous_format)
                    if not _in_place(head, weight):
                        raise RuntimeError("a head's weight came back from a saved-tensor hook in a form that it did not have")
            ref = ctypes.byref(head)
            d_loss = d_loss.to(torch.float32).contiguous()
            dx = torch.empty((head.rows, head.dim), dtype=ctx.x_dtype, device=dev) if want_x else None
            dw = torch.empty((head.classes, head.dim), dtype=ctx.w_dtype, device=dev) if want_w else None
            scratch = _buffer(_bytes(_L.na1d_head_backward_scratch(ref, want_x, want_w), "na1d_head_backward_scratch"), dev)
            check(_L.na1d_head_backward(ref, dx.data_ptr() if want_x else None, dw.data_ptr() if want_w else None, d_loss.data_ptr(), saved.data_ptr(),
                                        scratch.data_ptr(), ops._stream(saved)), "na1d_head_backward")
        return dx, dw, None, None, None, None


# ------------------------------------------------------------------ arguments
def _compute_type(x, weight):
    """Type of the products: x's own 16-bit type, or autocast's for float32 rows."""
    dt = x.dtype
    if dt == torch.float32 and torch.is_autocast_enabled(x.device.type):
        dt = torch.get_autocast_dtype(x.device.type)
    if dt not in (torch.bfloat16, torch.float16):
        raise TypeError("a head's rows are bfloat16 or float16 (float32 under autocast to one of them), got %s" % x.dtype)
    if weight.dtype not in (dt, torch.float32):
        raise TypeError("the weight of a head with %s rows is of that type or float32, got %s" % (dt, weight.dtype))
    return dt


def _rows(x, weight, reduction):
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("x and weight are tensors")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError("x (..., dim) and weight (classes, dim) do not go together: %s and %s" % (tuple(x.shape), tuple(weight.shape)))
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("a head needs a class and a channel, got a weight of %s" % (tuple(weight.shape),))
    if reduction not in _REDUCTION:
        raise ValueError("reduction is 'mean', 'sum' or 'none', got %r" % (reduction,))
    if torch.compiler.is_compiling():
        raise NotImplementedError("the losses of a head are eager operators")
    _no_tangents(x, weight)
    return _compute_type(x, weight)


def _no_tangents(*ts):
    """Forward-mode differentiation is refused: a tangent on an input that needs no gradient would be dropped without a word. (The C++ node does not
    take such inputs.)"""
    if any(isinstance(t, torch.Tensor) and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError("the losses of a head have no forward-mode derivative")


def _index(t, shape, name):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32):
        raise TypeError("%s are int64 or int32 tensors" % name)
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s have shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))


def _run(dt, x, weight, labels, teacher_logits, teacher_index, cfg, reduction):
    tensors = [t for t in (x, weight, labels, teacher_logits, teacher_index) if t is not None]
    ops._need_cuda(*tensors)
    if any(t.device != x.device for t in tensors):
        raise ValueError("the tensors of a head are on different devices: %s" % ", ".join(str(t.device) for t in tensors))
    shape = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1])
    if x2.shape[0] == 0:
        # no rows: a loss of zero that still belongs to the graph (of no row of the weight either: it may hold infinities)
        zero = x.sum(dtype=torch.float32) + weight[:0].sum(dtype=torch.float32)
        return zero if reduction != "none" else zero.expand(shape) + torch.zeros(shape, device=x.device)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    w = weight if weight.stride(1) == 1 or weight.shape[1] == 1 else weight.contiguous()
    cfg = (_CODE[dt],) + cfg + (_REDUCTION[reduction],)
    with torch.autocast(x.device.type, enabled=False):
        if torch.is_grad_enabled() and (x2.requires_grad or w.requires_grad):
            loss = _HeadFunction.apply(x2, w, labels, teacher_logits, teacher_index, cfg)
        else:
            loss = _forward(cfg, x2, w, labels, teacher_logits, teacher_index)[0]
    return loss.view(shape) if reduction == "none" else loss


def _labels_loss(x, weight, labels, cfg, reduction):
    """What the C++ node (``ops.native.head``) did not take: checks, conversions, the Python route."""
    dt = _rows(x, weight, reduction)
    _index(labels, x.shape[:-1], "labels")
    return _run(dt, x, weight, labels.reshape(-1).to(torch.int64).contiguous(), None, None, cfg, reduction)


def _numbers(**named):
    for name, v in named.items():
        if isinstance(v, torch.Tensor):   # (it would be read back from the device, and get no gradient)
            raise TypeError("%s is a number, got a tensor" % name)


def _tensors(*ts):
    return all(isinstance(t, torch.Tensor) for t in ts) and not torch.compiler.is_compiling()


# ------------------------------------------------------------------ the losses
def linear_cross_entropy(x, weight, labels, *, scale=1.0, ignore_index=-100, reduction="mean"):
    """``F.cross_entropy(scale * x @ weight.T, labels)`` without the logits.

    ``x`` (..., dim), ``weight`` (classes, dim), ``labels`` (...) int64 or int32. Rows labelled ``ignore_index`` do not count: nothing in
    them reaches the loss or a gradient, and no time goes into them; where no row counts the mean is 0. A label outside the classes makes
    its row's loss, and the gradients that depend on it, NaN (there is no synchronisation to raise an error from). ``reduction``: "mean" over
    the rows that count, "sum", or "none" (0 for the others; a float16 gradient of a logit is held relative to the largest factor of any row, and keeps all its digits
    down to 2^-28 of it, of cosines 2^-19). Differentiable once in ``x`` and ``weight``; same bits from run to run."""
    _numbers(scale=scale, ignore_index=ignore_index)
    loss = None
    if _tensors(x, weight, labels):
        loss = ops.native.head(x, weight, labels, None, None, scale, 0.0, 1.0, False, ignore_index, _REDUCTION.get(reduction, -1))
    return _labels_loss(x, weight, labels, (int(ignore_index), float(scale), 0.0, 1.0, False), reduction) if loss is None else loss


def angular_cross_entropy(x, weight, labels, *, margin=0.2, scale=30.0, ignore_index=-100, reduction="mean"):
    """AAM-softmax: cross entropy of ``scale`` times the cosines of rows and classes, the label's angle widened by ``margin`` radians
    (``model.AAMSoftmax``; cos(a + m) as cos a cos m - sin a sin m, the squared sine at least 2e-7). A row or class of zeros (or shorter than
    2^-126) has cosine 0 with all others and no gradient; one with an infinity is NaN. Where the weight is read in its place (16-bit, dense), a probability
    over its class's length below 2^-126 reaches the gradients with fewer digits. Otherwise as ``linear_cross_entropy``."""
    _numbers(margin=margin, scale=scale, ignore_index=ignore_index)
    loss = None
    if _tensors(x, weight, labels):
        loss = ops.native.head(x, weight, labels, None, None, scale, margin, 1.0, True, ignore_index, _REDUCTION.get(reduction, -1))
    return _labels_loss(x, weight, labels, (int(ignore_index), float(scale), float(margin), 1.0, True), reduction) if loss is None else loss


def linear_distillation(x, weight, teacher_logits, teacher_index, *, temperature=1.0, scale=1.0, normalize=False, reduction="mean"):
    """``temperature**2 * KL(q || p)``: p the softmax over all classes of ``scale * x @ weight.T / temperature`` (``normalize``: of scaled
    cosines), q that of a teacher's kept logits, ``teacher_logits / temperature``, over a row's entries.

    ``teacher_logits`` (..., k) of any floating type, ``teacher_index`` (..., k) int64 or int32: the entries' classes, negative where there is
    no entry (its logit is not read). Rows without an entry do not count; a class may come twice. k is at most 1024. No gradient
    goes to the teacher. Otherwise as ``linear_cross_entropy``."""
    _numbers(temperature=temperature, scale=scale)
    if _tensors(x, weight, teacher_logits, teacher_index):
        loss = ops.native.head(x, weight, None, teacher_logits, teacher_index, scale, 0.0, temperature, normalize, 0, _REDUCTION.get(reduction, -1))
        if loss is not None:
            return loss
    cfg = (0, float(scale), 0.0, float(temperature), bool(normalize))
    dt = _rows(x, weight, reduction)
    _no_tangents(teacher_logits)
    if not isinstance(teacher_index, torch.Tensor) or teacher_index.dim() != x.dim() or teacher_index.shape[-1] == 0:
        raise ValueError("teacher_index is (..., k) for x (..., dim), k at least 1")
    _index(teacher_index, x.shape[:-1] + teacher_index.shape[-1:], "a teacher's classes")
    if not isinstance(teacher_logits, torch.Tensor) or not teacher_logits.is_floating_point():
        raise TypeError("a teacher's logits are a floating tensor")
    if teacher_logits.shape != teacher_index.shape:
        raise ValueError("a teacher's logits %s and classes %s differ in shape" % (tuple(teacher_logits.shape), tuple(teacher_index.shape)))
    k = teacher_index.shape[-1]
    logits = teacher_logits.detach().reshape(-1, k).to(torch.float32).contiguous()
    index = teacher_index.reshape(-1, k).to(torch.int64).contiguous()
    return _run(dt, x, weight, None, logits, index, cfg, reduction)
