"""Losses of a classification head: refusals, on the host, before anything is launched."""
import ctypes
import math

import pytest
import torch

import pcf_nat_b200 as b200
from pcf_nat_b200 import _lib

L = _lib.lib()
BF = torch.bfloat16


def _args(x_dtype=BF, w_dtype=BF, x_shape=(4, 16), w_shape=(10, 16)):
    return torch.zeros(x_shape, dtype=x_dtype), torch.zeros(w_shape, dtype=w_dtype), torch.zeros(x_shape[:-1], dtype=torch.int64)


@pytest.mark.parametrize("f", [b200.linear_cross_entropy, b200.angular_cross_entropy])
def test_label_losses_refuse(f):
    x, w, y = _args()
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x, w, y)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        f(x.float(), w, y)
    with pytest.raises(TypeError, match="weight"):
        f(x, w.half(), y)
    with pytest.raises(ValueError, match="do not go together"):
        f(x, w[:, :8], y)
    with pytest.raises(ValueError, match="do not go together"):
        f(x, w[0], y)
    with pytest.raises(ValueError, match="a class"):
        f(x, w[:0], y)
    with pytest.raises(ValueError, match="reduction"):
        f(x, w, y, reduction="max")
    with pytest.raises(TypeError, match="labels"):
        f(x, w, y.float())
    with pytest.raises(ValueError, match="labels"):
        f(x, w, y[:3])


def test_numbers_that_are_tensors_are_refused():
    x, w, y = _args()
    one = torch.ones((), requires_grad=True)
    for f in (b200.linear_cross_entropy, b200.angular_cross_entropy):
        with pytest.raises(TypeError, match="scale is a number"):
            f(x, w, y, scale=one)
        with pytest.raises(TypeError, match="ignore_index is a number"):
            f(x, w, y, ignore_index=torch.tensor(3))
    with pytest.raises(TypeError, match="margin is a number"):
        b200.angular_cross_entropy(x, w, y, margin=one)
    t, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    for name in ("scale", "temperature"):
        with pytest.raises(TypeError, match=name + " is a number"):
            b200.linear_distillation(x, w, t, i, **{name: one})


def test_distillation_refuses():
    x, w, _ = _args()
    t, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        b200.linear_distillation(x, w, t, i)
    with pytest.raises(ValueError, match="k at least 1"):
        b200.linear_distillation(x, w, t[:, :0], i[:, :0])
    with pytest.raises(ValueError, match="k at least 1"):
        b200.linear_distillation(x, w, t[:, 0], i[:, 0])
    with pytest.raises(ValueError, match="differ in shape"):
        b200.linear_distillation(x, w, t[:, :2], i)
    with pytest.raises(ValueError, match="classes"):
        b200.linear_distillation(x, w, t[:3], i[:3])
    with pytest.raises(TypeError, match="floating"):
        b200.linear_distillation(x, w, i, i)
    with pytest.raises(TypeError, match="classes"):
        b200.linear_distillation(x, w, t, t)


P = 4096   # never dereferenced: validation fails first


def _head(**more):
    d = dict(rows=4, dim=16, classes=10, top=0, x=P, x_stride=16, weight=P, weight_stride=16, labels=P, teacher_logits=None, teacher_index=None,
             ignore_index=-100, scale=1.0, margin=0.0, temperature=1.0, normalize=0, reduction=0, dtype=0, x_type=0, weight_type=0)
    d.update(more)
    return _lib.Head(**d)


@pytest.mark.parametrize("more,status", [
    (dict(rows=0), -2), (dict(dim=0), -2), (dict(classes=0), -2), (dict(top=-1), -2), (dict(reduction=3), -2),
    (dict(rows=(1 << 22) + 1), -9), (dict(dim=(1 << 14) + 1), -9), (dict(classes=(1 << 24) + 1), -9),
    (dict(top=1025, teacher_logits=P, teacher_index=P), -9),
    (dict(dtype=2), -4), (dict(x_type=1), -4), (dict(weight_type=1), -4), (dict(x_type=3), -4),
    (dict(x_stride=-16), -11),
    (dict(scale=0.0), -13), (dict(scale=math.nan), -13), (dict(scale=math.inf), -13), (dict(margin=0.2), -13), (dict(margin=math.nan, normalize=1), -13),
    (dict(top=3, temperature=0.0, teacher_logits=P, teacher_index=P), -13),
    (dict(x=None), -1), (dict(weight=None), -1), (dict(labels=None), -1), (dict(top=3, teacher_logits=P), -1),
    (dict(x=P + 1), -6), (dict(weight=P + 2, weight_type=2), -6), (dict(labels=P + 4), -6),
])
def test_abi_refuses(more, status):
    h = ctypes.byref(_head(**more))
    assert L.na1d_head_saved_bytes(h) == status
    assert L.na1d_head_forward_scratch(h) == status
    assert L.na1d_head_backward_scratch(h, 1, 1) == status
    assert L.na1d_head_forward(h, P, P, P, None) == status
    assert L.na1d_head_backward(h, P, P, P, P, P, None) == status


def test_abi_refuses_buffers():
    h = ctypes.byref(_head())
    assert L.na1d_head_forward(None, P, P, P, None) == -1
    assert L.na1d_head_forward(h, None, P, P, None) == -1
    assert L.na1d_head_forward(h, P, P + 16, P, None) == -6
    assert L.na1d_head_backward(h, None, None, P, P, P, None) == -1
    assert L.na1d_head_backward(h, P + 8, P, P, P, P, None) == -6
    assert len(L.na1d_status_string(-13)) > 3


@pytest.mark.parametrize("rows,dim,classes", [(1, 1, 1), (256, 192, 5994), (8192, 1024, 50000), (1 << 20, 192, 5994)])
def test_buffers_stay_far_below_the_logits(rows, dim, classes):
    h = ctypes.byref(_head(rows=rows, dim=dim, classes=classes, x_stride=dim, weight_stride=(dim + 7) // 8 * 8))
    saved, back = L.na1d_head_saved_bytes(h), L.na1d_head_backward_scratch(h, 1, 1)
    padded = (rows + 255) // 256 * 256
    assert saved <= padded * (2 * (dim + 8) + 64) + 64 * (classes + 256) + 4096   # (a copy of the rows, a few words for each row and class)
    # a piece's gradients (at most 256 MB, or 1024 classes of them), and both products' partial sums
    assert back <= max(256 << 20, padded * 1024 * 2) + 33 * 4 * (dim + 8) * padded + 17 * 4 * (dim + 8) * (classes + 256) + 4096


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("op,dual", [(op, dual) for op in ("ce", "angular", "distill") for dual in ("x", "weight", "teacher") if dual != "teacher" or op == "distill"])
def test_forward_mode_is_refused(op, dual, requires_grad):
    """A tangent on any input, whether or not that input needs a gradient too."""
    x, w, y = _args()
    t, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    f = {"ce": lambda x, w, t: b200.linear_cross_entropy(x, w, y), "angular": lambda x, w, t: b200.angular_cross_entropy(x, w, y),
         "distill": lambda x, w, t: b200.linear_distillation(x, w, t, i)}[op]
    args = [x, w, t]
    n = ["x", "weight", "teacher"].index(dual)
    with torch.autograd.forward_ad.dual_level():
        args[n] = torch.autograd.forward_ad.make_dual(args[n].requires_grad_(requires_grad), torch.ones_like(args[n]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*args)
    args = [x, w, t]
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda a: f(*(a if j == n else b for j, b in enumerate(args))), (args[n].detach(),), (torch.ones_like(args[n]),))


@pytest.mark.parametrize("more,in_place", [
    (dict(), 1), (dict(weight_stride=24), 1), (dict(dtype=1, x_type=1, weight_type=1), 1), (dict(normalize=1), 1),
    (dict(dtype=1, x_type=1, weight_type=1, normalize=1), 0),         # (fp16 cosines: classes times powers of two)
    (dict(weight_type=2), 0), (dict(dim=15), 0), (dict(weight_stride=20), 0), (dict(weight_stride=8), 0), (dict(weight=P + 2), 0),
    (dict(classes=1, weight_stride=19), 0), (dict(scale=0.0), -13),
])
def test_where_the_weight_is_read(more, in_place):
    """The nodes keep the weight itself or rely on the copy in `saved` by this answer; the copy is what makes `saved` larger."""
    h = _head(**more)
    assert L.na1d_head_weight_in_place(ctypes.byref(h)) == in_place
    if in_place >= 0:
        dense = _head(**{**more, "weight": P, "weight_stride": 16, "weight_type": more.get("dtype", 0), "dim": 16, "dtype": 0, "x_type": 0, "weight_type": 0})
        assert (L.na1d_head_saved_bytes(ctypes.byref(h)) > L.na1d_head_saved_bytes(ctypes.byref(dense))) == (in_place == 0)


@pytest.mark.parametrize("rows,classes", [(6400, 200000), (6912, 57500), (7000, 57344), (1024, 200003), (3500, 38000), (256, 1 << 20), (1 << 20, 6000), (3, 1 << 24)])
def test_a_piece_stays_within_its_limit(rows, classes):
    """8 channels, so that nothing else counts: 33 and 17 partial sums of them a row and a class of the piece."""
    h = ctypes.byref(_head(rows=rows, dim=8, classes=classes, x_stride=8, weight_stride=8))
    padded = (rows + 255) // 256 * 256
    piece = max(256 << 20, padded * 1024 * 2)
    assert L.na1d_head_backward_scratch(h, 1, 1) <= piece + 33 * 4 * 8 * padded + 17 * 4 * 8 * (piece // (2 * padded) + 256) + 4096


@pytest.mark.parametrize("more", [
    dict(scale=1e-42), dict(scale=3e38), dict(scale=1e-20, temperature=1e18), dict(scale=1e20, temperature=1e-18), dict(temperature=1e19), dict(temperature=1e-19), dict(scale=1e25, temperature=1e15),
])
def test_scales_that_leave_fp32_together(more):
    """Each is positive and finite; the factor of a logit, the gradient's or the squared temperature is not, or nearly."""
    top = dict(top=3, teacher_logits=P, teacher_index=P)
    assert L.na1d_head_saved_bytes(ctypes.byref(_head(**top, **more))) == -13
    assert L.na1d_head_saved_bytes(ctypes.byref(_head(**top, scale=1e-10, temperature=1e10))) > 0
    if "temperature" not in more:
        assert (L.na1d_head_saved_bytes(ctypes.byref(_head(**more))) == -13) == (more["scale"] > 1)
    assert L.na1d_head_saved_bytes(ctypes.byref(_head(temperature=math.nan))) > 0       # (labels have none)
