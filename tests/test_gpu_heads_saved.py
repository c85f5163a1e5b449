"""What a head keeps for its backward pass, given back by saved-tensor hooks in other places and strides: the same gradients."""
import pytest
import torch

import pcf_nat_b200 as b200
from pcf_nat_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _same(step, unpack, python, monkeypatch):
    if python:
        monkeypatch.setattr(ops, "native", ops._PythonRoutes)
    want = step()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
        got = step()
    ops.device_status()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("classes", [1, 2, 500])
def test_weight_in_padded_rows_with_an_aligned_start(classes, python, monkeypatch):
    """A single row counts as contiguous whatever its stride is; a stride that the forward pass would have copied away is no sign of a copy."""
    g = torch.Generator(device=DEV).manual_seed(classes)
    x = torch.randn(200, 64, device=DEV, generator=g).bfloat16()
    w = (0.2 * torch.randn(classes, 64, device=DEV, generator=g)).bfloat16()
    y = torch.randint(0, classes, (200,), device=DEV, generator=g)

    def step():
        x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(b200.linear_cross_entropy(x1, w1, y), (x1, w1))

    def unpack(t):
        if t.dim() == 1:
            return t
        padded = torch.cat([t, t.new_full((t.shape[0], 3), float("nan"))], 1)[:, :64]
        assert padded.stride(0) == 67 and padded.data_ptr() % 16 == 0
        return padded
    _same(step, unpack, python, monkeypatch)


@pytest.mark.parametrize("python", [False, True])
def test_kept_buffer_with_a_stride(python, monkeypatch):
    """Every second byte of a larger tensor: rows, entries and places in it would be read as anything."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(200, 64, device=DEV, generator=g).bfloat16()
    w = (0.2 * torch.randn(500, 64, device=DEV, generator=g)).bfloat16()
    t, i = torch.randn(200, 5, device=DEV, generator=g), torch.randint(0, 500, (200, 5), device=DEV, generator=g)

    def step():
        x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(b200.linear_distillation(x1, w1, t, i), (x1, w1))

    def unpack(t):
        if t.dim() != 1:
            return t
        wide = t.new_zeros(2 * t.numel())
        wide[::2] = t
        assert wide[::2].stride(0) == 2 and wide.data_ptr() % 256 == 0
        return wide[::2]
    _same(step, unpack, python, monkeypatch)
