"""Losses of a head at the ends of their types' ranges: wide margins, lengths far apart, factors far apart."""
import math

import pytest
import torch

import pcf_nat_b200 as b200
from pcf_nat_b200 import ops
from oracle import head_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("margin", [0.5, 1.0, math.pi / 2, 2.5])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_wide_margins_at_a_sine_of_zero(dtype, sign, margin):
    """Rows along their class or opposite to it, every class there twice: the margin's slope reaches cos m + sin m / sqrt(2e-7) where rounding leaves the squared
    sine just above its floor, and the probability stays away from 1. The own class's part lies along the row and is projected away, so the gradients
    are of the others' size. What stays of it is fp32 rounding: V + D sums and 16 other operations of a term `slope` times as large. A cosine off by
    `off` also moves the sine, at its floor, and with it the label's logit and every probability of the row."""
    N, D, V = 4000, 64, 2000
    g = torch.Generator(device=DEV).manual_seed(5)
    half = torch.nn.functional.normalize(torch.randn(V // 2, D, device=DEV, generator=g), dim=1)
    half = half * (1.005 + 0.075 * torch.rand(V // 2, 1, device=DEV, generator=g))      # (products of inverse lengths a little below a power of two)
    w = torch.cat([half, half]).to(dtype)
    y = torch.randint(0, V, (N,), device=DEV, generator=g)
    x = sign * w[y]
    x, w = x.requires_grad_(), w.requires_grad_()
    b200.angular_cross_entropy(x, w, y, margin=margin, scale=20.0, reduction="sum").backward()
    ops.device_status()
    r = orc.evaluate(x.detach(), w.detach(), labels=y, scale=20.0, margin=margin, normalize=True, reduction="sum")
    slope = 1 + abs(math.sin(margin)) / math.sqrt(orc.FLOOR)
    u = torch.finfo(dtype).eps / 2
    off = (D + 16) * 2.0 ** -23
    moved = math.expm1(20.0 * abs(math.sin(margin)) * (math.sqrt(orc.FLOOR + 2 * off) - math.sqrt(orc.FLOOR)))
    rest = ((V + D + 16) * 2.0 ** -23 * slope + moved) * 20.0
    for got, ref, other, own in ((x.grad, r["dx"], w, x), (w.grad, r["dw"], x, w)):
        # terms of the other operand's rows over this one's length; the weight's rows have some N / V of them, 16 at most
        size = rest / own.detach().double().norm(dim=1) * (1 if own is x else 16)
        err, scale = (got.double() - ref).norm(dim=1), ref.norm(dim=1)
        assert bool(torch.isfinite(got).all())
        # (each gradient of a logit rounded once, up to 20 times the row's length; the result once more)
        parts = 20.0 / own.detach().double().norm(dim=1) * u * (1 if own is x else 16)
        assert bool((err <= size + parts + u * scale).all())
