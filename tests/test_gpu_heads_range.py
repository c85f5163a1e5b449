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


def _cosine_problem(op, N, D, V, seed):
    """Values that stay exact in both types when they are multiplied with powers of two down to 2^-8."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randint(-31, 32, (V, D), device=DEV, generator=g) / 16.0
    y = torch.randint(0, V // 2, (N,), device=DEV, generator=g)     # (the second half of the classes is no row's own)
    x = torch.randint(-15, 16, (N, D), device=DEV, generator=g) / 16.0 + w[y]
    t, i = torch.randn(N, 4, device=DEV, generator=g), (y[:, None] + torch.arange(4, device=DEV) * 7) % (V // 2)
    return x, w, y, t, i


def _cosine_loss(op, x, w, y, t, i, reduction="sum"):
    if op == "angular":
        return b200.angular_cross_entropy(x, w, y, margin=0.2, scale=30.0, reduction=reduction)
    return b200.linear_distillation(x, w, t, i, scale=30.0, normalize=True, reduction=reduction)


@pytest.mark.parametrize("op", ["angular", "distill"])
@pytest.mark.parametrize("row,cls", [(1e-5, 1.0), (1.0, 1e-5), (1e-3, 1e-3), (1e-4, 1e-4), (30.0, 1e-4)])
def test_one_length_far_from_the_others_in_fp16(op, row, cls):
    """A short row or class costs the others' gradients nothing. Each row's and each class's own error, against what rounding allows whatever the others' lengths are: half a
    step of fp16 (and the logits' fp32 errors) of each gradient of a logit, or half a subnormal step: 2^-25 / 2^5 of a probability."""
    N, D, V = 40, 32, 6000
    x, w, y, t, i = _cosine_problem(op, N, D, V, 1)
    x[3] *= row
    w[17] *= cls
    w[V - 5] *= cls
    x, w = x.half().float().requires_grad_(), w.half().float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.float16):
        _cosine_loss(op, x, w, y, t, i).backward()
    ops.device_status()
    kw = dict(labels=y, margin=0.2) if op == "angular" else dict(teacher_logits=t, teacher_index=i)
    r = orc.evaluate(x.detach().half(), w.detach().half(), scale=30.0, normalize=True, reduction="sum", **kw)
    z, _, ix, iw, slope = orc.logits(x.detach(), w.detach(), 30.0, True, kw.get("labels"), kw.get("margin", 0.0))
    h = torch.softmax(z, 1)
    if op == "angular":
        h.scatter_(1, y[:, None], (h.gather(1, y[:, None]) - 1) * slope[:, None])
    else:
        h.scatter_add_(1, i, -orc.teacher_probabilities(t, i, 1.0)[0])
    relative = 2.0 ** -11 + 4 * 30 * (D + 8) * 2.0 ** -23
    for got, ref, inverse, sums, terms in ((x.grad, r["dx"], ix, h.abs().sum(1), V), (w.grad, r["dw"], iw, h.abs().sum(0), N)):
        off = 30 * inverse * (sums * (relative + (terms + D + 16) * 2.0 ** -23) + terms * 2.0 ** -30)
        err = (got.double() - ref).norm(dim=1)
        assert bool((err <= off).all()), float((err / off).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("copy", [False, True])
@pytest.mark.parametrize("op", ["angular", "distill"])
def test_powers_of_two_of_single_rows_change_no_bits(op, copy, dtype):
    """Cosines do not know a row's length, nor do the other rows' gradients: the same bits, its own gradient times the inverse power."""
    N, D, V = 60, 64, 3000
    x, w, y, t, i = _cosine_problem(op, N, D, V, 2)
    a, b = torch.ones(N, 1, device=DEV), torch.ones(V, 1, device=DEV)
    a[5], a[6], b[9], b[V - 2] = 2.0 ** -8, 2.0 ** 4, 2.0 ** -7, 2.0 ** 5
    got = []
    for p, q in ((torch.ones_like(a), torch.ones_like(b)), (a, b)):
        u, v = (x * p).to(dtype), (w * q).to(dtype if not copy else torch.float32)
        assert torch.equal(u.float(), x * p) and torch.equal(v.float(), w * q)
        u, v = u.requires_grad_(), v.requires_grad_()
        loss = _cosine_loss(op, u, v, y, t, i, "none")
        gu, gv = torch.autograd.grad((loss * 2.0 ** -9).sum(), (u, v))    # (no gradient leaves fp16's range)
        got.append((loss.detach(), gu.float() * p, gv.float() * q))
    same = [torch.equal(s, r) for s, r in zip(*got)]
    if dtype == torch.float16:            # (results below 2^-14 have fewer bits)
        off = 2.0 ** -24 * torch.maximum(p, torch.ones_like(p)), 2.0 ** -24 * torch.maximum(q, torch.ones_like(q))
        near = [bool(((s - r).abs() <= o).all()) for s, r, o in zip(got[0][1:], got[1][1:], off)]
        same[1:] = [s or n for s, n in zip(same[1:], near)]
    assert same == [True] * 3


@pytest.mark.parametrize("copy", [False, True])
@pytest.mark.parametrize("D", [64, 57, 320])
@pytest.mark.parametrize("op", ["angular", "distill"])
def test_lengths_whose_squares_leave_fp32(op, D, copy):
    """bfloat16 rows and classes of 1e-27 to 1e27: as above, no bit changes but the powers of two and what falls into subnormals, which have a step of 2^-133 in bfloat16
    and 2^-149 in fp32. A gradient there is off by half a step, times the power that is taken out of it here. With the weight in its place a gradient of a logit is
    divided by the class's own length: half a step of 2^-133 of each, 30 times as large in the result, reaches dx times the class's elements (up to 2) and dw times the
    N kept rows' (up to 2). The projection at most adds sqrt(D) times that, and results that differ at all may be rounded apart, half a step each."""
    N, V = 60, 500
    x, w, y, t, i = _cosine_problem(op, N, D, V, 3)
    a, b = torch.ones(N, 1, device=DEV), torch.ones(V, 1, device=DEV)
    a[5], a[6], a[7], a[8] = 2.0 ** -90, 2.0 ** 90, 2.0 ** -64, 2.0 ** 66
    b[9], b[V - 2], b[11], b[V - 4] = 2.0 ** -90, 2.0 ** 90, 2.0 ** 70, 2.0 ** -62
    b[y[20]], b[y[21]] = 2.0 ** -90, 2.0 ** 88
    got = []
    for p, q in ((torch.ones_like(a), torch.ones_like(b)), (a, b)):
        u, v = (x * p).bfloat16().requires_grad_(), (w * q).to(torch.float32 if copy else torch.bfloat16).requires_grad_()
        loss = _cosine_loss(op, u, v, y, t, i, "none")
        gu, gv = torch.autograd.grad(loss.sum(), (u, v))
        got.append((loss.detach(), gu.float() * p, gv.float() * q))
    ops.device_status()
    assert torch.equal(got[0][0], got[1][0])
    for s, r, power, out, products in ((got[0][1], got[1][1], a, u.dtype, 2 * b[b > 1].sum()), (got[0][2], got[1][2], b, v.dtype, 2 * N * b * (b > 1))):
        f, power, products = torch.finfo(out), power.double(), products.double()
        off = f.tiny * f.eps / 2 * power + 2.0 ** -150 * power
        if not copy:
            moved = 30 * 2.0 ** -134 * products * (1 + D ** 0.5)
            off = off + moved + torch.where(moved > 0, f.eps * (s.abs() + moved), 0.0)
        assert bool(torch.isfinite(r).all()) and bool(((s - r).abs() <= off).all())


@pytest.mark.parametrize("copy", [False, True])
@pytest.mark.parametrize("op", ["angular", "distill"])
def test_rows_without_a_length(op, copy):
    """Shorter than 2^-126: as rows of zeros. An infinity: NaN, in the row's loss and gradient alone, or (in a class) in all."""
    N, D, V = 60, 64, 500
    x, w, y, t, i = _cosine_problem(op, N, D, V, 4)
    wt = torch.float32 if copy else torch.bfloat16

    def run(x, w):
        u, v = x.bfloat16().requires_grad_(), w.to(wt, copy=True).requires_grad_()
        loss = _cosine_loss(op, u, v, y, t, i, "none")
        return (loss.detach(),) + torch.autograd.grad(loss.sum(), (u, v))
    tiny, zero = [x.clone(), w.clone()], [x.clone(), w.clone()]
    for s, n in ((0, 5), (1, 9), (1, int(y[20]))):
        tiny[s][n] = 2.0 ** -133 * torch.randint(-1, 2, (D,), device=DEV)
        zero[s][n] = 0
    assert bool(tiny[0].bfloat16()[5].any()) and all(torch.equal(p, q) for p, q in zip(run(*tiny), run(*zero)))
    x[7, 3] = float("inf")
    loss, dx, dw = run(x, w)
    rows = torch.arange(N, device=DEV) == 7
    assert torch.equal(loss.isnan(), rows) and torch.equal(dx.isnan().all(1), rows) and torch.equal(dx.isnan().any(1), rows) and bool(dw.isnan().all())
    x[7, 3], w[400, 2] = 1.0, -float("inf")
    assert all(bool(g.isnan().all()) for g in run(x, w)[:2])


@pytest.mark.parametrize("op", ["ce", "angular"])
def test_tiny_factors_of_rows_in_fp16(op):
    """Factors of 2^-130 give 2^-130 times the gradients of factors of 1, to the fp32 weight: half a step of 2^-149 off, and for its two roundings the same again."""
    g = torch.Generator(device=DEV).manual_seed(6)
    x, w = torch.randn(50, 64, device=DEV, generator=g).half(), torch.randn(300, 64, device=DEV, generator=g).half().float().requires_grad_()
    y = torch.randint(0, 300, (50,), device=DEV, generator=g)
    f = b200.linear_cross_entropy if op == "ce" else b200.angular_cross_entropy
    (one,), (tiny,) = (torch.autograd.grad(f(x, w, y, reduction="none"), w, torch.full((50,), d, device=DEV)) for d in (1.0, 2.0 ** -130))
    # Gradients of logits are relative to 2^-120 then, ten bits fewer: half a subnormal step is 2^-25 / 2^(14 - 10), or 2^-25 / 2^(5 - 10) of cosines. Those above
    # are rounded in both, half a step of 2^-11 each. The projection at most doubles what lies along a class and adds it elsewhere: its length.
    z, _, ix, iw, slope = orc.logits(x, w.detach(), 1.0 if op == "ce" else 30.0, op != "ce", y, 0.0 if op == "ce" else 0.2)
    h = torch.softmax(z, 1)
    h.scatter_(1, y[:, None], (h.gather(1, y[:, None]) - 1) * slope[:, None])
    each = 2.0 ** -10 * h.abs() + (2.0 ** -29 if op == "ce" else 2.0 ** -20)
    if op == "ce":
        size = each.t() @ x.double().abs()
    else:
        size = 30 * iw[:, None] * (each.t() @ (x.double().abs() * ix[:, None]))
        size = size + size.norm(dim=1, keepdim=True)
    assert bool(torch.isfinite(tiny).all()) and bool(((tiny.double() * 2.0 ** 130 - one.double()).abs() <= size + 2.0 ** -149 * 2.0 ** 130).all())


@pytest.mark.parametrize("op", ["ce", "angular"])
@pytest.mark.parametrize("dtype", TYPES)
def test_an_infinite_factor_is_its_row_s_alone(op, dtype):
    """The other rows' gradients are those beside a factor of 0 there."""
    g = torch.Generator(device=DEV).manual_seed(7)
    x, w = torch.randn(50, 64, device=DEV, generator=g).requires_grad_(), torch.randn(300, 64, device=DEV, generator=g).to(dtype)
    y = torch.randint(0, 300, (50,), device=DEV, generator=g)
    f = b200.linear_cross_entropy if op == "ce" else b200.angular_cross_entropy
    d = 65536.0 * torch.rand(50, device=DEV, generator=g)
    got = []
    for v in (0.0, float("inf")):
        d[4] = v
        with torch.autocast("cuda", dtype=dtype):
            loss = f(x, w, y, reduction="none")
        got.append(torch.autograd.grad(loss, x, d)[0])
    rest = torch.arange(50, device=DEV) != 4
    assert bool(torch.isfinite(got[0][rest]).all()) and torch.equal(got[0][rest], got[1][rest]) and not bool(torch.isfinite(got[1][4]).any())
