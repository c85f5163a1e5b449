"""Losses of a classification head against their formulas in 64 bits. Bounds are derived in oracle/head_oracle.py."""
import pytest
import torch

import pcf_nat_b200 as b200
from pcf_nat_b200 import ops
from oracle import head_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def make(N, D, V, dtype, seed=0, cosine=False, k=0, ignored=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * N + 13 * D + V)
    w = (torch.randn(V, D, device=DEV, generator=g) * (0.05 if cosine else 2 * D ** -0.5)).to(dtype)
    y = torch.randint(0, V, (N,), device=DEV, generator=g)
    x = torch.randn(N, D, device=DEV, generator=g)
    x = (x + 0.4 * x.norm(dim=1, keepdim=True) * torch.nn.functional.normalize(w[y].float(), dim=1)).to(dtype)
    if ignored:
        y[torch.randperm(N, device=DEV, generator=g)[:ignored]] = -100
    if not k:
        return x, w, y
    t = 3 * torch.randn(N, k, device=DEV, generator=g)
    i = (y.clamp_min(0)[:, None] + torch.arange(k, device=DEV) * max(1, V // (k + 1))) % V
    return x, w, y, t, i


def near(got, ref, off, what):
    assert got.shape == ref.shape, what
    err = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all()), what
    worst = float((err / off).max()) if err.numel() else 0.0
    assert worst <= 1, "%s: %.3g times its bound (error %.3g)" % (what, worst, float(err.max()))


def compare(f, x, w, more, oracle, reduction="mean", d_loss=1.0):
    x, w = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = f(x, w, *more, reduction=reduction)
    assert loss.dtype == torch.float32
    d = torch.as_tensor(d_loss, dtype=torch.float32, device=DEV)
    loss.backward(d)
    r = orc.evaluate(x.detach(), w.detach(), reduction=reduction, d_loss=d if reduction == "none" else float(d), **oracle)
    ops.device_status()
    near(loss.detach(), r["loss"], r["loss_off"] + 2 ** -22 * r["loss"].abs(), "loss")
    near(x.grad, r["dx"], orc.rounded(r["dx"], r["dx_off"], x.dtype), "dx")
    near(w.grad, r["dw"], orc.rounded(r["dw"], r["dw_off"], w.dtype), "dw")
    return loss.detach(), x.grad, w.grad


SIZES = [(1, 192, 5994), (1, 8, 1), (2, 16, 2), (3, 40, 129), (17, 64, 127), (127, 72, 128), (128, 24, 257), (129, 192, 600), (255, 200, 255), (256, 256, 256),
         (257, 264, 1000), (300, 320, 513), (700, 520, 2100), (40, 1032, 300), (33, 57, 77), (5, 1, 9), (64, 191, 3001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", SIZES)
def test_cross_entropy(N, D, V, dtype):
    x, w, y = make(N, D, V, dtype)
    compare(b200.linear_cross_entropy, x, w, (y,), dict(labels=y))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", SIZES)
def test_angular(N, D, V, dtype):
    x, w, y = make(N, D, V, dtype, cosine=True)
    if D == 1:      # cosines of +-1: the margin's slope has no bound there
        x, w, y = make(N, 8, V, dtype, cosine=True)
    compare(b200.angular_cross_entropy, x, w, (y,), dict(labels=y, scale=30.0, margin=0.2, normalize=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cosine", [False, True])
@pytest.mark.parametrize("N,D,V,k,tau", [(1, 192, 5994, 8, 2.0), (3, 40, 129, 1, 1.0), (129, 192, 600, 32, 4.0), (257, 264, 1000, 33, 1.0), (65, 72, 64, 64, 2.0), (20, 57, 2100, 100, 1.0)])
def test_distillation(N, D, V, k, tau, cosine, dtype):
    x, w, _, t, i = make(N, D, V, dtype, cosine=cosine, k=k)
    scale = 20.0 if cosine else 1.0
    f = lambda x, w, t, i, reduction: b200.linear_distillation(x, w, t, i, temperature=tau, scale=scale, normalize=cosine, reduction=reduction)  # noqa: E731
    compare(f, x, w, (t, i), dict(teacher_logits=t, teacher_index=i, temperature=tau, scale=scale, normalize=cosine))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
def test_reductions_and_rows_that_do_not_count(op, reduction, dtype):
    N, D, V = 300, 96, 700
    x, w, y, t, i = make(N, D, V, dtype, cosine=op == "angular", k=5, ignored=120)
    off = y == -100
    x[off] = float("nan")          # nothing of these rows is read
    d = torch.randn(N, device=DEV) * torch.rand(N, device=DEV).mul(-6).exp2() if reduction == "none" else 3.0
    if op == "ce":
        f, more, o = b200.linear_cross_entropy, (y,), dict(labels=y)
    elif op == "angular":
        f, more, o = b200.angular_cross_entropy, (y,), dict(labels=y, scale=30.0, margin=0.2, normalize=True)
    else:
        t[off] = float("nan")
        i[off] = -1
        i[::3, 1] = -1             # and fewer entries in others
        t[::3, 1] = float("inf")
        f, more, o = b200.linear_distillation, (t, i), dict(teacher_logits=t, teacher_index=i)
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = f(x1, w1, *more, reduction=reduction)
    loss.backward(torch.as_tensor(d, device=DEV, dtype=torch.float32))
    clean = torch.where(off[:, None], torch.zeros_like(x), x)
    if op == "distill":
        o["teacher_logits"] = torch.where(i < 0, torch.zeros_like(t), t)
    r = orc.evaluate(clean, w, reduction=reduction, d_loss=d, **o)
    near(loss.detach(), r["loss"], r["loss_off"] + 2 ** -22 * r["loss"].abs(), "loss")
    near(x1.grad, r["dx"], orc.rounded(r["dx"], r["dx_off"], dtype), "dx")
    near(w1.grad, r["dw"], orc.rounded(r["dw"], r["dw_off"], dtype), "dw")
    assert not x1.grad[off].any()
    if reduction == "none":
        assert not loss[off].any()


@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_row_counts(op, reduction):
    N, D, V = 70, 64, 300
    x, w, y, t, i = make(N, D, V, torch.bfloat16, k=3, ignored=N)
    x, w = x.fill_(float("nan")).requires_grad_(), w.requires_grad_()
    if op == "distill":
        t[:35] = -float("inf")     # entries without probability, and rows without entries
        i[35:] = -1
        loss = b200.linear_distillation(x, w, t, i, reduction=reduction)
    else:
        f = b200.linear_cross_entropy if op == "ce" else b200.angular_cross_entropy
        loss = f(x, w, y, reduction=reduction)
    loss.sum().backward()
    assert not loss.any() and not x.grad.any() and not w.grad.any()
    assert loss.shape == (() if reduction != "none" else (N,))


def test_no_rows():
    x, w = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True), torch.randn(30, 64, device=DEV).bfloat16().requires_grad_()
    y = torch.zeros(0, dtype=torch.int64, device=DEV)
    loss = b200.linear_cross_entropy(x, w, y)
    loss.backward()
    assert float(loss) == 0 and not w.grad.any() and x.grad.shape == x.shape
    assert b200.linear_cross_entropy(x, w, y, reduction="none").shape == (0,)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_rows_of_a_weight_with_infinities(reduction):
    x, w = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True), torch.full((30, 64), float("inf"), device=DEV).bfloat16().requires_grad_()
    loss = b200.linear_cross_entropy(x, w, torch.zeros(0, dtype=torch.int64, device=DEV), reduction=reduction)
    assert not loss.any() and loss.shape == ((0,) if reduction == "none" else ())
    loss.sum().backward()
    assert w.grad.shape == w.shape and not w.grad.any()


@pytest.mark.parametrize("op", ["ce", "angular"])
def test_a_label_that_is_no_class_shows(op):
    x, w, y = make(40, 64, 100, torch.bfloat16)
    y[3], y[7], y[11] = 100, -5, 1 << 40
    f = b200.linear_cross_entropy if op == "ce" else b200.angular_cross_entropy
    x.requires_grad_()
    loss = f(x, w, y, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 7, 11]] = True
    assert bool((loss.isnan() == bad).all())
    loss.sum().backward()
    assert bool((x.grad.isnan().all(1) == bad).all()) and bool((x.grad.isnan().any(1) == bad).all())


def test_an_entry_that_is_no_class_shows():
    x, w, _, t, i = make(40, 64, 100, torch.bfloat16, k=4)
    i[3, 0], i[7, 3], t[9, 2] = 100, 1 << 40, float("nan")
    i[11, 1], t[11, 1] = -1, float("nan")
    loss = b200.linear_distillation(x, w, t, i, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 7, 9]] = True
    assert bool((loss.isnan() == bad).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_a_class_that_comes_twice(dtype):
    x, w, _, t, i = make(50, 64, 300, dtype, k=40)
    i[:, 7] = i[:, 3]
    i[::2, 39] = i[::2, 3]
    i[::5] = i[::5, :1]
    compare(b200.linear_distillation, x, w, (t, i), dict(teacher_logits=t, teacher_index=i))


def test_entries_without_probability():
    x, w, _, t, i = make(50, 64, 300, torch.bfloat16, k=6)
    t[:, 2] = -float("inf")
    t[:, 4] = -1e4
    compare(b200.linear_distillation, x, w, (t, i), dict(teacher_logits=t, teacher_index=i))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits(dtype):
    """Logits of hundreds: one class takes everything, the loss of rows that have it right is nearly 0."""
    x, w, y = make(200, 64, 500, dtype)
    f = lambda x, w, y, reduction: b200.linear_cross_entropy(x, w, y, scale=40.0, reduction=reduction)  # noqa: E731
    compare(f, x, w, (y,), dict(labels=y, scale=40.0), reduction="none", d_loss=torch.ones(200, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cosine", [False, True])
def test_small_losses_keep_their_relative_accuracy(cosine, dtype):
    """Rows that are sure of their class: the loss is the others' share, log1p(r), and off by no more than r is, relative to itself."""
    N, D, V = 300, 256, 200
    x, w, y = make(N, D, V, dtype, cosine=cosine)
    x = (x.float() + torch.linspace(0, 12, N, device=DEV)[:, None] * torch.nn.functional.normalize(w[y].float(), dim=1)).to(dtype)
    if cosine:
        loss = b200.angular_cross_entropy(x, w, y, margin=0.0, scale=30.0, reduction="none")
        r = orc.evaluate(x, w, labels=y, scale=30.0, normalize=True, reduction="none")
    else:
        loss = b200.linear_cross_entropy(x, w, y, reduction="none")
        r = orc.evaluate(x, w, labels=y, reduction="none")
    assert float(r["loss"].min()) < 1e-3
    near(loss, r["loss"], r["loss"] * (r["loss_off"] + 2.0 ** -22), "loss")


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_and_classes_of_zeros(dtype):
    x, w, y = make(60, 64, 100, dtype, cosine=True)
    x[5] = 0
    w[9] = 0
    y[6] = 9
    compare(b200.angular_cross_entropy, x, w, (y,), dict(labels=y, scale=30.0, margin=0.2, normalize=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_far_apart(dtype):
    """Normalised rows and classes whose lengths span a factor of a thousand."""
    x, w, y = make(120, 64, 300, dtype, cosine=True)
    x = (x.float() * torch.logspace(-1.5, 1.5, 120, device=DEV)[:, None]).to(dtype)
    w = (w.float() * torch.logspace(1, -1, 300, device=DEV)[:, None]).to(dtype)
    f = b200.angular_cross_entropy
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    f(x1, w1, y, reduction="sum").backward()
    r = orc.evaluate(x, w, labels=y, scale=30.0, margin=0.2, normalize=True, reduction="sum")
    near(x1.grad, r["dx"], orc.rounded(r["dx"], r["dx_off"], dtype), "dx")
    near(w1.grad, r["dw"], orc.rounded(r["dw"], r["dw_off"], dtype), "dw")


@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
def test_gradients_against_differences(op):
    """Differences of the formula's loss along random directions, steps of 1e-5."""
    N, D, V = 130, 72, 333
    x, w, y, t, i = make(N, D, V, torch.bfloat16, cosine=op == "angular", k=6)
    cfg = {"ce": dict(labels=y), "angular": dict(labels=y, scale=30.0, margin=0.2, normalize=True), "distill": dict(teacher_logits=t, teacher_index=i, temperature=2.0)}[op]
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    f = {"ce": lambda: b200.linear_cross_entropy(x1, w1, y), "angular": lambda: b200.angular_cross_entropy(x1, w1, y),
         "distill": lambda: b200.linear_distillation(x1, w1, t, i, temperature=2.0)}[op]
    f().backward()
    r = orc.evaluate(x, w, **cfg)
    value = lambda x, w: float(orc.total(*orc.losses(x, w, **cfg), "mean"))  # noqa: E731
    for s in range(3):
        g = torch.Generator(device=DEV).manual_seed(s)
        for name, a, grad in (("x", x, x1.grad), ("w", w, w1.grad)):
            d = torch.randn(a.shape, device=DEV, generator=g, dtype=torch.float64) * float(a.float().abs().mean())
            h = 1e-5
            up = [x.double(), w.double()]
            down = [x.double(), w.double()]
            j = "xw".index(name)
            up[j], down[j] = up[j] + h * d, down[j] - h * d
            slope = (value(*up) - value(*down)) / (2 * h)
            off = (orc.rounded(r["d" + name], r["d%s_off" % name], a.dtype) * d.abs()).sum() + 1e-7
            assert abs(float((grad.double() * d).sum()) - slope) <= off


@pytest.mark.parametrize("w_dtype", [torch.float32, None])
@pytest.mark.parametrize("dtype", TYPES)
def test_forms_of_the_inputs(dtype, w_dtype):
    """fp32 weights, strided and misaligned rows and weights, leading dimensions, int32 labels."""
    N, D, V = 120, 64, 200
    x, w, y = make(N, D, V, dtype)
    base_x, base_w = torch.zeros(N, 2 * D + 3, dtype=dtype, device=DEV), torch.zeros(V, D + 5, dtype=w_dtype or dtype, device=DEV)
    if w_dtype:
        w = w.float() + 1e-3 * torch.randn(V, D, device=DEV)
    w = w.to(w_dtype or dtype)
    w16 = w.to(dtype)
    ref = compare(b200.linear_cross_entropy, x, w16, (y,), dict(labels=y))
    base_x[:, 3:3 + D], base_w[:, 1:1 + D] = x, w
    for xs, ws in ((x.view(4, 30, D), w), (base_x[:, 3:3 + D], base_w[:, 1:1 + D]), (x.t().contiguous().t(), w.t().contiguous().t())):
        xs, ws = xs.detach().requires_grad_(), ws.detach().requires_grad_()
        loss = b200.linear_cross_entropy(xs, ws, y.view(xs.shape[:-1]).to(torch.int32))
        loss.backward()
        assert torch.equal(loss, ref[0]) and torch.equal(xs.grad.reshape(N, D), ref[1])
        assert ws.grad.dtype == ws.dtype and torch.equal(ws.grad.to(dtype), ref[2])
    # rows of 57 channels in rows of 64, nothing but NaN between them, the last one at the end of its storage
    gap = torch.full((V * 64 - 7,), float("nan"), dtype=dtype, device=DEV).as_strided((V, 57), (64, 1))
    gap.copy_(w16[:, :57])
    odd = gap.detach().requires_grad_()
    loss = b200.angular_cross_entropy(x[:, :57], odd, y)
    loss.backward()
    tight = w16[:, :57].contiguous().requires_grad_()
    ref57 = b200.angular_cross_entropy(x[:, :57].contiguous(), tight, y)
    ref57.backward()
    assert torch.equal(loss, ref57) and torch.equal(odd.grad, tight.grad)
    one = torch.randn(D, device=DEV).to(dtype)                    # a row broadcast to all: its gradient is the rows' sum
    a, b = one.clone().requires_grad_(), one.expand(N, D).contiguous().requires_grad_()
    b200.linear_cross_entropy(a.expand(N, D), w16, y, reduction="sum").backward()
    b200.linear_cross_entropy(b, w16, y, reduction="sum").backward()
    assert torch.equal(a.grad, b.grad.sum(0))
    single = b200.linear_cross_entropy(x[0], w16, y[0])           # (dim,) and a label
    assert torch.equal(single, b200.linear_cross_entropy(x[:1], w16, y[:1]))


def test_autocast_rounds_fp32_rows():
    x, w, y = make(64, 96, 150, torch.bfloat16)
    xf, wf = x.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = b200.angular_cross_entropy(xf, wf, y)
    loss.backward()
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    ref = b200.angular_cross_entropy(x1, w1, y)
    ref.backward()
    assert torch.equal(loss, ref) and xf.grad.dtype == torch.float32
    assert torch.equal(xf.grad.bfloat16(), x1.grad) and torch.equal(wf.grad.bfloat16(), w1.grad)


@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
def test_only_one_gradient(op):
    x, w, y, t, i = make(140, 96, 300, torch.bfloat16, cosine=op == "angular", k=4)
    f = {"ce": lambda x, w: b200.linear_cross_entropy(x, w, y), "angular": lambda x, w: b200.angular_cross_entropy(x, w, y),
         "distill": lambda x, w: b200.linear_distillation(x, w, t, i)}[op]
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    f(x1, w1).backward()
    x2, w2 = x.clone().requires_grad_(), w.clone().requires_grad_()
    a, b = f(x2, w), f(x, w2)
    a.backward()
    b.backward()
    r = lambda u, v: float((u.double() - v.double()).norm() / v.double().norm())  # noqa: E731
    # (other splits of the contraction: other fp32 roundings of the sums, seldom another 16-bit result)
    assert r(x2.grad, x1.grad) < 2 ** -10 and r(w2.grad, w1.grad) < 2 ** -10
    with torch.no_grad():
        assert torch.equal(f(x1, w1), a.detach())


def test_differentiated_once():
    x, w, y = make(20, 64, 100, torch.bfloat16)
    x.requires_grad_()
    (g,) = torch.autograd.grad(b200.linear_cross_entropy(x, w, y), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
def test_pieces_of_the_classes_and_same_bits(op):
    """Enough rows and classes for several pieces; twice the same bits, a kept graph included."""
    N, D, V = 2300, 136, 40011
    x, w, y, t, i = make(N, D, V, torch.bfloat16, cosine=op == "angular", k=9, ignored=300)
    if op == "distill":
        i[y == -100] = -1
    f = {"ce": lambda x, w: b200.linear_cross_entropy(x, w, y), "angular": lambda x, w: b200.angular_cross_entropy(x, w, y),
         "distill": lambda x, w: b200.linear_distillation(x, w, t, i, temperature=2.0)}[op]
    cfg = {"ce": dict(labels=y), "angular": dict(labels=y, scale=30.0, margin=0.2, normalize=True), "distill": dict(teacher_logits=t, teacher_index=i, temperature=2.0)}[op]
    x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = f(x1, w1)
    g1 = torch.autograd.grad(loss, (x1, w1), retain_graph=True)
    g2 = torch.autograd.grad(loss, (x1, w1))
    again = f(x1, w1)
    assert torch.equal(loss, again)
    for a, b in zip(g1, g2):
        assert torch.equal(a, b)
    r = orc.evaluate(x, w, **cfg)
    near(loss.detach(), r["loss"], r["loss_off"] + 2 ** -22 * r["loss"].abs(), "loss")
    near(g1[0], r["dx"], orc.rounded(r["dx"], r["dx_off"], x.dtype), "dx")
    near(g1[1], r["dw"], orc.rounded(r["dw"], r["dw_off"], x.dtype), "dw")


def test_other_stream_and_graph():
    x, w, y = make(300, 96, 700, torch.bfloat16)
    x, w = x.requires_grad_(), w.requires_grad_()
    def step():   # (no graph of an eager pass is left behind: its leaves belong to the stream that it ran on)
        loss = b200.linear_cross_entropy(x, w, y)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, w))
    ref = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    graphs = []
    for _ in range(2):            # two graphs, each with buffers of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    with torch.no_grad():
        x.mul_(0.5)
    ref = step()
    for g, _ in graphs:
        g.replay()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(ref, out))
    ops.device_status()


@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
def test_python_route_gives_the_same_bits(op, monkeypatch):
    N, D, V = 200, 57 if op == "ce" else 64, 500
    x, w, y, t, i = make(N, D, V, torch.bfloat16, cosine=op == "angular", k=4)
    f = {"ce": lambda x, w: b200.linear_cross_entropy(x, w, y, reduction="sum"), "angular": lambda x, w: b200.angular_cross_entropy(x, w, y),
         "distill": lambda x, w: b200.linear_distillation(x, w, t, i)}[op]

    def step():
        x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = f(x1, w1)
        return (loss.detach(), f(x, w), type(loss.grad_fn).__name__) + torch.autograd.grad(loss, (x1, w1))
    node = step()
    monkeypatch.setattr(ops, "native", ops._PythonRoutes)
    python = step()
    assert node[2] != python[2]
    assert all(torch.equal(a, b) for a, b in zip(node, python) if isinstance(a, torch.Tensor))


@pytest.mark.parametrize("python", [False, True])
def test_saved_tensors_moved_by_hooks(python, monkeypatch):
    if python:
        monkeypatch.setattr(ops, "native", ops._PythonRoutes)
    x, w, y = make(200, 64, 500, torch.bfloat16)

    def step():
        x1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(b200.linear_cross_entropy(x1, w1, y), (x1, w1))
    ref = step()

    def unpack(t):        # off every boundary, and with other strides
        if t.dim() == 1:
            return torch.cat([t.new_zeros(2), t])[2:]
        return torch.cat([t.new_zeros(t.shape[0], 3), t], 1)[:, 3:]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_weight_changed_between_the_passes():
    """As with any saved tensor: an error, not another gradient."""
    x, w, y = make(20, 64, 100, torch.bfloat16)
    w.requires_grad_()
    loss = b200.linear_cross_entropy(x, w, y)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
def test_transforms_are_refused(op, python, monkeypatch):
    """A tangent is not dropped, and the function transforms raise."""
    if python:
        monkeypatch.setattr(ops, "native", ops._PythonRoutes)
    x, w, y, t, i = make(20, 64, 100, torch.bfloat16, k=4)
    f = {"ce": lambda x, w, t: b200.linear_cross_entropy(x, w, y), "angular": lambda x, w, t: b200.angular_cross_entropy(x, w, y),
         "distill": lambda x, w, t: b200.linear_distillation(x, w, t, i)}[op]
    fwd = torch.autograd.forward_ad
    for n in range(3 if op == "distill" else 2):
        args = [x, w, t]
        with fwd.dual_level():
            args[n] = fwd.make_dual(args[n], torch.ones_like(args[n]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*args)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: f(a, w, t))(torch.stack([x, x]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: f(a, w, t))(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("scale", [33.2, 33.4, 64.0, 200.0])
@pytest.mark.parametrize("op", ["angular", "distill"])
def test_cosines_at_scales_with_a_running_maximum(op, scale, reduction, dtype):
    """Scales up to 33.27 (2^48) stand for the maximum themselves, larger ones take it from the products; with and without a teacher."""
    N, D, V, k = 150, 72, 700, 6
    x, w, y, t, i = make(N, D, V, dtype, cosine=True, k=k)
    w[11], x[9] = 0, 0                         # (a class and a row without a direction)
    d = torch.linspace(0.25, 4, N, device=DEV) if reduction == "none" else 1.0
    if op == "angular":
        f = lambda x, w, y, reduction: b200.angular_cross_entropy(x, w, y, margin=0.2, scale=scale, reduction=reduction)  # noqa: E731
        compare(f, x, w, (y,), dict(labels=y, scale=scale, margin=0.2, normalize=True), reduction, d)
    else:
        f = lambda x, w, t, i, reduction: b200.linear_distillation(x, w, t, i, scale=scale, normalize=True, reduction=reduction)  # noqa: E731
        compare(f, x, w, (t, i), dict(teacher_logits=t, teacher_index=i, scale=scale, normalize=True), reduction, d)


@pytest.mark.parametrize("cosine", [False, True])
@pytest.mark.parametrize("N,k,V", [(40, 1024, 1500), (40, 1024, 1024), (300, 777, 2000), (9, 1000, 100)])
def test_many_entries_of_a_teacher(N, k, V, cosine):
    """As many as there may be; more than there are classes, so that each comes ten times."""
    x, w, _, t, i = make(N, 64, V, torch.bfloat16, cosine=cosine, k=k)
    i[::3, k // 2:] = -1
    scale = 20.0 if cosine else 1.0
    f = lambda x, w, t, i, reduction: b200.linear_distillation(x, w, t, i, temperature=2.0, scale=scale, normalize=cosine, reduction=reduction)  # noqa: E731
    compare(f, x, w, (t, i), dict(teacher_logits=t, teacher_index=i, temperature=2.0, scale=scale, normalize=cosine))


@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
@pytest.mark.parametrize("dtype", TYPES)
def test_fp32_rows_and_weight_under_autocast(op, dtype):
    """What the extractor passes: gradients in fp32, whose only 16-bit rounding is that of the logits' gradients. (The oracle rounds a result; here it is not.)"""
    N, D, V = 200, 192, 900
    x, w, y, t, i = make(N, D, V, dtype, cosine=op != "ce", k=8)
    x1, w1 = x.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast("cuda", dtype=dtype):
        if op == "ce":
            loss, o = b200.linear_cross_entropy(x1, w1, y), dict(labels=y)
        elif op == "angular":
            loss, o = b200.angular_cross_entropy(x1, w1, y), dict(labels=y, scale=30.0, margin=0.2, normalize=True)
        else:
            loss, o = b200.linear_distillation(x1, w1, t, i, scale=30.0, normalize=True), dict(teacher_logits=t, teacher_index=i, scale=30.0, normalize=True)
    loss.backward()
    r = orc.evaluate(x, w, **o)
    near(loss.detach(), r["loss"], r["loss_off"] + 2 ** -22 * r["loss"].abs(), "loss")
    near(x1.grad, r["dx"], orc.rounded(r["dx"], r["dx_off"], torch.float32), "dx")
    near(w1.grad, r["dw"], orc.rounded(r["dw"], r["dw_off"], torch.float32), "dw")


def test_offsets_beyond_32_bits():
    """A weight of 2.2e9 elements, labels at both ends: the sums of all classes in pieces and in 64 bits; dx, and dw of the first and last classes. Bounds as the oracle's:
    half a step of 2^-8 for each gradient of a logit and for the result, (D + 8) 2^-23 of a logit's terms, V / 64 2^-24 for the sum."""
    N, D, V = 6, 192, 11_500_000
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.empty(V, D, device=DEV, dtype=torch.bfloat16).normal_(generator=g).mul_(0.125).requires_grad_()
    x = torch.randn(N, D, device=DEV, generator=g).bfloat16().requires_grad_()
    y = torch.tensor([0, 1, V // 2, V - 3, V - 2, V - 1], device=DEV)
    loss = b200.linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    ops.device_status()
    xd, parts, sums, sizes = x.detach().double(), [], torch.zeros(N, D, dtype=torch.float64, device=DEV), torch.zeros(N, D, dtype=torch.float64, device=DEV)
    size = 0.0
    for v in range(0, V, 500_000):
        wd = w.detach()[v:v + 500_000].double()
        z = xd @ wd.t()
        size = max(size, float((xd.abs() @ wd.abs().t()).max()))
        parts.append(torch.logsumexp(z, 1))
        sums += torch.exp(z) @ wd             # (logits of some units: nothing overflows)
        sizes += torch.exp(z) @ wd.abs()
    lse = torch.logsumexp(torch.stack(parts), 0)
    own = w.detach()[y].double()
    off = 2 * ((D + 8) * 2.0 ** -23 * size + V / 64 * 2.0 ** -24)
    assert bool(((loss.detach().double() - (lse - (xd * own).sum(1))).abs() <= off + 2.0 ** -22 * lse).all())
    p = torch.exp(-lse)[:, None]
    near(dx, sums * p - own, (2.0 ** -8 + off) * (sizes * p) + (off + 2.0 ** -20) * own.abs() + 2.0 ** -8 * (sums * p - own).abs(), "dx")
    for v in (slice(0, 600), slice(V // 2 - 300, V // 2 + 300), slice(V - 600, V)):
        G = torch.exp(xd @ w.detach()[v].double().t() - lse[:, None])
        G = G - (torch.arange(V, device=DEV)[v] == y[:, None]).double()
        ref = G.t() @ xd
        near(dw[v], ref, (2.0 ** -8 + off) * (G.abs().t() @ xd.abs()) + 2.0 ** -8 * ref.abs(), "dw")


@pytest.mark.parametrize("op", ["ce", "angular", "distill"])
def test_calls_at_once(op):
    """From several threads, each on a stream of its own: what one call gives."""
    import threading
    x, w, y, t, i = make(300, 96, 3000, torch.float16, cosine=op == "angular", k=5)
    f = {"ce": lambda x, w: b200.linear_cross_entropy(x, w, y), "angular": lambda x, w: b200.angular_cross_entropy(x, w, y),
         "distill": lambda x, w: b200.linear_distillation(x, w, t, i)}[op]

    def step():
        x1, w1 = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = f(x1, w1)
        return (loss.detach(),) + torch.autograd.grad(loss, (x1, w1))
    want, got = step(), [None] * 4
    torch.cuda.synchronize()

    def work(n):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[n] = step()
        s.synchronize()
    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
