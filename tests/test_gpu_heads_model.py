"""The losses of a head where the extractor uses them: its AAM-softmax, learning from a teacher, a captured training step."""
import pytest
import torch

from pcf_nat_b200 import ops
from pcf_nat_b200.model import AAMSoftmax, PCFNATExtractor
from oracle import head_oracle as orc

pytestmark = pytest.mark.gpu
KW = dict(frames=70, feat=24, dim=64, heads=2, win=7, stages=2, blocks=1, emb=32, classes=300)


def test_aam_softmax_fused_is_the_same_loss():
    """On values that 16 bits hold the two differ by fp32 sums alone: cosines off by at most (D + 16) 2^-23, twice that and the scale in a loss."""
    torch.manual_seed(0)
    plain, fused = AAMSoftmax(64, 500).cuda(), AAMSoftmax(64, 500, fused=True).cuda()
    with torch.no_grad():
        plain.weight.copy_(plain.weight.bfloat16().float())
        fused.load_state_dict(plain.state_dict())
    emb = torch.randn(90, 64, device="cuda").bfloat16().float()
    y = torch.randint(0, 500, (90,), device="cuda")
    a, b = emb.clone().requires_grad_(), emb.clone().requires_grad_()
    la, lb = plain(a, y), fused(b, y)
    la.backward()
    lb.backward()
    assert abs(float(la) - float(lb)) <= 2 * 30 * (64 + 16) * 2.0 ** -23 + 1e-6 * float(la)
    r = orc.evaluate(emb.bfloat16(), fused.weight.detach().bfloat16(), labels=y, scale=30.0, margin=0.2, normalize=True)
    assert b.grad.dtype == torch.float32 and fused.weight.grad.dtype == torch.float32
    assert bool(((b.grad.double() - r["dx"]).abs() <= orc.rounded(r["dx"], r["dx_off"], torch.bfloat16)).all())
    assert bool(((fused.weight.grad.double() - r["dw"]).abs() <= orc.rounded(r["dw"], r["dw_off"], torch.float32)).all())


def test_extractor_learns_from_labels_and_a_teacher_in_a_graph():
    """Both losses on one embedding, eagerly and captured: the same numbers, gradients in every parameter."""
    torch.manual_seed(1)
    teacher, student = PCFNATExtractor(**KW).cuda().eval(), PCFNATExtractor(head="fused", **KW).cuda()
    x, y = torch.randn(16, 24, 70, device="cuda"), torch.randint(0, 300, (16,), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        top, index = teacher.top_logits(x, 8)
    assert top.shape == index.shape == (16, 8) and bool((top[:, :-1] >= top[:, 1:]).all())
    params = list(student.parameters())
    for p in params:
        p.grad = torch.zeros_like(p)

    def step():
        torch._foreach_zero_([p.grad for p in params])
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            loss = student.distill(x, y, top, index, temperature=2.0, weight=0.5)
        loss.backward()
        return loss.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            eager = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(bool(torch.isfinite(p.grad).all()) and bool(p.grad.any()) for p in params if p.numel() > 300)
    head = student.loss.weight.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    graph.replay()
    torch.cuda.synchronize()
    ops.device_status()
    assert bool(torch.isfinite(loss)) and abs(float(loss) - float(eager)) <= 2.0 ** -7 * float(eager)   # (batch norm and 16-bit activations apart)
    assert float((student.loss.weight.grad - head).norm()) <= 2.0 ** -6 * float(head.norm())


def test_train_step_with_the_fused_head_and_a_teacher():
    from pcf_nat_b200.model_bench import TrainStep
    dev = torch.device("cuda", 0)
    for kw in (dict(head="fused"), dict(head="fused", teacher_top=4), dict(precision="bf16", head="fused")):
        ts = TrainStep(4, dev, 1, 0, frames=60, **kw)
        losses = [float(ts()) for _ in range(2)]
        assert all(l == l and l > 0 for l in losses) and ts.graph_a is not None
        del ts
        torch.cuda.synchronize()
    ops.device_status()


def test_two_losses_of_one_embedding_together():
    """Cross entropy and distillation of the same rows and weight: the gradients are the sum of the two losses'."""
    import pcf_nat_b200 as b200
    torch.manual_seed(2)
    x, w = torch.randn(100, 48, device="cuda").bfloat16(), (0.1 * torch.randn(400, 48, device="cuda")).bfloat16()
    y = torch.randint(0, 400, (100,), device="cuda")
    t, i = torch.randn(100, 6, device="cuda"), torch.stack([torch.randperm(400, device="cuda")[:6] for _ in range(100)])

    def grads(*fs):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        sum(f(a, b) for f in fs).backward()
        return a.grad, b.grad
    ce = lambda a, b: b200.linear_cross_entropy(a, b, y)  # noqa: E731
    kd = lambda a, b: b200.linear_distillation(a, b, t, i, temperature=2.0)  # noqa: E731
    both, one, two = grads(ce, kd), grads(ce), grads(kd)
    for s, p, q in zip(both, one, two):
        assert torch.equal(s, p + q)
