"""The losses of a classification head, as timed cases: what they are computed from, their plain forms, and their values in 64 bits.

Three operators on the rows ``x`` (rows, dim) that a network ends in and the ``weight`` (classes, dim) of its head, whose (rows, classes)
logits no caller needs:

* ``ce``       softmax cross entropy of the logits ``x weight^T``; rows labelled -100 do not count;
* ``angular``  the same on scaled cosines with an additive angular margin on the label's (the head of a speaker network);
* ``distill``  Kullback-Leibler divergence from a teacher of whose logits the top ones are known, at a temperature, on plain or cosine logits;
               rows have as many of the entries as the teacher kept, the others have index -1.

A training case returns the loss and the gradients of rows and weight, the others each row's loss.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
IGNORED = -100
FLOOR = 2e-7                                  # of the squared sine in the margin's formula
MOST_PRODUCTS = 8192 * 50000 * 1024           # rows x classes x dim of the largest listed case
MOST_LOGITS = 8192 * 50000                    # and its logits


def _case(name, op, rows, dim, classes, dtype="bf16", train=True, scale=1.0, ignored=0.0, reduction="mean"):
    return {"name": name, "op": op, "rows": rows, "dim": dim, "classes": classes, "dtype": dtype, "train": train, "scale": scale,
            "ignored": ignored, "reduction": reduction}


def _angular(name, rows, dim, classes, margin=0.2, scale=30.0, **more):
    return {**_case(name, "angular", rows, dim, classes, scale=scale, **more), "margin": margin}


def _distill(name, rows, dim, classes, top, temperature, cosine=False, ragged=False, **more):
    return {**_case(name, "distill", rows, dim, classes, scale=30.0 if cosine else 1.0, **more), "top": top, "temperature": temperature,
            "cosine": cosine, "ragged": ragged}


def listed():
    return [
        # One row: the latency of the whole forward and backward pass at the extractor's head (192-d embedding, 5994 speakers).
        _case("ce_row", "ce", 1, 192, 5994),
        # A linear head on the extractor's embeddings, a step's batch of utterances.
        _case("ce_head", "ce", 256, 192, 5994),
        # Validation loss over a few thousand tokens, some of them padding: each row's, forward only, an odd number of classes.
        _case("ce_validate", "ce", 3001, 512, 20011, dtype="fp16", train=False, ignored=0.25, reduction="none"),
        # A step on a long batch of tokens with a large vocabulary, a quarter of them padding.
        _case("ce_large", "ce", 8192, 1024, 50000, ignored=0.25),
        # The extractor's own head in training: AAM-softmax over 5994 speakers.
        _angular("angular_head", 256, 192, 5994),
        # Three classes for each speaker, as with speed perturbation, and every frame's row with a label; fp16.
        _angular("angular_frames", 4099, 192, 17982, dtype="fp16", margin=0.3, scale=32.0),
        # A head over many speakers, a large batch.
        _angular("angular_large", 1024, 256, 200003),
        # A few utterances' rows against a teacher's eight best.
        _distill("distill_few", 16, 192, 5994, 8, 2.0, cosine=True),
        # A smaller extractor that learns from a larger one: a step's batch, cosine logits.
        _distill("distill_head", 256, 192, 5994, 32, 4.0, cosine=True),
        # Rows with different numbers of entries, some with none; odd sizes, fp16, a sum over the rows.
        _distill("distill_ragged", 1003, 320, 12007, 20, 1.0, ragged=True, dtype="fp16", reduction="sum"),
        # Tokens against the 64 best of a large vocabulary.
        _distill("distill_large", 4096, 768, 32003, 64, 2.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ce", "angular", "distill"])
    dim = rng.choice([64, 128, 192, 192, 256, 512, 1024, 8 * _log_int(rng, 4, 128), 8 * _log_int(rng, 4, 128), _log_int(rng, 33, 1000)])
    classes = _log_int(rng, 200, 200000)
    rows = _log_int(rng, 1, max(1, min(8192, MOST_LOGITS // classes, MOST_PRODUCTS // (classes * dim))))
    more = {"dtype": rng.choice(["bf16", "bf16", "fp16"]), "train": rng.random() < 0.8, "reduction": rng.choice(["mean", "mean", "sum"])}
    if not more["train"]:
        more["reduction"] = "none"
    if op != "distill":
        more["ignored"] = rng.choice([0.0, 0.0, 0.1, 0.5])
    if op == "ce":
        case = _case("", "ce", rows, dim, classes, scale=rng.choice([1.0, 1.0, 0.5]), **more)
    elif op == "angular":
        case = _angular("", rows, dim, classes, margin=rng.choice([0.0, 0.2, 0.2, 0.3]), scale=rng.choice([16.0, 30.0, 32.0]), **more)
    else:
        case = _distill("", rows, dim, classes, _log_int(rng, 1, 100), rng.choice([1.0, 2.0, 4.0]), cosine=rng.random() < 0.5,
                        ragged=rows > 1 and rng.random() < 0.4, **more)
    case.pop("name")
    return case


def _counted(case):
    if case["op"] == "distill":
        return case["rows"] - -(-case["rows"] // (case["top"] + 1)) if case["ragged"] else case["rows"]
    return case["rows"] - int(case["rows"] * case["ignored"])


def prepare(case, seed):
    dev, dt = "cuda", DTYPES[case["dtype"]]
    N, D, V = case["rows"], case["dim"], case["classes"]
    g = torch.Generator(device=dev).manual_seed(seed)
    cosine = case["op"] == "angular" or case.get("cosine", False)
    # a weight as it is initialised (cosine heads) or with logits of about two standard units; rows lean towards their own class
    w = (torch.randn(V, D, device=dev, generator=g) * (0.01 if cosine else 2 * D ** -0.5)).to(dt)
    labels = torch.randint(0, V, (N,), device=dev, generator=g)
    toward = w[labels].float()
    toward = toward * (toward.square().sum(1, keepdim=True) + 1e-12).rsqrt()
    x = torch.randn(N, D, device=dev, generator=g) + toward * (0.5 * D ** 0.5 if cosine else 3.0)
    # what a training step multiplies the loss with: a mean in fp16 is scaled, since its gradients are small
    loss_scale = torch.tensor(1024.0 if case["dtype"] == "fp16" and case["reduction"] == "mean" else 1.0, device=dev)
    state = {"case": case, "x": x.to(dt).requires_grad_(case["train"]), "w": w.requires_grad_(case["train"]), "loss_scale": loss_scale}
    if case["op"] != "distill":
        labels[torch.randperm(N, device=dev, generator=g)[:N - _counted(case)]] = IGNORED
        state["labels"] = labels
        return state
    # the teacher's rows are the student's and some noise; what it kept of its logits comes sorted
    k = min(case["top"], V)
    t = (x + 0.5 * torch.randn(N, D, device=dev, generator=g)).to(dt)
    a, b = (t, w.detach()) if not cosine else (t * (D ** -0.5), w.detach() * (100 * D ** -0.5))
    top, index = (a @ b.t()).float().topk(k, dim=1)
    if cosine:
        top = top * 30.0
    if case["ragged"]:
        kept = (torch.arange(N, device=dev) % (k + 1))[torch.randperm(N, device=dev, generator=g)]
        index = index.masked_fill(torch.arange(k, device=dev) >= kept[:, None], -1)
    state["top"], state["index"] = top, index
    return state


# ------------------------------------------------------------------ plain forms
def _logits(case, x, w):
    """fp32 products of the rows and the weight (normalised ones where the logits are cosines), and what they are products of."""
    xf, wf = x.detach().float(), w.detach().float()
    if case["op"] == "angular" or case.get("cosine", False):
        xf, wf = xf / xf.square().sum(1, keepdim=True).sqrt(), wf / wf.square().sum(1, keepdim=True).sqrt()
    return xf @ wf.t(), xf, wf


def _softmax(z):
    """Probabilities (in the place of z) and the logarithm of the sum."""
    m = z.amax(1, keepdim=True)
    e = z.sub_(m).exp_()
    s = e.sum(1, keepdim=True)
    return e.div_(s), (s.log() + m).squeeze(1)


def _total(case, rows, counted):
    if case["reduction"] == "none":
        return rows
    return rows.sum() / counted.sum().clamp_min(1) if case["reduction"] == "mean" else rows.sum()


def _gradients(case, G, xf, wf, x, w, counted, loss_scale):
    """Gradients of rows and weight from that of the products, for rows that count."""
    G *= (counted * (loss_scale / counted.sum().clamp_min(1) if case["reduction"] == "mean" else loss_scale))[:, None]
    dx, dw = G @ wf, G.t() @ xf
    if case["op"] == "angular" or case.get("cosine", False):
        dx = (dx - xf * (xf * dx).sum(1, keepdim=True)) / x.detach().float().square().sum(1, keepdim=True).sqrt()
        dw = (dw - wf * (wf * dw).sum(1, keepdim=True)) / w.detach().float().square().sum(1, keepdim=True).sqrt()
    return dx.to(x.dtype), dw.to(w.dtype)


def _plain_labels(case, x, w, labels, loss_scale):
    z, xf, wf = _logits(case, x, w)
    counted = (labels != IGNORED).float()
    at = labels.clamp_min(0)[:, None]
    slope = 1.0
    if case["op"] == "angular":
        c = z.gather(1, at)
        sine2 = 1 - c * c
        sine = sine2.clamp_min(FLOOR).sqrt()
        z.scatter_(1, at, c * math.cos(case["margin"]) - sine * math.sin(case["margin"]))
        slope = math.cos(case["margin"]) + torch.where(sine2 > FLOOR, c / sine, 0.0) * math.sin(case["margin"])
    z *= case["scale"]
    target = z.gather(1, at)
    p, lse = _softmax(z)
    loss = _total(case, (lse - target.squeeze(1)) * counted, counted)
    if not case["train"]:
        return loss
    G = p.scatter_(1, at, (p.gather(1, at) - 1) * slope).mul_(case["scale"])
    return (loss,) + _gradients(case, G, xf, wf, x, w, counted, loss_scale)


def _plain_distill(case, x, w, top, index, loss_scale):
    z, xf, wf = _logits(case, x, w)
    tau = case["temperature"]
    z *= case["scale"] / tau
    there = index >= 0
    counted = there.any(1).float()
    t = torch.where(there, top / tau, -torch.inf)
    q = torch.where(there, (t - t.amax(1, keepdim=True)).exp(), 0.0)
    q = q / q.sum(1, keepdim=True).clamp_min(1e-30)
    at = index.clamp_min(0)
    kept = z.gather(1, at)
    p, lse = _softmax(z)
    terms = torch.where(q > 0, q * (q.clamp_min(1e-38).log() - kept + lse[:, None]), 0.0)
    loss = _total(case, terms.sum(1) * counted * tau ** 2, counted)
    if not case["train"]:
        return loss
    G = p.scatter_add_(1, at, -q).mul_(tau * case["scale"])
    return (loss,) + _gradients(case, G, xf, wf, x, w, counted, loss_scale)


def run(state):
    case, x, w = state["case"], state["x"], state["w"]
    if not own:
        if case["op"] == "distill":
            return _plain_distill(case, x, w, state["top"], state["index"], state["loss_scale"])
        return _plain_labels(case, x, w, state["labels"], state["loss_scale"])
    import pcf_nat_b200 as b200
    if case["op"] == "ce":
        loss = b200.linear_cross_entropy(x, w, state["labels"], scale=case["scale"], ignore_index=IGNORED, reduction=case["reduction"])
    elif case["op"] == "angular":
        loss = b200.angular_cross_entropy(x, w, state["labels"], margin=case["margin"], scale=case["scale"], ignore_index=IGNORED,
                                          reduction=case["reduction"])
    else:
        loss = b200.linear_distillation(x, w, state["top"], state["index"], temperature=case["temperature"], scale=case["scale"],
                                        normalize=case["cosine"], reduction=case["reduction"])
    if not case["train"]:
        return loss
    return (loss.detach(),) + torch.autograd.grad(loss, (x, w), state["loss_scale"])


def work(case):
    N, D, V, n = case["rows"], case["dim"], case["classes"], _counted(case)
    inputs = 2 * n * D + 2 * V * D + (8 * N if case["op"] != "distill" else 12 * N * min(case["top"], V))
    if not case["train"]:
        return {"bytes": inputs + 4 * N, "flops": 2 * n * V * D}
    return {"bytes": inputs + 4 + 2 * N * D + 2 * V * D, "flops": 6 * n * V * D}


def exact(case, seed):
    """From the definition in 64 bits; gradients by the framework's differentiation of the forward formula."""
    s = prepare(case, seed)
    x, w = (s[n].detach().double().requires_grad_(case["train"]) for n in ("x", "w"))
    z = x @ w.t()
    if case["op"] == "angular" or case.get("cosine", False):
        z = z / (x.norm(dim=1)[:, None] * w.norm(dim=1)[None, :])
    if case["op"] == "distill":
        tau, there = case["temperature"], s["index"] >= 0
        rows = there.any(1).nonzero().squeeze(1)
        there, at = there[rows], s["index"][rows].clamp_min(0)
        log_q = torch.log_softmax((s["top"][rows].double() / tau).masked_fill(~there, -1e300), dim=1)
        log_p = torch.log_softmax(z[rows] * (case["scale"] / tau), dim=1).gather(1, at)
        each = tau * tau * (log_q.exp() * (log_q - log_p)).masked_fill(~there, 0.0).sum(1)
    else:
        rows = (s["labels"] != IGNORED).nonzero().squeeze(1)
        at, z = s["labels"][rows], z[rows]
        own_class = torch.zeros_like(z, dtype=torch.bool).scatter_(1, at[:, None], True)
        if case["op"] == "angular":
            angle = torch.acos(z.gather(1, at[:, None]))
            z = torch.where(own_class, torch.cos(angle + case["margin"]), z)
        each = -torch.log_softmax(z * case["scale"], dim=1).gather(1, at[:, None]).squeeze(1)
    if not case["train"]:
        return torch.zeros(case["rows"], dtype=torch.float64, device="cuda").index_put((rows,), each)
    loss = each.sum() / max(1, len(rows)) if case["reduction"] == "mean" else each.sum()
    return (loss.detach(),) + torch.autograd.grad(loss, (x, w), s["loss_scale"].double())
