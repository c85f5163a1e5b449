"""The losses of a classification head in 64 bits, with their gradients by formula and bounds on what 16-bit products may be off.

Test infrastructure. ``losses`` has the formulas alone; ``evaluate`` adds gradients and bounds."""
import math

import torch

FLOOR = 2e-7


def teacher_probabilities(teacher_logits, teacher_index, temperature):
    """(q (N, k), rows that count)."""
    there = teacher_index >= 0
    t = torch.where(there, teacher_logits.double() / temperature, -math.inf)
    counted = (t > -math.inf).any(1)
    q = torch.softmax(torch.where(counted[:, None], t, torch.zeros_like(t)), 1)
    return torch.where(there & counted[:, None], q, 0.0), counted


def logits(x, w, scale, normalize, labels=None, margin=0.0):
    """z (N, V), cosines or products c, factors ix, iw and the margin's slope at the label."""
    x, w = x.double(), w.double()
    ix = iw = None
    c = x @ w.t()
    if normalize:
        inverse = lambda t: torch.where(t > 0, 1 / t.clamp_min(1e-300), 0.0)   # noqa: E731
        ix, iw = inverse(x.norm(dim=1)), inverse(w.norm(dim=1))
        c = c * ix[:, None] * iw[None, :]
    z, slope = c, torch.ones(len(x), dtype=torch.float64, device=x.device)
    if labels is not None and margin:
        at = labels.clamp(0, w.shape[0] - 1)[:, None]
        own = c.gather(1, at)
        sine2 = 1 - own * own
        sine = sine2.clamp_min(FLOOR).sqrt()
        z = c.scatter(1, at, own * math.cos(margin) - sine * math.sin(margin))
        slope = (math.cos(margin) + torch.where(sine2 > FLOOR, own / sine, 0.0) * math.sin(margin)).squeeze(1)
    return z * scale, c, ix, iw, slope


def losses(x, w, labels=None, teacher_logits=None, teacher_index=None, scale=1.0, margin=0.0, normalize=False, temperature=1.0, ignore=-100):
    """(each row's loss, rows that count)."""
    z = logits(x, w, scale, normalize, labels, margin)[0]
    if labels is not None:
        counted = labels != ignore
        at = labels.clamp(0, w.shape[0] - 1)[:, None]
        others = torch.logsumexp(z.scatter(1, at, -math.inf), 1) - z.gather(1, at).squeeze(1)   # (small losses keep their digits)
        each = torch.logaddexp(others, torch.zeros_like(others))
    else:
        q, counted = teacher_probabilities(teacher_logits, teacher_index, temperature)
        log_p = torch.log_softmax(z / temperature, 1).gather(1, teacher_index.clamp_min(0))
        each = temperature ** 2 * torch.where(q > 0, q * (q.clamp_min(1e-300).log() - log_p), 0.0).sum(1)
    return torch.where(counted, each, 0.0), counted


def total(each, counted, reduction):
    return each if reduction == "none" else each.sum() / (max(1, int(counted.sum())) if reduction == "mean" else 1)


def evaluate(x, w, labels=None, teacher_logits=None, teacher_index=None, scale=1.0, margin=0.0, normalize=False, temperature=1.0, ignore=-100,
             reduction="mean", d_loss=1.0):
    """loss, dx, dw and how far an implementation may be from them that multiplies 16-bit values with fp32 sums.

    u: half a step of x's type. Products are exact in fp32, a sum of D of them is off by at most D 2^-23 times the sum of their magnitudes (truncating
    adders included): `off` below, times the scale that turns it into a logit. exp2, the fma of its argument and the sums of exponentials add a
    few fp32 steps of the largest exponent. A probability is then off by a factor 1 + 2 `loss_off`. The gradient of a logit is rounded once,
    |H| u, and its products' sums are off like the logits'; the result is rounded once more."""
    xd, wd = x.double(), w.double()
    u = torch.finfo(x.dtype).eps / 2
    z, c, ix, iw, slope = logits(x, w, scale, normalize, labels, margin)
    each, counted = losses(x, w, labels, teacher_logits, teacher_index, scale, margin, normalize, temperature, ignore)
    N, D = x.shape
    V = w.shape[0]
    on = counted.nonzero().squeeze(1)
    tau = temperature if labels is None else 1.0
    p = torch.softmax(z / tau, 1)
    H, Hoff = p.clone(), None
    # logits
    size = (xd.abs() @ wd.abs().t())
    if normalize:
        size = size * ix[:, None] * iw[None, :]
    size = size[on]
    off = (D + 8) * 2.0 ** -23 * float(size.max()) * scale / tau if len(on) else 0.0
    if normalize:
        off += 8 * 2.0 ** -23 * scale / tau      # the inverse lengths, rounded, and their sums of squares
    top = float(z[on].abs().max()) / tau if len(on) else 0.0
    loss_off = 2 * off + 16 * 2.0 ** -24 * (1 + top) + V / 128 * 2.0 ** -24 + 40 * 2.0 ** -24
    relative = 2 * loss_off
    if labels is not None:
        at = labels.clamp(0, V - 1)[:, None]
        own = p.gather(1, at)
        H.scatter_(1, at, (own - 1) * slope[:, None])
        Hoff = p * relative
        own_c = c.gather(1, at)
        sine = (1 - own_c * own_c).clamp_min(FLOOR).sqrt()
        steep = (1 + abs(math.sin(margin)) / sine ** 3) * (D + 16) * 2.0 ** -23 if margin else torch.zeros_like(own)
        loss_off = loss_off + (2 * float((steep * scale)[on].max()) if margin and len(on) else 0.0)
        Hoff.scatter_(1, at, own * slope[:, None].abs() * (relative + loss_off) + (1 - own) * slope[:, None].abs() * (relative + loss_off) + steep * (1 - own))
        factor = scale
    else:
        q, _ = teacher_probabilities(teacher_logits, teacher_index, temperature)
        H.scatter_add_(1, teacher_index.clamp_min(0), -q)
        Hoff = p * relative
        Hoff.scatter_add_(1, teacher_index.clamp_min(0), q * 32 * 2.0 ** -24 * (1 + float(torch.where(q > 0, teacher_logits.double().abs(), 0.0).max()) / tau))
        loss_off = tau ** 2 * (2 * loss_off + 2.0 ** -20)
        factor = scale * tau
    if reduction == "none":
        row = counted.double() * (torch.as_tensor(d_loss, dtype=torch.float64, device=x.device))
    else:
        row = counted.double() * float(d_loss) / (max(1, int(counted.sum())) if reduction == "mean" else 1)
    H = torch.where(counted[:, None], H, 0.0) * factor * row[:, None]
    Hoff = torch.where(counted[:, None], Hoff, 0.0) * factor * row.abs()[:, None]
    if normalize:
        H, Hoff = H * ix[:, None] * iw[None, :], Hoff * ix[:, None] * iw[None, :]
    # Below 2^-14 fp16 has steps of 2^-24. Gradients of logits are stored times 2^14 (products; relative to the largest of `row` where each row has
    # its own), or times a power of two that leaves the largest ix iw between 32 and 64 (cosines): half a step of 2^-25 is 2^-39, or
    # 2^-30 of that largest one.
    small = 0.0
    if x.dtype == torch.float16 and len(on):
        small = factor * float(row.abs().max()) * (2.0 ** -30 * float(ix[on].max() * iw.max()) if normalize else 2.0 ** -39)
    if len(on):   # a power below 2^-126 is 0
        small += 2.0 ** -125 * factor * float(row.abs().max()) * (float(ix[on].max() * iw.max()) if normalize else 1.0)
    Hoff = Hoff + H.abs() * u * 1.01 + small * counted[:, None]
    xs, ws = torch.where(counted[:, None], xd, 0.0), wd

    def project(d, d_off, own, inverse):
        if not normalize:
            return d, d_off
        n = own * inverse[:, None]
        return d - n * (n * d).sum(1, keepdim=True), d_off + n.abs() * (n.abs() * d_off).sum(1, keepdim=True) + (D + 16) * 2.0 ** -23 * (d.abs() + n.abs() * (n * d).abs().sum(1, keepdim=True))

    def both(H, Hoff, other, own, inverse, terms):
        d = H @ other
        d_off = Hoff @ other.abs() + (terms + 8) * 2.0 ** -23 * (H.abs() @ other.abs())
        return project(d, d_off, own, inverse)

    dx, dx_off = both(H, Hoff, ws, xs, ix, V)
    dw, dw_off = both(H.t(), Hoff.t(), xs, ws, iw, N)
    return {"loss": total(each, counted, reduction), "dx": dx, "dw": dw, "loss_off": loss_off * (1 if reduction != "sum" else max(1, len(on))),
            "dx_off": dx_off, "dw_off": dw_off, "counted": counted}


def rounded(value, off, dtype):
    """`off` and the rounding of a result to `dtype`."""
    f = torch.finfo(dtype)
    return off + (value.abs() + off) * (f.eps / 2) + f.tiny * f.eps / 2
