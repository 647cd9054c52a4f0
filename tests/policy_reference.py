"""The policy operators' definitions in 64 bits, and how far a kernel of a given type may be off (test infrastructure)."""
import math

import torch


def choice(logits, mask=None):
    """(allowed, empty, log p with 0 for an empty row and -inf where not allowed, p, entropy)"""
    x = logits.detach().double().cpu()
    allowed = x != -math.inf
    if mask is not None:
        allowed = allowed & (mask.cpu() != 0).expand(x.shape)
    empty = ~allowed.any(1)
    m = x.masked_fill(~allowed, -math.inf).amax(1, keepdim=True).masked_fill(empty[:, None], 0.0)
    z = (x - m).masked_fill(~allowed, -math.inf)
    e = z.exp()
    s = e.sum(1, keepdim=True).masked_fill(empty[:, None], 1.0)
    logp = z - s.log()
    p = e / s
    h = -(p * logp.masked_fill(p == 0, 0.0)).sum(1)
    return allowed, empty, logp, p, h


def given_log_probs(logp, empty, ids):
    v = logp.shape[1]
    ids = ids.cpu()
    out = logp.gather(1, ids.clamp(0, v - 1))
    out = out.masked_fill(empty[:, None], 0.0)
    out = out.masked_fill(ids == -1, 0.0)
    return out.masked_fill((ids < -1) | (ids >= v), math.nan)


def choice_gradient(allowed, p, logp, h, lists, d_entropy=None):
    """lists: (ids, d) pairs"""
    n, v = p.shape
    grad = torch.zeros(n, v, dtype=torch.float64)
    if d_entropy is not None:
        grad -= d_entropy.double().cpu()[:, None] * p * (logp.masked_fill(~allowed | (p == 0), 0.0) + h[:, None])
    size = grad.abs()
    for ids, d in lists:
        ids, d = ids.cpu(), d.double().cpu()
        ok = (ids >= 0) & (ids < v)
        ok &= allowed.gather(1, ids.clamp(0, v - 1))
        d = d * ok
        grad -= p * d.sum(1, keepdim=True)
        size += p * d.abs().sum(1, keepdim=True)
        grad.scatter_add_(1, ids.clamp(0, v - 1), d)
        size.scatter_add_(1, ids.clamp(0, v - 1), d.abs())
    return grad * allowed, size


def log_prob_error(logp, h, v):
    """What float32 arithmetic may add to a log-probability: the subtraction and the final one round to 2^-24 of their
    values, an exponential to 2^-22 of itself per unit of its argument's logarithm (whose mean over p is at most ln v), and
    a sum over v terms, of which one lane adds at most v / 64, to (8 + v / 512) 2^-24 (2048 terms and more are shared by
    512 lanes or more; below that v / 512 < 4 only understates what 8 covers)."""
    lv = math.log(v) + 1
    return 2.0 ** -24 * (2 * logp.abs().nan_to_num(0, 0, 0) + 8 * lv + 8 + v / 512)


def attention(q, k, v, allowed, scale, d_out=None):
    """float64 results and, for each, the bound of tests/test_gpu_policy_ops.py: (out, dq, dk, dv), (their bounds)"""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    w = 0.0 if dt == torch.float32 else u  # P and dS are rounded to the type on their way into the second product
    f = 2.0 ** -24
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    g = h // hk
    qh = q.view(b, lq, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, lq * g, d)
    kh, vh = k.permute(0, 2, 1, 3).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    if allowed is None:
        allowed = torch.ones(b, lk, dtype=torch.bool)
    keep = allowed.cpu()[:, None, :, None]
    kh, vh = kh.masked_fill(~keep, 0.0), vh.masked_fill(~keep, 0.0)
    n = allowed.cpu().sum(1).view(b, 1, 1, 1).double()
    mm = lambda x, y: torch.matmul(x, y.contiguous())
    s = mm(qh, kh.transpose(2, 3)) * scale
    s = s.masked_fill(~keep.transpose(2, 3), -math.inf)
    top = s.amax(3, keepdim=True).masked_fill(n == 0, 0.0) if lk else torch.zeros(b, hk, lq * g, 1, dtype=torch.float64)
    p = (s - top).exp()
    p = p / p.sum(3, keepdim=True).masked_fill(n == 0, 1.0)
    back = lambda x: x.view(b, hk, lq, g, d).permute(0, 2, 1, 3, 4).reshape(b, lq, h, d)
    backk = lambda x: x.permute(0, 2, 1, 3)
    o = mm(p, vh)
    # the score's rounding (a sum of d products, each to 2^-24 of the sum of magnitudes at worst), the exponent's, the sums'
    mag = mm(qh.abs(), kh.abs().transpose(2, 3)) * scale
    big = mag.amax() if mag.numel() else torch.zeros(())
    es = float((d / 2 + 8) * f * big + (16 + float(n.max() if n.numel() else 0) / 32) * f)
    pv = mm(p, vh.abs())
    e_out = u * o.abs() + (w + 2 * es) * pv + 1e-30
    if d_out is None:
        return (back(o),), (back(e_out),)
    do = d_out.detach().double().cpu().view(b, lq, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, lq * g, d)
    dv = mm(p.transpose(2, 3), do)
    e_dv = u * dv.abs() + (w + 2 * es) * mm(p.transpose(2, 3), do.abs())
    dp = mm(do, vh.transpose(2, 3))
    dd = (p * dp).sum(3, keepdim=True)
    ds = p * (dp - dd)
    e_dp = (d / 2 + 8) * f * mm(do.abs(), vh.abs().transpose(2, 3))
    few = (n <= 32).double()  # D is summed from P dP where the keys are few, else from the rounded output
    e_dd = (do.abs() * e_out).sum(3, keepdim=True) * (1 - few) + ((2 * es + 32 * f) * p * dp.abs() + p * e_dp).sum(3, keepdim=True) * few
    e_ds = (w + 2 * es) * ds.abs() + p * (e_dp + e_dd)
    dq = mm(ds, kh) * scale
    e_dq = u * dq.abs() + mm(e_ds, kh.abs()) * scale + 1e-30
    dk = mm(ds.transpose(2, 3), qh) * scale
    e_dk = u * dk.abs() + mm(e_ds.transpose(2, 3), qh.abs()) * scale + 1e-30
    if dt == torch.float16:  # results below the normal range are rounded to 2^-25
        e_out, e_dq, e_dk, e_dv = (e + 2.0 ** -25 for e in (e_out, e_dq, e_dk, e_dv))
    return (back(o), back(dq), backk(dk), backk(dv)), (back(e_out), back(e_dq), backk(e_dk), backk(e_dv + 1e-30))
