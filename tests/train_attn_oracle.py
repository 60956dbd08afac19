"""Attention with a gradient from its definition in 64 bits, and how far 16-bit operands and 32-bit sums may be off."""
import math

import torch


def visible(Sq, Skv, causal, window, key_mask, B, device):
    last = torch.arange(Sq, device=device).view(-1, 1) + (Skv - Sq)
    key = torch.arange(Skv, device=device).view(1, -1)
    see = torch.ones(B, 1, Sq, Skv, dtype=torch.bool, device=device)
    if causal:
        see = see & (key <= last)
    if window:
        see = see & (key > last - window)
    return see if key_mask is None else see & key_mask[:, None, None, :]


def attention(q, k, v, g, scale, causal, window, key_mask):
    """{"out", "dq", "dk", "dv"}: (exact value, tolerance)."""
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    n = Hq // Hkv
    eps = torch.finfo(q.dtype).eps / 2
    small = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134
    see = visible(Sq, Skv, causal, window, key_mask, B, q.device)
    if key_mask is not None:
        k, v = (t.masked_fill(~key_mask[:, None, :, None], 0.0) for t in (k, v))
    q, k, v, g = (t.detach().double() for t in (q, k, v, g))
    kk, vv = k.repeat_interleave(n, 1), v.repeat_interleave(n, 1)
    s = (q @ kk.transpose(-1, -2) * scale).masked_fill(~see, -math.inf)
    some = see.any(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(~some, 0.0), -1).masked_fill(~see, 0.0)
    o = p @ vv
    dp = g @ vv.transpose(-1, -2)
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    fold = lambda t: t.reshape(B, Hkv, n, Skv, D).sum(2)
    got = {"out": o, "dq": ds @ kk * scale, "dk": fold(ds.transpose(-1, -2) @ q) * scale, "dv": fold(p.transpose(-1, -2) @ g)}
    # A product over D adds D / 16 groups to a 32-bit sum, which may cut off instead of rounding: (D / 16 + 2) 2^-23 of the sum
    # of magnitudes.  That is the error of a score, relative to e^score that of a probability, once in s and once in its row's
    # L; the exponential's own errors are below 2^-20.
    steps = (D / 16 + 2) * 2.0 ** -23
    a_max = float((q.abs() @ kk.abs().transpose(-1, -2) * scale).masked_fill(~see, 0.0).max())
    rel = 2 * steps * a_max + 2.0 ** -20
    # probabilities are rounded to 16 bits on their way into a product (in fp16 by at least half of the smallest subnormal, of
    # numbers whose row has a largest one of 1 or more), sums over rows cut off like those over D
    sums = (max(Sq, Skv) / 16 + 2) * 2.0 ** -23
    pv = p @ vv.abs()
    seen_v = see.double() @ vv.abs()
    tol = {"out": (eps + rel + sums) * pv + small * seen_v + eps * o.abs()}
    tol["dv"] = fold((eps + rel + sums) * (p.transpose(-1, -2) @ g.abs()) + small * (see.double().transpose(-1, -2) @ g.abs()))
    # dS: delta's error comes from the rounded o (and its own error), dP's from its sum
    e = (g.abs() * (tol["out"] + eps * o.abs())).sum(-1, keepdim=True) + steps * (g.abs() * o.abs()).sum(-1, keepdim=True) \
        + steps * float((g.abs() @ vv.abs().transpose(-1, -2)).max())
    size = (eps + rel + sums) * ds.abs() + p * e * (1 + eps)
    # fp16: dS is stored times a power of two that puts 2 max|dO| max|v| between 2^14 and 2^15
    floor = small * 2.0 ** -14 * 2 * float(g.norm(dim=-1).max() * vv.norm(dim=-1).max()) * see.double()
    tol["dq"] = ((size + floor) @ kk.abs()) * scale
    tol["dk"] = fold((size + floor).transpose(-1, -2) @ q.abs()) * scale
    for name in ("dq", "dk", "dv", "out"):
        tol[name] = tol[name] * 1.02 + eps * got[name].abs() * 1.02 + small
    return {name: (got[name], tol[name]) for name in got}
