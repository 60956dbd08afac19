"""Preference and policy losses from their definitions in 64 bits, with gradients by autograd, and how far the kernels may be off."""
import math

import torch

import token_loss_oracle as tokens

U = tokens.U


def _logprobs(x, t, temperature, ignore):
    real = t != ignore
    y = torch.where(real.unsqueeze(-1), x, 0.0) / temperature          # rows without a target take no part, whatever they hold
    logp = y - torch.logsumexp(y, dim=-1, keepdim=True)
    return torch.where(real, logp.gather(-1, t.masked_fill(~real, 0).unsqueeze(-1)).squeeze(-1), 0.0), real


def preference(logits, targets, reference=None, beta=0.1, form="sigmoid", label_smoothing=0.0, margin=0.0, average=False,
               temperature=1.0, ignore_index=-100, g=None, g_seq=None):
    """(loss, logprob, dlogits) and the tolerances of each."""
    x, t = logits.detach().double().cpu().requires_grad_(), targets.cpu()
    lp, real = _logprobs(x, t, temperature, ignore_index)
    n = real.sum(1)
    share = 1.0 / n.clamp(min=1) if average else torch.ones_like(n, dtype=torch.float64)
    s = lp.sum(1) * share
    P = len(s) // 2
    h = s if reference is None else s - reference.double().cpu()
    h = h[:P] - h[P:]
    if form == "ipo":
        loss, slope, curve = (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta), 2.0
    elif form == "hinge":
        loss, slope, curve = torch.relu(1 - beta * h), torch.where(beta * h < 1, -beta, 0.0), 0.0
    else:
        z = beta * h - margin
        loss = -((1 - label_smoothing) * torch.nn.functional.logsigmoid(z) + label_smoothing * torch.nn.functional.logsigmoid(-z))
        slope = beta * (label_smoothing * torch.sigmoid(z) - (1 - label_smoothing) * torch.sigmoid(-z))
        curve = beta * beta / 4
    total = 0.0
    if g is not None:
        total = total + (loss * g.double().cpu()).sum()
    if g_seq is not None:
        total = total + (s * g_seq.double().cpu()).sum()
    dx, = torch.autograd.grad(total, x)
    V = logits.shape[-1]
    # sums over a sequence are in 64 bits: their terms' errors add up
    s_tol = torch.where(real, tokens.value_tol(V, lp.detach(), temperature), 0.0).sum(1) * share + U * s.detach().abs()
    h_tol = s_tol[:P] + s_tol[P:]
    loss_tol = slope.detach().abs() * h_tol + curve * h_tol ** 2 + 2 * U * loss.detach().abs() + 1e-37
    # what reaches a row: the slope, with what the error of h makes of it
    by = torch.zeros(2 * P, dtype=torch.float64)
    more = torch.zeros(2 * P, dtype=torch.float64)
    if g is not None:
        by += (slope.detach().abs() * g.double().cpu().abs()).repeat(2)
        more += (curve * h_tol * g.double().cpu().abs()).repeat(2)
    if g_seq is not None:
        by += g_seq.double().cpu().abs()
    by, more = (v * share for v in (by, more))
    dx_tol = tokens.grad_tol(dx, torch.float32 if logits.dtype == torch.float64 else logits.dtype, V, (by * 1.01).view(-1, 1, 1), temperature) + more.view(-1, 1, 1) / temperature
    return (loss.detach(), loss_tol), (s.detach(), s_tol), (dx, dx_tol)


def policy(logits, targets, advantages, old=None, ref=None, clip=(0.2, 0.2), kl_weight=0.0, temperature=1.0, ignore_index=-100, g=None):
    """(loss, logprob, kl, dlogits) and the tolerances of each, and which are clipped."""
    x, t = logits.detach().double().cpu().requires_grad_(), targets.cpu()
    lp, real = _logprobs(x, t, temperature, ignore_index)
    w = torch.exp(lp - (lp.detach() if old is None else old.double().cpu()))
    a = advantages.double().cpu().expand(t.shape)
    inside = w.clamp(1 - clip[0], 1 + clip[1])
    clipped = (inside * a < w * a) & real
    loss = -torch.where(clipped, inside.detach() * a, w * a)
    kl = torch.zeros_like(lp)
    if ref is not None:
        d = ref.double().cpu() - lp
        kl = torch.expm1(d) - d
        loss = loss + kl_weight * kl
    loss, kl = torch.where(real, loss, 0.0), torch.where(real, kl, 0.0)
    dx, = torch.autograd.grad((loss * g.double().cpu()).sum(), x)
    V = logits.shape[-1]
    lp_tol = torch.where(real, tokens.value_tol(V, lp.detach(), temperature), 0.0)
    with torch.no_grad():
        rise = torch.zeros_like(lp) if ref is None else torch.expm1(d).abs()
        kl_tol = rise * lp_tol + (rise + 1) * lp_tol ** 2 + 2 * U * kl
        slope = torch.where(clipped, 0.0, (a * w).abs()) + kl_weight * rise
        loss_tol = slope * lp_tol * 1.01 + kl_weight * (rise + 1) * lp_tol ** 2 + 2 * U * loss.abs()
        # the slope's own change with log p
        more = (torch.where(clipped, 0.0, (a * w).abs()) + kl_weight * (rise + 1)) * lp_tol * 1.01 * g.double().cpu().abs()
        size = torch.where(real, slope * g.double().cpu().abs() * 1.01, 0.0).unsqueeze(-1)
        dx_tol = tokens.grad_tol(dx, torch.float32 if logits.dtype == torch.float64 else logits.dtype, V, size, temperature) + torch.where(real, more, 0.0).unsqueeze(-1) / temperature
    return (loss.detach(), torch.where(real, loss_tol, 0.0) + 1e-37), (lp.detach(), lp_tol), (kl.detach(), kl_tol + 1e-37), (dx, dx_tol), clipped


def near_border(logits, targets, old, clip, temperature, ignore_index=-100):
    """Rows whose ratio is so near a border that rounding may decide: both sides are right there."""
    lp, real = _logprobs(logits.detach().double().cpu(), targets.cpu(), temperature, ignore_index)
    d = lp - old.double().cpu()
    tol = tokens.value_tol(logits.shape[-1], lp, temperature)
    edge = [math.log(b) if b > 0 else -math.inf for b in (1 - clip[0], 1 + clip[1])]
    return real & (((d - edge[0]).abs() <= tol) | ((d - edge[1]).abs() <= tol))
