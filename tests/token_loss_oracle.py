"""Log probabilities, entropies and divergences from their definitions in 64 bits, with gradients by autograd, and how far the
kernels' 32-bit sums may be off."""
import math

import torch

U = 2.0 ** -24           # half a step of 32 bits


def logprobs(logits, targets, temperature, g=None, g_ent=None, ignore=-100):
    x = logits.detach().double().cpu().requires_grad_()
    t = targets.cpu()
    y = x / temperature
    logp = y - torch.logsumexp(y, dim=-1, keepdim=True)
    real = t != ignore
    lp = torch.where(real, logp.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1), 0.0)
    ent = torch.where(real, -(logp.exp() * logp.masked_fill(logp == -math.inf, 0.0)).sum(-1), 0.0)
    dx = None
    if g is not None:
        loss = (lp * g.double().cpu()).sum() + (ent * g_ent.double().cpu()).sum()
        dx, = torch.autograd.grad(loss, x)
    return lp.detach(), ent.detach(), logp.detach(), dx


def distill(logits, ids, values, temperature, lse=None, g=None):
    x = logits.detach().double().cpu().requires_grad_()
    ids, values = ids.cpu(), values.double().cpu()
    y = x / temperature
    logp = y - torch.logsumexp(y, dim=-1, keepdim=True)
    loss = torch.zeros(x.shape[:-1], dtype=torch.float64)
    flat, fl = logp.reshape(-1, x.shape[-1]), []
    for r in range(flat.shape[0]):
        i, v = ids.reshape(-1, ids.shape[-1])[r], values.reshape(-1, ids.shape[-1])[r] / temperature
        i, v = i[i >= 0], v[i >= 0]
        if len(i) == 0:
            fl.append(flat[r].sum() * 0)
            continue
        logq = v - (torch.logsumexp(v, 0) if lse is None else lse.double().cpu().reshape(-1)[r])
        q = logq.exp()
        loss = (q * (logq - flat[r][i])).sum()
        if lse is not None:
            rest = (1 - q.sum()).clamp(min=0)
            other = torch.ones(x.shape[-1], dtype=torch.bool)
            other[i] = False
            if rest > 0 and bool(other.any()):
                loss = loss + rest * (rest.log() - torch.logsumexp(flat[r][other], 0))
        fl.append(loss * temperature ** 2)
    out = torch.stack(fl).reshape(x.shape[:-1])
    dx = None
    if g is not None:
        dx, = torch.autograd.grad((out * g.double().cpu()).sum(), x)
    return out.detach(), dx


def sum_steps(V):
    """Roundings on the way into a row's sum, in units of U, from above: a thread adds batches of up to 32 terms (each an
    exponential of 2 ulp with a rounded argument) to its sum, V / 7168 of them (V / 512 is more than enough), then come trees of
    5 + 16 + 8 joins of two factors each."""
    return V / 512 + 32 + 8 + 3 * 29


def value_tol(V, logp_like, temperature):
    """An absolute bound for log probabilities and entropies: the sum's relative error, and a few roundings of the numbers
    themselves.  The exponentials' arguments d / T carry up to |d / T| roundings, which their weight p bounds: p |d / T| sums to
    less than ln V."""
    return U * (2 * sum_steps(V) + 4 * math.log(V) + 8 * logp_like.abs().masked_fill(logp_like.isinf(), 0.0) + 8)


def grad_tol(exact, dtype, V, size, temperature):
    """Half a step of the type for the last rounding (and half of the smallest subnormal), and the 32-bit errors in front of
    it, for factors up to `size`: of p as above, of log p + H (up to |log p| + ln V, times p: below 2 ln V)."""
    f = torch.finfo(dtype)
    small = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}[dtype]
    return f.eps / 2 * exact.abs() * 1.01 + small + U * (2 * sum_steps(V) + 16 * math.log(V) + 16) * size / temperature
