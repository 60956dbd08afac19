"""AdamW from its definition in 64 bits, and how far 32-bit arithmetic may be off."""
import math

import torch

U = 2.0 ** -24           # half a step of 32 bits


def step(p, g, m, v, t, lr, betas, eps, decay, norm=None, max_norm=0.0):
    """Parameters and moments behind step number ``t`` in 64 bits, each with its tolerance.

    The clipped gradient x has two roundings (of the factor, of the product).  m is a sum of two products with rounded factors: three
    roundings of each product at most beside x's own, one of the sum.  v likewise, with x twice.  The divisor has half of v's relative
    error, and roundings of the root, its factor, the product and the sum; the rate, its product and the quotient are rounded; p has
    its rounded factor (a rounding of 1), the product and the difference."""
    (b1, b2), p, g, m, v = betas, *(x.detach().double().cpu() for x in (p, g, m, v))
    x = g if norm is None else g * min(1.0, max_norm / (norm + 1e-6))
    m1, v1 = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    m_tol = (4 * (b1 * m).abs() + 6 * ((1 - b1) * x).abs()) * U
    v_tol = (4 * b2 * v + 9 * (1 - b2) * x * x) * U
    rate, d = lr / (1 - b1 ** t), v1.sqrt() / math.sqrt(1 - b2 ** t) + eps
    change = rate * m1 / d
    p1 = p * (1 - lr * decay) - change
    p_tol = 3 * U * p.abs() + rate * m_tol / d + change.abs() * (10 * U + 0.5 * v_tol / v1.clamp(min=1e-300)) + U * p1.abs()
    small = 2.0 ** -148      # the smallest 32-bit numbers are this far apart, and may come out of several products
    return (p1, p_tol * 1.01 + small), (m1, m_tol * 1.01 + small), (v1, v_tol * 1.01 + small)


def with_rounding(tol, want, dtype):
    """A tolerance with the last rounding to ``dtype``."""
    if dtype == torch.float32:
        return tol
    info = torch.finfo(dtype)
    return tol + (want.abs() * info.eps / 2).clamp(min=info.smallest_normal * info.eps / 2) * 1.01


def norm(grads):
    return math.sqrt(sum(float(g.detach().double().cpu().square().sum()) for g in grads if g is not None))


def norm_tol(want):
    """The kernel adds eight squares in 32 bits, each sum rounded once (at most half a step of a number not above the last one: 8 U of
    it in all), and takes everything else in 64: half of that is the root's, and its rounding to 32 bits is one more U."""
    return want * (4 + 1) * U * 1.01
