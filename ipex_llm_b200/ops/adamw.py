"""The optimizer's part of a step (``adamw.cu``): AdamW over many tensors at once, with moments in 32 or in 8 bits, and the norm of
all gradients.

On CUDA tensors the package's own kernels run, on the current stream of the tensors' device; on the CPU it is the same arithmetic in
plain PyTorch, operation by operation, so that both give the same bits (but for a root or a power of the factors common to all, and
the last bits of changes below 2^-62).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from ..native.lib import calls
from ..utils.common import invalidInputError

BLOCK = 256              # elements of a tensor are counted in these, and 8-bit moments share an exponent in each
DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_LOW, _HIGH = 32, 254    # exponents of a block


class AdamWState(NamedTuple):
    """What AdamW keeps of a list of parameters, in flat buffers: parameter i's elements begin behind those of the ones before it,
    each taking its number of elements rounded up to 256.  Zeros are the state of parameters that no step has seen."""
    exp_avg: torch.Tensor                            # 32-bit, or float8_e4m3fn
    exp_avg_sq: torch.Tensor                         # 32-bit, or float8_e5m2
    step: torch.Tensor                               # int64: [1] for all parameters, or one for each
    exp_avg_scale: Optional[torch.Tensor] = None     # uint8, one for each 256: an exponent
    exp_avg_sq_scale: Optional[torch.Tensor] = None
    rest: Optional[torch.Tensor] = None              # int16: the 16 bits below bf16; 32-bit: copies of 16-bit parameters


def flat_size(sizes: Sequence[int]) -> int:
    """Elements of a flat buffer for tensors of these sizes."""
    return sum(-(-n // BLOCK) * BLOCK for n in sizes)


def _in_memory_order(t: torch.Tensor) -> Optional[torch.Tensor]:
    """The tensor's elements as they lie, in one dimension; None where others lie between them."""
    if t.is_contiguous():
        return t.reshape(-1)
    dims = sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1)
    want = 1
    for s, n in dims:
        if s != want:
            return None
        want *= n
    return t.as_strided((t.numel(),), (1,))


def _is_dense(t: torch.Tensor) -> bool:
    return t.is_contiguous() or _in_memory_order(t) is not None


def _like(g: torch.Tensor, p: torch.Tensor) -> torch.Tensor:
    """A gradient whose elements lie as the parameter's do."""
    if (p.is_contiguous() and g.is_contiguous()) or (g.stride() == p.stride()):
        return g
    return torch.empty_strided(p.shape, p.stride(), dtype=g.dtype, device=g.device).copy_(g)


def _check_gradients(grads, what):
    """The gradients that are there, of one type on one device."""
    have = [g for g in grads if g is not None]
    if have:
        dtype, dev = have[0].dtype, have[0].device
        for g in have:
            if g.layout != torch.strided:
                invalidInputError(False, f"{what}: sparse gradients are not supported")
            if g.dtype != dtype or g.device != dev:
                invalidInputError(False, f"{what}: all gradients should be of one type on one device, got {dtype} on {dev} and {g.dtype} "
                                         f"on {g.device}")
        if dtype not in DTYPES and (dev.type == "cuda" or dtype != torch.float64):
            invalidInputError(False, f"{what}: gradients of type {dtype} are not supported")
    return have


@torch.no_grad()
def grad_norm(grads: Sequence[Optional[torch.Tensor]]) -> torch.Tensor:
    """The 2-norm of all gradients together (32-bit, no dimension), ``None`` among them left out; 0 of none.  Sums are held in 64
    bits and added up in an order that depends on the sizes and the device alone."""
    norm = calls().grad_norm(grads) if any(g is not None and g.is_cuda for g in grads[:1]) else None
    if norm is not None:
        return norm
    have = _check_gradients(grads, "grad_norm")
    if not have:
        return torch.zeros((), dtype=torch.float32)
    if have[0].is_cuda:
        return calls().grad_norm([g if _is_dense(g) else g.contiguous() for g in have])
    return sum(g.double().square().sum() for g in have).sqrt().float()


def adamw_state(params: Sequence[torch.Tensor], bits: int = 32, rest: Optional[str] = None, each: bool = False) -> AdamWState:
    """A fresh state for ``adamw_step``: ``bits`` (32 or 8) of the moments; ``rest``: what is kept of 16-bit parameters beside
    themselves, so that steps below half of their last place are not lost: "low" (of bf16: the 16 bits that it leaves of a 32-bit
    number; the parameters are taken as they are) or "copy" (in 32 bits); ``each``: a step counter for each parameter, else one."""
    what = "adamw_state"
    params = list(params)
    invalidInputError(len(params) > 0, f"{what}: no parameters")
    invalidInputError(bits in (8, 32), f"{what}: moments have 32 or 8 bits, got {bits}")
    invalidInputError(rest in (None, "low", "copy"), f"{what}: rest should be None, 'low' or 'copy', got {rest!r}")
    dev, dtype = params[0].device, params[0].dtype
    _check_params(params, what)
    n = flat_size([p.numel() for p in params])
    small = bits == 8
    kw = dict(device=dev)
    kept = None
    if rest == "low":
        invalidInputError(dtype == torch.bfloat16, f"{what}: 'low' is what bf16 leaves, parameters of {dtype} take a copy")
        kept = torch.zeros(n, dtype=torch.int16, **kw)
    elif rest == "copy":
        invalidInputError(dtype in (torch.bfloat16, torch.float16), f"{what}: copies are for 16-bit parameters")
        kept = torch.zeros(n, dtype=torch.float32, **kw)
        at = 0
        for p in params:
            kept[at:at + p.numel()].copy_(_in_memory_order(p.detach()))
            at += flat_size([p.numel()])
    return AdamWState(torch.zeros(n, dtype=torch.uint8, **kw).view(torch.float8_e4m3fn) if small else torch.zeros(n, **kw),
                      torch.zeros(n, dtype=torch.uint8, **kw).view(torch.float8_e5m2) if small else torch.zeros(n, **kw),
                      torch.zeros(len(params) if each else 1, dtype=torch.int64, **kw),
                      torch.zeros(n // BLOCK, dtype=torch.uint8, **kw) if small else None,
                      torch.zeros(n // BLOCK, dtype=torch.uint8, **kw) if small else None, kept)


def _check_params(params, what):
    dtype, dev = params[0].dtype, params[0].device
    if dtype not in DTYPES:
        invalidInputError(False, f"{what}: parameters of type {dtype} are not supported")
    for p in params:
        if p.dtype != dtype or p.device != dev:
            invalidInputError(False, f"{what}: all parameters should be of one type on one device, got {dtype} on {dev} and {p.dtype} on "
                                     f"{p.device}")
        if not _is_dense(p):
            invalidInputError(False, f"{what}: a parameter's elements should lie one behind the other, got strides {p.stride()}")


def _check_buffer(t, name, dtype, n, dev):
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous() or t.device != dev or t.data_ptr() & 15:
        invalidInputError(False, f"adamw_step: {name} should be a contiguous, aligned {dtype} of {n} elements on {dev}, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]], exp_avg: torch.Tensor,
               exp_avg_sq: torch.Tensor, step: torch.Tensor, *, lr: Union[float, torch.Tensor],
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
               exp_avg_scale: Optional[torch.Tensor] = None, exp_avg_sq_scale: Optional[torch.Tensor] = None,
               rest: Optional[torch.Tensor] = None, grad_norm: Optional[torch.Tensor] = None, max_grad_norm: float = 0.0,
               seed: int = 0) -> None:
    """One step of AdamW, in place, on parameters of one 16-bit or 32-bit type, with gradients of the same type and shapes.

    ``exp_avg`` and the other flat buffers are those of an ``AdamWState`` (where the elements of a parameter lie one behind the other
    in another order than that of its dimensions, the buffers have them in that order).  A parameter whose gradient is None is left as
    it is, with its moments and, where each has one, its step counter; a common counter moves if any has a gradient.  ``step`` and,
    where it is a tensor (32-bit, on the device), ``lr`` are read by the kernels: a step that is captured into a graph counts on with
    each replay.  With ``max_grad_norm`` > 0 gradients are taken times ``min(1, max_grad_norm / (grad_norm + 1e-6))``; ``grad_norm``
    (32-bit, on the device) is theirs as ``grad_norm()`` gives it.

    Moments in 8 bits are rounded at random with the right mean, by a hash of ``seed``, the step and the element's place in the buffer,
    so that equal calls give equal results; a NaN or an infinity stays in its place.
    """
    what = "adamw_step"
    if len(params) != len(grads):
        invalidInputError(False, f"{what}: {len(params)} parameters and {len(grads)} gradients")
    if not len(params):
        return
    b1, b2 = float(betas[0]), float(betas[1])
    lr_at = lr if isinstance(lr, torch.Tensor) else None
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and weight_decay >= 0.0 and (lr_at is not None or lr >= 0.0)):
        invalidInputError(False, f"{what}: betas should lie in [0, 1), lr, eps and weight_decay not below 0; got {betas}, {lr}, {eps}, "
                                 f"{weight_decay}")
    if not (max_grad_norm and max_grad_norm > 0.0):
        grad_norm, max_grad_norm = None, 0.0
    elif grad_norm is None:
        invalidInputError(False, f"{what}: max_grad_norm needs the gradients' norm")
    elif all(g is None for g in grads):
        grad_norm = None                                      # of none: it is on no device
    buffers = (exp_avg, exp_avg_sq, step, exp_avg_scale, exp_avg_sq_scale, rest, grad_norm)
    numbers = (float(max_grad_norm), 0.0 if lr_at is not None else float(lr), lr_at, b1, b2, float(eps), float(weight_decay),
               int(seed) & 0xFFFFFFFF)
    cuda = params[0].is_cuda
    if cuda and calls().adamw_step(params, grads, *buffers, *numbers):
        return
    grads = _checked(params, grads, *buffers, lr_at)          # says what is wrong, or lays the gradients out as the parameters lie
    if not cuda:
        with torch.no_grad():
            _step_plain(params, grads, *buffers, *numbers)
        torch.autograd.graph.increment_version(params)
    elif not calls().adamw_step(list(params), grads, *buffers, *numbers):
        invalidInputError(False, f"{what}: these tensors are not supported")


def _checked(params, grads, exp_avg, exp_avg_sq, step, exp_avg_scale, exp_avg_sq_scale, rest, grad_norm, lr_at):
    what = "adamw_step"
    dtype, dev = params[0].dtype, params[0].device
    _check_params(params, what)
    seen = set()
    gs = []
    for p, g in zip(params, grads):
        if g is None:
            gs.append(None)
            continue
        if g.layout != torch.strided:
            invalidInputError(False, f"{what}: sparse gradients are not supported")
        if g.dtype != dtype or g.device != dev or g.shape != p.shape:
            invalidInputError(False, f"{what}: a gradient should be like its parameter, {dtype} {tuple(p.shape)} on {dev}, got {g.dtype} "
                                     f"{tuple(g.shape)} on {g.device}")
        if p.numel():
            if p.data_ptr() in seen:
                invalidInputError(False, f"{what}: a parameter occurs twice")
            seen.add(p.data_ptr())
        gs.append(_like(g, p))
    n = flat_size([p.numel() for p in params])
    small = exp_avg.dtype == torch.float8_e4m3fn
    _check_buffer(exp_avg, "exp_avg", torch.float8_e4m3fn if small else torch.float32, n, dev)
    _check_buffer(exp_avg_sq, "exp_avg_sq", torch.float8_e5m2 if small else torch.float32, n, dev)
    if small:
        if exp_avg_scale is None or exp_avg_sq_scale is None:
            invalidInputError(False, f"{what}: 8-bit moments come with their exponents")
        for t, name in ((exp_avg_scale, "exp_avg_scale"), (exp_avg_sq_scale, "exp_avg_sq_scale")):
            if t.dtype != torch.uint8 or t.numel() != n // BLOCK or not t.is_contiguous() or t.device != dev:
                invalidInputError(False, f"{what}: {name} should be a contiguous uint8 of {n // BLOCK} elements on {dev}")
    kind = 0
    if rest is not None:
        kind = 1 if rest.dtype == torch.int16 else 2
        if (kind == 1 and dtype != torch.bfloat16) or dtype == torch.float32:
            invalidInputError(False, f"{what}: parameters of {dtype} have no rest of {rest.dtype}")
        _check_buffer(rest, "rest", torch.int16 if kind == 1 else torch.float32, n, dev)
    if step.dtype != torch.int64 or step.numel() not in (1, len(params)) or not step.is_contiguous() or step.device != dev:
        invalidInputError(False, f"{what}: step should be an int64 of 1 or {len(params)} elements on {dev}")
    for t, name in ((lr_at, "lr"), (grad_norm, "grad_norm")):
        if t is not None and (t.dtype != torch.float32 or t.numel() != 1 or t.device != dev):
            invalidInputError(False, f"{what}: {name} should be one 32-bit number on {dev}")
    return gs


# ---- 8-bit moments and the rest of bf16, in plain PyTorch --------------------------------------------------------------------
def _power(e: torch.Tensor) -> torch.Tensor:
    """2^e for e from -126 to 127, each for 256 elements."""
    return ((e.int() + 127) << 23).view(torch.float32).repeat_interleave(BLOCK)


def _held_exponents(e: torch.Tensor) -> torch.Tensor:
    return e.int().clamp(_LOW, _HIGH)


def _block_exponents(x: torch.Tensor) -> torch.Tensor:
    """Of the largest finite number of each 256."""
    top = torch.where(x.isfinite(), x.abs(), 0.0).view(-1, BLOCK).amax(dim=1)
    return _held_exponents(top.view(torch.int32) >> 23)


def moments(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, exp_avg_scale: Optional[torch.Tensor] = None,
            exp_avg_sq_scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The moments of an ``AdamWState`` in 32 bits."""
    if exp_avg.dtype == torch.float32:
        return exp_avg, exp_avg_sq
    return (exp_avg.float() * _power(_held_exponents(exp_avg_scale) - 134),
            exp_avg_sq.float() * _power(_held_exponents(exp_avg_sq_scale) - 141))


def _mixed(x):
    x = ((x ^ (x >> 16)) * 0xBB67AE85) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _chances(at: int, n: int, step: int, seed: int):
    """16 random bits for each moment of ``n`` elements from place ``at`` on."""
    key = _mixed((_mixed(step & 0xFFFFFFFF) + seed * 0x9E3779B1) & 0xFFFFFFFF)
    i = torch.arange(at, at + n)
    h = _mixed(((i & 0xFFFFFFFF) * 0x9E3779B1 + (i >> 32) * 0xBB67AE85 + key) & 0xFFFFFFFF)
    return h & 0xFFFF, h >> 16


def _to_small(m, v, chance_m, chance_v):
    """Moments in 32 bits as (codes, exponents) of each."""
    em, ev = _block_exponents(m), _block_exponents(v)
    bits = (m.abs() * _power(134 - em) * 2.0 ** -120).view(torch.int32).long()
    cm = (bits + (chance_m << 4) + 8) >> 20
    cm = torch.where(m.isfinite(), torch.where(m.signbit(), cm + 128, cm), 0x7F)
    bits = (v * _power(141 - ev) * 2.0 ** -112).view(torch.int32).long()
    cv = (bits + (chance_v << 5) + 16) >> 21
    cv = torch.where(v > 0, cv.clamp(min=1), cv)
    cv = torch.where(v.isfinite(), cv, torch.where(v == math.inf, 0x7C, 0x7F))
    return cm.to(torch.uint8).view(torch.float8_e4m3fn), em.to(torch.uint8), cv.to(torch.uint8).view(torch.float8_e5m2), ev.to(torch.uint8)


def _as_signed(x, bits):
    return torch.where(x >= 1 << (bits - 1), x - (1 << bits), x)


def _split(wide):
    bits = wide.view(torch.int32).long() & 0xFFFFFFFF
    high = (bits + 0x8000) >> 16
    rest = torch.where(wide.isnan(), 0, bits - (high << 16)).to(torch.int16)
    high = torch.where(wide.isnan(), 0x7FFF, high & 0xFFFF)
    return _as_signed(high, 16).to(torch.int16).view(torch.bfloat16), rest


def _joined(high, rest):
    bits = ((high.view(torch.int16).long() << 16) + rest.long()) & 0xFFFFFFFF
    return _as_signed(bits, 32).to(torch.int32).view(torch.float32)


def _step_plain(params, grads, m, v, step, m_scale, v_scale, rest, norm, max_norm, lr, lr_at, b1, b2, eps, decay, seed):
    lr = float(lr_at) if lr_at is not None else lr
    kind = 0 if rest is None else 1 if rest.dtype == torch.int16 else 2
    # by a tensor: of a number and a tensor, the library takes the reciprocal and a product, which round twice
    clip = None if norm is None else (norm.new_tensor(max_norm) / (norm + 1e-6)).clamp(max=1.0).reshape(())
    counted = set()
    at = 0
    for i, (p, g) in enumerate(zip(params, grads)):
        n, size = p.numel(), flat_size([p.numel()])
        here, blocks = slice(at, at + size), slice(at // BLOCK, (at + size) // BLOCK)
        at += size
        if g is None or n == 0:
            continue
        c = i if step.numel() == len(params) else 0
        if c not in counted:
            step[c] += 1
            counted.add(c)
        t = int(step[c])
        rate = torch.tensor(lr / (1.0 - b1 ** t) if lr else 0.0, dtype=torch.float64).float()
        root = torch.tensor(1.0 / math.sqrt(1.0 - b2 ** t), dtype=torch.float64).float()
        grad = torch.zeros(size)
        grad[:n] = _in_memory_order(g).float()
        if clip is not None:
            grad = grad * clip
        scales = (m_scale[blocks], v_scale[blocks]) if m_scale is not None else (None, None)
        mm, vv = moments(m[here], v[here], *scales)
        mm = mm * b1 + grad * (1.0 - b1)
        vv = vv * b2 + (grad * grad) * (1.0 - b2)
        flat = _in_memory_order(p)
        w = torch.zeros(size)
        w[:n] = flat.float() if kind == 0 else rest[here][:n] if kind == 2 else _joined(flat, rest[here][:n])
        w = w * (1.0 - lr * decay) - (mm * rate) / (vv.double().sqrt().float() * root + eps)      # the library's 32-bit root is not always the nearest
        mm[n:], vv[n:], w[n:] = 0.0, 0.0, 0.0
        if m_scale is not None:
            mm, em, vv, ev = _to_small(mm, vv, *_chances(at - size, size, t, seed))
            m_scale[blocks].copy_(em)
            v_scale[blocks].copy_(ev)
        m[here].copy_(mm)
        v[here].copy_(vv)
        if kind == 1:
            w, low = _split(w)
            rest[here].copy_(low)
        elif kind == 2:
            rest[here].copy_(w)
        flat.copy_(w[:n])
