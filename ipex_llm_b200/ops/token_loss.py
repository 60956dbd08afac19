"""What stands behind an output layer (``token_loss.cu``): log probabilities of given tokens with their entropy and the best
alternatives, and the divergence from a teacher's top logits, each with the gradient of the logits.

On a CUDA tensor every function calls the package's own kernels on the current stream of the tensor's device, in the logits'
type with 32-bit sums, and no copy of the logits in 32 bits is made; on the CPU it is plain PyTorch.  Logits may be a view with
any strides between rows.  Gradients are those of a backward pass; on the GPU tangents of forward-mode differentiation are
refused.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from ..native import cuda_api as api
from ..native.lib import current_stream, ptr, stream_lib
from ..utils.common import invalidInputError
from .cuda_ops import error_flag
from .gradients import on, refuse_tangents

MAX_TOP = 32             # alternatives of a row
MAX_TEACHER = 1024       # tokens of a teacher's row
MAX_TAIL_VOCAB = 1 << 19
IGNORE = -100
_NO_TOKEN = -2.0 ** 127   # a row whose largest logit is not above this has no token
_NOTHING = 2.0 ** -100    # a probability of all other tokens that counts as none


class TokenLogprobs(NamedTuple):
    """``logprob`` and ``entropy`` have a gradient; the alternatives have none."""
    logprob: torch.Tensor                          # [...]
    entropy: Optional[torch.Tensor]                # [...], None unless asked for
    top_logprobs: Optional[torch.Tensor]           # [..., top], largest first
    top_ids: Optional[torch.Tensor]                # [..., top]; of equal ones the lower index first


def _rows(logits: torch.Tensor):
    """The logits with unit stride along the vocabulary, and (outer stride, inner stride, rows to an outer index)."""
    if logits.dim() > 3:
        logits = logits.reshape(-1, *logits.shape[-2:])
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if logits.dim() == 3:
        return logits, logits.stride(0), logits.stride(1), logits.shape[1]
    return logits, 0, logits.stride(0) if logits.dim() == 2 else 0, logits.shape[0] if logits.dim() == 2 else 1


def _check_logits(logits: torch.Tensor, temperature: float, what: str):
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= 1 << 30:
        invalidInputError(False, f"{what}: logits need a vocabulary of 1 to 2^30 tokens, got shape {tuple(logits.shape)}")
    if logits.dtype not in (torch.float16, torch.bfloat16, torch.float32) and (logits.is_cuda or logits.dtype != torch.float64):
        invalidInputError(False, f"{what}: logits of type {logits.dtype} are not supported")
    if logits.is_cuda and logits.numel() // logits.shape[-1] > 1 << 27:
        invalidInputError(False, f"{what}: more than 2^27 rows")
    if not 1e-6 <= temperature <= 1e6:
        invalidInputError(False, f"{what}: the temperature should lie between 1e-6 and 1e6, got {temperature}")


def _check_like(t: torch.Tensor, shape, device, what: str, whole: bool):
    if t.shape != shape:
        invalidInputError(False, f"{what} should have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        invalidInputError(False, f"{what} should be on {device}, like the logits, got {t.device}")
    if (t.is_floating_point() == whole) or t.is_complex() or t.dtype == torch.bool:
        invalidInputError(False, f"{what} should hold {'token ids' if whole else 'floating-point numbers'}, got {t.dtype}")


def _token_logprobs(logits, targets, temperature, entropy, top, ignore, keep):
    """The results, and with ``keep`` each row's statistics for the backward pass."""
    x, s0, s1, n1 = _rows(logits)
    shape, V, dev = targets.shape, logits.shape[-1], logits.device
    rows = targets.numel()
    logprob = torch.empty(shape, dtype=torch.float32, device=dev)
    ent = torch.empty_like(logprob) if entropy else None
    stats = torch.empty((rows, 4), dtype=torch.float32, device=dev) if keep else None
    top_lp = torch.empty((*shape, top), dtype=torch.float32, device=dev) if top else None
    top_id = torch.empty((*shape, top), dtype=torch.int64, device=dev) if top else None
    if rows:
        with on(dev):
            rc = stream_lib("token_loss").ipex_token_logprobs(
                ptr(x), s0, s1, n1, ptr(targets), ptr(logprob), ptr(ent), ptr(stats), ptr(top_lp), ptr(top_id), rows, V, top, ignore,
                temperature, api.dtype_code(x.dtype), ptr(error_flag(dev)), current_stream())
        api.check(rc, "token_logprobs")
    return (logprob, ent, top_lp, top_id), stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, entropy, top, ignore):
        ctx.set_materialize_grads(False)
        out, stats = _token_logprobs(logits, targets, temperature, entropy, top, ignore, True)
        if top:
            ctx.mark_non_differentiable(*out[2:])
        ctx.save_for_backward(logits, targets, stats)
        ctx.temperature, ctx.ignore = temperature, ignore
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_ent, _lp, _id):
        if g is None and g_ent is None:
            return (None,) * 6
        logits, targets, stats = ctx.saved_tensors
        x, s0, s1, n1 = _rows(logits)
        dev, rows = logits.device, targets.numel()
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        g = None if g is None else g.float().contiguous()
        g_ent = None if g_ent is None else g_ent.float().contiguous()
        if rows:
            with on(dev):
                rc = stream_lib("token_loss").ipex_token_logprobs_grad(
                    ptr(x), s0, s1, n1, ptr(targets), ptr(stats), ptr(g), ptr(g_ent), ptr(dx), rows, x.shape[-1], ctx.ignore,
                    ctx.temperature, api.dtype_code(x.dtype), current_stream())
            api.check(rc, "token_logprobs_grad")
        return dx, None, None, None, None, None


def _wide(logits: torch.Tensor) -> torch.Tensor:
    return logits if logits.dtype == torch.float64 else logits.float()


def _hidden_to_zero(logp: torch.Tensor) -> torch.Tensor:
    """Log probabilities with 0 for hidden tokens: what multiplies their probability of 0."""
    return logp.masked_fill(logp == -math.inf, 0.0)


def _token_logprobs_plain(logits, targets, temperature, entropy, top, ignore):
    y = _wide(logits) / temperature
    real = targets != ignore
    none = logits.detach().amax(dim=-1) <= _NO_TOKEN                # rows without any token
    logp = torch.log_softmax(y.masked_fill(none.unsqueeze(-1), 0.0), dim=-1)
    lp = logp.gather(-1, targets.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    lp = torch.where(real, torch.where(none, -math.inf, lp), 0.0)
    ent = top_lp = top_id = None
    if entropy:
        ent = -(logp.exp() * _hidden_to_zero(logp)).sum(dim=-1)
        ent = torch.where(real & ~none, ent, 0.0)
    if top:
        order = torch.sort(logits.detach(), dim=-1, descending=True, stable=True).indices
        top_id = order[..., :top].contiguous()
        top_lp = logp.detach().gather(-1, top_id).masked_fill(none.unsqueeze(-1), -math.inf)
    return lp, ent, top_lp, top_id


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0, entropy: bool = False, top: int = 0,
                   ignore_index: int = IGNORE) -> TokenLogprobs:
    """Log probabilities of ``targets [...]`` under softmax(``logits [..., V]`` / temperature).

    ``entropy``: that of each row as well; ``top`` (up to 32): the best tokens of each row with their log probabilities.  All
    results but the ids are 32-bit (64 for 64-bit logits on the CPU).  Rows whose target is ``ignore_index`` give a log
    probability and an entropy of 0 and no gradient, whatever their logits hold, and their alternatives all the same.  A logit
    of -inf hides its token, as the lowest value of bf16 or 32 bits does; a row of nothing else gives a log probability of -inf,
    an entropy of 0 and no gradient.  A target
    outside of the vocabulary raises on the CPU; on the GPU its results are NaN, and ``cuda_ops.check_error_flag`` reports 61.

    16-bit and 32-bit logits; the gradient has the logits' type.
    """
    _check_logits(logits, temperature, "token_logprobs")
    _check_like(targets, logits.shape[:-1], logits.device, "token_logprobs: targets", True)
    most = min(MAX_TOP, logits.shape[-1])
    if not 0 <= top <= most:
        invalidInputError(False, f"token_logprobs: top should be between 0 and {most}, got {top}")
    if logits.is_cuda:
        refuse_tangents("token_logprobs", logits)
        args = (logits, targets.to(torch.int64).contiguous(), float(temperature), bool(entropy), int(top), int(ignore_index))
        if logits.requires_grad and torch.is_grad_enabled():
            return TokenLogprobs(*_TokenLogprobs.apply(*args))
        return TokenLogprobs(*_token_logprobs(*args, False)[0])
    outside = (targets != ignore_index) & ((targets < 0) | (targets >= logits.shape[-1]))
    if bool(outside.any()):
        invalidInputError(False, "token_logprobs: a target lies outside of the vocabulary")
    return TokenLogprobs(*_token_logprobs_plain(logits, targets.long(), temperature, entropy, top, ignore_index))


def _distill(logits, ids, values, lse, temperature, keep):
    """The loss, and with ``keep`` each row's statistics for the backward pass."""
    x, s0, s1, n1 = _rows(logits)
    dev, V, K = logits.device, logits.shape[-1], ids.shape[-1]
    loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
    rows = loss.numel()
    stats = torch.empty((rows, 8), dtype=torch.float32, device=dev) if keep else None
    if rows:
        with on(dev):
            rc = stream_lib("token_loss").ipex_distill(
                ptr(x), s0, s1, n1, ptr(ids), ptr(values), ptr(lse), ptr(loss), ptr(stats), rows, V, K, temperature,
                api.dtype_code(x.dtype), ptr(error_flag(dev)), current_stream())
        api.check(rc, "distill")
    return loss, stats


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, values, lse, temperature):
        loss, stats = _distill(logits, ids, values, lse, temperature, True)
        ctx.save_for_backward(logits, ids, values, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, ids, values, stats = ctx.saved_tensors
        x, s0, s1, n1 = _rows(logits)
        dev = logits.device
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        g = g.float().contiguous()
        if g.numel():
            with on(dev):
                rc = stream_lib("token_loss").ipex_distill_grad(
                    ptr(x), s0, s1, n1, ptr(ids), ptr(values), ptr(stats), ptr(g), ptr(dx), g.numel(), x.shape[-1], ids.shape[-1],
                    ctx.temperature, api.dtype_code(x.dtype), current_stream())
            api.check(rc, "distill_grad")
        return dx, None, None, None, None


def _distill_plain(logits, ids, values, lse, temperature):
    y = _wide(logits) / temperature
    none = logits.detach().amax(dim=-1, keepdim=True) <= _NO_TOKEN
    logp = torch.log_softmax(y.masked_fill(none, 0.0), dim=-1)
    given = ids >= 0
    at = ids.clamp(min=0)
    t = (values.to(y.dtype) / temperature).masked_fill(~given, -math.inf)
    empty = ~(t > -math.inf).any(dim=-1, keepdim=True)             # rows without a teacher's token
    logq = t - (torch.logsumexp(t.masked_fill(empty, 0.0), dim=-1, keepdim=True) if lse is None else lse.to(y.dtype).unsqueeze(-1))
    q = torch.exp(logq)
    own = logp.masked_fill(none, -math.inf).gather(-1, at)
    loss = torch.where(q != 0, q * (logq - torch.where(q != 0, own, 0.0)), 0.0).sum(dim=-1, keepdim=True)
    if lse is not None:
        rest = (1.0 - q.sum(dim=-1, keepdim=True)).clamp(min=0.0)
        hide = torch.zeros(logits.shape, dtype=torch.int32, device=logits.device).scatter_add_(-1, at, given.int()) > 0
        left = torch.exp(logp).masked_fill(hide, 0.0).sum(dim=-1, keepdim=True)
        some = (rest > 0) & (left > _NOTHING)
        loss = loss + torch.where(some, rest * (torch.log(rest.clamp(min=1e-38)) - torch.log(torch.where(some, left, 1.0))), 0.0)
    loss = torch.where(empty, 0.0, loss)
    return (loss * (temperature * temperature)).squeeze(-1)


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, temperature: float = 1.0,
                 teacher_logsumexp: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Divergence ``[...]`` (32-bit) of the student's softmax(``logits [..., V]`` / temperature) from a teacher of which the top
    tokens are kept: ``temperature^2 * sum_k q_k (log q_k - log p_k)`` with q = softmax(``teacher_logits [..., K]`` /
    temperature) at ``teacher_ids [..., K]`` (K up to 1024).

    With ``teacher_logsumexp [...]``, the logsumexp of all the teacher's logits / temperature, q_k are the teacher's own
    probabilities, and what they leave is compared with what the student gives to all other tokens together (left out where that
    is nothing: less than 2^-100).  Ids below 0 are padding; a row of nothing else gives 0 and no gradient.  An id that occurs
    twice counts twice.  An id past the vocabulary raises on the CPU; on the GPU its row is NaN, and
    ``cuda_ops.check_error_flag`` reports 61.

    The gradient goes to the logits alone (in their type: 16 or 32 bits); the teacher is a constant.
    """
    _check_logits(logits, temperature, "distill_loss")
    if teacher_ids.dim() != logits.dim() or not 1 <= teacher_ids.shape[-1] <= MAX_TEACHER:
        invalidInputError(False, f"distill_loss: teacher_ids should hold 1 to {MAX_TEACHER} tokens for each row, got shape "
                                 f"{tuple(teacher_ids.shape)}")
    rows = logits.shape[:-1]
    shape = (*rows, teacher_ids.shape[-1])
    _check_like(teacher_ids, shape, logits.device, "distill_loss: teacher_ids", True)
    _check_like(teacher_logits, shape, logits.device, "distill_loss: teacher_logits", False)
    lse = teacher_logsumexp
    if lse is not None:
        _check_like(lse, rows, logits.device, "distill_loss: teacher_logsumexp", False)
        if logits.shape[-1] > MAX_TAIL_VOCAB:
            invalidInputError(False, f"distill_loss: teacher_logsumexp takes vocabularies up to {MAX_TAIL_VOCAB}")
    if logits.is_cuda:
        refuse_tangents("distill_loss", logits)
        args = (logits, teacher_ids.to(torch.int64).contiguous(), teacher_logits.detach().float().contiguous(),
                None if lse is None else lse.detach().float().contiguous(), float(temperature))
        if logits.requires_grad and torch.is_grad_enabled():
            return _Distill.apply(*args)
        return _distill(*args, False)[0]
    if bool((teacher_ids >= logits.shape[-1]).any()):
        invalidInputError(False, "distill_loss: an id lies outside of the vocabulary")
    return _distill_plain(logits, teacher_ids.long(), teacher_logits.detach(), None if lse is None else lse.detach(), temperature)
