"""Attention with a gradient (``attn_train_tcgen05.cu``): forward keeps one number for each row, backward computes the
probabilities from it again, so that nothing of the size of queries x keys is ever held.

On a CUDA tensor the package's own kernels run, on the current stream of the tensor's device; on the CPU it is plain PyTorch.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ..native import cuda_api as api
from ..native.lib import current_stream, ptr, stream_lib
from ..utils.common import invalidInputError
from .cuda_ops import error_flag
from .gradients import on, refuse_tangents

MAX_DIM = 128
MAX_HEADS = 65535       # of queries and keys together
MAX_TOKENS = 1 << 22
_TILE = 128


def _fit(t: torch.Tensor):
    """The tensor as the kernels' 4-D maps take it, rows contiguous, aligned to 16 bytes, and other strides positive multiples of
    16 bytes (copied where it is not), behind its pointer and strides.  The stride of a dimension of size 1 is never taken: 8
    stands for it."""
    (B, H, S, _), (b, h, s, d) = t.shape, t.stride()
    b, h, s = b if B > 1 else 8, h if H > 1 else 8, s if S > 1 else 8
    at = t.data_ptr()
    if d != 1 or at & 15 or (b | h | s) & 7 or not (b and h and s):
        return _fit(t.clone(memory_format=torch.contiguous_format))          # a contiguous one may still lie at any address
    return at, b, h, s, t


def _forward(q, k, v, key_mask, scale, causal, window, keep: bool):
    """The outputs [B, Sq, Hq, D] and, with ``keep``, what the backward pass needs."""
    lib, dev = stream_lib("train_attn"), q.device
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    *q_at, q = _fit(q)
    *k_at, k = _fit(k)
    *v_at, v = _fit(v)
    sizes = (B, Hq, Hkv, Sq, Skv, D, int(causal), window, scale, api.dtype_code(q.dtype))
    out = torch.empty((B, Sq, Hq, D), dtype=q.dtype, device=dev)
    stats = low = words = None
    if keep:
        stats = torch.empty((B, Hq, -(-Sq // _TILE) * _TILE), dtype=torch.float32, device=dev)
        low = torch.empty_like(out)
    with on(dev):
        st, err = current_stream(), ptr(error_flag(dev))
        if key_mask is not None:
            words = torch.empty((B, -(-Skv // _TILE) * (_TILE // 32)), dtype=torch.int32, device=dev)
            k, v = torch.empty((2, B, Skv, Hkv, D), dtype=q.dtype, device=dev).transpose(2, 3).unbind(0)
            api.check(lib.ipex_attn_hide(ptr(key_mask), *key_mask.stride(), *k_at, *v_at, ptr(k), ptr(v), ptr(words), B, Hkv, Skv, D,
                                         st), "attn_hide")
            *k_at, k = _fit(k)
            *v_at, v = _fit(v)
        api.check(lib.ipex_attn_train_fwd(*q_at, *k_at, *v_at, ptr(words), ptr(out), ptr(low), ptr(stats), *sizes, err, st),
                  "attn_train_fwd")
    return out, (q, k, v, out, low, stats, words), sizes


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, scale, causal, window):
        out, kept, ctx.sizes = _forward(q, k, v, key_mask, scale, causal, window, True)
        ctx.save_for_backward(*kept)
        return out.transpose(1, 2)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, out, low, stats, words = ctx.saved_tensors
        B, Hq, Hkv, Sq, Skv, D = ctx.sizes[:6]
        dev = q.device
        *q_at, q = _fit(q)
        *k_at, k = _fit(k)
        *v_at, v = _fit(v)
        *g_at, g = _fit(g)
        dq = torch.empty_like(out)
        dk = torch.empty((B, Skv, Hkv, D), dtype=q.dtype, device=dev)
        dv = torch.empty_like(dk)
        work = torch.empty(9 * stats.numel() + 2 * B * Hkv, dtype=torch.float32, device=dev)
        with on(dev):
            rc = stream_lib("train_attn").ipex_attn_train_bwd(
                *q_at, *k_at, *v_at, ptr(words), ptr(out), ptr(low), ptr(stats), *g_at, ptr(work), ptr(dq), ptr(dk), ptr(dv),
                *ctx.sizes, ptr(error_flag(dev)), current_stream())
        api.check(rc, "attn_train_bwd")
        return dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2), None, None, None, None


def _visible(Sq, Skv, causal, window, key_mask, device):
    last = torch.arange(Sq, device=device).view(-1, 1) + (Skv - Sq)
    key = torch.arange(Skv, device=device).view(1, -1)
    see = torch.ones(Sq, Skv, dtype=torch.bool, device=device)
    if causal:
        see = see & (key <= last)
    if window:
        see = see & (key > last - window)
    return see if key_mask is None else see & key_mask[:, None, None, :]


def _attention_plain(q, k, v, key_mask, scale, causal, window):
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    see = _visible(Sq, Skv, causal, window, key_mask, q.device)
    if key_mask is not None:                       # what hidden rows hold takes no part, not even times 0
        k, v = (torch.where(key_mask[:, None, :, None], t, torch.zeros((), dtype=t.dtype)) for t in (k, v))
    qg = q.to(wide).reshape(B, Hkv, Hq // Hkv, Sq, D)
    kf, vf = k.to(wide).unsqueeze(2), v.to(wide).unsqueeze(2)
    see = see if see.dim() == 2 else see.unsqueeze(2)
    s = (qg @ kf.transpose(-1, -2) * scale).masked_fill(~see, -math.inf)
    p = torch.softmax(s.masked_fill(~see.any(dim=-1, keepdim=True), 0.0), dim=-1).masked_fill(~see, 0.0)
    return (p @ vf).reshape(B, Hq, Sq, D).to(q.dtype).transpose(1, 2).contiguous().transpose(1, 2)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
              window: int = 0, key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(``q`` ``k``^T * scale) ``v`` with gradients of all three: ``q [B, Hq, Sq, D]``, ``k`` and ``v [B, Hkv, Skv, D]``,
    each key head shared by Hq / Hkv query heads.  Returns ``[B, Hq, Sq, D]`` as a view of ``[B, Sq, Hq, D]``.

    ``causal``: query i sees keys up to i + Skv - Sq (the queries are the last of the keys' sequence); ``window``: and only so
    many, itself among them.  ``key_mask [B, Skv]``: True (or not 0) for real keys, as a tokenizer's attention mask; what hidden
    rows hold, NaN included, takes no part.  A query that sees no key gives zeros and gets no gradient.  ``scale`` (1e-4 to
    1e4) defaults to D^-1/2.

    GPU: backward gradients alone (a tangent of forward-mode differentiation is refused), fp16 or bf16, D a multiple of 8 up to
    128, any strides (rows that are not contiguous, or not aligned to 16 bytes, are copied).  Scores, sums and gradients are
    summed in 32 bits; probabilities and their gradients are rounded to 16 bits where they enter a product (twice as many bits
    for queries of few keys).  In fp16 the backward pass takes scores up to 2^30 * scale, and rows whose outputs and gradients
    have a product up to 2^30 (NaN past 2^31).  The results do not depend on the order in which anything runs.  A causal limit or
    a window hides a key by a probability of 0: NaN and infinities in such a row may spread to earlier queries, as they do in the
    formula; behind ``key_mask`` they do not.  Those of a query, or of its output's gradient, spread to dk and dv even where the
    query sees nothing.
    """
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        invalidInputError(False, f"attention: q, k and v should be [batch, heads, tokens, dim], k and v alike; got {tuple(q.shape)}, "
                                 f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, Hq, Sq, D = q.shape
    _, Hkv, Skv, _ = k.shape
    if k.shape[0] != B or k.shape[3] != D or D < 1 or Hkv < 1 or Hq < 1 or Hq % Hkv != 0:
        invalidInputError(False, f"attention: keys {tuple(k.shape)} do not fit queries {tuple(q.shape)}")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        invalidInputError(False, "attention: q, k and v should have one type and lie on one device")
    scale, window = D ** -0.5 if scale is None else float(scale), int(window)
    if not 1e-4 <= scale <= 1e4:
        invalidInputError(False, f"attention: the scale should lie between 1e-4 and 1e4, got {scale}")
    if not 0 <= window < 1 << 31 or (window and not causal):
        invalidInputError(False, f"attention: a window of {window} tokens needs causal attention and has to be positive (0: none)")
    if key_mask is not None:
        if key_mask.shape != (B, Skv) or key_mask.device != q.device or key_mask.is_floating_point() or key_mask.is_complex():
            invalidInputError(False, f"attention: key_mask should be [{B}, {Skv}] truth values on {q.device}, got "
                                     f"{tuple(key_mask.shape)} of {key_mask.dtype} on {key_mask.device}")
        key_mask = key_mask if key_mask.dtype == torch.bool else key_mask != 0
    if not q.is_cuda:
        invalidInputError(q.is_floating_point(), "attention: inputs should be floating-point numbers")
        return _attention_plain(q, k, v, key_mask, scale, causal, window)
    refuse_tangents("attention", q, k, v)
    if q.dtype not in (torch.float16, torch.bfloat16):
        invalidInputError(False, f"attention: {q.dtype} is not supported on the GPU (float16 and bfloat16 are)")
    if D > MAX_DIM or D % 8:
        invalidInputError(False, f"attention: heads of {D} are not supported (multiples of 8 up to {MAX_DIM} are)")
    if Hq + Hkv > MAX_HEADS:
        invalidInputError(False, f"attention: {Hq} and {Hkv} heads are too many ({MAX_HEADS} together are not)")
    if B > 65535 or Sq > MAX_TOKENS or Skv > MAX_TOKENS:
        invalidInputError(False, f"attention: {B} sequences of {Sq} queries and {Skv} keys are too many (65535 of {MAX_TOKENS} "
                                 "are not)")
    if q.numel() == 0 or k.numel() == 0:
        zeros = q.masked_fill(torch.ones_like(q, dtype=torch.bool), 0.0) + (k.sum() + v.sum()) * 0
        return zeros.transpose(1, 2).contiguous().transpose(1, 2)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, key_mask, scale, bool(causal), window)
    return _forward(q, k, v, key_mask, scale, bool(causal), window, False)[0].transpose(1, 2)
