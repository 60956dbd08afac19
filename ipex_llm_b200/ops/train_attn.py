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

MAX_DIM = 128
_TILE = 128


def _fit(t: torch.Tensor) -> torch.Tensor:
    """The tensor as the kernels' 4-D maps take it: rows contiguous, other strides positive multiples of 16 bytes."""
    ok = t.stride(3) == 1 and t.data_ptr() % 16 == 0 and \
        all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:3], t.stride()[:3]))
    return t if ok else t.contiguous()


def _strided(t: torch.Tensor):
    """Pointer and strides; that of a dimension of size 1 is never taken."""
    return (ptr(t), *(8 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, scale, causal, window):
        lib, dev = stream_lib("train_attn"), q.device
        B, Hq, Sq, D = q.shape
        Hkv, Skv = k.shape[1], k.shape[2]
        grad = any(ctx.needs_input_grad[:3])
        q, k, v = _fit(q.detach()), _fit(k.detach()), _fit(v.detach())
        sizes = (B, Hq, Hkv, Sq, Skv, D, int(causal), window, scale, api.dtype_code(q.dtype))
        out = torch.empty(B, Sq, Hq, D, dtype=q.dtype, device=dev)
        stats = torch.empty(B, Hq, -(-Sq // _TILE) * _TILE, dtype=torch.float32, device=dev) if grad else None
        words = None
        with torch.cuda.device(dev):
            st = current_stream()
            if key_mask is not None:
                words = torch.empty(B, -(-Skv // _TILE) * (_TILE // 32), dtype=torch.int32, device=dev)
                kv = torch.empty(2, B, Skv, Hkv, D, dtype=q.dtype, device=dev)
                api.check(lib.ipex_attn_hide(ptr(key_mask), *key_mask.stride(), *_strided(k), *_strided(v), ptr(kv[0]), ptr(kv[1]),
                                             ptr(words), B, Hkv, Skv, D, st), "attn_hide")
                k, v = kv[0].transpose(1, 2), kv[1].transpose(1, 2)
            api.check(lib.ipex_attn_train_fwd(*_strided(q), *_strided(k), *_strided(v), ptr(words), ptr(out), ptr(stats), *sizes,
                                              ptr(error_flag(dev)), st), "attn_train_fwd")
        if grad:
            ctx.save_for_backward(q, k, v, out, stats, words)
            ctx.sizes = sizes
        return out.transpose(1, 2)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, out, stats, words = ctx.saved_tensors
        B, Hq, Hkv, Sq, Skv, D = ctx.sizes[:6]
        dev = q.device
        g = _fit(g)
        dq = torch.empty(B, Sq, Hq, D, dtype=q.dtype, device=dev)
        dk = torch.empty(B, Skv, Hkv, D, dtype=q.dtype, device=dev)
        dv = torch.empty(B, Skv, Hkv, D, dtype=q.dtype, device=dev)
        delta = torch.empty_like(stats)
        with torch.cuda.device(dev):
            bound = torch.zeros(B, Hkv, 2, dtype=torch.int32, device=dev) if q.dtype == torch.float16 else None
            rc = stream_lib("train_attn").ipex_attn_train_bwd(
                *_strided(q), *_strided(k), *_strided(v), ptr(words), ptr(out), ptr(stats), *_strided(g), ptr(delta), ptr(bound),
                ptr(dq), ptr(dk), ptr(dv), *ctx.sizes, ptr(error_flag(dev)), current_stream())
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
    return (p @ vf).reshape(B, Hq, Sq, D).to(q.dtype)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
              window: int = 0, key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(``q`` ``k``^T * scale) ``v`` with gradients of all three: ``q [B, Hq, Sq, D]``, ``k`` and ``v [B, Hkv, Skv, D]``,
    each key head shared by Hq / Hkv query heads.  Returns ``[B, Hq, Sq, D]`` as a view of ``[B, Sq, Hq, D]``.

    ``causal``: query i sees keys up to i + Skv - Sq (the queries are the last of the keys' sequence); ``window``: and only so
    many, itself among them.  ``key_mask [B, Skv]``: True (or not 0) for real keys, as a tokenizer's attention mask; what hidden
    rows hold, NaN included, takes no part.  A query that sees no key gives zeros and gets no gradient.  ``scale`` (positive)
    defaults to D^-1/2.

    GPU: fp16 or bf16, D a multiple of 8 up to 128, any strides (rows that are not contiguous, or not aligned to 16 bytes, are
    copied).  Scores, sums and gradients are summed in 32 bits; probabilities and their gradients are rounded to 16 bits
    where they enter a product.  The results do not depend on the order in which anything runs.
    """
    invalidInputError(q.dim() == 4 and k.dim() == 4 and tuple(k.shape) == tuple(v.shape),
                      f"attention: q, k and v should be [batch, heads, tokens, dim], k and v alike; got {tuple(q.shape)}, "
                      f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, Hq, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    invalidInputError(k.shape[0] == B and k.shape[3] == D and Hkv >= 1 and Hq >= 1 and Hq % Hkv == 0,
                      f"attention: keys {tuple(k.shape)} do not fit queries {tuple(q.shape)}")
    invalidInputError(q.dtype == k.dtype == v.dtype and q.device == k.device == v.device,
                      "attention: q, k and v should have one type and lie on one device")
    scale = D ** -0.5 if scale is None else float(scale)
    invalidInputError(0.0 < scale < 1e30, f"attention: the scale has to be positive and finite, got {scale}")
    window = int(window)
    invalidInputError(0 <= window < 1 << 31 and (causal or window == 0),
                      f"attention: a window of {window} tokens needs causal attention and has to be positive (0: none)")
    if key_mask is not None:
        invalidInputError(tuple(key_mask.shape) == (B, Skv) and key_mask.device == q.device and
                          not (key_mask.is_floating_point() or key_mask.is_complex()),
                          f"attention: key_mask should be [{B}, {Skv}] truth values on {q.device}, got {tuple(key_mask.shape)} of "
                          f"{key_mask.dtype} on {key_mask.device}")
        key_mask = key_mask if key_mask.dtype == torch.bool else key_mask != 0
    if not q.is_cuda:
        invalidInputError(q.is_floating_point(), f"attention: inputs of type {q.dtype} are not supported")
        return _attention_plain(q, k, v, key_mask, scale, causal, window)
    invalidInputError(q.dtype in (torch.float16, torch.bfloat16), f"attention: {q.dtype} is not supported on the GPU (float16 and "
                                                                  "bfloat16 are)")
    invalidInputError(8 <= D <= MAX_DIM and D % 8 == 0, f"attention: heads of {D} are not supported (multiples of 8 up to 128 are)")
    invalidInputError(B <= 65535 and max(Sq, Skv) < 1 << 23, "attention: too many sequences or tokens")
    if q.numel() == 0 or k.numel() == 0:
        return q.masked_fill(torch.ones_like(q, dtype=torch.bool), 0.0) + (k.sum() + v.sum()) * 0
    return _Attention.apply(q, k, v, key_mask, scale, bool(causal), window)
