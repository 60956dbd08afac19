"""The attention with a gradient behind the transformers attention interface, for finetuning: a decoder whose attention goes
through the registry runs ``ops.train_attn.attention`` where that can compute it, and the package's usual path elsewhere
(soft-capped scores, dropout, masks that are neither padding nor a window, other types and head sizes, single tokens).

Masks: a causal mask, with or without a window, stays what it is, and padding stays ``[batch, keys]`` truth values; no mask of
the size of queries x keys is made for them.
"""
from __future__ import annotations

import torch

from ..ops.train_attn import MAX_DIM, MAX_HEADS, attention
from .common import _uses_attention_registry, attention_interface

TRAIN_INTERFACE_NAME = "ipex_llm_train"


def _is_window(mask_function, q_length: int, kv_length: int, window: int, device) -> bool:
    """Is this mask causal attention to the last ``window`` keys, at every query and key?"""
    q = torch.arange(q_length, device=device).view(1, 1, -1, 1) + (kv_length - q_length)
    key = torch.arange(kv_length, device=device).view(1, 1, 1, -1)
    zero = torch.zeros((1, 1, 1, 1), dtype=torch.long, device=device)
    try:
        own = mask_function(zero, zero, q, key)
    except Exception:  # noqa: BLE001  (a function that takes single indices only)
        return False
    return torch.is_tensor(own) and bool(((key <= q) & (key > q - window) == own).all())


def _mask(batch_size, q_length, kv_length, q_offset=0, kv_offset=0, mask_function=None, attention_mask=None, **kwargs):
    """None or the padding mask [batch, keys] for causal attention over all keys or a window of them; else the mask that the usual
    path takes."""
    from transformers.masking_utils import causal_mask_function, sdpa_mask
    window, device = kwargs.get("local_size"), kwargs.get("device", "cpu")
    if attention_mask is not None:
        device = attention_mask.device
    ends = not torch.is_tensor(q_offset) and q_length > 1 and kv_offset == 0 and q_offset + q_length == kv_length
    if ends and (attention_mask is None or attention_mask.shape == (batch_size, kv_length)):
        if mask_function is causal_mask_function:
            return attention_mask
        if window and _is_window(mask_function, q_length, kv_length, window, device):
            return attention_mask
    return sdpa_mask(batch_size=batch_size, q_length=q_length, kv_length=kv_length, q_offset=q_offset, kv_offset=kv_offset,
                     mask_function=mask_function, attention_mask=attention_mask, **kwargs)


def _whole_mask(key_mask, q_length: int, causal: bool, window: int):
    """The mask [batch, 1, queries, keys] that a padding mask stands for."""
    kv_length = key_mask.shape[1]
    see = key_mask.bool()[:, None, None, :].expand(-1, 1, q_length, -1)
    if causal:
        q = torch.arange(q_length, device=key_mask.device).view(-1, 1) + (kv_length - q_length)
        key = torch.arange(kv_length, device=key_mask.device)
        see = see & (key <= q)
        if window:
            see = see & (key > q - window)
    return see


def train_attention_interface(module, query, key, value, attention_mask=None, dropout: float = 0.0, scaling=None,
                              is_causal=None, softcap=None, sliding_window=None, **kwargs):
    """``attention_interface``, with the gradient's own kernels where they apply."""
    q, k, v = query, key, value
    if q.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    Hq, Sq, D = q.shape[1:]
    Hkv, Skv = k.shape[1:3]
    causal = getattr(module, "is_causal", True) if is_causal is None else bool(is_causal)
    window = int(sliding_window or 0) if causal and (sliding_window or 0) < Skv else 0
    padding = attention_mask is not None and attention_mask.dim() == 2
    causal = causal or padding
    scale = D ** -0.5 if scaling is None else float(scaling)
    fits = (attention_mask is None or padding) and (torch.is_grad_enabled() or module.training) and Sq > 1 \
        and Sq <= Skv and not softcap and not (dropout and module.training) and k.shape == v.shape and Hq % Hkv == 0 \
        and 1e-4 <= scale <= 1e4 and q.dtype == k.dtype == v.dtype and q.device == k.device == v.device \
        and not any(torch.is_tensor(t) for n, t in kwargs.items() if n in ("position_bias", "s_aux", "sinks"))
    if fits and q.is_cuda:
        fits = q.dtype in (torch.float16, torch.bfloat16) and D <= MAX_DIM and D % 8 == 0 and Hq + Hkv <= MAX_HEADS
    if fits:
        return attention(q, k, v, scale, causal, window, attention_mask if padding else None).transpose(1, 2), None
    if padding:
        attention_mask = _whole_mask(attention_mask, Sq, causal, window)
    return attention_interface(module, query, key, value, attention_mask, dropout, scaling, is_causal, softcap, sliding_window,
                               **kwargs)


def use_train_attention(model) -> bool:
    """Point every sub-model whose attention goes through the registry at ``train_attention_interface``; the others keep theirs.
    False when there is none."""
    try:
        from transformers import AttentionInterface, AttentionMaskInterface
    except ImportError:
        return False
    AttentionInterface.register(TRAIN_INTERFACE_NAME, train_attention_interface)
    AttentionMaskInterface.register(TRAIN_INTERFACE_NAME, _mask)
    found = {}
    for mod in model.modules():
        cfg = getattr(mod, "config", None)
        if cfg is not None and hasattr(cfg, "to_dict") and _uses_attention_registry(mod):
            found[id(cfg)] = cfg
    for cfg in found.values():
        cfg._attn_implementation = TRAIN_INTERFACE_NAME
    return bool(found)
