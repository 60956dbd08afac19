"""The attention with a gradient behind the transformers attention interface, for finetuning: a decoder whose attention goes
through the registry, or through this package's own decoder forward, runs ``ops.train_attn.attention`` where that can compute
it, and the package's usual path elsewhere (soft-capped scores, dropout, masks that are neither padding nor a window, other
types and head sizes, single tokens).

Masks: a causal mask, with or without a window, stays what it is, and padding stays ``[batch, keys]``; no mask of the size of
queries x keys is kept for them (a window's function is looked at, some rows at a time).  Padding and windows travel in a type
that no arithmetic takes (``_compact``): a module that would use such a mask in a way of its own raises, where truth values
``[batch, keys]`` would pass for a mask of scores without a causal limit.
"""
from __future__ import annotations

import torch

from ..ops.train_attn import MAX_DIM, MAX_HEADS, attention
from .common import TRAIN_INTERFACE_NAME, _uses_attention_registry, attention_interface
from .decoder import decoder_attention_forward

_LOOKED_AT = 1 << 24               # pairs of a query and a key at a time, where a mask function is looked at
_CARRIER = torch.float8_e5m2       # the bytes of truth values; sums, products, comparisons with other types and SDPA refuse it


def _compact(padding, window: int = 0, kv_length: int = 0, device=None):
    """What this interface's masks are, beside None (causal attention over all keys): truth values [batch, keys], and with a
    window [batch, keys, window] of stride 0, or [0, keys, window] where no key is hidden.  The window has to come with the mask:
    not every attention module hands it on, and it goes through whatever passes a tensor's shape on."""
    if padding is None:
        return torch.empty((0, kv_length, window), dtype=_CARRIER, device=device) if window else None
    padding = (padding if padding.dtype == torch.bool else padding != 0).view(_CARRIER)
    return padding.unsqueeze(2).expand(-1, -1, window) if window else padding


def is_compact(mask) -> bool:
    return mask is not None and mask.dtype == _CARRIER


def _parts(mask):
    """The truth values [batch, keys] (None: all keys) and the window (0: none) of a compact mask."""
    if mask.dim() == 2:
        return mask.view(torch.bool), 0
    return mask[..., 0].view(torch.bool) if mask.shape[0] else None, mask.shape[2]


def whole_mask(mask, q_length: int):
    """The truth values [batch or 1, 1, queries, keys] that one of this interface's masks stands for; other masks as they are."""
    if not is_compact(mask):
        return mask
    padding, window = _parts(mask)
    kv_length = mask.shape[1]
    q = torch.arange(q_length, device=mask.device).view(-1, 1) + (kv_length - q_length)
    key = torch.arange(kv_length, device=mask.device)
    see = (key <= q) & (key > q - window) if window else key <= q
    return see[None, None] if padding is None else padding[:, None, None, :] & see


def _is_window(mask_function, q_length: int, kv_length: int, window: int, device, batch_size: int = 1) -> bool:
    """Is this mask causal attention to the last ``window`` keys, in every sequence, at every query and key?  Looked at some rows at
    a time."""
    rows = max(1, _LOOKED_AT // (kv_length * batch_size))
    key = torch.arange(kv_length, device=device).view(1, 1, 1, -1)
    batch = torch.arange(batch_size, device=device).view(-1, 1, 1, 1)
    head = torch.zeros((1, 1, 1, 1), dtype=torch.long, device=device)
    same = []
    try:
        for first in range(0, q_length, rows):
            q = torch.arange(first, min(first + rows, q_length), device=device).view(1, 1, -1, 1) + (kv_length - q_length)
            same.append(((key <= q) & (key > q - window) == mask_function(batch, head, q, key)).all())
    except Exception:  # noqa: BLE001  (a function that takes single indices only)
        return False
    return bool(torch.stack(same).all())


def _mask(batch_size, q_length, kv_length, q_offset=0, kv_offset=0, mask_function=None, attention_mask=None, **kwargs):
    """None or a compact mask for causal attention over all keys or a window of them; else the mask that the usual path takes."""
    from transformers.masking_utils import causal_mask_function, sdpa_mask
    window, device = kwargs.get("local_size"), kwargs.get("device", "cpu")
    if attention_mask is not None:
        device = attention_mask.device
    ends = not torch.is_tensor(q_offset) and q_length > 1 and kv_offset == 0 and q_offset + q_length == kv_length
    if ends and (attention_mask is None or attention_mask.shape == (batch_size, kv_length)):
        if mask_function is causal_mask_function:
            return _compact(attention_mask)
        if window and _is_window(mask_function, q_length, kv_length, window, device, batch_size):
            return _compact(attention_mask, window if window < kv_length else 0, kv_length, device)
    return sdpa_mask(batch_size=batch_size, q_length=q_length, kv_length=kv_length, q_offset=q_offset, kv_offset=kv_offset,
                     mask_function=mask_function, attention_mask=attention_mask, **kwargs)


def train_attention_interface(module, query, key, value, attention_mask=None, dropout: float = 0.0, scaling=None,
                              is_causal=None, softcap=None, sliding_window=None, **kwargs):
    """``attention_interface``, with the gradient's own kernels where they apply."""
    q, k, v = query, key, value
    if q.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    Hq, Sq, D = q.shape[1:]
    Hkv, Skv = k.shape[1:3]
    compact, padding = is_compact(attention_mask), None
    causal = compact or bool(getattr(module, "is_causal", True) if is_causal is None else is_causal)
    window = int(sliding_window or 0)
    if compact:
        padding, own = _parts(attention_mask)
        window = own or window
    window = window if causal and window < Skv else 0
    scale = D ** -0.5 if scaling is None else float(scaling)
    fits = (attention_mask is None or compact) and (torch.is_grad_enabled() or module.training) and Sq > 1 \
        and Sq <= Skv and not softcap and not (dropout and module.training) and k.shape == v.shape and Hq % Hkv == 0 \
        and 1e-4 <= scale <= 1e4 and q.dtype == k.dtype == v.dtype and q.device == k.device == v.device \
        and not any(torch.is_tensor(t) for n, t in kwargs.items() if n in ("position_bias", "s_aux", "sinks"))
    if fits and q.is_cuda:
        fits = q.dtype in (torch.float16, torch.bfloat16) and D <= MAX_DIM and D % 8 == 0 and Hq + Hkv <= MAX_HEADS
    if fits:
        return attention(q, k, v, scale, causal, window, padding).transpose(1, 2), None
    if compact:
        if padding is None:
            attention_mask, is_causal, sliding_window = None, True, window or None
        else:
            if attention_mask.dim() == 2 and window:
                attention_mask = _compact(padding, window)
            attention_mask = whole_mask(attention_mask, Sq)
    return attention_interface(module, query, key, value, attention_mask, dropout, scaling, is_causal, softcap, sliding_window,
                               **kwargs)


def _dispatches(mod) -> bool:
    """Does the attention of this module reach the interface: by the registry, or by this package's decoder forward (which a model
    that was optimised has bound to its attention modules)?  With linear attention biases it has masks of its own.  What a hook
    has wrapped counts as what is inside (``_old_forward``)."""
    if getattr(mod.config, "ipex_alibi", False) or not _uses_attention_registry(mod):
        return False
    for m in mod.modules():
        if "forward" in m.__dict__ and "Attention" in type(m).__name__:
            f = getattr(m, "_old_forward", m.forward)
            if getattr(f, "__func__", f) not in (decoder_attention_forward, type(m).forward):
                return False
    return True


def use_train_attention(model) -> bool:
    """Point every sub-model whose attention reaches it at ``train_attention_interface``; the others keep theirs.  False when
    there is none."""
    try:
        from transformers import AttentionInterface, AttentionMaskInterface
    except ImportError:
        return False
    AttentionInterface.register(TRAIN_INTERFACE_NAME, train_attention_interface)
    AttentionMaskInterface.register(TRAIN_INTERFACE_NAME, _mask)
    found = {}
    for mod in model.modules():
        cfg = getattr(mod, "config", None)
        if cfg is not None and hasattr(cfg, "to_dict"):
            found.setdefault(id(cfg), []).append(mod)
    found = [mods[0].config for mods in found.values() if any(map(_uses_attention_registry, mods)) and
             all(_dispatches(m) for m in mods if _uses_attention_registry(m))]
    for cfg in found:
        cfg._attn_implementation = TRAIN_INTERFACE_NAME
    return bool(found)
