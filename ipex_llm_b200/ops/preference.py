"""Losses of preference and policy finetuning straight from an output layer's logits (``preference.cu``): preferred over rejected
sequences, and the clipped policy loss with a KL term, each with the gradient of the logits.

On a CUDA tensor the package's own kernels run, on the current stream of the tensor's device: logits of rows without a target are
never read, no copy of the logits is made, and the gradient is written once, in their type.  On the CPU it is plain PyTorch.  Logits
may be a view with any strides between rows.  Gradients are those of a backward pass; on the GPU tangents of forward-mode
differentiation are refused.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from ..native.lib import calls
from ..utils.common import invalidInputError
from .cuda_ops import error_flag
from .gradients import refuse_tangents
from .token_loss import IGNORE, _check_like, _check_logits, token_logprobs

FORMS = ("sigmoid", "hinge", "ipo")
_FORM_CODES = {f: i for i, f in enumerate(FORMS)}


class PreferenceLoss(NamedTuple):
    """Both have a gradient."""
    loss: torch.Tensor           # [pairs]
    logprob: torch.Tensor        # [2 pairs]: of each sequence, the sum (or the mean) over its targets


class PolicyLoss(NamedTuple):
    """``loss`` has a gradient; the others tell how the step goes."""
    loss: torch.Tensor           # [...]
    logprob: torch.Tensor        # [...]: of the targets
    kl: torch.Tensor             # [...]: the estimate e^d - d - 1, d = ref - logprob (0 without a reference)
    clipped: torch.Tensor        # [...]: True where the ratio lies outside and the loss does not move with it


def _preference_plain(logits, targets, reference, beta, form, smooth, margin, average, temperature, ignore):
    s = token_logprobs(logits, targets, temperature, ignore_index=ignore).logprob.double().sum(dim=1)
    if average:
        s = s / (targets != ignore).sum(dim=1).clamp(min=1)
    h = s if reference is None else s - reference.double()
    h = h[:len(h) // 2] - h[len(h) // 2:]
    if form == "ipo":
        loss = (h - 0.5 / beta).square()
    elif form == "hinge":
        loss = (1.0 - beta * h).relu()                  # its gradient at 0 is 0
    else:
        z = beta * h - margin
        loss = -(1.0 - smooth) * torch.nn.functional.logsigmoid(z)
        if smooth:
            loss = loss - smooth * torch.nn.functional.logsigmoid(-z)
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    return PreferenceLoss(loss.to(wide), s.to(wide))


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, reference: Optional[torch.Tensor] = None, beta: float = 0.1,
                    form: str = "sigmoid", label_smoothing: float = 0.0, margin: float = 0.0, average: bool = False,
                    temperature: float = 1.0, ignore_index: int = IGNORE) -> PreferenceLoss:
    """Losses ``[pairs]`` of preferred over rejected sequences: ``logits [2 pairs, tokens, V]`` and ``targets [2 pairs, tokens]`` hold
    the preferred ones first, then the rejected ones in the same order.

    A sequence's log probability is the sum (``average``: the mean) of its targets' under softmax(logits / temperature); targets of
    ``ignore_index`` (a prompt, padding) take no part, and their logits are not read.  With h the preferred one's less the rejected
    one's, each less that of a ``reference [2 pairs]`` (the same sums under the model that finetuning began with; None: 0),

    - "sigmoid": ``-(1 - e) log sigmoid(z) - e log sigmoid(-z)``, z = beta h - margin, e = ``label_smoothing``
    - "hinge": ``max(0, 1 - beta h)``
    - "ipo": ``(h - 1 / (2 beta))^2``

    The gradient goes to the logits alone (in their type: 16 or 32 bits), from the losses and from the sequences' log probabilities.
    A hidden target (a logit of -inf) makes its sequence's log probability -inf, and a loss that compares two such numbers NaN.  A target
    outside of the vocabulary raises on the CPU; on the GPU its pair's results are NaN, and ``cuda_ops.check_error_flag`` reports 61.
    """
    what = "preference_loss"
    cuda = logits.is_cuda
    if cuda:
        refuse_tangents(what, logits)
        got = calls().preference(logits, targets, reference, beta, _FORM_CODES.get(form, -1), label_smoothing, margin, average, temperature,
                                 ignore_index, error_flag(logits.device).data_ptr())
        if got is not None:
            return PreferenceLoss(*got)
    _check_logits(logits, temperature, what)
    if logits.dim() != 3 or logits.shape[0] % 2 or not logits.shape[0]:
        invalidInputError(False, f"{what}: logits should be [2 pairs, tokens, vocabulary], got {tuple(logits.shape)}")
    if not logits.shape[1]:
        invalidInputError(False, f"{what}: no tokens")
    _check_like(targets, logits.shape[:2], logits.device, f"{what}: targets", True)
    if reference is not None:
        _check_like(reference, logits.shape[:1], logits.device, f"{what}: reference", False)
    if form not in FORMS:
        invalidInputError(False, f"{what}: form should be one of {', '.join(FORMS)}, got {form!r}")
    if not (0.0 < beta < math.inf and 0.0 <= label_smoothing <= 1.0 and math.isfinite(margin)):
        invalidInputError(False, f"{what}: beta should be above 0, label_smoothing between 0 and 1, margin finite; got {beta}, "
                                 f"{label_smoothing}, {margin}")
    if form != "sigmoid" and (label_smoothing or margin):
        invalidInputError(False, f"{what}: label_smoothing and margin belong to the form 'sigmoid'")
    if cuda:
        invalidInputError(False, f"{what}: these tensors are not supported")
    return _preference_plain(logits, targets, None if reference is None else reference.detach(), beta, form, label_smoothing, margin,
                             average, temperature, ignore_index)


def _apart(a, b):
    """a - b: 0, and without a gradient, where both are the same infinity."""
    same = (a == b) & a.isinf()
    return a.masked_fill(same, 0.0) - b.masked_fill(same, 0.0)


def _policy_plain(logits, targets, advantages, old, ref, lo, hi, weight, temperature, ignore):
    lp = token_logprobs(logits, targets, temperature, ignore_index=ignore).logprob
    real = targets != ignore
    wide = lp.double()
    ratio = torch.exp(_apart(wide, wide.detach() if old is None else old.double()))
    a = advantages.double()
    held = ratio.clamp(1.0 - lo, 1.0 + hi)
    clipped = held * a < ratio * a
    loss = -torch.where(clipped, held.detach() * a, ratio * a)
    kl = torch.zeros_like(wide)
    if ref is not None:
        d = _apart(ref.double(), wide)
        far = d.detach() == math.inf
        kl = torch.where(far, math.inf, torch.expm1(d.masked_fill(far, 0.0)) - d.masked_fill(far, 0.0))
        loss = loss + weight * kl if weight else loss
    return PolicyLoss(torch.where(real, loss, 0.0).to(lp.dtype), lp.detach(), torch.where(real, kl, 0.0).detach().to(lp.dtype), clipped & real)


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, advantages: torch.Tensor, old_logprobs: Optional[torch.Tensor] = None,
                ref_logprobs: Optional[torch.Tensor] = None, clip: Tuple[float, float] = (0.2, 0.2), kl_weight: float = 0.0,
                temperature: float = 1.0, ignore_index: int = IGNORE) -> PolicyLoss:
    """Loss of each of the ``targets [...]`` that a policy drew, from its ``logits [..., V]`` now.

    With lp its log probability under softmax(logits / temperature), w = e^(lp - ``old_logprobs``) and A the ``advantages``
    (broadcast to the targets: one a token, or ``[batch, 1]``),

    ``-min(w A, clamp(w, 1 - clip[0], 1 + clip[1]) A) + kl_weight (e^d - d - 1)``, d = ``ref_logprobs`` - lp.

    Without ``old_logprobs`` they are lp itself (one step for each batch): w is 1 and still has its gradient.  Targets of
    ``ignore_index`` give 0 and no gradient, and their logits are not read.  The gradient goes to the logits alone (in their type: 16
    or 32 bits).  A hidden target (a logit of -inf) has no gradient; its w is 0, or 1 without ``old_logprobs`` and where they hide it,
    too, and its KL term is infinite, or 0 where the reference hides it, too.  A target outside of the vocabulary raises on the CPU; on
    the GPU its results are NaN, and ``cuda_ops.check_error_flag`` reports 61.
    """
    what = "policy_loss"
    lo, hi = float(clip[0]), float(clip[1])
    cuda = logits.is_cuda
    if cuda:
        refuse_tangents(what, logits)
        got = calls().policy(logits, targets, advantages, old_logprobs, ref_logprobs, lo, hi, kl_weight, temperature, ignore_index,
                             error_flag(logits.device).data_ptr())
        if got is not None:
            return PolicyLoss(*got)
    _check_logits(logits, temperature, what)
    _check_like(targets, logits.shape[:-1], logits.device, f"{what}: targets", True)
    for t, name in ((old_logprobs, "old_logprobs"), (ref_logprobs, "ref_logprobs")):
        if t is not None:
            _check_like(t, targets.shape, logits.device, f"{what}: {name}", False)
    if advantages.device != logits.device or not advantages.is_floating_point():
        invalidInputError(False, f"{what}: advantages should hold floating-point numbers on {logits.device}, got {advantages.dtype} on "
                                 f"{advantages.device}")
    fits = advantages.dim() <= targets.dim() and all(
        m in (1, n) for m, n in zip(reversed(advantages.shape), reversed(targets.shape)))
    if not fits:
        invalidInputError(False, f"{what}: advantages of shape {tuple(advantages.shape)} do not fit targets of {tuple(targets.shape)}")
    if not (0.0 <= lo <= 1.0 and 0.0 <= hi and 0.0 <= kl_weight < math.inf):
        invalidInputError(False, f"{what}: clip should hold a number in [0, 1] and one not below 0, kl_weight be finite and not below 0; "
                                 f"got {clip}, {kl_weight}")
    if kl_weight and ref_logprobs is None:
        invalidInputError(False, f"{what}: kl_weight needs ref_logprobs")
    if cuda:
        invalidInputError(False, f"{what}: these tensors are not supported")
    old, ref = (None if t is None else t.detach() for t in (old_logprobs, ref_logprobs))
    return _policy_plain(logits, targets, advantages.detach(), old, ref, lo, hi, kl_weight, temperature, ignore_index)
