"""Losses of causal language models on the output layer's logits as they are: no shifted copy, no copy in 32 bits, and the
gradient is written once, in the logits' type (``ops.token_loss``)."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ..ops.preference import policy_loss, preference_loss
from ..ops.token_loss import IGNORE, distill_loss, token_logprobs
from ..utils.common import invalidInputError


class TeacherTokens(NamedTuple):
    """What is kept of a teacher's distribution at each position: as a student's ``distill_lm_loss`` takes it."""
    teacher_ids: torch.Tensor            # [..., top]
    teacher_logits: torch.Tensor         # [..., top]: temperature x log probability
    teacher_logsumexp: torch.Tensor      # [...]: 0, as these are normalised


def next_tokens(labels: torch.Tensor) -> torch.Tensor:
    """The label that each position predicts: ``labels [batch, tokens]`` moved on by one, -100 at the end."""
    out = torch.full_like(labels, IGNORE, dtype=torch.int64)
    out[..., :-1] = labels[..., 1:]
    return out


def _check(logits, labels, what):
    if logits.dim() != 3 or labels.shape != logits.shape[:2]:
        invalidInputError(False, f"{what}: logits should be [batch, tokens, vocabulary] and labels [batch, tokens]; got "
                                 f"{tuple(logits.shape)} and {tuple(labels.shape)}")


def causal_lm_loss(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Mean negative log probability of each next label; labels of -100 take no part.  0 where none is left."""
    _check(logits, labels, "causal_lm_loss")
    targets = next_tokens(labels)
    logprob = token_logprobs(logits, targets).logprob
    return -logprob.sum() / (targets != IGNORE).sum().clamp(min=1)


def distill_lm_loss(logits: torch.Tensor, labels: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                    teacher_logsumexp: Optional[torch.Tensor] = None, temperature: float = 1.0) -> torch.Tensor:
    """Mean divergence from the teacher over the positions that predict a label; the teacher's row t belongs to the logits' row t,
    and ids below 0 pad it.  0 where no position is left."""
    _check(logits, labels, "distill_lm_loss")
    real = next_tokens(labels) != IGNORE
    ids = teacher_ids.masked_fill(~real.unsqueeze(-1), -1) if teacher_ids.shape[:-1] == real.shape else teacher_ids
    loss = distill_loss(logits, ids, teacher_logits, temperature, teacher_logsumexp)
    return loss.sum() / real.sum().clamp(min=1)


@torch.no_grad()
def teacher_tokens(logits: torch.Tensor, top: int = 32, temperature: float = 1.0) -> TeacherTokens:
    """A teacher's ``top`` best tokens (up to 32) at each position of ``logits [..., V]``, with what is left of its distribution
    known: for ``distill_lm_loss`` at the same temperature."""
    best = token_logprobs(logits, torch.zeros(logits.shape[:-1], dtype=torch.int64, device=logits.device), temperature, top=top)
    return TeacherTokens(best.top_ids, best.top_logprobs.float() * temperature,
                         torch.zeros(logits.shape[:-1], dtype=torch.float32, device=logits.device))


@torch.no_grad()
def sequence_logprobs(logits: torch.Tensor, labels: torch.Tensor, average: bool = False) -> torch.Tensor:
    """Log probability of each sequence's labels, ``[batch]`` (``average``: the mean over them): what ``preference_lm_loss`` takes of a
    reference model."""
    _check(logits, labels, "sequence_logprobs")
    targets = next_tokens(labels)
    total = token_logprobs(logits, targets).logprob.double().sum(dim=1)
    return (total / (targets != IGNORE).sum(dim=1).clamp(min=1) if average else total).float()


def preference_lm_loss(logits: torch.Tensor, labels: torch.Tensor, reference: Optional[torch.Tensor] = None, beta: float = 0.1,
                       form: str = "sigmoid", label_smoothing: float = 0.0, margin: float = 0.0, average: bool = False,
                       likelihood_weight: float = 0.0) -> torch.Tensor:
    """Mean loss of preferred over rejected sequences (``ops.preference.preference_loss``): the first half of the batch is preferred to
    the second, in order; labels of -100 (prompts, padding) take no part.  ``likelihood_weight`` of the preferred sequences' mean
    negative log probability a token is added."""
    _check(logits, labels, "preference_lm_loss")
    targets = next_tokens(labels)
    got = preference_loss(logits, targets, reference, beta, form, label_smoothing, margin, average)
    loss = got.loss.mean()
    if likelihood_weight:
        pairs = got.loss.shape[0]
        likely = got.logprob[:pairs]
        if not average:
            likely = likely / (targets[:pairs] != IGNORE).sum(dim=1).clamp(min=1)
        loss = loss - likelihood_weight * likely.mean()
    return loss


def policy_lm_loss(logits: torch.Tensor, labels: torch.Tensor, advantages: torch.Tensor, old_logprobs: Optional[torch.Tensor] = None,
                   ref_logprobs: Optional[torch.Tensor] = None, clip: Tuple[float, float] = (0.2, 0.2), kl_weight: float = 0.0,
                   temperature: float = 1.0) -> torch.Tensor:
    """Mean clipped policy loss (``ops.preference.policy_loss``) over the positions that predict a label.  What belongs to a token stands
    in the row that predicts it: ``old_logprobs``, ``ref_logprobs`` and ``advantages [batch, tokens]`` (or ``[batch, 1]``).  0 where no
    position is left."""
    _check(logits, labels, "policy_lm_loss")
    targets = next_tokens(labels)
    loss = policy_loss(logits, targets, advantages, old_logprobs, ref_logprobs, clip, kl_weight, temperature).loss
    return loss.sum() / (targets != IGNORE).sum().clamp(min=1)
