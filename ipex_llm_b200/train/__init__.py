"""Finetuning: trainer, callbacks, optimizers (reference: HF Trainer + peft + DeepSpeed driven by the example
scripts under python/llm/example/GPU/LLM-Finetuning)."""
from .losses import (TeacherTokens, causal_lm_loss, distill_lm_loss, next_tokens, policy_lm_loss,  # noqa: F401
                     preference_lm_loss, sequence_logprobs, teacher_tokens)
from .optim import MultiTensorAdamW  # noqa: F401
from .trainer import Trainer, TrainerCallback, TrainerControl, TrainerState, default_collator  # noqa: F401
from ..parallel.dp import FusedLoraAdamW, PagedAdamW  # noqa: F401
