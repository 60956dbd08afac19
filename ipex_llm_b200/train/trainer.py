"""A small causal-LM trainer for adapter finetuning (the reference drives HF ``Trainer``;
python/llm/example/GPU/LLM-Finetuning/QLoRA/alpaca-qlora/alpaca_qlora_finetuning.py:242-278).

One process per GPU.  Data parallelism is built in: every rank runs its micro-batches, the optimizer
(``FusedLoraAdamW``) averages gradients and updates parameters in one fused kernel.  Checkpoints hold the adapter
weights, the optimizer shards, the step, the RNG state and the data cursor, so ``resume_from_checkpoint`` continues
bit-for-bit on the same world size.
"""
from __future__ import annotations

import inspect
import json
import math
import os
import time
from typing import Callable, Dict, List, Optional

import torch
import torch.distributed as dist

from ..parallel.dp import FusedLoraAdamW, PagedAdamW
from ..utils.common import invalidInputError
from .losses import TeacherTokens, causal_lm_loss, distill_lm_loss, policy_lm_loss, preference_lm_loss, sequence_logprobs
from .optim import MultiTensorAdamW

TEACHER_COLUMNS = TeacherTokens._fields
POLICY_COLUMNS = ("advantages", "old_logprobs", "ref_logprobs")


class TrainerCallback:
    """Hook points (same names as HF ``TrainerCallback`` for the ones used by ReLoRA / LISA)."""

    folds_adapters = False               # True: adapters are folded into their base while it trains

    def on_train_begin(self, args, state, control, **kw): ...
    def on_step_begin(self, args, state, control, **kw): ...
    def on_step_end(self, args, state, control, **kw): ...
    def on_save(self, args, state, control, **kw): ...
    def on_train_end(self, args, state, control, **kw): ...


class TrainerState:
    def __init__(self):
        self.global_step = 0
        self.epoch = 0.0
        self.log_history: List[Dict] = []
        self.data_cursor = 0


class TrainerControl:
    def __init__(self):
        self.should_training_stop = False
        self.should_save = False


def _lr_lambda(kind: str, warmup: int, total: int) -> Callable[[int], float]:
    def f(step):
        if warmup > 0 and step < warmup:
            return (step + 1) / warmup
        if kind == "constant":
            return 1.0
        prog = (step - warmup) / max(1, total - warmup)
        if kind == "cosine":
            return 0.5 * (1.0 + math.cos(math.pi * min(1.0, prog)))
        return max(0.0, 1.0 - prog)   # linear
    return f


class Trainer:
    def __init__(self, model, args, train_dataset=None, data_collator=None, callbacks: Optional[list] = None,
                 optimizers=(None, None), tokenizer=None, eval_dataset=None):
        self.model, self.args = model, args
        self.train_dataset, self.collate = train_dataset, data_collator or default_collator
        self.callbacks = list(callbacks or [])
        self.optimizer, self.lr_scheduler = optimizers
        self.state, self.control = TrainerState(), TrainerControl()
        self.rank = dist.get_rank() if dist.is_initialized() else 0
        self.world = dist.get_world_size() if dist.is_initialized() else 1
        self.device = next(p for p in model.parameters()).device
        self._folds = None               # how often adapters had been folded into their base, at the first loss that compares with it
        pairs = bool(getattr(args, "preference_form", None))
        invalidInputError(not pairs or getattr(args, "fused_loss", False), "preference_form needs fused_loss=True")
        first = _first_of(train_dataset) if data_collator is None else None
        if isinstance(first, dict):
            paired = "chosen_input_ids" in first
            invalidInputError(pairs or not paired, "pairs of samples need preference_form")
            invalidInputError(paired or not pairs, "preference_form needs pairs of samples (chosen_input_ids, rejected_input_ids)")

    # ------------------------------------------------------------------------------------------------
    def create_optimizer(self):
        a = self.args
        params = [p for p in self.model.parameters() if p.requires_grad]
        kw = dict(lr=a.learning_rate, betas=(a.adam_beta1, a.adam_beta2), eps=a.adam_epsilon,
                  weight_decay=a.weight_decay)
        if a.optim == "adamw_torch":
            invalidInputError(self.world == 1, "adamw_torch has no gradient averaging: use fused_lora_adamw")
            self.optimizer = torch.optim.AdamW(params, **kw)
        elif a.optim in ("adamw_multi", "adamw_8bit") and self.world == 1:      # ranks share moments in 32 bits among them
            self.optimizer = MultiTensorAdamW(params, max_grad_norm=a.max_grad_norm, bits=8 if a.optim == "adamw_8bit" else 32,
                                              seed=a.seed, **kw)
        elif a.optim == "paged_adamw" and self.world == 1 and self.device.type == "cuda" and \
                sum(p.numel() for p in params) > (1 << 28):
            self.optimizer = PagedAdamW(params, **kw)
        else:
            self.optimizer = FusedLoraAdamW(params, max_grad_norm=a.max_grad_norm, **kw)
        return self.optimizer

    def _batches(self, start_cursor: int):
        """Rank-strided micro-batches over the dataset, resumable from a cursor (in samples)."""
        a = self.args
        n = len(self.train_dataset)
        bs = a.per_device_train_batch_size
        g = torch.Generator().manual_seed(a.seed)
        cursor = start_cursor
        epoch = cursor // n
        while True:
            g.manual_seed(a.seed + epoch)
            perm = torch.randperm(n, generator=g).tolist()
            pos = cursor % n
            while pos + bs * self.world <= n:
                idx = perm[pos + self.rank * bs: pos + (self.rank + 1) * bs]
                yield self.collate([self.train_dataset[i] for i in idx]), cursor + bs * self.world
                pos += bs * self.world
                cursor += bs * self.world
            cursor = (epoch + 1) * n
            epoch += 1

    def _check_columns(self, model, batch):
        """Columns of a policy's or of pairs' batches belong to their losses: a model that takes any would pass over them."""
        fused, form = getattr(self.args, "fused_loss", False), getattr(self.args, "preference_form", None)
        given = [k for k in (*POLICY_COLUMNS, "reference_logprobs") if k in batch]
        if given and not fused:
            named = inspect.signature(model.forward).parameters      # of a model that has a loss for them
            given = [k for k in given if k not in named]
            invalidInputError(not given, f"{', '.join(given)} in the batch: this loss needs fused_loss=True")
        if not (given and fused):
            return
        invalidInputError(not form or given == ["reference_logprobs"], f"{', '.join(given)} in the batch: preference_form is for pairs")
        invalidInputError(form or "reference_logprobs" not in given, "reference_logprobs in the batch: pairs need preference_form")
        if not form:
            invalidInputError("advantages" in batch, f"{', '.join(given)} in the batch, without advantages")
            invalidInputError(not any(k in batch for k in TEACHER_COLUMNS), "a policy's batch takes no teacher's tokens")

    def compute_loss(self, model, batch):
        self._check_columns(model, batch)
        batch = {k: v.to(self.device, non_blocking=True) for k, v in batch.items()}
        if getattr(self.args, "fused_loss", False):
            return self._fused_loss(model, batch)
        out = model(**batch)
        return out.loss if hasattr(out, "loss") and out.loss is not None else out[0]

    def _fused_loss(self, model, batch):
        """The loss by ``causal_lm_loss``; with a teacher's tokens in the batch, ``distill_weight`` of it by ``distill_lm_loss``.  With
        ``preference_form`` batches are pairs, and the loss ``preference_lm_loss``; with advantages in the batch it is
        ``policy_lm_loss``."""
        if getattr(self.args, "preference_form", None):
            return self._preference_loss(model, batch)
        if "advantages" in batch:
            return self._policy_loss(model, batch)
        teacher = {k: batch.pop(k) for k in TEACHER_COLUMNS if k in batch}
        invalidInputError("labels" in batch, "fused_loss: the batch has no labels")
        labels = batch.pop("labels")
        out = model(**batch)
        logits = out.logits if hasattr(out, "logits") else out[0]
        w = float(getattr(self.args, "distill_weight", 0.5)) if teacher else 0.0
        invalidInputError(0.0 <= w <= 1.0, f"distill_weight should lie between 0 and 1, got {w}")
        loss = causal_lm_loss(logits, labels) * (1.0 - w) if w < 1.0 else 0.0
        if w > 0.0:
            invalidInputError("teacher_ids" in teacher and "teacher_logits" in teacher,
                              "a teacher's tokens need the columns teacher_ids and teacher_logits")
            loss = loss + w * distill_lm_loss(logits, labels, temperature=float(getattr(self.args, "distill_temperature", 1.0)),
                                              **teacher)
        return loss

    def _check_base(self, model):
        """The model without its adapters is a reference as long as nothing moves it."""
        how = "give the pairs reference_logprobs (or preference_reference=False)"
        invalidInputError(hasattr(model, "disable_adapter_layers"), f"preference_form: there are no adapters to disable: {how}")
        folds = getattr(model, "adapter_folds", 0)
        if self._folds is None:
            self._folds = folds
        if folds != self._folds or any(getattr(cb, "folds_adapters", False) for cb in self.callbacks):
            invalidInputError(False, f"preference_form: adapters are folded into their base, which is no reference any more: {how}")
        for name, p in model.named_parameters():
            if p.requires_grad and "lora_" not in name:
                invalidInputError(False, f"preference_form: outside of the adapters {name} is trained, too, and the base is no reference: {how}")

    def _preference_loss(self, model, batch):
        a = self.args
        invalidInputError("labels" in batch, "preference_form: the batch has no labels")
        labels, reference = batch.pop("labels"), batch.pop("reference_logprobs", None)
        average = bool(getattr(a, "preference_average", False))
        if reference is None and getattr(a, "preference_reference", True):
            self._check_base(model)
            model.disable_adapter_layers(True)
            try:
                with torch.no_grad():
                    reference = sequence_logprobs(_logits_of(model(**batch)), labels, average)
            finally:
                model.disable_adapter_layers(False)
        return preference_lm_loss(_logits_of(model(**batch)), labels, reference, float(getattr(a, "preference_beta", 0.1)),
                                  a.preference_form, float(getattr(a, "preference_label_smoothing", 0.0)),
                                  float(getattr(a, "preference_margin", 0.0)), average,
                                  float(getattr(a, "preference_likelihood_weight", 0.0)))

    def _policy_loss(self, model, batch):
        a = self.args
        invalidInputError("labels" in batch, "a policy's batch has no labels")
        given = {k: batch.pop(k) for k in POLICY_COLUMNS if k in batch}
        labels = batch.pop("labels")
        return policy_lm_loss(_logits_of(model(**batch)), labels, clip=tuple(getattr(a, "policy_clip", (0.2, 0.2))),
                              kl_weight=float(getattr(a, "policy_kl_weight", 0.0)),
                              temperature=float(getattr(a, "policy_temperature", 1.0)), **given)

    def train(self, resume_from_checkpoint: Optional[str] = None):
        a = self.args
        torch.manual_seed(a.seed + self.rank)
        if self.optimizer is None:
            self.create_optimizer()
        steps_per_epoch = max(1, len(self.train_dataset) // (a.per_device_train_batch_size * self.world *
                                                              a.gradient_accumulation_steps))
        total = a.max_steps if a.max_steps > 0 else int(math.ceil(a.num_train_epochs * steps_per_epoch))
        warmup = a.warmup_steps or int(a.warmup_ratio * total)
        sched = _lr_lambda(a.lr_scheduler_type, warmup, total)
        base_lr = a.learning_rate
        resume = resume_from_checkpoint or a.resume_from_checkpoint
        if resume:
            self._load_checkpoint(resume)
        for cb in self.callbacks:
            cb.on_train_begin(a, self.state, self.control, model=self.model, optimizer=self.optimizer)
        self.model.train()
        it = self._batches(self.state.data_cursor)
        t0 = time.time()
        tokens = 0
        self.optimizer.zero_grad()
        while self.state.global_step < total and not self.control.should_training_stop:
            for cb in self.callbacks:
                cb.on_step_begin(a, self.state, self.control, model=self.model, optimizer=self.optimizer)
            for g in self.optimizer.param_groups:
                # callbacks may install a per-group multiplier (ReLoRA's re-warm-up after each restart)
                g["lr"] = base_lr * sched(self.state.global_step) * g.get("relora_scale", 1.0)
            loss_acc = 0.0
            for _ in range(a.gradient_accumulation_steps):
                batch, cursor = next(it)
                ctx = torch.autocast("cuda", dtype=torch.bfloat16) if (self.device.type == "cuda" and a.bf16) \
                    else _null()
                with ctx:
                    loss = self.compute_loss(self.model, batch) / a.gradient_accumulation_steps
                loss.backward()
                loss_acc += float(loss.detach())
                tokens += int(batch["input_ids"].numel())
                self.state.data_cursor = cursor
            clips = isinstance(self.optimizer, FusedLoraAdamW) or (isinstance(self.optimizer, MultiTensorAdamW) and
                                                                   self.optimizer.max_grad_norm)
            if not clips and a.max_grad_norm and a.max_grad_norm > 0:
                torch.nn.utils.clip_grad_norm_([p for p in self.model.parameters() if p.requires_grad],
                                               a.max_grad_norm)
            self.optimizer.step()
            self.optimizer.zero_grad()
            self.state.global_step += 1
            self.state.epoch = self.state.global_step / steps_per_epoch
            if a.logging_steps and self.state.global_step % a.logging_steps == 0:
                rec = {"step": self.state.global_step, "loss": loss_acc, "lr": self.optimizer.param_groups[0]["lr"],
                       "epoch": round(self.state.epoch, 4)}
                self.state.log_history.append(rec)
                if self.rank == 0:
                    print(rec, flush=True)
            for cb in self.callbacks:
                cb.on_step_end(a, self.state, self.control, model=self.model, optimizer=self.optimizer)
            if (a.save_steps and self.state.global_step % a.save_steps == 0) or self.control.should_save:
                self.save_checkpoint()
                self.control.should_save = False
        dt = time.time() - t0
        for cb in self.callbacks:
            cb.on_train_end(a, self.state, self.control, model=self.model, optimizer=self.optimizer)
        metrics = {"train_runtime": dt, "train_steps_per_second": self.state.global_step / max(dt, 1e-9),
                   "train_tokens_per_second": tokens * self.world / max(dt, 1e-9),
                   "train_loss": self.state.log_history[-1]["loss"] if self.state.log_history else None}
        return metrics

    # ------------------------------------------------------------------------------------------------
    def _ckpt_dir(self):
        return os.path.join(self.args.output_dir, f"checkpoint-{self.state.global_step}")

    def save_checkpoint(self):
        d = self._ckpt_dir()
        os.makedirs(d, exist_ok=True)
        if self.rank == 0:
            if hasattr(self.model, "save_pretrained") and hasattr(self.model, "peft_config"):
                self.model.save_pretrained(d)
            else:
                torch.save({k: v.cpu() for k, v in self.model.state_dict().items()
                            if v.is_floating_point() and "lora_" in k}, os.path.join(d, "trainable.bin"))
            with open(os.path.join(d, "trainer_state.json"), "w") as f:
                json.dump({"global_step": self.state.global_step, "epoch": self.state.epoch,
                           "data_cursor": self.state.data_cursor, "log_history": self.state.log_history}, f)
        torch.save({"optimizer": self.optimizer.state_dict(), "rng": torch.get_rng_state(),
                    "cuda_rng": torch.cuda.get_rng_state() if self.device.type == "cuda" else None},
                   os.path.join(d, f"optimizer_rank{self.rank}.pt"))
        for cb in self.callbacks:
            cb.on_save(self.args, self.state, self.control, model=self.model)
        if dist.is_initialized():
            dist.barrier()
        self._rotate()
        return d

    def _rotate(self):
        lim = self.args.save_total_limit
        if not lim or self.rank != 0:
            return
        import shutil
        cks = sorted((int(n.split("-")[1]), n) for n in os.listdir(self.args.output_dir)
                     if n.startswith("checkpoint-") and n.split("-")[1].isdigit())
        for _, n in cks[:-lim]:
            shutil.rmtree(os.path.join(self.args.output_dir, n), ignore_errors=True)

    def _load_checkpoint(self, d):
        if d is True:
            cks = sorted(int(n.split("-")[1]) for n in os.listdir(self.args.output_dir) if n.startswith("checkpoint-"))
            invalidInputError(len(cks) > 0, f"no checkpoint under {self.args.output_dir}")
            d = os.path.join(self.args.output_dir, f"checkpoint-{cks[-1]}")
        with open(os.path.join(d, "trainer_state.json")) as f:
            st = json.load(f)
        self.state.global_step, self.state.epoch = st["global_step"], st["epoch"]
        self.state.data_cursor, self.state.log_history = st["data_cursor"], st["log_history"]
        from ..transformers.qlora import ADAPTER_WEIGHTS, set_peft_model_state_dict
        if os.path.exists(os.path.join(d, ADAPTER_WEIGHTS)):
            set_peft_model_state_dict(self.model, torch.load(os.path.join(d, ADAPTER_WEIGHTS), map_location="cpu",
                                                             weights_only=True))
        else:
            self.model.load_state_dict(torch.load(os.path.join(d, "trainable.bin"), map_location="cpu",
                                                  weights_only=True), strict=False)
        blob = torch.load(os.path.join(d, f"optimizer_rank{self.rank}.pt"), map_location="cpu", weights_only=False)
        self.optimizer.load_state_dict(blob["optimizer"])
        torch.set_rng_state(blob["rng"])
        if blob.get("cuda_rng") is not None and self.device.type == "cuda":
            torch.cuda.set_rng_state(blob["cuda_rng"])

    def save_model(self, output_dir=None):
        d = output_dir or self.args.output_dir
        if self.rank == 0 and hasattr(self.model, "save_pretrained"):
            self.model.save_pretrained(d)


class _null:
    def __enter__(self): return None
    def __exit__(self, *a): return False


def _first_of(dataset):
    """A dataset's first sample; None where it is empty, or has no length or no places."""
    try:
        return dataset[0] if len(dataset) else None
    except (TypeError, NotImplementedError):
        return None


def _logits_of(out):
    return out.logits if hasattr(out, "logits") else out[0]


def _pad_teacher(rows, n: int, ids: bool):
    rows = [torch.as_tensor(r, dtype=torch.long if ids else torch.float32).cpu() for r in rows]
    top = [max(r.shape[1] for r in rows)] if rows[0].dim() == 2 else []
    out = torch.full((len(rows), n, *top), -1 if ids else 0, dtype=rows[0].dtype)
    for o, r in zip(out, rows):
        o[tuple(slice(0, s) for s in r.shape)] = r
    return out


def default_collator(samples):
    """Pads ``input_ids`` / ``labels`` / ``attention_mask`` lists to the longest sample (labels padded with -100); a teacher's
    rows (``TeacherTokens``: lists or tensors [tokens, top] and [tokens]) likewise, ids with -1, and a policy's numbers (advantages may
    be one for each sample, or for some of them) with 0.

    Pairs, with ``chosen_input_ids`` and ``rejected_input_ids`` (and labels of either name, -100 for the prompt), become a batch of the
    chosen samples, then of the rejected ones; ``reference_logprobs`` hold two numbers, the chosen one's first."""
    for k in (*POLICY_COLUMNS, "reference_logprobs"):
        have = sum(k in s for s in samples)
        invalidInputError(have in (0, len(samples)), f"{k} of some samples of a batch, but not of all")
    if "chosen_input_ids" in samples[0]:
        return _pairs(samples)
    keys = samples[0].keys()
    n = max(len(s["input_ids"]) for s in samples)
    out = {}
    for k in keys:
        if k in TEACHER_COLUMNS:
            out[k] = _pad_teacher([s[k] for s in samples], n, k == "teacher_ids")
            continue
        if k in POLICY_COLUMNS:
            rows = [torch.as_tensor(s[k], dtype=torch.float32).cpu().reshape(-1) for s in samples]
            one = k == "advantages" and all(r.numel() == 1 for r in rows)
            if k == "advantages" and not one:
                rows = [r.expand(len(s["input_ids"])) if r.numel() == 1 else r for r, s in zip(rows, samples)]
            out[k] = torch.stack(rows) if one else _pad_teacher(rows, n, False)
            continue
        pad = -100 if k == "labels" else 0
        out[k] = torch.tensor([list(s[k]) + [pad] * (n - len(s[k])) for s in samples], dtype=torch.long)
    if "labels" not in out:
        out["labels"] = out["input_ids"].clone()
    return out


def _pairs(samples):
    both = []
    for name in ("chosen", "rejected"):
        for s in samples:
            ids = list(s[f"{name}_input_ids"])
            both.append({"input_ids": ids, "labels": list(s.get(f"{name}_labels", ids)),
                         "attention_mask": list(s.get(f"{name}_attention_mask", [1] * len(ids)))})
    out = default_collator(both)
    if "reference_logprobs" in samples[0]:
        out["reference_logprobs"] = torch.tensor([[float(x) for x in s["reference_logprobs"]] for s in samples]).t().reshape(-1)
    return out
