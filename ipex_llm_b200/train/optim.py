"""AdamW over separately allocated parameters of any sizes, with moments in 32 or in 8 bits (``ops.adamw``)."""
from __future__ import annotations

from typing import Dict, List, Optional, Union

import torch

from ..ops.adamw import AdamWState, adamw_state, adamw_step, flat_size, grad_norm, moments
from ..utils.common import invalidInputError


class MultiTensorAdamW(torch.optim.Optimizer):
    """AdamW whose step takes all parameters of a type in one launch (a few, from some 600 on), whatever their number, and reads each
    number once.

    ``bits``: of the moments, 32, or 8 with an exponent for each 256 (2 bytes a parameter instead of 8).  ``rest``: what is kept of
    16-bit parameters, so that small steps are not lost: "auto" (the 16 bits below bf16, a 32-bit copy of fp16), "copy" or None.
    ``max_grad_norm`` > 0 clips by the norm of all gradients together.  Parameters without a gradient are left alone, and each counts
    its own steps.  One process: gradients are not averaged over ranks (``FusedLoraAdamW`` does that).

    Whoever changes parameters between steps calls ``parameters_changed``.
    """

    def __init__(self, params, lr: Union[float, torch.Tensor] = 2e-4, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 max_grad_norm: float = 0.0, bits: int = 32, rest: Optional[str] = "auto", seed: int = 0):
        invalidInputError(bits in (8, 32), f"MultiTensorAdamW: moments have 32 or 8 bits, got {bits}")
        invalidInputError(rest in ("auto", "copy", None), f"MultiTensorAdamW: rest should be 'auto', 'copy' or None, got {rest!r}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.max_grad_norm, self.bits, self.rest, self.seed = max_grad_norm, bits, rest, seed
        self._buckets: Optional[List[Dict]] = None

    def add_param_group(self, group):
        invalidInputError(getattr(self, "_buckets", None) is None, "MultiTensorAdamW: groups are added before the first step")
        super().add_param_group(group)

    def _rest_of(self, dtype) -> Optional[str]:
        if dtype == torch.float32 or self.rest is None:
            return None
        return "low" if dtype == torch.bfloat16 and self.rest == "auto" else "copy"

    def buckets(self) -> List[Dict]:
        """The parameters of each group, type and device, with their state."""
        if self._buckets is None:
            self._buckets = []
            for g in self.param_groups:
                by = {}
                for p in g["params"]:
                    by.setdefault((p.dtype, p.device), []).append(p)
                for (dtype, _), ps in by.items():
                    self._buckets.append(dict(group=g, params=ps, state=adamw_state(ps, self.bits, self._rest_of(dtype), each=True)))
        return self._buckets

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        buckets = self.buckets()
        grads = [[p.grad for p in b["params"]] for b in buckets]
        norms = {}
        if self.max_grad_norm and self.max_grad_norm > 0.0:
            parts = [grad_norm(g) for g in grads if any(x is not None for x in g)]
            if parts:
                dev = parts[0].device
                norm = parts[0] if len(parts) == 1 else torch.stack([x.to(dev) for x in parts]).double().square().sum().sqrt().float()
                norms = {b["params"][0].device: norm.to(b["params"][0].device) for b in buckets}
        for i, (b, g) in enumerate(zip(buckets, grads)):
            if all(x is None for x in g):
                continue
            o, s = b["group"], b["state"]
            norm = norms.get(b["params"][0].device)
            adamw_step(b["params"], g, s.exp_avg, s.exp_avg_sq, s.step, lr=o["lr"], betas=o["betas"], eps=o["eps"],
                       weight_decay=o["weight_decay"], exp_avg_scale=s.exp_avg_scale, exp_avg_sq_scale=s.exp_avg_sq_scale, rest=s.rest,
                       grad_norm=norm, max_grad_norm=self.max_grad_norm if norm is not None else 0.0, seed=self.seed + i)
        return loss

    @torch.no_grad()
    def parameters_changed(self):
        """Takes the parameters as they are now for what is kept of them beside themselves."""
        for b in self.buckets():
            s = b["state"]
            if s.rest is not None:
                s.rest.copy_(adamw_state(b["params"], 32, "low" if s.rest.dtype == torch.int16 else "copy").rest)

    @torch.no_grad()
    def prune_moments(self, ratio: float):
        """Zeroes the smallest ``ratio`` of each kind of moment (with what equals the last one of them)."""
        for b in self.buckets():
            s, sizes = b["state"], [p.numel() for p in b["params"]]
            k = int(ratio * sum(sizes))
            if k > 0:
                for codes, wide in zip(s[:2], moments(s.exp_avg, s.exp_avg_sq, s.exp_avg_scale, s.exp_avg_sq_scale)):
                    # the zeros that fill a parameter's last 256 are none of its moments
                    real = [x[:n] for x, n in zip(wide.split([flat_size([n]) for n in sizes]), sizes)]
                    limit = torch.kthvalue(torch.cat(real).abs().cpu(), k).values.to(wide.device)
                    bits = codes.view(torch.uint8 if codes.element_size() == 1 else torch.int32)
                    bits.mul_((wide.abs() > limit).to(bits.dtype))

    def _sizes(self):
        return [[p.numel() for p in b["params"]] for b in self.buckets()]

    # state for checkpoint / resume -------------------------------------------------------------------
    def state_dict(self):
        """The state as it is now: copies, on the CPU, that later steps do not change."""
        return {"bits": self.bits, "seed": self.seed, "sizes": self._sizes(),
                "buckets": [[None if t is None else t.to("cpu", copy=True) for t in b["state"]] for b in self.buckets()],
                "param_groups": [{k: v.detach().to("cpu", copy=True) if isinstance(v, torch.Tensor) else v for k, v in g.items()
                                  if k != "params"} for g in self.param_groups]}

    @torch.no_grad()
    def load_state_dict(self, sd):
        mine = self.buckets()
        fits = len(sd["buckets"]) == len(mine) and len(sd["param_groups"]) == len(self.param_groups) and \
            sd.get("sizes", self._sizes()) == self._sizes() and all(
            (a is None) == (t is None) and (t is None or (a.shape == t.shape and a.dtype == t.dtype))
            for saved, b in zip(sd["buckets"], mine) for a, t in zip(saved, b["state"]))
        invalidInputError(fits, "MultiTensorAdamW: the state was saved for other parameters, or with other bits")
        for saved, b in zip(sd["buckets"], mine):
            for a, t in zip(saved, b["state"]):
                if t is not None:
                    raw = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()]
                    t.view(raw).copy_(a.view(raw))
        self.seed = sd.get("seed", self.seed)
        for g, s in zip(self.param_groups, sd["param_groups"]):
            rate = g["lr"]
            g.update(s)
            if isinstance(rate, torch.Tensor):               # steps that were captured read it where it is
                g["lr"] = rate.fill_(float(s["lr"]))
            else:
                g["lr"] = float(s["lr"])


__all__ = ["AdamWState", "MultiTensorAdamW"]
