"""The AdamW step over many tensors at once, with the clipping of the gradients' norm in
it, on the kernels of optim_kernels.cu: two launches for all tensors of a group (three
with clipping, up to 400 tensors each), and states in 32 bits or in 8.

`AdamW` is a torch optimizer to use in place of clip_grad_norm_ and torch.optim.AdamW;
`adamw_step` is its one step on tensors that the caller keeps.

States in 8 bits take 2 bytes and 1/128 of an element instead of 8: e4m3 codes with a
power-of-two scale per 256 elements.  They, and bf16 parameters, are rounded up or down by
random bits drawn from (seed, step, the element's number): steps that are smaller than the
type's own are kept in the mean, and every run gives the same bits.

Everything that changes from step to step -- the step count, the norm, a learning rate
given as a tensor -- lives on the device, so a step can be captured in a CUDA graph, once
the parameters have their states.  A replay does not raise the parameters' versions, by which
the networks know that their bf16 weights are old: `torch.autograd.graph.increment_version`
does (ppo.GraphedPpoStep calls it)."""
from __future__ import annotations

from typing import Any, Iterable

import torch

from .ext import load_update

_STATES = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")


def _capturing(device: torch.device) -> bool:
    """Whether the device's current stream records a CUDA graph."""
    if device.type != "cuda":
        return False
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def adamw_step(params: list[torch.Tensor], grads: list[torch.Tensor],
               exp_avgs: list[torch.Tensor], exp_avg_sqs: list[torch.Tensor], step: torch.Tensor, *,
               lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, max_grad_norm: float | None = None,
               seed: int = 0, exp_avg_scales: list[torch.Tensor] | None = None,
               exp_avg_sq_scales: list[torch.Tensor] | None = None) -> torch.Tensor | None:
    """One AdamW step, in place:

      g = g min(1, max_grad_norm / (|g| + 1e-6))    (|g| over all tensors; returned)
      m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
      p = (1 - lr weight_decay) p - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)

    with t = step + 1, which is stored back (int64, one value on the device).  params: fp32
    or bf16; grads: fp32 or bf16; all contiguous, one type per list; parameters, states and
    step share no memory with any other tensor of the call.  exp_avgs, exp_avg_sqs: fp32; or,
    with the lists of scales (uint8 or float8_e8m0fnu, ceil(size / 256) each), e4m3 codes
    (uint8 or float8_e4m3fn).  States start as zeros.  lr: a number, or one fp32 value on the
    device.  A norm that is infinite or NaN makes the step NaN, as clip_grad_norm_ does."""
    rate = (0.0, lr) if torch.is_tensor(lr) else (lr, None)
    return load_update().adamw(params, grads, exp_avgs, exp_avg_sqs, step, *rate, *betas, eps, weight_decay,
                               max_grad_norm, seed, exp_avg_scales, exp_avg_sq_scales)


class AdamW(torch.optim.Optimizer):
    """AdamW on one kernel per group.  The arguments are torch.optim.AdamW's, and

      state_bits     32 or 8 (see above)
      max_grad_norm  clips the norm of each group's gradients inside the step (None: not);
                     the latest norms, before clipping, are in group["grad_norm"]
      seed           of the rounding by random bits

    A group holds contiguous parameters of one type (fp32 or bf16) on one device; its tensors
    share one step count, and the ones without a gradient are left out of a step."""

    def __init__(self, params: Iterable, lr: float | torch.Tensor = 1e-3,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32,
                 max_grad_norm: float | None = None, seed: int = 0) -> None:
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, max_grad_norm=max_grad_norm, seed=seed,
                                      grad_norm=None))

    def add_param_group(self, group: dict[str, Any]) -> None:
        super().add_param_group(group)
        ps = self.param_groups[-1]["params"]
        if any(p.dtype not in (torch.float32, torch.bfloat16) or p.dtype != ps[0].dtype
               or p.device != ps[0].device or not p.is_contiguous() for p in ps):
            self.param_groups.pop()
            raise ValueError("a group's parameters must be contiguous, fp32 or all bf16, on one device")

    @property
    def clips(self) -> bool:
        """Whether every group's gradients are clipped inside the step."""
        return all(g["max_grad_norm"] is not None for g in self.param_groups)

    def _new_state(self, p: torch.Tensor, bits: int, step: torch.Tensor) -> dict[str, torch.Tensor]:
        if bits == 32:
            return {"step": step, "exp_avg": torch.zeros_like(p, dtype=torch.float32),
                    "exp_avg_sq": torch.zeros_like(p, dtype=torch.float32)}

        def zeros(shape):
            return torch.zeros(shape, dtype=torch.uint8, device=p.device)

        blocks = -(-p.numel() // 256)
        return {"step": step, "exp_avg": zeros(p.shape), "exp_avg_sq": zeros(p.shape),
                "exp_avg_scale": zeros(blocks), "exp_avg_sq_scale": zeros(blocks)}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            ps = [p for p in group["params"] if p.grad is not None]
            if not ps:
                continue
            if any(p.grad.is_sparse for p in ps):
                raise RuntimeError("adamw: sparse gradients are not supported")
            shared = next((self.state[p]["step"] for p in group["params"] if self.state.get(p)), None)
            for p in ps:
                if not self.state.get(p):  # none, or an entry that a look has left
                    if _capturing(p.device):
                        raise RuntimeError("adamw: a replay would set new states to 0 again: take a step "
                                           "with every parameter before it is captured")
                    if shared is None:
                        shared = torch.zeros(1, dtype=torch.int64, device=p.device)
                    self.state[p] = self._new_state(p, group["state_bits"], shared)
            states = [self.state[p] for p in ps]
            eight = group["state_bits"] == 8
            group["grad_norm"] = adamw_step(
                ps, [p.grad for p in ps], [s["exp_avg"] for s in states],
                [s["exp_avg_sq"] for s in states], shared, lr=group["lr"], betas=group["betas"],
                eps=group["eps"], weight_decay=group["weight_decay"],
                max_grad_norm=group["max_grad_norm"], seed=group["seed"],
                exp_avg_scales=[s["exp_avg_scale"] for s in states] if eight else None,
                exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if eight else None)
        return loss

    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        """torch's, which would turn every state into the parameter's type: the states keep
        the types they were saved in, and a group's tensors share their step count again."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        for group, old in zip(self.param_groups, state_dict["param_groups"]):
            group["grad_norm"] = None
            shared = None
            for p, key in zip(group["params"], old["params"]):
                if not saved.get(key):
                    continue
                if shared is None:
                    shared = saved[key]["step"].detach().to(p.device, torch.int64).clone().reshape(1)
                self.state[p] = {"step": shared, **{
                    k: saved[key][k].detach().to(p.device).clone() for k in _STATES if k in saved[key]}}
