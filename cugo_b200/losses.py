"""Losses of a policy over rows of logits, on the kernels of loss_kernels.cu: the
log-probabilities of given actions (`action_logp`), the clipped policy loss with an
entropy bonus and a KL term (`policy_loss`, and `policy_loss_grad` for steps without
autograd), and the preference loss over pairs of lines of play (`preference_loss`).

They go beside the 179-action loss of the PPO update (`ext.ppo_loss`), and take what that
one does not: any number of entries, fp32, bf16 or fp16 logits, rows of any stride, weights
(0 for padded rows), bounds of the clip that differ, a reference policy, and autograd.

Rows.  logits [rows, entries] with unit column stride; legal bool of the same shape (or
one mask expanded over the rows), or None; actions int64 [rows].  An entry that is not
legal has probability 0, and so has one at or below -2^30 (-inf, -1e30, the lowest value of
fp32 and bf16; fp16's, -65,504, is an entry); legal entries are taken to lie below 2^30.
What stands in a masked place is not used, NaN included.  A row does not count -- log p,
entropy and gradients are 0 -- where its action is outside the entries or masked, or its
weight is 0; so a row that its mask leaves empty never counts.  log p is never above 0 and
the entropy never below; an action that is a row's only open entry has both 0.

Everything is computed in 32 bits from the logits' own type; sums over rows in 64 bits and
in a fixed order, so every run gives the same bits.  The calls enqueue on the current
stream of the logits' device, do not wait for it, and can be captured in CUDA graphs.
A backward that is captured needs a graph of its own leaves' making: torch ties a leaf's
accumulation to the stream of the graph that still holds it, so eager graphs of the same
leaves have to be gone by then.  Backwards of backwards, forward-mode derivatives and
traces are not built: such calls raise."""
from __future__ import annotations

from typing import NamedTuple

import torch
from .ext import load_update

STATS = ("loss", "policy", "entropy", "kl", "kl_old", "clip_fraction", "used")


class PolicyLoss(NamedTuple):
    """loss: scalar; stats: fp32 [7], in the order of STATS -- the loss, the means of the
    clipped surrogate's negative, the entropy, the KL to the reference, the estimate
    (r - 1) - log r of the KL to the behaviour policy, the share of ratios outside the
    clip's bounds, and the share of rows (by weight) that count; logp: fp32 [rows]."""
    loss: torch.Tensor
    stats: torch.Tensor
    logp: torch.Tensor


class PreferenceLoss(NamedTuple):
    """loss: scalar; margin: fp32 [pairs], beta times the difference of the scores; logp:
    fp32 [2 pairs], the sequences' log-probabilities; accuracy: the share of margins above
    0.  Only the loss is differentiable."""
    loss: torch.Tensor
    margin: torch.Tensor
    logp: torch.Tensor
    accuracy: torch.Tensor


def action_logp(logits: torch.Tensor, actions: torch.Tensor,
                legal: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(log p of each row's action, entropy of each row's distribution), fp32 [rows] each,
    differentiable in the logits."""
    return load_update().action_logp(logits, actions, legal)


def _options(clip_low, clip_high, kl_coef, entropy_coef, denominator) -> tuple:
    """The binding's arguments from the clip to the denominator (0: found from the rows)."""
    if denominator is not None and not denominator > 0.0:
        raise RuntimeError("policy_loss: the denominator must be positive")
    kl = (1.0, kl_coef) if torch.is_tensor(kl_coef) else (kl_coef, None)
    entropy = (1.0, entropy_coef) if torch.is_tensor(entropy_coef) else (entropy_coef, None)
    return (clip_low, clip_low if clip_high is None else clip_high, *kl, *entropy, denominator or 0.0)


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, logp_old: torch.Tensor,
                adv: torch.Tensor, *, legal: torch.Tensor | None = None,
                weight: torch.Tensor | None = None, ref_logits: torch.Tensor | None = None,
                ref_logp: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float | None = None, kl_coef: float | torch.Tensor = 0.0,
                entropy_coef: float | torch.Tensor = 0.0,
                denominator: float | None = None) -> PolicyLoss:
    """The clipped policy loss, differentiable in the logits:

      r = exp(log p(action) - logp_old)
      loss = sum w (-min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A)
                    - entropy_coef H + kl_coef K) / D

    K: KL(p | q) over the legal entries, q from ref_logits (infinite, and the row's gradient
    with it, where q masks an entry that p does not; with a coefficient of 0 it takes no part
    in loss and gradient); or, from ref_logp (the
    reference's log p of the actions), the estimate exp(d) - 1 - d with d = ref_logp - log p,
    which is never negative and right in the mean; or 0.  D: the sum of the weights (the
    rows without weights; 0 gives a loss of 0), or `denominator` (a data-parallel job's
    total, say).  logp_old, adv, weight, ref_logp: fp32 [rows]; clip_high defaults to
    clip_low; kl_coef and entropy_coef may be one fp32 value on the device (a schedule that a
    captured graph follows)."""
    return PolicyLoss(*load_update().policy_loss(
        logits, actions, logp_old, adv, legal, weight, ref_logits, ref_logp,
        *_options(clip_low, clip_high, kl_coef, entropy_coef, denominator)))


def policy_loss_grad(logits: torch.Tensor, actions: torch.Tensor, logp_old: torch.Tensor,
                     adv: torch.Tensor, *, legal: torch.Tensor | None = None,
                     weight: torch.Tensor | None = None, ref_logits: torch.Tensor | None = None,
                     ref_logp: torch.Tensor | None = None, clip_low: float = 0.2,
                     clip_high: float | None = None, kl_coef: float | torch.Tensor = 0.0,
                     entropy_coef: float | torch.Tensor = 0.0, denominator: float | None = None,
                     grad_scale: float | torch.Tensor = 1.0, grad_dtype: torch.dtype | None = None,
                     dlogits: torch.Tensor | None = None) -> tuple[PolicyLoss, torch.Tensor]:
    """policy_loss and grad_scale (a number, or one fp32 value on the device) times its
    gradient, in one pass over the logits, for a step that runs its backward without
    autograd.  The gradient goes to dlogits [rows, >= entries] (columns past the entries
    are set to 0: the padded operand of a head's GEMM; memory of its own), or to a new tensor of grad_dtype
    (the logits' type)."""
    scale, scale_dev = (1.0, grad_scale) if torch.is_tensor(grad_scale) else (grad_scale, None)
    loss, stats, logp, grad = load_update().policy_loss_grad(
        logits, actions, logp_old, adv, legal, weight, ref_logits, ref_logp,
        *_options(clip_low, clip_high, kl_coef, entropy_coef, denominator), scale, scale_dev, grad_dtype, dlogits)
    return PolicyLoss(loss, stats, logp), grad


def preference_loss(logits: torch.Tensor, actions: torch.Tensor, offsets: torch.Tensor,
                    ref_logp: torch.Tensor, *, legal: torch.Tensor | None = None,
                    weight: torch.Tensor | None = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, average: bool = False) -> PreferenceLoss:
    """The preference loss over pairs of sequences of decisions, differentiable in the logits.

    The rows of all sequences lie one after another: sequence j holds rows offsets[j] ..
    offsets[j + 1] - 1 (offsets int64 [2 pairs + 1] on the device, not decreasing; an empty
    sequence scores 0), and pair i prefers sequence 2 i to sequence 2 i + 1 -- the better and
    the worse line of a duplicate deal, say.  ref_logp: fp32 [rows], log p of the actions
    under the frozen policy (`action_logp`); weight: fp32 [rows], 0 for rows that are not the
    policy's own.

      score = sum w (log p - ref_logp), over sum w with `average`
      m = beta (score of the preferred - score of the other)
      loss = mean of -(1 - label_smoothing) log sigmoid(m) - label_smoothing log sigmoid(-m)

    A margin needs all its rows first, so the backward reads the logits a second time."""
    return PreferenceLoss(*load_update().preference_loss(logits, actions, offsets, ref_logp, legal, weight,
                                                         beta, label_smoothing, average))
