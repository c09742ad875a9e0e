"""Losses of a policy over rows of logits, on the kernels of loss_kernels.cu: the
log-probabilities of given actions (`action_logp`), the clipped policy loss with an
entropy bonus and a KL term (`policy_loss`, and `policy_loss_grad` for steps without
autograd), and the preference loss over pairs of lines of play (`preference_loss`).

They go beside the 179-action loss of the PPO update (`ext.ppo_loss`), and take what that
one does not: any number of entries, fp32, bf16 or fp16 logits, rows of any stride, weights
(0 for padded rows), bounds of the clip that differ, a reference policy, and autograd.

Rows.  logits [rows, entries] with unit column stride; legal bool of the same shape (or
one mask expanded over the rows), or None; actions int64 [rows].  An entry that is not
legal has probability 0, and so has one at or below -2^30 (-inf, -1e30, the type's lowest
value).  What stands in such a place is not used, NaN included.  A row does not count --
log p, entropy and gradients are 0 -- where its action is outside the entries or masked,
or its weight is 0; so a row that its mask leaves empty never counts.

Everything is computed in 32 bits from the logits' own type; sums over rows in 64 bits and
in a fixed order, so every run gives the same bits.  The calls enqueue on the current
stream of the logits' device, do not wait for it, and can be captured in CUDA graphs.
Backwards of backwards are not built."""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .ext import load_extension

_EXT = None


def _ext():
    """The extension, looked up once: these calls are short enough for the look to count."""
    global _EXT
    if _EXT is None:
        _EXT = load_extension()
    return _EXT


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


class _ActionLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, legal):
        logp, entropy, lse, _ = _ext().action_logp(logits, actions, legal, backward=True)
        ctx.save_for_backward(logits, actions, legal, lse, entropy)
        ctx.set_materialize_grads(False)
        return logp, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logp, d_entropy):
        if d_logp is None and d_entropy is None:
            return None, None, None
        logits, actions, legal, lse, entropy = ctx.saved_tensors
        d_logp = d_logp if d_logp is None else d_logp.contiguous()
        d_entropy = d_entropy if d_entropy is None else d_entropy.contiguous()
        return _ext().action_logp_backward(logits, actions, legal, lse, entropy, d_logp,
                                                     d_entropy), None, None


def action_logp(logits: torch.Tensor, actions: torch.Tensor,
                legal: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(log p of each row's action, entropy of each row's distribution), fp32 [rows] each,
    differentiable in the logits."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return _ActionLogp.apply(logits, actions, legal)
    logp, entropy, _, _ = _ext().action_logp(logits, actions, legal)
    return logp, entropy


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, logp_old, adv, legal, weight, ref_logits, ref_logp, coefs):
        loss, stats, logp, _ = _ext().policy_loss(
            logits, actions, logp_old, adv, legal, weight, ref_logits, ref_logp, *coefs)
        ctx.save_for_backward(logits, actions, logp_old, adv, legal, weight, ref_logits, ref_logp)
        ctx.coefs, ctx.denominator = coefs, stats[7:]
        stats = stats[:7]
        ctx.mark_non_differentiable(stats, logp)
        ctx.set_materialize_grads(False)
        return loss, stats, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss, *_):
        if d_loss is None:
            return (None,) * 9
        logits = ctx.saved_tensors[0]
        # With the denominator that the forward found; the logits are read once more.
        d = _ext().policy_loss(*ctx.saved_tensors, *ctx.coefs[:4], 0.0, ctx.denominator,
                               grad_scale_dev=d_loss, grad_dtype=logits.dtype, stats=False)[3]
        return (d,) + (None,) * 8


def _coefs(clip_low, clip_high, kl_coef, entropy_coef, denominator):
    clip_high = clip_low if clip_high is None else clip_high
    if clip_low < 0.0 or clip_high < 0.0:
        raise RuntimeError("policy_loss: the clip's bounds must not be negative")
    if denominator is not None and not denominator > 0.0:
        raise RuntimeError("policy_loss: the denominator must be positive")
    kl_coef, entropy_coef = (c if torch.is_tensor(c) else float(c) for c in (kl_coef, entropy_coef))
    return (float(clip_low), float(clip_high), kl_coef, entropy_coef,
            0.0 if denominator is None else float(denominator))


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

    K: KL(p | q) over the legal entries, q from ref_logits; or, from ref_logp (the
    reference's log p of the actions), the estimate exp(d) - 1 - d with d = ref_logp - log p,
    which is never negative and right in the mean; or 0.  D: the sum of the weights (the
    rows without weights; 0 gives a loss of 0), or `denominator` (a data-parallel job's
    total, say).  logp_old, adv, weight, ref_logp: fp32 [rows]; clip_high defaults to
    clip_low; kl_coef and entropy_coef may be one fp32 value on the device (a schedule that a
    captured graph follows)."""
    coefs = _coefs(clip_low, clip_high, kl_coef, entropy_coef, denominator)
    if torch.is_grad_enabled() and logits.requires_grad:
        return PolicyLoss(*_PolicyLoss.apply(logits, actions, logp_old, adv, legal, weight, ref_logits,
                                             ref_logp, coefs))
    loss, stats, logp, _ = _ext().policy_loss(logits, actions, logp_old, adv, legal, weight, ref_logits,
                                              ref_logp, *coefs)
    return PolicyLoss(loss, stats[:7], logp)


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
    are set to 0: the padded operand of a head's GEMM), or to a new tensor of grad_dtype
    (the logits' type)."""
    coefs = _coefs(clip_low, clip_high, kl_coef, entropy_coef, denominator)
    if dlogits is None:
        grad_dtype = grad_dtype or logits.dtype
    elif grad_dtype is not None and grad_dtype != dlogits.dtype:
        raise RuntimeError("policy_loss: dlogits is not of grad_dtype")
    scale, scale_dev = (1.0, grad_scale) if torch.is_tensor(grad_scale) else (float(grad_scale), None)
    loss, stats, logp, dlogits = _ext().policy_loss(
        logits, actions, logp_old, adv, legal, weight, ref_logits, ref_logp, *coefs, None, scale, scale_dev,
        dlogits, grad_dtype)
    return PolicyLoss(loss, stats[:7], logp), dlogits


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, offsets, ref_logp, legal, weight, options):
        out, lse, d_logp = _preference(logits, actions, offsets, ref_logp, legal, weight, options, True)
        ctx.save_for_backward(logits, actions, legal, lse, d_logp)
        ctx.mark_non_differentiable(*out[1:])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss, *_):
        if d_loss is None:
            return (None,) * 7
        logits, actions, legal, lse, d_logp = ctx.saved_tensors
        d = _ext().action_logp_backward(logits, actions, legal, lse, None, d_logp, None,
                                                  scale=d_loss)
        return (d,) + (None,) * 6


def _preference(logits, actions, offsets, ref_logp, legal, weight, options, grad):
    """((loss, margin, sequences' log p, accuracy), and what the backward needs)."""
    ext = _ext()
    logp, _, lse, d_logp = ext.action_logp(logits, actions, legal, weight, entropy=False,
                                           backward=True, zeros=grad)
    return ext.preference_pairs(logp, ref_logp, weight, lse, offsets, *options,
                                d_logp=d_logp), lse, d_logp


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
    options = (float(beta), float(label_smoothing), bool(average))
    if torch.is_grad_enabled() and logits.requires_grad:
        return PreferenceLoss(*_PreferenceLoss.apply(logits, actions, offsets, ref_logp, legal, weight,
                                                     options))
    out, _, _ = _preference(logits, actions, offsets, ref_logp, legal, weight, options, False)
    return PreferenceLoss(*out)
