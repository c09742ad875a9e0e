"""The operators of a policy update from their definitions, in 64 bits with plain torch
operations and autograd: what the kernels of loss_kernels.cu and optim_kernels.cu are
tested against.  Rows that do not count are dropped, masked entries are left out."""
from __future__ import annotations

import torch

MASKED = -float(2 ** 30)


def rows64(logits, actions, legal=None, weight=None):
    """(leaf logits in 64 bits, log p of every entry with 0 where p is 0, p, which rows count)."""
    leaf = logits.detach().double().requires_grad_()
    n, v = leaf.shape
    open_ = torch.ones((n, v), dtype=torch.bool, device=leaf.device) if legal is None else legal.expand(n, v)
    open_ = open_ & ~(leaf.detach() <= MASKED)
    used = (actions >= 0) & (actions < v)
    used &= open_.gather(1, actions.clamp(0, v - 1)[:, None])[:, 0]
    if weight is not None:
        used &= weight != 0
    x = torch.where(open_, leaf, torch.full_like(leaf, -float("inf")))
    x = torch.where(used[:, None], x, torch.zeros_like(leaf))  # a uniform row in its place
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    lp = torch.where(p > 0, lp, torch.zeros_like(lp)) if not bool(torch.isnan(lp).any()) else lp
    return leaf, lp, p, used


def _zero(used, t):
    return torch.where(used, t, torch.zeros_like(t))


def action_logp64(logits, actions, legal=None, weight=None):
    """(leaf, log p of the actions, entropy, p, which rows count)."""
    leaf, lp, p, used = rows64(logits, actions, legal, weight)
    logp = _zero(used, lp.gather(1, actions.clamp(0, lp.shape[1] - 1)[:, None])[:, 0])
    return leaf, logp, _zero(used, -(p * lp).sum(1)), p.detach(), used


def policy64(logits, actions, logp_old, adv, legal=None, weight=None, ref_logits=None, ref_logp=None,
             clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0, denominator=None):
    """(gradient, stats [7], logp, p, which rows count)."""
    leaf, lp, p, used = rows64(logits, actions, legal, weight)
    logp = _zero(used, lp.gather(1, actions.clamp(0, lp.shape[1] - 1)[:, None])[:, 0])
    w = torch.ones_like(logp) if weight is None else weight.double()
    d = float(w.sum()) if denominator is None else denominator
    w = _zero(used, w)
    log_ratio = _zero(used, logp - logp_old.double())
    ratio = log_ratio.exp()
    a = adv.double()
    gain = torch.minimum(ratio * a, ratio.clamp(1 - clip_low, 1 + clip_high) * a)
    kl = torch.zeros_like(logp)
    if ref_logp is not None:
        diff = _zero(used, ref_logp.double() - logp)
        kl = diff.exp() - 1 - diff
    if ref_logits is not None:
        lq = rows64(ref_logits, actions, legal, weight)[1].detach()
        kl = (p * (lp - lq)).sum(1)
    each = torch.stack((-gain, -(p * lp).sum(1), kl, ratio - 1 - log_ratio,
                        ((ratio < 1 - clip_low) | (ratio > 1 + clip_high)).double(), torch.ones_like(w)))
    means = (_zero(used, each) * w).sum(1) / d if d else each.sum(1) * 0
    loss = means[0] - entropy_coef * means[1] + kl_coef * means[2]
    grad = torch.autograd.grad(loss, leaf)[0]
    return grad, torch.cat((loss[None], means)).detach(), logp.detach(), p.detach(), used


def preference64(logits, actions, offsets, ref_logp, legal=None, weight=None, beta=0.1, smoothing=0.0,
                 average=False):
    """(gradient, loss, margin, sequences' log p, accuracy)."""
    leaf, logp, _, _, used = action_logp64(logits, actions, legal, weight)
    w = _zero(used, torch.ones_like(logp) if weight is None else weight.double())
    o = offsets.tolist()
    score, seq = [], []
    for i, j in zip(o, o[1:]):
        n = w[i:j].sum() if average and bool(w[i:j].sum() != 0) else 1.0
        score.append((w[i:j] * (logp - ref_logp.double())[i:j]).sum() / n)
        seq.append((w[i:j] * logp[i:j]).sum() / n)
    m = beta * (torch.stack(score[0::2]) - torch.stack(score[1::2]))
    f = torch.nn.functional.logsigmoid
    loss = (-(1 - smoothing) * f(m) - smoothing * f(-m)).mean()
    grad = torch.autograd.grad(loss, leaf)[0]
    return grad, loss.detach(), m.detach(), torch.stack(seq).detach(), (m > 0).double().mean()


def adamw64(p, g, m, v, t, lr, b1, b2, eps, decay, clip=1.0):
    """One step on 64-bit tensors: (p, m, v)."""
    g = g * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * decay) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
    return p, m, v


# ---- the rounding by random bits ------------------------------------------------------------

def mix32(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(first_block, n, step, seed, device):
    """The 32 random bits of elements 0 .. n - 1 of a tensor before which `first_block`
    blocks of 256 were counted."""
    e = torch.arange(n, dtype=torch.int64, device=device) + first_block * 256
    key = int(mix32(torch.tensor((seed + step * 0x9E3779B9) & 0xFFFFFFFF)))
    return mix32((e & 0xFFFFFFFF) ^ ((key + (e >> 32) * 0x9E3779B9) & 0xFFFFFFFF))


def e4m3_step(x):
    """The distance of e4m3's grid points around |x| (at most 448)."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)


def block_scale(x):
    """[blocks] the power of two that keeps each block of 256 at or below 448 (flat x, 64 bits)."""
    pad = torch.zeros(-(-x.numel() // 256) * 256, dtype=x.dtype, device=x.device)
    pad[:x.numel()] = x
    a = pad.view(-1, 256).abs().amax(1)
    k = torch.where(a > 0, torch.ceil(torch.log2(a / 448)), torch.full_like(a, -100.0))
    return torch.exp2(k.clamp(-100, 120))


def decode(codes, scale):
    """8-bit states (flat uint8 codes, uint8 scales) as 64-bit values."""
    s = torch.exp2(scale.double() - 127).repeat_interleave(256)[:codes.numel()]
    return codes.view(torch.float8_e4m3fn).double() * s
