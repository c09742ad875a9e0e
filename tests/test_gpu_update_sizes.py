"""GPU: the policy update's kernels at sizes where a warp or a block goes round more than
once: short rows in three turns and more, the AdamW step with several blocks of 256 elements
a warp and more tiles than its grid.  The tolerances are those of test_gpu_losses.py and
test_gpu_optim.py."""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_losses import chain, grad_tol, make, near, policy_case, policy_tols
from tests.test_gpu_optim import HYPER, U, expected, p_tolerance, step, tensors
from tests.test_gpu_optim import near as near_flat
from tests.update_reference import action_logp64, block_scale, decode, e4m3_step, policy64, random_bits

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")

# Rows that a launch's warps take in three turns or more: four blocks an SM at most, of 16
# rows (up to 192 entries), 8 or 4 (above 384).
TURNS = [(30001, 179), (30001, 30), (16001, 300), (8001, 1000)]


@pytest.mark.parametrize("rows,vocab", TURNS)
@pytest.mark.parametrize("masks", ["own", "one", "none"])
@pytest.mark.parametrize("kl,weights,pad", [("full", True, 0), ("sampled", False, 5), ("none", True, 200)])
def test_short_rows_in_many_turns(rows, vocab, masks, kl, weights, pad):
    from cugo_b200.losses import policy_loss_grad
    dtype = torch.float32
    x, actions, old, adv, k = policy_case(rows, vocab, dtype, masks == "own", pad, kl, weights)
    if masks == "one":
        one = torch.arange(vocab, device=DEV) % 3 != 1
        actions = torch.where(one[actions], actions, actions - actions % 3)
        k["legal"] = one.expand(rows, vocab)
        old = torch.full((rows,), -4.0, device=DEV) + 1e-3 * adv
    want, stats, logp, p, _ = policy64(x, actions, old, adv, **k)
    worst, size = policy_tols(vocab, x, actions, k, adv, p, stats, rows)
    if masks == "one":  # the ratios lie anywhere: those within a rounding of the clip decide nothing here
        ratio = (logp - old.double()).exp()
        size = size * ratio.clamp_min(1.0)
        worst = worst * float(ratio.max())
        edge = torch.minimum((ratio - 0.8).abs(), (ratio - 1.28).abs()) < 1e-4 * (1 + ratio)
        keep = ~edge
    else:
        keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    out, d = policy_loss_grad(x, actions, old, adv, **k)
    near(out.logp, logp, chain(vocab) * U * (1 + logp.abs()), "logp")
    near(d[keep], want[keep], grad_tol(vocab, p, actions, size, dtype, want)[keep], "gradient, rows one after another")
    if bool(keep.all()):
        near(out.stats, stats, worst * (1 + stats.abs()), "stats")
    room = torch.full((rows, vocab + 9), 7.0, dtype=torch.bfloat16, device=DEV)
    again, same = policy_loss_grad(x, actions, old, adv, **k, dlogits=room[:, 1:vocab + 4])
    assert torch.equal(again.logp, out.logp) and torch.equal(again.stats, out.stats)
    near(same[keep, :vocab], want[keep], grad_tol(vocab, p, actions, size, torch.bfloat16, want)[keep], "rows apart")
    assert not bool(same[:, vocab:].any())
    assert bool((room[:, 0] == 7).all()) and bool((room[:, vocab + 4:] == 7).all())


@pytest.mark.parametrize("rows,vocab", TURNS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_in_many_turns(rows, vocab, dtype):
    from cugo_b200.losses import action_logp
    rows = 2 * rows + 1
    x, actions, mask, _ = make(rows, vocab, dtype, 6, True, 3)
    _, want, want_h, _, _ = action_logp64(x, actions, mask)
    logp, entropy = action_logp(x, actions, mask)
    c = chain(vocab) * U
    near(logp, want.detach(), c * (1 + want.detach().abs()), "log p")
    near(entropy, want_h.detach(), c * (1 + 2 * want_h.detach().abs() + math.log(vocab)), "entropy")


def rounded_p(want, first_block, step_count, seed):
    """bf16 parameters from their fp32 values before the rounding, by the random bits."""
    r = random_bits(first_block, want.numel(), step_count, seed, DEV)
    return (r * 0x2C1B3C6D & 0xFFFFFFFF) >> 16


def check_bf16(p, new, tol, first_block, now, name):
    """Each on one of the two values around, the one that the bits say (off the border).

    What is rounded is the kernel's fp32 value, which is off the definition's by tol (fp32
    parameters' bound): of a parameter that the step brings close to 0, p (1 - lr wd) - update
    cancels, and tol, of the size of its terms, is more than a step of the small result.  So
    the bound is a step, and tol for where the value lay and which step it had."""
    unit = torch.exp2(torch.floor(torch.log2(new.abs().clamp_min(1e-30))) - 7)
    near_flat(p, new, unit * (1 + 1e-3) + 2 * tol, name)
    low = torch.floor(new.abs() / unit)
    share = new.abs() / unit - low
    up = share + (rounded_p(new, first_block, now, 11).double()) / 65536
    clear = ((up - 1.0).abs() > 2e-3 + tol / unit) & (tol < 1e-3 * unit)
    want = torch.copysign((low + (up >= 1.0)) * unit, new)
    assert torch.equal(p.double()[clear], want[clear]) and float(clear.double().mean()) > 0.9, name


def check_codes(codes, scales, want, bits, name):
    """8-bit states: scales and codes as the definition and the random bits say."""
    n = want.numel()
    scale, stored = block_scale(want), torch.exp2(scales.double() - 127)
    top = torch.zeros(scale.numel() * 256, dtype=torch.float64, device=DEV)
    top[:n] = want.abs()
    top = top.view(-1, 256).amax(1) / scale
    edge = ((top - 448).abs() < 448 * 8 * U) | ((top - 224).abs() < 224 * 8 * U)
    assert bool(((stored == scale) | edge).all()), name
    unit = stored.repeat_interleave(256)[:n]
    x, got = want / unit, decode(codes, scales) / unit
    grid = e4m3_step(x)
    low = torch.floor(x.abs() / grid) * grid
    up = (x.abs() - low) / grid + (bits.double() + 0.5) / 65536
    clear = (up - 1.0).abs() > 1e-3
    code = torch.copysign(low + (up >= 1.0) * grid, x)
    if name == "v":
        code = torch.where((x > 0) & (code == 0), 2.0 ** -9, code)
    assert torch.equal(got[clear], code[clear]), name


def check_step(sizes, p_type, g_type, bits, clip, offset, odd=()):
    t = tensors(sizes, p_type, g_type, bits, 3, offset)
    for k in odd:  # tensors that begin between two 16-byte boundaries, among others that do not
        for name in ("p", "g", "m", "v"):
            wide = torch.empty(sizes[k] + 3, dtype=t[name][k].dtype, device=DEV)
            wide[3:] = t[name][k]
            t[name][k] = wide[3:]
    old, new, norm, c = expected(t, clip)
    got = step(t, clip)
    if clip is not None:
        assert abs(float(got) - norm) <= 4 * U * norm
    number, now = 0, int(t["step"])
    for k, n in enumerate(sizes):
        if bits == 32:
            g = (old[k][1] * c).abs()
            near_flat(t["m"][k], new[k][1], 6 * U * (old[k][2].abs() + g), "m")
            near_flat(t["v"][k], new[k][2], 12 * U * (old[k][3] + g * g), "v")
        elif n:
            r = random_bits(number, n, now, 11, DEV)
            check_codes(t["m"][k], t["ms"][k], new[k][1], r & 0xFFFF, "m")
            check_codes(t["v"][k], t["vs"][k], new[k][2], r >> 16, "v")
        if p_type == torch.float32:
            near_flat(t["p"][k], new[k][0], p_tolerance(old[k], new[k], HYPER), "p")
        elif n:
            check_bf16(t["p"][k], new[k][0], p_tolerance(old[k], new[k], HYPER), number, now, k)
        number += -(-n // 256)


@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [2047, 2048, 2049, 0, 5], [720 * 64, 64, 64 * 64, 64]])
@pytest.mark.parametrize("g_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip,offset", [(None, 0), (0.05, 0), (100.0, 3)])
def test_bf16_parameters_with_32_bit_states(sizes, g_type, clip, offset):
    check_step(sizes, torch.bfloat16, g_type, 32, clip, offset)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p_type,g_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                           (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("sizes,odd", [([10_000_003, 257, 5000, 1, 70001], (2, 4)), ([300, 9_800_000, 9_900_001], (1,))])
def test_several_blocks_a_warp(bits, p_type, g_type, sizes, odd):
    """Above 9.7 million elements a warp takes four blocks; the norm's grid goes round."""
    check_step(sizes, p_type, g_type, bits, 0.05, 0, odd)


@pytest.mark.parametrize("bits,p_type", [(32, torch.float32), (8, torch.float32), (8, torch.bfloat16)])
def test_more_tiles_than_blocks(bits, p_type):
    """Above 78 million elements the step's grid goes round."""
    check_step([80_000_000, 1_000_003, 77], p_type, p_type, bits, 0.05, 0, (1,))
