"""GPU: masks at the edge of what they can be -- references that mask what the policy does
not, rows with one open entry."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 179, 900, 2500, 60000, 131072])
@pytest.mark.parametrize("value", [-INF, -1e30])
@pytest.mark.parametrize("masked", [False, True])
def test_a_reference_that_masks_an_open_entry(vocab, dtype, value, masked):
    """KL(p | q) is infinite where q is 0 and p is not -- also where p is 0 in 32 bits -- in
    that row and no other; with a coefficient of 0 it takes no part in loss or gradient."""
    from cugo_b200.losses import policy_loss, policy_loss_grad
    if dtype == torch.float16 and value != -INF:
        pytest.skip("not a value of fp16")
    rows = 300 if vocab < 60000 else 6
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn((rows, vocab), device=DEV, generator=g).to(dtype)
    q = torch.randn((rows, vocab), device=DEV, generator=g).to(dtype)
    actions = torch.randint(vocab - 8, (rows,), device=DEV, generator=g)
    legal = None
    if masked:
        legal = torch.rand((rows, vocab), device=DEV, generator=g) < 0.5
        legal.scatter_(1, actions[:, None], True)
        legal[:, -2:] = True
    x[:, -3] = q[:, -3] = value              # masked on both sides: no part
    f = torch.zeros(rows, device=DEV)
    k = dict(legal=legal, ref_logits=q, clip_low=0.2)
    clean, dc = policy_loss_grad(x, actions, f, f + 1, **k, kl_coef=0.5)
    assert bool(torch.isfinite(clean.stats).all())
    for row, far in ((rows // 2, False), (rows - 1, True)):
        bad, y = q.clone(), x.clone()
        bad[row, -1] = value
        if far:
            y[row, -1] = -200.0
        for out in (policy_loss(y, actions, f, f + 1, **{**k, "ref_logits": bad}, kl_coef=0.5),
                    policy_loss_grad(y, actions, f, f + 1, **{**k, "ref_logits": bad}, kl_coef=0.5)[0]):
            assert float(out.stats[3]) == INF and float(out.loss) == INF
            assert bool(torch.isfinite(out.stats[[1, 2, 4, 5, 6]]).all())
        _, d = policy_loss_grad(y, actions, f, f + 1, **{**k, "ref_logits": bad}, kl_coef=0.5)
        keep = [i for i in range(rows) if i != row]
        # (Rows behind one with masked entries may be added up another way: a rounding apart.)
        off = (d.float() - dc.float())[keep].abs().max()
        assert float(off) <= 2.0 ** -7 * float(dc.float().abs().max())
        assert not bool(torch.isfinite(d[row, actions[row]]))
        zero = torch.zeros((), device=DEV)
        for coef in (0.0, zero):
            out, d = policy_loss_grad(y, actions, f, f + 1, **{**k, "ref_logits": bad}, kl_coef=coef)
            plain, want = policy_loss_grad(y, actions, f, f + 1, legal=legal)
            assert bool(torch.isfinite(out.loss)) and bool(torch.isfinite(d).all())
            assert abs(float(out.loss) - float(plain.loss)) < 1e-5 * (1 + abs(float(plain.loss)))
            assert float((d.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 33, 179, 700, 2500, 40000])
def test_a_single_open_entry_is_certain(vocab, dtype):
    """Forced moves: log p and entropy are 0, the ratio to a behaviour policy's log p of 0 is
    1, whatever the logit is; by mask and by value.  And log p is never above 0, the entropy
    never below."""
    from cugo_b200.losses import action_logp, policy_loss, policy_loss_grad
    rows = 900
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = (torch.randn((rows, vocab), device=DEV, generator=g) * 20).to(dtype)
    x[:8] = 0
    actions = torch.randint(vocab, (rows,), device=DEV, generator=g)
    legal = torch.zeros((rows, vocab), dtype=torch.bool, device=DEV).scatter_(1, actions[:, None], True)
    zero = torch.zeros(rows, device=DEV)
    for y, mask in ((x, legal), (x.masked_fill(~legal, -INF), None), (x.masked_fill(~legal, -INF), legal)):
        logp, entropy = action_logp(y, actions, mask)
        assert not bool(logp.any()) and not bool(entropy.any())
        for out in (policy_loss(y, actions, zero, zero + 1, legal=mask, ref_logits=y),
                    policy_loss_grad(y, actions, zero, zero + 1, legal=mask)[0]):
            assert not bool(out.logp.any())
            assert out.stats[1:3].tolist() == [-1.0, 0.0] and float(out.stats[4]) == 0.0
    # Nearly all of the weight at one entry.
    sharp = x.clone().scatter_(1, actions[:, None], x.amax(1, keepdim=True) + 14)
    logp, entropy = action_logp(sharp, actions)
    assert float(logp.max()) <= 0.0 and float(entropy.min()) >= 0.0
