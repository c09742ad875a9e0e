"""GPU: how the policy update's calls get along with what goes on around them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_statistics_may_be_changed_before_the_backward():
    """An in-place all-reduce of the statistics, say: the gradient is the same."""
    from cugo_b200.losses import policy_loss
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((50, 179), device=DEV, generator=g).requires_grad_()
    actions = torch.randint(179, (50,), device=DEV, generator=g)
    f = torch.zeros(50, device=DEV)
    grads = []
    for change in (False, True):
        out = policy_loss(x, actions, f - 5.0, f + 1.0, weight=f + 0.5)
        if change:
            out.stats.mul_(7.0)
            out.logp.zero_()
        grads += torch.autograd.grad(out.loss, x)
    assert torch.equal(*grads) and bool(grads[0].any())


def test_transforms_are_refused():
    """torch.func's transforms and torch.jit.trace do not see into the calls: errors, not results
    without derivatives or without the call."""
    from cugo_b200.losses import action_logp
    x, t = torch.zeros((4, 9), device=DEV), torch.ones((4, 9), device=DEV)
    i = torch.zeros(4, dtype=torch.int64, device=DEV)
    for call in (lambda: torch.func.jvp(lambda y: action_logp(y, i)[0], (x,), (t,)),
                 lambda: torch.func.grad(lambda y: action_logp(y, i)[0].sum())(x),
                 lambda: torch.func.vmap(lambda y: action_logp(y, i)[0])(x.expand(2, 4, 9)),
                 lambda: torch.jit.trace(lambda y: action_logp(y, i), (x,))):
        with pytest.raises(RuntimeError):
            call()
