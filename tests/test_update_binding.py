"""CPU: what the policy update's Python calls refuse before they look at a device."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from cugo_b200 import losses, optim

X, T = torch.zeros((4, 9)), torch.ones((4, 9))
I, F, O = torch.zeros(4, dtype=torch.int64), torch.zeros(4), torch.tensor([0, 2, 4])


def test_forward_mode_derivatives_are_refused():
    """The kernels see a dual tensor's primal only: its tangent would be lost without a word."""
    with fwd.dual_level():
        x, f = fwd.make_dual(X, T), fwd.make_dual(F, F + 1)
        one = fwd.make_dual(torch.zeros(()), torch.ones(()))
        calls = [
            lambda: losses.action_logp(x, I),
            lambda: losses.policy_loss(x, I, F, F),
            lambda: losses.policy_loss(X, I, f, F),
            lambda: losses.policy_loss(X, I, F, f),
            lambda: losses.policy_loss(X, I, F, F, weight=f),
            lambda: losses.policy_loss(X, I, F, F, ref_logits=x),
            lambda: losses.policy_loss(X, I, F, F, ref_logp=f),
            lambda: losses.policy_loss(X, I, F, F, kl_coef=one),
            lambda: losses.policy_loss(X, I, F, F, entropy_coef=one),
            lambda: losses.policy_loss_grad(x, I, F, F),
            lambda: losses.policy_loss_grad(X, I, F, F, grad_scale=one),
            lambda: losses.policy_loss_grad(X, I, F, F, dlogits=x),
            lambda: losses.preference_loss(x, I, O, F),
            lambda: losses.preference_loss(X, I, O, f),
            lambda: losses.preference_loss(X, I, O, F, weight=f),
            lambda: optim.adamw_step([f], [F], [F], [F], I[:1]),
            lambda: optim.adamw_step([F], [f], [F], [F], I[:1]),
            lambda: optim.adamw_step([F], [F], [F], [F], I[:1], lr=one),
        ]
        for k, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
                pytest.fail(f"call {k}")
        with pytest.raises(RuntimeError, match="CUDA tensor"):  # beside duals, not of them
            losses.action_logp(X, I)


def test_a_trace_is_refused():
    """torch.jit.trace would record the outputs' allocation and not the call."""
    calls = [
        lambda x: losses.action_logp(x, I),
        lambda x: losses.policy_loss(x, I, F, F).loss,
        lambda x: losses.policy_loss_grad(x, I, F, F)[1],
        lambda x: losses.preference_loss(x, I, O, F).loss,
        lambda x: optim.adamw_step([x], [X], [X], [X], I[:1], max_grad_norm=1.0),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (X,))
