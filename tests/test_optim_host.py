"""CPU: what optim.AdamW does before it calls its kernels, whose call is replaced here by one
that records its arguments."""
from __future__ import annotations

import pytest
import torch

from cugo_b200 import optim


@pytest.fixture
def calls(monkeypatch):
    made = []

    def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, **k):
        made.append((params, grads, exp_avgs, exp_avg_sqs, step, k))
        step += 1

    monkeypatch.setattr(optim, "adamw_step", adamw_step)
    return made


def _parameters(count=3):
    ps = [torch.nn.Parameter(torch.zeros(300 + k)) for k in range(count)]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_was_looked_up_before_the_first_step(calls, bits):
    """torch's state is a defaultdict: a look leaves an empty entry."""
    ps = _parameters()
    opt = optim.AdamW(ps, state_bits=bits)
    assert opt.state[ps[0]] == {} and opt.state[ps[2]] == {}
    opt.step()
    opt.step()
    (params, _, avgs, _, step, k), _ = calls
    assert params == ps and [a.shape for a in avgs] == [p.shape for p in ps] and int(step) == 2
    assert all(opt.state[p]["step"] is step for p in ps)
    assert (k["exp_avg_scales"] is None) == (bits == 32)
    # Saved and loaded with an empty entry among the others.
    opt.state[ps[1]].clear()
    other = optim.AdamW(_parameters(), state_bits=bits)
    other.load_state_dict(opt.state_dict())
    other.step()
    assert int(calls[-1][4]) == 3 and len(calls[-1][2]) == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_states_are_not_made_inside_a_capture(calls, monkeypatch, bits):
    """A replay would set them to 0 again: the first step of a parameter is refused there."""
    ps = _parameters(2)
    opt = optim.AdamW(ps, state_bits=bits)
    ps[1].grad, grad = None, ps[1].grad
    opt.step()  # ps[0] has a state
    ps[1].grad = grad
    monkeypatch.setattr(optim, "_capturing", lambda device: True)
    with pytest.raises(RuntimeError, match="before it is captured"):
        opt.step()
    ps[1].grad = None
    opt.step()
    assert len(calls) == 2 and ps[1] not in opt.state
