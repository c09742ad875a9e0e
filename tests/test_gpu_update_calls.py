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


def test_tensors_that_share_memory_are_refused():
    """What the AdamW step writes is no other tensor of the call, in whole or in part; what it
    only reads may be there twice, and neighbours in one buffer are apart."""
    from cugo_b200.optim import adamw_step

    def new(*sizes):
        return [torch.full((n,), 0.5, device=DEV) for n in sizes]

    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    p, g, m, v = (new(300, 700) for _ in range(4))
    flat = torch.full((2000,), 0.5, device=DEV)
    codes = [torch.zeros(1000, dtype=torch.uint8, device=DEV) for _ in range(4)]
    eight = [[c[:300], c[300:]] for c in codes[:2]]
    scales = [[c[:2], c[2:5]] for c in codes[2:]]
    bad = [
        (p, g, m, m),
        ([p[0], p[0]], [g[0], g[0]], new(300, 300), new(300, 300)),
        ([flat[:300], flat[200:900]], g, m, v),
        (p, p, m, v),
        (p, [g[0], p[1]], m, v),
        (p, [flat[:300], flat[400:1100]], [flat[1200:1500], flat[700:1400]], v),
        ([flat[0:300], flat[1000:1700]], g, [flat[299:599], m[1]], v),
        (p, g, eight[0], [eight[1][0], codes[0][200:900]], *scales),
        (p, g, *eight, scales[0], scales[0]),
        (p, g, *eight, [codes[0][:2], scales[0][1]], scales[1]),
    ]
    before = [t.clone() for t in (*p, *m, *v, flat, *codes)]
    for k, args in enumerate(bad):
        more = dict(exp_avg_scales=args[4], exp_avg_sq_scales=args[5]) if len(args) > 4 else {}
        with pytest.raises(RuntimeError, match="twice"):
            adamw_step(*args[:4], step, **more)
            pytest.fail(f"call {k}")
    with pytest.raises(RuntimeError, match="twice"):
        adamw_step([p[0], flat[:1]], [g[0], flat[1:2]], [m[0], flat[2:3]], [v[0], flat[3:4]], step, lr=flat[0])
    assert int(step) == 0 and all(torch.equal(a, b) for a, b in zip(before, (*p, *m, *v, flat, *codes)))
    cut = list(flat.split([300, 700, 300, 700]))
    adamw_step(cut[:2], [g[1][:300], g[1]], cut[2:], v, step)
    adamw_step([*p, flat[:0]], [*g, flat[:0]], [*eight[0], codes[0][:0]], [*eight[1], codes[1][:0]], step,
               exp_avg_scales=[*scales[0], codes[2][:0]], exp_avg_sq_scales=[*scales[1], codes[3][:0]])
    assert int(step) == 2
