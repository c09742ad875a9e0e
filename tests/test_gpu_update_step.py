"""GPU: the operators of a policy update used together -- a minibatch step held to a
reference policy with the AdamW step, as the trainer runs it, and a step on preferred
lines of play -- against the same steps composed in torch."""
from __future__ import annotations

import copy

import pytest
import torch

from tests.test_gpu_ppo import _minibatch, _twins
from tests.update_reference import adamw64, policy64, preference64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _networks(seed=2):
    actor, _ = _twins(720, 179, seed=seed)
    critic, _ = _twins(770, 1, seed=seed + 1, squeeze=True)
    reference, _ = _twins(720, 179, seed=seed + 20)
    return actor, critic, reference


def _adamw(actor, critic, **k):
    from cugo_b200.optim import AdamW
    return AdamW([{"params": list(n.parameters())} for n in (actor, critic)],
                 **{**dict(lr=3e-4, eps=1e-5, max_grad_norm=1.0, weight_decay=0.01), **k})


def test_native_step_with_a_reference():
    """The policy loss with its KL term in NativePpoStep: statistics and the head's gradient
    against the definition on the step's own logits, the step against the definition on the
    step's own gradients, and the autograd step's gradients beside them.

    The logits, of fp32, are the same on both sides, so the statistics differ by fp32 sums
    (1e-5); the head's bias gradient is the column sums of bf16-rounded rows: 2^-8 of the
    rows' sizes, added up."""
    from cugo_b200.ppo import NativePpoStep, PpoStep, train_forward
    actor, critic, reference = _networks()
    mb = _minibatch(4096, 4)
    twins = copy.deepcopy(actor), copy.deepcopy(critic)
    step = NativePpoStep(actor, critic, _adamw(actor, critic), reference=reference, kl_coef=0.3)
    step.entropy_coef.fill_(0.05)
    logits, _ = train_forward(actor, mb.features)
    with torch.no_grad():
        ref_logits = reference(mb.features).float()
    grad, stats, _, _, _ = policy64(logits, mb.actions, mb.logp_old, mb.adv, legal=mb.legal,
                                    ref_logits=ref_logits, kl_coef=0.3, entropy_coef=0.05)
    before = [p.detach().double() for p in list(actor.parameters()) + list(critic.parameters())]
    step.step(mb)
    for at, want in zip((0, 2, 3, 4, 7), stats[[1, 2, 4, 5, 3]].tolist()):
        assert abs(float(step.sums[at]) - want) < 1e-5 * (1 + abs(want)), at
    assert int(step.sums[5]) == 1 and abs(float(step.last_kl) - float(stats[4])) < 1e-5 * (1 + float(stats[4]))
    # (The gradients in .grad are as the backward left them: the clip is in the step.)
    bias = actor.out.bias.grad.double()
    assert bool(((bias - grad.sum(0)).abs() <= 2.0 ** -8 * grad.abs().sum(0) + 1e-7).all())
    for net, old in ((actor, before[:len(list(actor.parameters()))]), (critic, before[len(list(actor.parameters())):])):
        norm = torch.linalg.vector_norm(torch.cat([p.grad.double().flatten() for p in net.parameters()]))
        clip = min(1.0, 1.0 / (float(norm) + 1e-6))
        for p, q in zip(net.parameters(), old):
            zero = torch.zeros_like(q)
            want, _, _ = adamw64(q, p.grad.double(), zero, zero, 1, 3e-4, 0.9, 0.999, 1e-5, 0.01, clip)
            assert float((p.detach().double() - want).abs().max()) < 1e-7 + 3e-4 * 1e-4
    # Autograd's step on the same networks: gradients alike (its weight gradients are rounded
    # to bf16 on the way).
    eager = PpoStep(*twins, _adamw(*twins), reference=reference, kl_coef=0.3)
    eager.entropy_coef.fill_(0.05)
    eager.step(mb)
    assert bool(((eager.sums - step.sums).abs() <= 1e-2 * step.sums.abs() + 1e-4).all())
    for net, other in zip((actor, critic), twins):
        a, b = (torch.cat([p.grad.flatten() for p in n.parameters()]) for n in (net, other))
        assert float(torch.dot(a, b) / (a.norm() * b.norm())) >= 0.999


@pytest.mark.parametrize("bits", [32, 8])
def test_graphed_step_equals_eager_step(bits):
    """The whole step -- both networks, the reference, the losses, the AdamW step with its
    clipping and random rounding -- captured and replayed: the same parameters and states.
    The scalar head's and the losses' kernels add in a fixed order but for the value loss's
    statistics, so the parameters are equal bit for bit."""
    from cugo_b200.ppo import GraphedPpoStep, NativePpoStep
    runs = []
    for _ in range(2):
        actor, critic, reference = _networks(5)
        opt = _adamw(actor, critic, state_bits=bits)
        runs.append((actor, critic, opt, NativePpoStep(actor, critic, opt, reference=reference, kl_coef=0.1)))
    batches = [_minibatch(2048, 10 + i) for i in range(3)]
    graphed = GraphedPpoStep(runs[1][3], batches[0])
    for i, mb in enumerate(batches):
        for r in runs:  # a schedule that the graph follows
            r[3].entropy_coef.fill_(0.05 - 0.01 * i)
            r[3].kl_coef.fill_(0.1 + 0.05 * i)
        runs[0][3].step(mb)
        graphed(mb)
    torch.cuda.synchronize()
    for a, b in zip(runs[0][2].param_groups, runs[1][2].param_groups):
        for p, q in zip(a["params"], b["params"]):
            assert torch.equal(p, q)
            for k, v in runs[0][2].state[p].items():
                assert torch.equal(v, runs[1][2].state[q][k]), k
            assert int(runs[1][2].state[q]["step"]) == 3
    assert torch.allclose(runs[0][3].sums, runs[1][3].sums, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_trainer_iteration(ext, optimizer):
    """train.iteration with the AdamW step and a reference policy: runs, moves both networks,
    reports the KL to the reference, and reads the weights that the step has written."""
    from cugo_b200.ppo import fused_actor, fused_critic
    from cugo_b200.train import PpoTrainer, RolloutStorage, iteration
    torch.manual_seed(1)
    actor, critic = fused_actor(hidden=256, blocks=2).to(DEV), fused_critic(hidden=256, blocks=2).to(DEV)
    reference = copy.deepcopy(actor)
    before = [p.detach().clone() for n in (actor, critic) for p in n.parameters()]
    trainer = PpoTrainer(actor, critic, minibatch=4096, use_graph=False, optimizer=optimizer,
                         weight_decay=0.01, reference=reference, kl_coef=0.2)
    storage = RolloutStorage(1 << 16, DEV)
    for k in range(2):
        st = iteration(ext, trainer, storage, 2048, 5 + k, epochs=1, target_kl=0.0)["stats"]
        for v in (st.policy_loss, st.value_loss, st.entropy, st.kl, st.clipfrac, st.ref_kl):
            assert v == v and abs(v) < 1e6
    assert st.ref_kl > 0.0  # the second iteration starts away from the reference
    after = [p for n in (actor, critic) for p in n.parameters()]
    assert all(not torch.equal(a, b) for a, b in zip(before, after) if a.numel() > 1)
    x = torch.rand((64, 720), device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        got = actor(x)
        fresh = fused_actor(hidden=256, blocks=2).to(DEV)
        fresh.load_state_dict(actor.state_dict())
        assert torch.equal(got, fresh(x))


def test_trainer_refuses_what_it_does_not_know():
    from cugo_b200.ppo import fused_actor, fused_critic
    from cugo_b200.train import PpoTrainer
    nets = fused_actor(hidden=64, blocks=1).to(DEV), fused_critic(hidden=64, blocks=1).to(DEV)
    with pytest.raises(ValueError, match="optimizer"):
        PpoTrainer(*nets, optimizer="sgd")
    with pytest.raises(ValueError, match="weight_decay"):
        PpoTrainer(*nets, weight_decay=0.1)


def test_a_step_on_preferred_lines():
    """A frozen actor scores recorded decisions (action_logp), the actor learns from pairs of
    lines by preference_loss under autograd, AdamW takes the step.  The head's gradient
    against the definition on the same logits: its bias's is the column sums of bf16-rounded
    rows (2^-8 of their sizes, added up)."""
    from cugo_b200.losses import action_logp, preference_loss
    actor, _, reference = _networks(9)
    mb = _minibatch(600, 3)
    lengths = [20, 25, 30, 1, 100, 124, 150, 150]
    offsets = torch.tensor([0] + lengths, device=DEV).cumsum(0)
    with torch.no_grad():
        ref_logp, _ = action_logp(reference(mb.features).float(), mb.actions, mb.legal)
    logits = actor(mb.features)
    out = preference_loss(logits, mb.actions, offsets, ref_logp, legal=mb.legal, beta=0.5, label_smoothing=0.1)
    out.loss.backward()
    grad, loss, margin, _, _ = preference64(logits, mb.actions, offsets, ref_logp, legal=mb.legal, beta=0.5,
                                            smoothing=0.1)
    assert float((out.margin - margin).abs().max()) < 1e-3 and abs(float(out.loss.detach()) - float(loss)) < 1e-3
    bias = actor.out.bias.grad.double()
    assert bool(((bias - grad.sum(0)).abs() <= 2.0 ** -8 * grad.abs().sum(0) + 1e-6).all())
    from cugo_b200.optim import AdamW
    opt = AdamW(actor.parameters(), lr=1e-4, max_grad_norm=1.0)
    before = [p.detach().clone() for p in actor.parameters()]
    opt.step()
    assert all(not torch.equal(a, b) for a, b in zip(before, actor.parameters()))
