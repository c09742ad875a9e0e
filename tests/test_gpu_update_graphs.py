"""GPU: update steps as captured graphs -- what their replays read, and what eager calls
beside them see of what a replay has written."""
from __future__ import annotations

import copy

import pytest
import torch

from tests.test_gpu_ppo import _minibatch, _twins
from tests.test_gpu_update_step import _adamw, _networks

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("optimizer", ["adam", "adamw", "adamw8"])
def test_networks_read_the_weights_of_the_latest_replay(ext, optimizer):
    """After each of three iterations of graphed updates both networks' inference and
    training forwards give the bits of fresh networks with the same parameters."""
    from cugo_b200.ppo import fused_actor, fused_critic, train_forward
    from cugo_b200.train import PpoTrainer, RolloutStorage, iteration
    torch.manual_seed(1)
    actor, critic = fused_actor(hidden=256, blocks=2).to(DEV), fused_critic(hidden=256, blocks=2).to(DEV)
    trainer = PpoTrainer(actor, critic, minibatch=4096, optimizer=optimizer)
    storage = RolloutStorage(1 << 16, DEV)
    x = torch.rand((64, 776), device=DEV).to(torch.bfloat16)
    for k in range(3):
        assert iteration(ext, trainer, storage, 2048, 5 + k, epochs=1, target_kl=0.0)["stats"].updates >= 1
        for net, make, width in ((actor, fused_actor, 720), (critic, fused_critic, 770)):
            fresh = make(hidden=256, blocks=2).to(DEV)
            fresh.load_state_dict(net.state_dict())
            with torch.no_grad():
                assert torch.equal(net(x[:, :width]), fresh(x[:, :width])), (k, width)
            assert torch.equal(train_forward(net, x[:, :width])[0], train_forward(fresh, x[:, :width])[0]), (k, width)


def _pair_of_steps(seed=5, native=True):
    """An eager step and a graphed one of equal networks, each with a reference of its own."""
    from cugo_b200.ppo import NativePpoStep, PpoStep
    steps = []
    for _ in range(2):
        actor, critic, reference = _networks(seed)
        make = NativePpoStep if native else PpoStep
        steps.append(make(actor, critic, _adamw(actor, critic), reference=reference, kl_coef=0.3))
    return steps


def _assert_equal_steps(eager, graphed):
    torch.cuda.synchronize()
    for a, b in zip(eager.groups, graphed.groups):
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    assert torch.allclose(eager.sums, graphed.sums, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("native", [True, False])
def test_a_reference_that_changes_between_replays(native):
    """The reference takes other weights in place, is called eagerly, other memory is written:
    the graphed step goes on as the eager one does."""
    from cugo_b200.ppo import GraphedPpoStep
    eager, step = _pair_of_steps(native=native)
    batches = [_minibatch(2048, 10 + i) for i in range(4)]
    graphed = GraphedPpoStep(step, batches[0])
    for i, mb in enumerate(batches):
        if i in (1, 3):
            state = _twins(720, 179, seed=60 + i)[0].state_dict()
            for s in (eager, step):
                s.reference.load_state_dict(state)
            with torch.no_grad():
                step.reference(mb.features)
            junk = [torch.full((k, 720), float("nan"), dtype=torch.bfloat16, device=DEV) for k in (179, 512, 720, 512)]
        eager.step(mb)
        graphed(mb)
        _assert_equal_steps(eager, step)
    del junk


def test_another_reference_between_replays():
    """Another network in the reference's place, and other tensors in its parameters'."""
    from cugo_b200.ppo import GraphedPpoStep
    eager, step = _pair_of_steps(6)
    batches = [_minibatch(2048, 30 + i) for i in range(3)]
    graphed = GraphedPpoStep(step, batches[0])
    for i, mb in enumerate(batches):
        if i == 1:
            for s in (eager, step):
                s.reference = _twins(720, 179, seed=70)[0]
        if i == 2:
            state = _twins(720, 179, seed=71)[0].state_dict()
            for s in (eager, step):
                s.reference.load_state_dict({k: v.clone() for k, v in state.items()}, assign=True)
        eager.step(mb)
        graphed(mb)
        _assert_equal_steps(eager, step)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_loaded_optimizer_between_replays(bits):
    """States that are loaded between two replays are the ones that the next one goes on with."""
    from cugo_b200.ppo import GraphedPpoStep, NativePpoStep
    steps = []
    for _ in range(2):
        actor, critic, _ = _networks(9)
        steps.append(NativePpoStep(actor, critic, _adamw(actor, critic, state_bits=bits)))
    eager, step = steps
    batches = [_minibatch(2048, 40 + i) for i in range(3)]
    graphed = GraphedPpoStep(step, batches[0])
    saved = None
    for i, mb in enumerate(batches):
        if i == 2:
            for s in steps:
                s.optimizer.load_state_dict(saved)
        eager.step(mb)
        graphed(mb)
        if i == 0:
            torch.cuda.synchronize()
            saved = copy.deepcopy(eager.optimizer.state_dict())
        _assert_equal_steps(eager, step)
    assert all(int(s["step"]) == 2 for s in step.optimizer.state.values())


def test_a_capture_leaves_the_step_count_of_parameters_with_states():
    """The warm-up before a capture is undone also where only some of a group's parameters
    had states: the count that they share stays."""
    from cugo_b200.ppo import GraphedPpoStep, NativePpoStep
    actor, critic, _ = _networks(8)
    opt = _adamw(actor, critic)
    mb = _minibatch(2048, 50)
    step = NativePpoStep(actor, critic, opt)
    step.step(mb)
    last = list(actor.parameters())[-1]
    del opt.state[last]
    before = [p.detach().clone() for p in actor.parameters()]
    graphed = GraphedPpoStep(step, mb)
    graphed(mb)
    assert int(opt.state[next(actor.parameters())]["step"]) == 2 and int(opt.state[last]["step"]) == 2
    assert any(not torch.equal(p, q) for p, q in zip(actor.parameters(), before))


def test_a_capture_after_a_look_at_the_states():
    """The empty entries that a look leaves in the optimizer's states are no states."""
    from cugo_b200.ppo import GraphedPpoStep, NativePpoStep
    actor, critic, _ = _networks(8)
    opt = _adamw(actor, critic)
    assert all(opt.state[p] == {} for p in actor.parameters())
    mb = _minibatch(2048, 50)
    GraphedPpoStep(NativePpoStep(actor, critic, opt), mb)(mb)
    assert all(int(opt.state[p]["step"]) == 1 for n in (actor, critic) for p in n.parameters())


def test_a_first_step_is_not_captured():
    """Refused, and nothing is left behind: a step, then the capture, go on from there."""
    from cugo_b200.optim import AdamW
    p, q = (torch.nn.Parameter(torch.ones(500, device=DEV)) for _ in range(2))
    opts = [AdamW([x], lr=0.1) for x in (p, q)]
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(graph):
            opts[0].step()
    for opt in opts:
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for _ in range(2):
        graph.replay()
        opts[1].step()
    torch.cuda.synchronize()
    assert torch.equal(p, q) and int(opts[0].state[p]["step"]) == 3


def test_a_reference_that_is_an_inference_policy():
    """A ResidualMlpPolicy as the reference: its weights and biases may change in place between
    replays too, and be replaced."""
    from cugo_b200.policy import ResidualMlpPolicy
    from cugo_b200.ppo import GraphedPpoStep
    eager, step = _pair_of_steps(11)
    for s in (eager, step):
        s.reference = ResidualMlpPolicy.from_state_dict(_twins(720, 179, seed=80)[0].state_dict(), 3, device=DEV)
    batches = [_minibatch(2048, 60 + i) for i in range(4)]
    graphed = GraphedPpoStep(step, batches[0])
    for i, mb in enumerate(batches):
        for s in (eager, step) if i == 1 else ():
            for t in (*s.reference.weights, *s.reference.biases):
                t.mul_(1.5)
        if i == 2:
            with torch.no_grad():
                step.reference(mb.features)
            for s in (eager, step):
                s.reference.biases = [b * 0.5 for b in s.reference.biases]
        eager.step(mb)
        graphed(mb)
        _assert_equal_steps(eager, step)


def test_options_that_change_between_replays():
    """A learning rate given as a number, the clip of the ratios, a decay: the next replay goes
    by the new ones."""
    from cugo_b200.ppo import GraphedPpoStep
    eager, step = _pair_of_steps(12)
    batches = [_minibatch(2048, 70 + i) for i in range(4)]
    graphed = GraphedPpoStep(step, batches[0])
    for i, mb in enumerate(batches):
        for s in (eager, step):
            for g in s.optimizer.param_groups if i in (1, 3) else ():
                g["lr"], g["weight_decay"] = 1e-3 / i, 0.1 * i
            if i == 2:
                s.clip, s.value_coef = 0.05, 2.0
        eager.step(mb)
        graphed(mb)
        _assert_equal_steps(eager, step)
