"""GPU: update steps as captured graphs -- what their replays read, and what eager calls
beside them see of what a replay has written."""
from __future__ import annotations

import pytest
import torch

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
