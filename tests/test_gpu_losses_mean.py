"""GPU: the mean of log p's error.  Sums of log p over long sequences add up what is alike in
every row; each row's own error is bounded in test_gpu_losses.py."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(262144, 179), (65536, 1000), (65536, 2500), (16384, 16384)])
def test_the_mean_error_of_log_p(rows, vocab, dtype):
    """The hardware's 2^y is 3.0e-8 of itself too small in the mean, which log p corrects: the
    mean error stays below that number (without the correction it would be about it, with the
    wrong sign twice it), give or take four standard errors of the rows' mean."""
    from cugo_b200.losses import action_logp
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = (torch.randn((rows, vocab), device=DEV, generator=g) * 2).to(dtype)
    actions = torch.randint(vocab, (rows,), device=DEV, generator=g)
    got, _ = action_logp(x, actions)
    step = (1 << 26) // vocab
    want = torch.cat([torch.log_softmax(x[i:i + step].double(), 1).gather(1, actions[i:i + step, None])[:, 0]
                      for i in range(0, rows, step)])
    off = got.double() - want
    assert abs(float(off.mean())) < 3.0e-8 + 4 * float(off.std()) / rows ** 0.5
