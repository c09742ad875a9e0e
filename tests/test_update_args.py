"""CPU: the host-side argument checks of the policy losses and of the AdamW step.  Every
call here returns before any CUDA call: fake, never dereferenced device pointers."""
from __future__ import annotations

import ctypes

import pytest
import torch

from cugo_b200 import load_library

OK, ARG, ALIGN, CAPACITY = 0, -1, -2, -4
P = 0x10000


@pytest.fixture(scope="module")
def lib():
    return load_library()


def _logp(lib, logits=P, ld=180, dtype=0, legal=None, ldm=0, actions=P, weight=None, rows=8, vocab=179,
          logp=P, entropy=P, lse=P, zeros=None):
    return lib.cugo_b200_action_logp(logits, ld, dtype, legal, ldm, actions, weight, rows, vocab, logp,
                                     entropy, lse, zeros, None)


def test_action_logp_arguments(lib):
    assert _logp(lib, rows=0, logits=None, actions=None) == OK
    assert _logp(lib, rows=-1) == ARG
    assert _logp(lib, vocab=0) == ARG
    assert _logp(lib, vocab=1 << 31) == ARG
    assert _logp(lib, vocab=(1 << 30) + 1, ld=1 << 31) == ARG
    assert _logp(lib, dtype=3) == ARG
    assert _logp(lib, logits=None) == ARG
    assert _logp(lib, actions=None) == ARG
    assert _logp(lib, ld=178) == ARG
    assert _logp(lib, legal=P, ldm=100) == ARG
    assert _logp(lib, logp=None, entropy=None, lse=None) == ARG
    assert _logp(lib, logits=P + 2) == ALIGN
    assert _logp(lib, logits=P + 1, dtype=1) == ALIGN
    assert _logp(lib, lse=P + 4) == ALIGN


def _back(lib, lse=P, entropy=P, d_entropy=P, dlogits=P, ldd=180, dtype=0, rows=8, vocab=179):
    return lib.cugo_b200_action_logp_backward(P, 180, 0, None, 0, P, lse, entropy, P, d_entropy, None, rows,
                                              vocab, dlogits, ldd, dtype, None)


def test_action_logp_backward_arguments(lib):
    assert _back(lib, rows=0) == OK
    assert _back(lib, lse=None) == ARG
    assert _back(lib, entropy=None) == ARG
    assert _back(lib, dlogits=None) == ARG
    assert _back(lib, ldd=178) == ARG
    assert _back(lib, dtype=-1) == ARG
    assert _back(lib, dlogits=P + 2) == ALIGN
    assert _back(lib, rows=1 << 40) == CAPACITY


def _policy(lib, rows=8, ref=None, ref_logp=None, low=0.2, high=0.2, dlogits=P, ldd=184, width=184, gdt=1,
            stats=P, loss=None, scratch=P, nbytes=None, logp_old=P, adv=P, vocab=179):
    need = lib.cugo_b200_policy_loss_scratch_bytes(rows) if nbytes is None else nbytes
    return lib.cugo_b200_policy_loss(P, 180, 0, ref, 180, None, 0, P, logp_old, adv, None, ref_logp, rows, vocab,
                                     low, high, 0.0, 0.0, None, None, 0.0, None, 1.0, None, dlogits, ldd, gdt, width, P,
                                     stats, loss, scratch, need, None)


def test_policy_loss_arguments(lib):
    q = lib.cugo_b200_policy_loss_scratch_bytes
    assert q(0) == 0 and q(-3) == 0 and 0 < q(1) <= q(100) <= q(1 << 40)
    assert q(1 << 40) < 1 << 20  # however many rows
    assert _policy(lib, rows=-1) == ARG
    assert _policy(lib, ref=P, ref_logp=P) == ARG
    assert _policy(lib, low=-0.1) == ARG
    assert _policy(lib, high=float("nan")) == ARG
    assert _policy(lib, stats=None, dlogits=None) == ARG
    assert _policy(lib, stats=None, loss=P) == ARG
    assert _policy(lib, logp_old=None) == ARG
    assert _policy(lib, adv=None) == ARG
    assert _policy(lib, width=178) == ARG
    assert _policy(lib, width=(1 << 30) + 1, ldd=1 << 31) == ARG
    assert _policy(lib, ldd=180, width=184) == ARG
    assert _policy(lib, gdt=5) == ARG
    assert _policy(lib, dlogits=P + 1) == ALIGN
    assert _policy(lib, scratch=P + 4) == ALIGN
    assert _policy(lib, scratch=None) == CAPACITY
    assert _policy(lib, nbytes=q(8) - 1) == CAPACITY


def _pairs(lib, pairs=4, rows=8, logp=P, offsets=P, margin=P, loss=P, smoothing=0.0, scratch=P, nbytes=None, lse=P):
    need = lib.cugo_b200_preference_pairs_scratch_bytes(pairs) if nbytes is None else nbytes
    return lib.cugo_b200_preference_pairs(logp, P, None, lse, offsets, pairs, rows, 0.1, smoothing, 0, margin, P,
                                          None, loss, P, scratch, need, None)


def test_preference_pairs_arguments(lib):
    assert lib.cugo_b200_preference_pairs_scratch_bytes(0) == 0
    assert _pairs(lib, pairs=-1) == ARG
    assert _pairs(lib, rows=-1) == ARG
    assert _pairs(lib, logp=None) == ARG
    assert _pairs(lib, offsets=None) == ARG
    assert _pairs(lib, margin=None) == ARG
    assert _pairs(lib, loss=None) == ARG
    assert _pairs(lib, smoothing=1.5) == ARG
    assert _pairs(lib, smoothing=float("nan")) == ARG
    assert _pairs(lib, lse=P + 4) == ALIGN
    assert _pairs(lib, nbytes=0) == CAPACITY


def _adamw(lib, sizes=(10, 0, 300), params=None, grads=None, m=None, ms=None, bits=32, pdt=0, gdt=0, lr=1e-3,
           b1=0.9, b2=0.99, eps=1e-8, decay=0.0, norm=None, max_norm=0.0, step=P, scratch=P, nbytes=None,
           count=None):
    n = len(sizes)
    vp = ctypes.c_void_p

    def arr(values):
        return (vp * n)(*(values or [P] * n))

    count = n if count is None else count
    need = lib.cugo_b200_adamw_scratch_bytes(max(count, 0)) if nbytes is None else nbytes
    scales = (arr(ms), arr(None)) if bits == 8 else (None, None)
    return lib.cugo_b200_adamw(count, arr(params), arr(grads), arr(m), arr(None), *scales,
                               (ctypes.c_int64 * n)(*sizes), pdt, gdt, bits, lr, None, b1, b2, eps, decay, max_norm,
                               0, step, norm, scratch, need, None)


def test_adamw_arguments(lib):
    q = lib.cugo_b200_adamw_scratch_bytes
    assert 0 < q(0) <= q(40) <= q(41) <= q(10000)
    assert _adamw(lib, count=-1) == ARG
    assert _adamw(lib, pdt=2) == ARG
    assert _adamw(lib, gdt=-1) == ARG
    assert _adamw(lib, bits=16) == ARG
    assert _adamw(lib, step=None) == ARG
    assert _adamw(lib, b1=1.0) == ARG
    assert _adamw(lib, b2=float("nan")) == ARG
    assert _adamw(lib, eps=-1.0) == ARG
    assert _adamw(lib, decay=-1.0) == ARG
    assert _adamw(lib, lr=float("nan")) == ARG
    assert _adamw(lib, norm=P, max_norm=-1.0) == ARG
    assert _adamw(lib, sizes=(10, -1)) == ARG
    assert _adamw(lib, sizes=(10, 5), params=[P, None]) == ARG
    assert _adamw(lib, sizes=(10, 5), grads=[None, P]) == ARG
    assert _adamw(lib, sizes=(10, 5), bits=8, ms=[P, None]) == ARG
    assert _adamw(lib, params=[P + 2, P, P]) == ALIGN
    assert _adamw(lib, m=[P, P, P + 1]) == ALIGN
    assert _adamw(lib, scratch=P + 4) == ALIGN
    assert _adamw(lib, scratch=None) == CAPACITY
    assert _adamw(lib, nbytes=q(3) - 1) == CAPACITY


def test_tensors_off_the_gpu_are_refused():
    from cugo_b200 import losses, optim
    x, i, f = torch.zeros((4, 9)), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    for call in (lambda: losses.action_logp(x, i), lambda: losses.policy_loss(x, i, f, f),
                 lambda: losses.policy_loss_grad(x, i, f, f), lambda: losses.preference_loss(x, i, i[:1], f),
                 lambda: losses.action_logp(x.clone().requires_grad_(), i)):
        with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="step must be one int64 value on a CUDA device"):
        optim.adamw_step([f], [f], [f], [f], i[:1])


def test_optimizer_groups_are_checked():
    from cugo_b200.optim import AdamW
    p = torch.nn.Parameter
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([p(torch.zeros(3)), p(torch.zeros(3, dtype=torch.bfloat16))])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([p(torch.zeros(3, dtype=torch.float16))])
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([p(torch.zeros(3))], state_bits=4)
    opt = AdamW([{"params": [p(torch.zeros(3))], "max_grad_norm": 1.0}, {"params": [p(torch.zeros(2))]}])
    assert not opt.clips
    opt.step()  # no gradients, nothing to do
