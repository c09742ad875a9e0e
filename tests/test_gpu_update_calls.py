"""GPU: how the policy update's calls get along with what goes on around them."""
from __future__ import annotations

import ctypes
import subprocess

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


def test_threads_with_rows_of_two_lengths(ext, tmp_path):
    """C callers on four threads whose rows take two amounts of shared memory of the same
    kernel: every call runs."""
    from cugo_b200 import load_library
    from cugo_b200.build import ROOT
    helper = tmp_path / "loss_threads.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-pthread",
                    str(ROOT / "tests" / "native" / "loss_threads.cpp"), "-o", str(helper)], check=True)
    lib, run = load_library(), ctypes.CDLL(str(helper)).loss_threads
    run.restype = ctypes.c_int64
    rows, vocabs = 160, (22000, 36000, 22000, 36000)
    need = lib.cugo_b200_policy_loss_scratch_bytes(rows)
    x, d = ([torch.zeros((rows, v), dtype=torch.bfloat16, device=DEV) for v in vocabs] for _ in range(2))
    scratch = [torch.zeros(need, dtype=torch.uint8, device=DEV) for _ in vocabs]
    actions, zeros = torch.zeros(rows, dtype=torch.int64, device=DEV), torch.zeros(rows, device=DEV)
    streams = [torch.cuda.Stream() for _ in vocabs]

    def pointers(values):
        return (ctypes.c_void_p * len(vocabs))(*values)

    torch.cuda.synchronize()
    failed = run(ctypes.cast(lib.cugo_b200_policy_loss, ctypes.c_void_p), len(vocabs), 5000, ctypes.c_int64(rows),
                 (ctypes.c_int64 * len(vocabs))(*vocabs), pointers(t.data_ptr() for t in x),
                 pointers(t.data_ptr() for t in d), pointers(t.data_ptr() for t in scratch), ctypes.c_int64(need),
                 pointers(s.cuda_stream for s in streams), ctypes.c_void_p(actions.data_ptr()),
                 ctypes.c_void_p(zeros.data_ptr()))
    torch.cuda.synchronize()
    assert failed == 0


@pytest.mark.parametrize("vocab", [179, 40000])
def test_a_launch_that_failed_is_not_reported_twice(ext, vocab):
    """A launch into a stream whose capture has been invalidated is refused on the host; the
    next call, on a good stream, knows nothing of it."""
    from cugo_b200 import load_library
    lib = load_library()
    cu = ctypes.CDLL("libcuda.so.1")
    rows = 300
    x = torch.zeros((rows, vocab), device=DEV)
    actions = torch.zeros(rows, dtype=torch.int64, device=DEV)
    out = torch.zeros(rows, device=DEV)
    lse, d = torch.zeros((rows, 2), device=DEV), torch.zeros((rows, vocab), device=DEV)
    torch.cuda.synchronize()

    def forward(stream):
        return lib.cugo_b200_action_logp(x.data_ptr(), vocab, 0, None, 0, actions.data_ptr(), None, rows, vocab,
                                         out.data_ptr(), None, lse.data_ptr(), None, stream)

    def backward(stream):
        return lib.cugo_b200_action_logp_backward(x.data_ptr(), vocab, 0, None, 0, actions.data_ptr(), lse.data_ptr(),
                                                  None, out.data_ptr(), None, None, rows, vocab, d.data_ptr(), vocab,
                                                  0, stream)

    stream = torch.cuda.Stream()
    handle = ctypes.c_void_p(stream.cuda_stream)
    good = torch.cuda.current_stream().cuda_stream
    assert forward(good) == 0
    assert cu.cuStreamBeginCapture_v2(handle, 2) == 0  # relaxed
    assert cu.cuStreamSynchronize(handle) != 0         # not allowed here: the capture is void
    assert forward(stream.cuda_stream) == -3
    graph = ctypes.c_void_p()
    assert cu.cuStreamEndCapture(handle, ctypes.byref(graph)) != 0
    assert backward(good) == 0
    torch.cuda.synchronize()
