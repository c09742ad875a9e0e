"""GPU: the AdamW step (cugo_b200.optim) against its definition in 64 bits
(update_reference.py).

Tolerances.  u = 2^-24.  m and v take three roundings of fp32 each (3 u of their terms);
the update lr m / (sqrt(v) + eps) one approximate root and quotient (2^-21 together, with
what m and v carry); p three more roundings.  The clip's factor c is off by 4 u."""
from __future__ import annotations

import copy
import math

import pytest
import torch

from tests.update_reference import adamw64, block_scale, decode, e4m3_step, random_bits

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
SIZES = [[1], [255, 256, 257], [2047, 2048, 2049, 0, 5], [720 * 64, 64, 64 * 64, 64, 179 * 64, 179]]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)


def tensors(sizes, p_type, g_type, bits, seed=0, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def new(n, std, dtype):
        flat = torch.randn(n + offset, device=DEV, generator=g) * std
        return flat.to(dtype)[offset:]

    t = {"p": [new(n, 0.1, p_type) for n in sizes], "g": [new(n, 1e-2, g_type) for n in sizes],
         "step": torch.full((1,), 4, dtype=torch.int64, device=DEV)}
    if bits == 32:
        t["m"] = [new(n, 1e-2, torch.float32) for n in sizes]
        t["v"] = [new(n, 1e-2, torch.float32).square() for n in sizes]
        return t
    for name in ("m", "v"):
        t[name] = [torch.zeros(n + offset, dtype=torch.uint8, device=DEV)[offset:] for n in sizes]
        t[name + "s"] = [torch.zeros(-(-n // 256), dtype=torch.uint8, device=DEV) for n in sizes]
    return t


def step(t, clip=None, seed=11, **over):
    from cugo_b200.optim import adamw_step
    return adamw_step(t["p"], t["g"], t["m"], t["v"], t["step"], max_grad_norm=clip, seed=seed,
                      exp_avg_scales=t.get("ms"), exp_avg_sq_scales=t.get("vs"), **{**HYPER, **over})


def before(t):
    """The tensors' values in 64 bits, one flat tensor per list entry."""
    def value(name, k):
        if name + "s" in t:
            return decode(t[name][k], t[name + "s"][k])
        return t[name][k].double()
    n = len(t["p"])
    return [(t["p"][k].double(), t["g"][k].double(), value("m", k), value("v", k)) for k in range(n)]


def near(got, want, tol, name):
    off = (got.double() - want).abs() - tol
    assert not off.numel() or float(off.max()) <= 0.0, (name, float(off.max()))


def expected(t, clip, **over):
    h = {**HYPER, **over}
    old = before(t)
    norm = math.sqrt(sum(float(g.square().sum()) for _, g, _, _ in old))
    c = 1.0 if clip is None else min(1.0, clip / (norm + 1e-6))
    new = [adamw64(p, g, m, v, int(t["step"]) + 1, h["lr"], *h["betas"], h["eps"], h["weight_decay"], c)
           for p, g, m, v in old]
    return old, new, norm, c


def p_tolerance(old, new, h):
    p0, _, _, _ = old
    p1 = new[0]
    return 4 * U * (p0.abs() + p1.abs()) + 2.0 ** -19 * (p1 - p0 * (1 - h["lr"] * h["weight_decay"])).abs() + 1e-12


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("g_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip,offset", [(None, 0), (0.05, 0), (100.0, 3)])
def test_32_bit_states(sizes, g_type, clip, offset):
    t = tensors(sizes, torch.float32, g_type, 32, 1, offset)
    old, new, norm, c = expected(t, clip)
    version = t["p"][0]._version
    got = step(t, clip)
    assert int(t["step"]) == 5 and t["p"][0]._version > version
    assert (got is None) == (clip is None)
    if clip is not None:
        assert abs(float(got) - norm) <= 4 * U * norm
    for k in range(len(sizes)):
        g = (old[k][1] * c).abs()
        near(t["m"][k], new[k][1], 6 * U * (old[k][2].abs() + g), "m")
        near(t["v"][k], new[k][2], 12 * U * (old[k][3] + g * g), "v")
        near(t["p"][k], new[k][0], p_tolerance(old[k], new[k], HYPER), "p")


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("p_type,g_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                           (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("clip,offset", [(None, 0), (0.05, 1)])
def test_8_bit_states(sizes, p_type, g_type, clip, offset):
    """Codes are one of the two grid points around the value, the one that the random bits
    say; scales are the definition's; the step itself knows no rounding of states."""
    t = tensors(sizes, p_type, g_type, 8, 2, offset)
    for round_ in range(3):  # from zero states on
        old, new, _, _ = expected(t, clip)
        step(t, clip)
        number, now = 0, int(t["step"])
        for k, n in enumerate(sizes):
            r = random_bits(number, n, now, 11, DEV)
            number += -(-n // 256)
            if n == 0:
                continue
            for name, want, bits in (("m", new[k][1], r & 0xFFFF), ("v", new[k][2], r >> 16)):
                scale = block_scale(want)
                stored = torch.exp2(t[name + "s"][k].double() - 127)
                # A largest value within rounding of 448 may take either scale.
                top = torch.zeros(scale.numel() * 256, dtype=torch.float64, device=DEV)
                top[:n] = want.abs()
                edge = (top.view(-1, 256).amax(1) / scale - 448).abs() < 448 * 8 * U
                edge |= (top.view(-1, 256).amax(1) / scale - 224).abs() < 224 * 8 * U
                assert bool(((stored == scale) | edge).all()), name
                unit = stored.repeat_interleave(256)[:n]
                x, got = want / unit, decode(t[name][k], t[name + "s"][k]) / unit
                grid = e4m3_step(x)
                assert float(((got - x).abs() / grid).max()) <= 1.0 + 1e-4, name
                # Rounded up exactly where the bits say (off the border of one in 2^16).
                low = torch.floor(x.abs() / grid) * grid
                share = (x.abs() - low) / grid
                up = share + (bits.double() + 0.5) / 65536 >= 1.0
                clear = (share + (bits.double() + 0.5) / 65536 - 1.0).abs() > 1e-3
                want_code = torch.copysign(low + up * grid, x)
                if name == "v":
                    want_code = torch.where((x > 0) & (want_code == 0), 2.0 ** -9, want_code)
                    assert bool(((got > 0) | (want == 0)).all())
                assert torch.equal(got[clear], want_code[clear]), name
            if p_type == torch.float32:
                near(t["p"][k], new[k][0], p_tolerance(old[k], new[k], HYPER), "p")
            else:
                step_ = torch.exp2(torch.floor(torch.log2(new[k][0].abs().clamp_min(1e-30))) - 7)
                near(t["p"][k], new[k][0], step_ * (1 + 1e-3), "p")


def test_rounding_is_right_in_the_mean():
    """bf16 parameters and both 8-bit states: over many elements the roundings cancel.  A
    rounding by 16 random bits of a value that lies at the share f of a step has the
    variance f (1 - f) <= 1/4 steps^2: the mean of n of them stays within 5 / (2 sqrt n)."""
    n = 1 << 20
    t = tensors([n], torch.bfloat16, torch.float32, 8, 5)
    old, new, _, _ = expected(t, None)
    step(t)
    p_step = torch.exp2(torch.floor(torch.log2(new[0][0].abs())) - 7)
    assert abs(float(((t["p"][0].double() - new[0][0]) / p_step).mean())) < 2.5 / math.sqrt(n)
    for name, want in (("m", new[0][1]), ("v", new[0][2])):
        unit = torch.exp2(t[name + "s"][0].double() - 127).repeat_interleave(256)
        off = (decode(t[name][0], t[name + "s"][0]) - want) / unit / e4m3_step(want / unit)
        if name == "v":  # the smallest are kept above 0 on purpose
            off = off[want / unit > 2.0 ** -8]
        assert abs(float(off.mean())) < 2.5 / math.sqrt(off.numel())


def test_a_still_second_moment_keeps_its_mean():
    """1,000 steps with the same gradient: v's mean follows the definition although every
    step moves it by far less than a code (rounding to nearest would leave it)."""
    n = 4096
    t = tensors([n], torch.float32, torch.float32, 8, 6)
    t["step"].zero_()
    t["g"][0].copy_(torch.where(torch.rand(n, device=DEV) < 0.5, 0.01, -0.01) * (0.5 + torch.rand(n, device=DEV)))
    g2 = t["g"][0].double().square()
    for _ in range(1000):
        step(t, betas=(0.9, 0.999), lr=0.0)
    want = g2 * (1 - 0.999 ** 1000)
    got = decode(t["v"][0], t["vs"][0])
    # Of a value the noise is about 0.2 of itself (sqrt(f) steps of 1/8 to 1/16, f the share
    # of a step it moves, over the 1,000 steps that the mean spans); of the mean of 4,096
    # values a 64th of that.
    assert abs(float((got / want).mean()) - 1.0) < 5 * 0.3 / 64
    assert float((decode(t["m"][0], t["ms"][0]) / t["g"][0].double() - 1).abs().mean()) < 0.2


def test_many_tensors_take_several_launches():
    """More tensors than a launch holds: as one call per tensor would, with the norm of all."""
    sizes = [1 + (37 * k) % 700 for k in range(1000)]
    t = tensors(sizes, torch.float32, torch.float32, 32, 7)
    old, new, norm, c = expected(t, 0.5)
    assert abs(float(step(t, 0.5)) - norm) <= 4 * U * norm
    for k in range(0, 1000, 97):
        near(t["p"][k], new[k][0], p_tolerance(old[k], new[k], HYPER), k)
    near(t["p"][999], new[999][0], p_tolerance(old[999], new[999], HYPER), "last")


def test_neighbours_are_left_alone():
    """Nothing outside the tensors is written: parameters and states inside larger buffers."""
    sizes = [3, 257, 1000]
    for bits in (32, 8):
        t = tensors(sizes, torch.float32, torch.float32, bits, 8)
        buffers = []
        for name in ("p", "m", "v") + (("ms", "vs") if bits == 8 else ()):
            for k, x in enumerate(t[name]):
                buf = torch.full((x.numel() + 64,), 77, dtype=x.dtype, device=DEV)
                buf[32:32 + x.numel()] = x
                buffers.append((buf, x.numel()))
                t[name][k] = buf[32:32 + x.numel()]
        step(t, 1.0)
        for buf, n in buffers:
            assert bool((buf[:32] == 77).all()) and bool((buf[32 + n:] == 77).all())


def test_infinite_and_nan_gradients():
    for bits in (32, 8):
        t = tensors([600], torch.float32, torch.float32, bits, 9)
        t["g"][0][5], t["g"][0][300] = float("nan"), float("inf")
        step(t)  # not clipped: those elements alone
        bad = torch.zeros(600, dtype=torch.bool, device=DEV)
        bad[5] = bad[300] = True
        assert torch.equal(~torch.isfinite(t["p"][0]), bad)
        values = before(t)[0]
        assert bool(torch.isfinite(values[2][~bad]).all()) and bool(torch.isfinite(values[3][~bad]).all())
        assert not bool(torch.isfinite(values[2][bad]).any())
        t = tensors([600], torch.float32, torch.float32, bits, 9)
        t["g"][0][5] = float("nan")
        assert bool(torch.isnan(step(t, 1.0))) and bool(torch.isnan(t["p"][0]).all())


def test_no_tensors_no_elements():
    from cugo_b200.optim import adamw_step
    s = torch.zeros(1, dtype=torch.int64, device=DEV)
    assert float(adamw_step([], [], [], [], s, max_grad_norm=1.0)) == 0.0 and int(s) == 1
    e = [torch.empty(0, device=DEV)]
    assert adamw_step(e, e, e, e, s) is None and int(s) == 2


def model(seed=0, dtype=torch.float32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(50, 70), torch.nn.ReLU(), torch.nn.Linear(70, 179)).to(DEV, dtype)


def backward(net, x):
    net.zero_grad()
    net(x).square().mean().backward()


def test_optimizer_follows_torch():
    """AdamW in 32 bits against torch's clip_grad_norm_ and AdamW over 20 steps, a
    learning rate on the device among them.  Each step differs by fp32 rounding: 2^-19 of
    lr per step and element, which the steps add up, and the gradients that differ by it."""
    from cugo_b200.optim import AdamW
    a, b = model(), model()
    lr = torch.tensor(1e-3, device=DEV)
    ours = AdamW([{"params": list(a.parameters())}], lr=lr, weight_decay=0.1, max_grad_norm=0.1)
    theirs = torch.optim.AdamW(b.parameters(), lr=1e-3, weight_decay=0.1)
    x = torch.randn(64, 50, device=DEV)
    for k in range(20):
        backward(a, x)
        backward(b, x)
        norm = torch.nn.utils.clip_grad_norm_(b.parameters(), 0.1)
        ours.step()
        theirs.step()
        assert abs(float(ours.param_groups[0]["grad_norm"]) - float(norm)) < 1e-4 * float(norm)
    for p, q in zip(a.parameters(), b.parameters()):
        assert float((p - q).detach().abs().max()) < 20 * 1e-3 * 1e-2


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_and_graph(bits, dtype):
    """A saved and loaded optimizer, and a captured step, go on bit for bit."""
    from cugo_b200.optim import AdamW
    net = model(1, dtype)
    opt = AdamW(net.parameters(), lr=1e-3, state_bits=bits, max_grad_norm=1.0, seed=5)
    x = torch.randn(32, 50, device=DEV, dtype=dtype)
    for _ in range(3):
        backward(net, x)
        opt.step()
    twin = copy.deepcopy(net)
    other = AdamW(twin.parameters(), lr=1e-3, state_bits=bits, max_grad_norm=1.0, seed=5)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p, q in zip(net.parameters(), twin.parameters()):
        for k, v in opt.state[p].items():
            assert other.state[q][k].dtype == v.dtype and torch.equal(other.state[q][k], v), k
    for p, q in zip(net.parameters(), twin.parameters()):
        q.grad = p.grad.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        other.step()
    for _ in range(4):
        opt.step()
        graph.replay()
    torch.cuda.synchronize()
    assert int(next(iter(opt.state.values()))["step"]) == 7
    for p, q in zip(net.parameters(), twin.parameters()):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            assert torch.equal(other.state[q][k], v), k


def test_parameters_without_gradients_are_left_out():
    from cugo_b200.optim import AdamW
    net = model(2)
    opt = AdamW(net.parameters(), state_bits=8)
    x = torch.randn(8, 50, device=DEV)
    backward(net, x)
    first = next(net.parameters())
    first.grad = None
    kept = first.detach().clone()
    opt.step()
    assert torch.equal(first, kept) and first not in opt.state
    for p in net.parameters():
        p.grad = None
    opt.step()


def test_refusals():
    from cugo_b200.optim import AdamW, adamw_step
    t = tensors([10, 20], torch.float32, torch.float32, 32)
    e = tensors([10, 20], torch.float32, torch.float32, 8)
    s = t["step"]
    bad = [
        (lambda: adamw_step(t["p"], t["g"][:1], t["m"], t["v"], s), "one tensor each"),
        (lambda: adamw_step(t["p"], t["g"][::-1], t["m"], t["v"], s), "wrong sizes"),
        (lambda: adamw_step([x.half() for x in t["p"]], t["g"], t["m"], t["v"], s), "fp32 or bf16"),
        (lambda: adamw_step(t["p"], [x.half() for x in t["g"]], t["m"], t["v"], s), "fp32 or bf16"),
        (lambda: adamw_step(t["p"], t["g"], [x.bfloat16() for x in t["m"]], t["v"], s), "contiguous"),
        (lambda: adamw_step([t["p"][0], t["p"][1].bfloat16()], t["g"], t["m"], t["v"], s), "of one type"),
        (lambda: adamw_step([t["p"][0], t["p"][0]], [t["g"][0]] * 2, [t["m"][0], t["m"][0].clone()],
                            [t["v"][0], t["v"][0].clone()], s), "twice"),
        (lambda: adamw_step(t["p"], t["g"], [x.cpu() for x in t["m"]], t["v"], s), "on cuda"),
        (lambda: adamw_step(t["p"], t["g"], t["m"], t["v"], s.int()), "step"),
        (lambda: adamw_step(e["p"], e["g"], e["m"], e["v"], s, exp_avg_scales=e["ms"]), "both lists"),
        (lambda: adamw_step(e["p"], e["g"], t["m"], e["v"], s, exp_avg_scales=e["ms"],
                            exp_avg_sq_scales=e["vs"]), "contiguous"),
        (lambda: adamw_step(t["p"], t["g"], t["m"], t["v"], s, lr=-1.0), "lr"),
        (lambda: adamw_step(t["p"], t["g"], t["m"], t["v"], s, betas=(0.9, 1.0)), "betas"),
        (lambda: adamw_step(t["p"], t["g"], t["m"], t["v"], s, max_grad_norm=-1.0), "max_grad_norm"),
        (lambda: adamw_step(t["p"], t["g"], t["m"], t["v"], s, lr=torch.tensor(1e-3)), "lr"),
    ]
    for call, words in bad:
        with pytest.raises(RuntimeError, match=words):
            call()
    assert int(s) == 4  # nothing ran
    p = torch.nn.Parameter(torch.zeros(4, 6, device=DEV).t())
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([p])
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([torch.nn.Parameter(torch.zeros(3, device=DEV))], state_bits=16)
