"""GPU: the losses over rows of logits (cugo_b200.losses) against their definitions in 64
bits (update_reference.py).

Tolerances.  u = 2^-24 is half a step of fp32.  A row's sums run over chains of at most
k = 32 (short rows: one lane's entries) or vocab / 128 + 16 additions, after which the
lanes and warps join in 10 steps; the base-2 exponential is off by 2^-22 and by |y| u from
its argument.  So a sum is off by c u relative, c = k + 16 + 4 + Y with Y the largest |y|
that carries weight (below 32 for these logits), log p and the entropy by c u times
(1 + their own size), and an entry's gradient by 2 c u times its terms' sizes, plus half
a step of the type it is stored in."""
from __future__ import annotations

import math

import pytest
import torch

from tests.update_reference import action_logp64, policy64, preference64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# Half a step of a stored value, relative, and of the type's smallest values.
HALF = {torch.float32: (U, 0.0), torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25)}
VOCABS = [1, 2, 31, 33, 179, 180, 1000, 1024, 1025, 4099, 20001]


def chain(vocab):
    return (32 if vocab <= 1024 else vocab // 128 + 16) + 16 + 4 + 32


def make(rows, vocab, dtype, seed=0, legal=False, pad=0, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * rows + vocab)
    x = torch.randn((rows, vocab + pad), device=DEV, generator=g) * std
    x = x.to(dtype)[:, :vocab]
    actions = torch.randint(vocab, (rows,), device=DEV, generator=g)
    mask = None
    if legal:
        mask = torch.rand((rows, vocab), device=DEV, generator=g) < 0.3
        mask.scatter_(1, actions[:, None], True)
    return x, actions, mask, g


def near(got, want, tol, name):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, name
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), name
    off = torch.where(torch.isnan(want), torch.zeros_like(want), (got - want).abs() - tol)
    assert float(off.max() if off.numel() else 0.0) <= 0.0, (name, float(off.max()))


def grad_tol(vocab, p, actions, size, dtype, want):
    """size [rows]: the sizes of a row's gradient terms, added up."""
    hot = torch.zeros_like(p).scatter_(1, actions.clamp(0, vocab - 1)[:, None], 1.0)
    rel, least = HALF[dtype]
    return 2 * chain(vocab) * U * size[:, None] * (p + hot) + rel * want.abs() + least + 1e-37


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows,legal,pad", [(1, False, 0), (5, True, 0), (67, True, 3), (300, False, 8)])
def test_action_logp(vocab, dtype, rows, legal, pad):
    from cugo_b200.losses import action_logp
    x, actions, mask, g = make(rows, vocab, dtype, 1, legal, pad)
    d1 = torch.randn(rows, device=DEV, generator=g)
    d2 = torch.randn(rows, device=DEV, generator=g)
    leaf, logp, entropy, p, used = action_logp64(x, actions, mask)
    want, = torch.autograd.grad((logp * d1).sum() + (entropy * d2).sum(), leaf)
    c = chain(vocab) * U
    y = x.detach().requires_grad_()
    got_logp, got_entropy = action_logp(y, actions, mask)
    near(got_logp.detach(), logp.detach(), c * (1 + logp.detach().abs()), "logp")
    near(got_entropy.detach(), entropy.detach(), c * (1 + 2 * entropy.detach().abs() + math.log(vocab)), "entropy")
    got, = torch.autograd.grad((got_logp, got_entropy), y, (d1, d2))
    size = d1.double().abs() + d2.double().abs() * (1 + 2 * math.log(vocab) + 16)
    near(got, want, grad_tol(vocab, p, actions, size, dtype, want), "gradient")
    with torch.no_grad():  # the forward alone gives the same bits
        again = action_logp(x, actions, mask)
    assert torch.equal(again[0], got_logp) and torch.equal(again[1], got_entropy)


def policy_case(rows, vocab, dtype, legal, pad, kl, weights, seed=3):
    x, actions, mask, g = make(rows, vocab, dtype, seed, legal, pad)
    _, logp, _, _, _ = action_logp64(x, actions, mask)
    shift = 0.3 * torch.randn(rows, device=DEV, generator=g, dtype=torch.float64)
    for border in (math.log(0.8), math.log(1.28)):  # no row where rounding decides the clip
        shift = torch.where((shift - border).abs() < 1e-2, border + 2e-2, shift)
    k = dict(legal=mask, clip_low=0.2, clip_high=0.28, entropy_coef=0.01)
    if kl != "none":
        k["kl_coef"] = 0.1
    if kl == "sampled":
        k["ref_logp"] = (logp.detach() + 0.3 * torch.randn(rows, device=DEV, generator=g)).float()
    if kl == "full":
        k["ref_logits"] = (x.float() + 0.5 * torch.randn((rows, vocab), device=DEV, generator=g)).to(dtype)
    if weights:
        k["weight"] = torch.rand(rows, device=DEV, generator=g) * (torch.rand(rows, device=DEV, generator=g) < 0.7)
        k["weight"][0] = 0.5
    old = (logp.detach() - shift).float()
    adv = torch.randn(rows, device=DEV, generator=g)
    return x, actions, old, adv, k


def policy_tols(vocab, x, actions, k, adv, p, stats_ref, rows):
    c = chain(vocab) * U
    w = torch.ones(rows, device=DEV) if k.get("weight") is None else k["weight"]
    share = w.double() / w.double().sum()
    # A ratio is off by what log p is (log p below 24 here), times e; the means weigh that.
    a = adv.double().abs()
    span = 24 + 2 * math.log(max(vocab, 2))
    worst = c * span * 4 * (share * (2 + a)).sum() + 1e-7
    size = share * 4 * span * (a + 1)
    return worst, size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [2, 179, 180, 1024, 1025, 5001, 20000])
@pytest.mark.parametrize("rows,legal,pad,kl,weights", [
    (1, False, 0, "full", False), (9, True, 1, "sampled", True), (130, True, 5, "full", True),
    (301, False, 8, "none", False)])
def test_policy_loss(vocab, dtype, rows, legal, pad, kl, weights):
    from cugo_b200.losses import policy_loss, policy_loss_grad
    x, actions, old, adv, k = policy_case(rows, vocab, dtype, legal, pad, kl, weights)
    want, stats, logp, p, used = policy64(x, actions, old, adv, **k)
    worst, size = policy_tols(vocab, x, actions, k, adv, p, stats, rows)
    out, d = policy_loss_grad(x, actions, old, adv, **k)
    near(out.stats, stats, worst * (1 + stats.abs()), "stats")
    assert float(out.loss) == float(out.stats[0])
    near(out.logp, logp, chain(vocab) * U * (1 + logp.abs()), "logp")
    near(d, want, grad_tol(vocab, p, actions, size, dtype, want), "one pass")
    y = x.detach().requires_grad_()
    again = policy_loss(y, actions, old, adv, **k)
    if vocab <= 1024:
        assert torch.equal(again.stats, out.stats) and torch.equal(again.logp, out.logp)
    else:
        # Without its gradient a long row goes over other threads, which add in another order:
        # each of the two is within its bound of the definition (above), so they are within
        # twice that of one another.
        near(again.stats, out.stats.double(), 2 * worst * (1 + stats.abs()), "stats of the loss alone")
        near(again.logp, out.logp.double(), 2 * chain(vocab) * U * (1 + logp.abs()), "logp of the loss alone")
    g, = torch.autograd.grad(again.loss * 3.0, y)
    near(g, 3 * want, 3 * grad_tol(vocab, p, actions, size, dtype, want), "autograd")
    # Into a wider buffer of another type, scaled by a device value.
    wide = torch.full((rows, vocab + 5), 7.0, dtype=torch.bfloat16, device=DEV)
    scale = torch.tensor([0.5], device=DEV)
    _, same = policy_loss_grad(x, actions, old, adv, **k, dlogits=wide, grad_scale=scale)
    assert same is wide and not bool(wide[:, vocab:].any())
    near(wide[:, :vocab], 0.5 * want, 0.5 * grad_tol(vocab, p, actions, size, torch.bfloat16, want), "wide")


@pytest.mark.parametrize("vocab", [40, 2000])
def test_gradient_by_differences(vocab):
    """The 64-bit definition's gradient, and with it the kernel's, against differences of
    the kernel's own loss: a step of 2^-4 along the gradient in fp32."""
    from cugo_b200.losses import policy_loss, policy_loss_grad
    x, actions, old, adv, k = policy_case(64, vocab, torch.float32, True, 0, "full", True)
    adv = torch.full_like(adv, 0.5)
    old = old + 5.0  # ratios far below the clip: A > 0, unclipped, smooth
    _, d = policy_loss_grad(x, actions, old, adv, **k)
    along = torch.randn_like(x)
    h = 2.0 ** -6
    up = policy_loss(x + h * along, actions, old, adv, **k).loss.double()
    down = policy_loss(x - h * along, actions, old, adv, **k).loss.double()
    slope = float((d.double() * along.double()).sum())
    # The second-order error is h^2 / 6 times a third derivative of order 1, the
    # subtraction's 2 c u / (2 h).
    assert abs(float(up - down) / (2 * h) - slope) < h * h + 4 * chain(vocab) * U / h


@pytest.mark.parametrize("vocab", [179, 3001])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count(vocab, dtype):
    """Empty masks, actions outside or masked, weights of 0: zeros, whatever the row holds;
    NaN and infinities in masked places are not seen; NaN in a legal place stays in its row."""
    from cugo_b200.losses import action_logp, policy_loss_grad
    rows = 12
    x, actions, mask, g = make(rows, vocab, dtype, 5, True)
    mask = mask.clone()
    low = torch.finfo(dtype).min
    mask[0] = False                                     # nothing legal
    mask[1, actions[1]] = False                         # the action is masked
    actions[2], actions[3] = -1, vocab                  # outside
    actions[4] = 1 << 40
    x = x.clone()
    x[5][~mask[5]] = float("nan")                       # masked places
    x[6][~mask[6]] = float("inf")
    x[7][mask[7]] = -float("inf")                       # every legal entry -inf
    x[8, actions[8]] = -float("inf")                    # the action's own
    other = (actions[9] + 1) % vocab
    mask[9, other] = True
    x[9, other] = -float("inf")                         # one legal entry -inf
    x[10, other] = low                                  # the type's lowest
    mask[10, other] = True
    weight = torch.ones(rows, device=DEV)
    weight[11] = 0.0
    x[11] = float("nan")
    unused = [0, 1, 2, 3, 4, 7, 8, 11]
    old = torch.full((rows,), -2.0, device=DEV)
    adv = torch.ones(rows, device=DEV)
    out, d = policy_loss_grad(x, actions, old, adv, legal=mask, weight=weight, entropy_coef=0.1)
    clean = x.clone()
    clean[~mask] = 0.0
    clean[11] = 0.0
    want, stats, logp, p, used = policy64(clean, actions, old, adv, legal=mask, weight=weight, entropy_coef=0.1)
    assert [i for i in range(rows) if not bool(used[i])] == unused
    assert not bool(d[unused].any()) and not bool(out.logp[unused].any())
    worst, size = policy_tols(vocab, x, actions, {"weight": weight}, adv, p, stats, rows)
    near(out.stats, stats, worst * (1 + stats.abs()), "stats")
    near(d, want, grad_tol(vocab, p, actions, size, dtype, want), "gradient")
    logp1, entropy1 = action_logp(x[:11], actions[:11], mask[:11])
    assert not bool(logp1[unused[:-1]].any()) and not bool(entropy1[unused[:-1]].any())
    # NaN in a legal place: that row, and the means.
    x[9, actions[9]] = float("nan")
    out, d = policy_loss_grad(x, actions, old, adv, legal=mask, weight=weight)
    assert bool(torch.isnan(d[9][mask[9]]).all()) and bool(torch.isnan(out.loss)) and bool(torch.isnan(out.logp[9]))
    keep = [i for i in range(rows) if i != 9]
    assert not bool(torch.isnan(d[keep]).any()) and not bool(torch.isnan(out.logp[keep]).any())


@pytest.mark.parametrize("vocab", [33, 2500])
def test_masks_by_value(vocab):
    """-1e30, -inf and the lowest value mask an entry as `legal` does; -1e9 is far below any
    other entry but an entry: a row of nothing else is uniform."""
    from cugo_b200.losses import action_logp
    x, actions, mask, _ = make(50, vocab, torch.float32, 9, True)
    want = action_logp(x, actions, mask)
    for value in (-1e30, -float("inf"), torch.finfo(torch.float32).min):
        got = action_logp(x.masked_fill(~mask, value), actions)
        # Long rows bring in a new maximum at other places where a mask is read, so each of
        # the two is off by its own rounding: twice the bound of one.
        c = 2 * chain(vocab) * U
        near(got[0], want[0].double(), c * (1 + want[0].double().abs()), "logp")
        near(got[1], want[1].double(), c * (1 + 2 * want[1].double() + math.log(vocab)), "entropy")
    flat = torch.full((3, vocab), -1e9, device=DEV)
    logp, entropy = action_logp(flat, torch.zeros(3, dtype=torch.int64, device=DEV))
    assert float((logp + math.log(vocab)).abs().max()) < 2e-5 and float((entropy - math.log(vocab)).abs().max()) < 2e-5


def test_one_mask_for_all_rows_and_large_logits():
    from cugo_b200.losses import action_logp
    x, actions, _, g = make(40, 200, torch.float32, 2)
    x = x + 3000.0  # the differences count, exact here
    one = torch.rand(200, device=DEV, generator=g) < 0.5
    one[actions] = True
    for mask in (one.expand(40, 200), one.expand(40, 200).contiguous()):
        logp, entropy = action_logp(x, actions, mask)
        _, want, want_h, _, _ = action_logp64(x, actions, mask)
        near(logp, want.detach(), chain(200) * U * (1 + want.detach().abs()), "logp")
        near(entropy, want_h.detach(), chain(200) * U * (8 + 2 * want_h.detach()), "entropy")


@pytest.mark.parametrize("vocab", [179, 4000])
def test_no_rows_and_no_weight(vocab):
    from cugo_b200.losses import action_logp, policy_loss, policy_loss_grad, preference_loss
    x = torch.empty((0, vocab), device=DEV)
    i, f = torch.empty(0, dtype=torch.int64, device=DEV), torch.empty(0, device=DEV)
    assert action_logp(x, i)[0].shape == (0,)
    out, d = policy_loss_grad(x, i, f, f)
    assert float(out.loss) == 0.0 and not bool(out.stats.any()) and d.shape == (0, vocab)
    o = torch.zeros(1, dtype=torch.int64, device=DEV)
    assert float(preference_loss(x, i, o, f).loss) == 0.0
    o = torch.zeros(3, dtype=torch.int64, device=DEV)  # a pair of empty sequences
    out = preference_loss(x, i, o, f)
    assert abs(float(out.loss) - math.log(2)) < 1e-6 and float(out.margin[0]) == 0.0
    # All weights 0: no mean, no gradient, no NaN.
    x, actions, _, _ = make(5, vocab, torch.float32)
    x.requires_grad_()
    z = torch.zeros(5, device=DEV)
    out = policy_loss(x, actions, z, z + 1, weight=z, entropy_coef=0.1)
    d, = torch.autograd.grad(out.loss, x)
    assert float(out.loss.detach()) == 0.0 and not bool(d.any())


def test_denominator_of_a_larger_batch():
    """Two halves with the whole's denominator add up to the whole."""
    from cugo_b200.losses import policy_loss_grad
    x, actions, old, adv, k = policy_case(5000, 30, torch.float32, False, 0, "none", True)
    _, _, _, p, _ = policy64(x, actions, old, adv, **k)
    _, size = policy_tols(30, x, actions, k, adv, p, None, 5000)
    out, d = policy_loss_grad(x, actions, old, adv, **k)
    total = float(k["weight"].double().sum())
    weight = k.pop("weight")
    parts = [policy_loss_grad(x[s], actions[s], old[s], adv[s], weight=weight[s], denominator=total, **k)
             for s in (slice(0, 1700), slice(1700, 5000))]
    near(parts[0][0].stats + parts[1][0].stats, out.stats.double(), 1e-6 * (1 + out.stats.double().abs()), "stats")
    # Where the action's p is near 1 its gradient is the difference of two larger terms, hot
    # and p c_0: each is rounded to u of its own size, not of the result's, and the two
    # runs' scales (1 / D from 64 and from 32 bits) round differently.  So the bound is the
    # one of the terms' sizes.
    near(torch.cat([q[1] for q in parts]), d.double(), grad_tol(30, p, actions, size, torch.float32, d.double()),
         "gradient")


def pairs_case(lengths, vocab, dtype, legal, weights, pad=0):
    rows = sum(lengths)
    x, actions, mask, g = make(rows, vocab, dtype, 4, legal, pad)
    _, logp, _, _, _ = action_logp64(x, actions, mask)
    ref = (logp.detach() + 0.5 * torch.randn(rows, device=DEV, generator=g)).float()
    offsets = torch.tensor([0] + lengths, device=DEV).cumsum(0)
    weight = (torch.rand(rows, device=DEV, generator=g) < 0.6).float() if weights else None
    return x, actions, offsets, ref, dict(legal=mask, weight=weight)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,vocab,legal,weights", [
    ([1, 1], 179, True, False), ([0, 3, 5, 0], 2, False, False), ([7] * 2 + [13] * 10, 179, True, True),
    ([700, 300], 40, False, True), ([3, 1, 4, 1, 5, 9, 2, 6], 2049, True, True),
    ([5] * 1400, 33, False, False), ([40] * 900, 17, False, True)])
@pytest.mark.parametrize("beta,smoothing,average", [(0.1, 0.0, False), (2.0, 0.2, True)])
def test_preference_loss(lengths, vocab, legal, weights, dtype, beta, smoothing, average):
    from cugo_b200.losses import preference_loss
    x, actions, offsets, ref, k = pairs_case(lengths, vocab, dtype, legal, weights)
    want, loss, margin, seq, acc = preference64(x, actions, offsets, ref, beta=beta, smoothing=smoothing,
                                                average=average, **k)
    y = x.detach().requires_grad_()
    out = preference_loss(y, actions, offsets, ref, beta=beta, label_smoothing=smoothing, average=average, **k)
    c, longest = chain(vocab) * U, 1 if average else max(lengths)
    span = 24 + 2 * math.log(max(vocab, 2))
    near(out.logp, seq, c * span * longest + 2 * U * seq.abs(), "sequences")
    m_tol = 2 * beta * c * span * longest + 2 * U * margin.abs()
    near(out.margin, margin, m_tol, "margin")
    near(out.loss, loss, m_tol.max() + 2 * U * loss.abs(), "loss")
    assert abs(float(out.accuracy) - float(acc)) < 1e-6 or float(margin.abs().min()) < float(m_tol.max())
    d, = torch.autograd.grad(out.loss, y, torch.tensor(2.0, device=DEV))
    _, _, _, p, _ = action_logp64(x, actions, k["legal"], k["weight"])
    slope = 2 * beta / (len(lengths) // 2) * torch.ones(len(x), device=DEV, dtype=torch.float64)
    near(d, 2 * want, grad_tol(vocab, p, actions, slope * (1 + float(m_tol.max()) / (2 * chain(vocab) * U)),
                               dtype, 2 * want), "gradient")
    plain = preference_loss(x, actions, offsets, ref, beta=beta, label_smoothing=smoothing, average=average, **k)
    assert torch.equal(plain.loss, out.loss.detach()) and torch.equal(plain.margin, out.margin)


def test_rows_outside_the_sequences():
    """Offsets that leave rows out, and offsets past the rows: no gradient, no access."""
    from cugo_b200.losses import preference_loss
    x, actions, _, _ = make(20, 50, torch.float32)
    ref = torch.zeros(20, device=DEV)
    y = x.detach().requires_grad_()
    o = torch.tensor([3, 8, 15], device=DEV)
    d, = torch.autograd.grad(preference_loss(y, actions, o, ref).loss, y)
    assert not bool(d[:3].any()) and not bool(d[15:].any()) and bool(d[3:15].any(1).all())
    o = torch.tensor([-5, 8, 1 << 40], device=DEV)
    out = preference_loss(x, actions, o, ref)
    same = preference_loss(x, actions, torch.tensor([0, 8, 20], device=DEV), ref)
    assert torch.equal(out.margin, same.margin)


def test_strides_streams_graphs_and_the_same_bits():
    from cugo_b200.losses import action_logp, policy_loss_grad, preference_loss
    x, actions, old, adv, k = policy_case(500, 179, torch.float32, True, 1, "full", True)
    out, d = policy_loss_grad(x, actions, old, adv, **k)
    flat = k | {"ref_logits": k["ref_logits"].contiguous()}
    again, d2 = policy_loss_grad(x.contiguous(), actions, old, adv, **flat)
    assert torch.equal(d, d2) and torch.equal(out.stats, again.stats)
    # Rows of a larger matrix, every other one.
    big = torch.zeros((1000, 200), device=DEV)
    big[::2, 3:182] = x
    sub, d3 = policy_loss_grad(big[::2, 3:182], actions, old, adv, **k)
    # (Rows apart are added up in another order than rows one after another.)
    want, stats, logp, p, _ = policy64(x, actions, old, adv, **k)
    worst, size = policy_tols(179, x, actions, k, adv, p, stats, 500)
    near(d3, want, grad_tol(179, p, actions, size, torch.float32, want), "rows apart")
    near(sub.stats, stats, worst * (1 + stats.abs()), "rows apart")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other, d4 = policy_loss_grad(x, actions, old, adv, **k)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(d, d4) and torch.equal(out.stats, other.stats)
    # A captured step replayed on new inputs; two graphs of the same op share nothing.
    sx, sa = x.clone(), adv.clone()
    offsets = torch.tensor([0, 100, 250, 260, 500], device=DEV)
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = policy_loss_grad(sx, actions, old, sa, **k)
            leaf = sx.detach().requires_grad_()
            pref = preference_loss(leaf, actions, offsets, old, legal=k["legal"])
            dp, = torch.autograd.grad(pref.loss, leaf)
        graphs.append((graph, res, pref, dp))
    x2, adv2 = torch.randn_like(x), torch.randn_like(adv)
    sx.copy_(x2)
    sa.copy_(adv2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st, (graph, _, _, _) in zip(streams, graphs):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            graph.replay()
    torch.cuda.synchronize()
    want, dw = policy_loss_grad(sx, actions, old, adv2, **k)
    leaf = sx.detach().requires_grad_()
    pw = preference_loss(leaf, actions, offsets, old, legal=k["legal"])
    dpw, = torch.autograd.grad(pw.loss, leaf)
    for _, (res, dg), pref, dp in graphs:
        assert torch.equal(res.stats, want.stats) and torch.equal(dg, dw) and torch.equal(res.logp, want.logp)
        assert torch.equal(pref.loss.detach(), pw.loss.detach()) and torch.equal(dp, dpw)
    logp, _ = action_logp(sx, actions, k["legal"])
    assert logp.shape == (500,)


def test_the_loss_can_be_scaled_in_place_and_differentiated_twice():
    from cugo_b200.losses import policy_loss
    x, actions, old, adv, k = policy_case(64, 179, torch.float32, True, 0, "sampled", False)
    y = x.detach().requires_grad_()
    loss = policy_loss(y, actions, old, adv, **k).loss
    loss /= 4
    a, = torch.autograd.grad(loss, y, retain_graph=True)
    b, = torch.autograd.grad(loss, y)
    assert torch.equal(a, b) and bool(a.any())


def test_an_entry_past_32_bits_of_offset():
    """The last rows of logits of more than 2^32 bytes, and of more than 2^31 entries."""
    from cugo_b200.losses import action_logp
    rows, vocab = 8200, 1 << 18
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=DEV)
    x[-1].normal_()
    actions = torch.full((rows,), 77, device=DEV)
    y = x.requires_grad_()
    logp, entropy = action_logp(y, actions)
    _, want, _, _, _ = action_logp64(x[-1:], actions[-1:])
    near(logp[-1:].detach(), want.detach(), chain(vocab) * U * 20, "last row")
    assert float((logp[:-1] + math.log(vocab)).abs().max()) < 1e-3
    d_logp = torch.zeros(rows, device=DEV)
    d_logp[-1] = 1.0
    d, = torch.autograd.grad(logp, y, d_logp)
    assert abs(float(d[-1].double().sum())) < 2e-2 and float(d[-1, 77]) > 0.99 and not bool(d[-2].any())


@pytest.mark.parametrize("vocab", [1 << 17, 131071])
def test_few_long_rows(vocab):
    """A row over several blocks: the same sums as the definition's."""
    from cugo_b200.losses import policy_loss_grad
    for rows, kl in ((1, "full"), (3, "sampled"), (40, "none")):
        x, actions, old, adv, k = policy_case(rows, vocab, torch.bfloat16, False, 0, kl, False)
        want, stats, logp, p, _ = policy64(x, actions, old, adv, **k)
        worst, size = policy_tols(vocab, x, actions, k, adv, p, stats, rows)
        out, d = policy_loss_grad(x, actions, old, adv, **k)
        near(out.stats, stats, worst * (1 + stats.abs()), "stats")
        near(d, want, grad_tol(vocab, p, actions, size, torch.bfloat16, want), "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(3, 131072), (700, 2501), (1000, 1501), (4000, 2501), (950, 9001), (500, 33000),
                                        (400, 50000), (300, 100001)])
def test_masked_entries_turn_up_late(rows, vocab, dtype):
    """Long rows of which some, not the first ones, have entries of -inf, and one a NaN: each
    plan for such rows, with and without a reference, forward and backward."""
    from cugo_b200.losses import action_logp, policy_loss_grad
    for kl in ("none", "full"):
        x, actions, old, adv, k = policy_case(rows, vocab, dtype, False, 0, kl, False)
        g = torch.Generator(device=DEV).manual_seed(rows)
        shut = torch.rand((rows, vocab), device=DEV, generator=g) < 0.3
        shut &= torch.rand((rows, 1), device=DEV, generator=g) < 0.3
        shut.scatter_(1, actions[:, None], False)
        shut[0] = False
        shut[rows - 1] = True                                   # a row that does not count
        x = x.masked_fill(shut, -float("inf"))
        if kl == "full":
            k["ref_logits"] = k["ref_logits"].masked_fill(shut, -float("inf"))
        out, d = policy_loss_grad(x, actions, old, adv, **k)
        want, stats, logp, p, used = policy64(x, actions, old, adv, **k)
        assert not bool(used[rows - 1])
        worst, size = policy_tols(vocab, x, actions, k, adv, p, stats, rows)
        near(out.stats, stats, worst * (1 + stats.abs()), "stats")
        near(out.logp, logp, chain(vocab) * U * (1 + logp.abs()), "logp")
        near(d, want, grad_tol(vocab, p, actions, size, dtype, want), "gradient")
        # The same as a mask, whatever stands in the masked places.
        k["legal"] = ~shut
        noisy = torch.where(shut, torch.full_like(x, float("nan")), x)
        if kl == "full":
            k["ref_logits"] = torch.where(shut, torch.full_like(x, float("inf")), k["ref_logits"])
        out, d = policy_loss_grad(noisy, actions, old, adv, **k)
        near(out.stats, stats, worst * (1 + stats.abs()), "stats, masked")
        near(d, want, grad_tol(vocab, p, actions, size, dtype, want), "gradient, masked")
    y = x.requires_grad_()
    got, entropy = action_logp(y, actions)
    leaf, want, want_h, p, _ = action_logp64(x, actions)
    near(got.detach(), want.detach(), chain(vocab) * U * (1 + want.detach().abs()), "log p")
    near(entropy.detach(), want_h.detach(), chain(vocab) * U * (1 + 2 * want_h.detach() + math.log(vocab)), "entropy")
    d, = torch.autograd.grad(got.sum() + 0.5 * entropy.sum(), y)
    want_d, = torch.autograd.grad(want.sum() + 0.5 * want_h.sum(), leaf)
    size = torch.full((rows,), 2.0 + 2 * (24 + 2 * math.log(vocab)), device=DEV, dtype=torch.float64)
    near(d, want_d, grad_tol(vocab, p, actions, size, dtype, want_d), "backward")
    bad = x.detach().clone()
    bad[1, 5] = float("nan")
    worse, _ = action_logp(bad, actions)
    assert bool(torch.isnan(worse[1])) and int(torch.isnan(worse).sum()) == 1
    near(worse[2:], got[2:].detach().double(), 2 * chain(vocab) * U * (1 + want.detach()[2:].abs()), "beside a NaN")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [3, 30, 64, 179, 384, 1000, 1500, 4100])
def test_rows_far_apart_and_masks_anywhere(vocab, dtype):
    """Rows, reference rows, masks and gradients with strides of their own, flags that begin at
    any byte; what lies between the gradient's rows stays as it was."""
    from cugo_b200.losses import policy_loss_grad
    rows = 37
    for shift, gap in ((0, 77), (1, 100), (3, 33), (6, 0)):
        x, actions, old, adv, k = policy_case(rows, vocab, dtype, True, 0, "full", True)
        g = torch.Generator(device=DEV).manual_seed(shift)

        def apart(t, more):
            wide = torch.zeros((rows, vocab + more + shift), dtype=t.dtype, device=DEV)
            if t.dtype != torch.bool:
                wide.fill_(float("nan"))
            wide[:, shift:shift + vocab] = t
            return wide[:, shift:shift + vocab]

        want, stats, _, p, _ = policy64(x, actions, old, adv, **k)
        worst, size = policy_tols(vocab, x, actions, k, adv, p, stats, rows)
        k["legal"], k["ref_logits"] = apart(k["legal"], gap), apart(k["ref_logits"], 2 * gap + 1)
        room = torch.full((rows, vocab + 9 + shift), 7.0, dtype=dtype, device=DEV)
        out, d = policy_loss_grad(apart(x, gap), actions, old, adv, **k, dlogits=room[:, shift:shift + vocab + 2])
        near(out.stats, stats, worst * (1 + stats.abs()), "stats")
        near(d[:, :vocab], want, grad_tol(vocab, p, actions, size, dtype, want), "gradient")
        assert not bool(d[:, vocab:].any())
        assert bool((room[:, :shift] == 7).all()) and bool((room[:, shift + vocab + 2:] == 7).all())


def test_a_given_gradient_is_a_new_version():
    """What autograd has kept of the tensor that the gradient goes to is out of date."""
    from cugo_b200.losses import policy_loss_grad
    x, actions, _, _ = make(6, 20, torch.float32, 0)
    f, d = torch.zeros(6, device=DEV), torch.ones((6, 24), device=DEV)
    w = torch.ones((6, 24), device=DEV, requires_grad=True)
    y = (w * d).sum()
    policy_loss_grad(x, actions, f, f, dlogits=d)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("rows", [1, 5, 600])
def test_one_mask_gives_the_bits_of_many(rows):
    from cugo_b200.losses import policy_loss_grad
    for vocab in (30, 179, 700, 1500):
        x, actions, old, adv, _ = policy_case(rows, vocab, torch.float32, False, 0, "none", False)
        one = torch.rand(vocab, device=DEV) < 0.4
        one[actions[::2]] = True
        a, da = policy_loss_grad(x, actions, old, adv, legal=one.expand(rows, vocab), entropy_coef=0.1)
        b, db = policy_loss_grad(x, actions, old, adv, legal=one.repeat(rows, 1), entropy_coef=0.1)
        assert torch.equal(a.stats, b.stats) and torch.equal(a.logp, b.logp) and torch.equal(da, db)


def test_refusals():
    from cugo_b200.losses import action_logp, policy_loss, policy_loss_grad, preference_loss
    x, actions, mask, _ = make(6, 20, torch.float32, 0, True)
    f = torch.zeros(6, device=DEV)
    bad = [
        (lambda: action_logp(x.double(), actions), "fp32, bf16 or fp16"),
        (lambda: action_logp(x[0], actions), "logits must be"),
        (lambda: action_logp(x.t().contiguous().t(), actions), "row-major"),
        (lambda: action_logp(x[:1].expand(6, 20), actions), "row-major"),
        (lambda: action_logp(x, actions.int()), "actions"),
        (lambda: action_logp(x, actions[:5]), "actions"),
        (lambda: action_logp(x, actions.cpu()), "actions"),
        (lambda: action_logp(x, actions, mask[:, :19]), "legal"),
        (lambda: action_logp(x, actions, mask.int()), "legal"),
        (lambda: policy_loss(x, actions, f.half(), f), "logp_old"),
        (lambda: policy_loss(x, actions, f, f[:5]), "adv"),
        (lambda: policy_loss(x, actions, f, f, weight=f.double()), "weight"),
        (lambda: policy_loss(x, actions, f, f, ref_logits=x.half()), "ref_logits"),
        (lambda: policy_loss(x, actions, f, f, ref_logits=x, ref_logp=f), "not both"),
        (lambda: policy_loss(x, actions, f, f, clip_low=-0.1), "clip"),
        (lambda: policy_loss(x, actions, f, f, denominator=0.0), "denominator"),
        (lambda: policy_loss_grad(x, actions, f, f, dlogits=x[:, :19].clone()), "dlogits"),
        (lambda: policy_loss_grad(x, actions, f, f, dlogits=x.double()), "dlogits"),
        (lambda: policy_loss_grad(x, actions, f, f, dlogits=x.clone(), grad_dtype=torch.half), "grad_dtype"),
        (lambda: policy_loss(x, actions, f, f, denominator=1e-60), "denominator"),
        (lambda: policy_loss_grad(x, actions, f, f, dlogits=x), "share memory"),
        (lambda: policy_loss_grad(x[:5], actions[:5], f[:5], f[:5], dlogits=x[1:]), "share memory"),
        (lambda: policy_loss_grad(x, actions, f, f, ref_logits=x.clone(), dlogits=x[:, :]), "share memory"),
        (lambda: preference_loss(x, actions, torch.zeros(2, dtype=torch.int64, device=DEV), f), "offsets"),
        (lambda: preference_loss(x, actions, torch.zeros(3, dtype=torch.int32, device=DEV), f), "offsets"),
        (lambda: preference_loss(x, actions, torch.zeros(3, dtype=torch.int64, device=DEV), f,
                                 label_smoothing=1.5), "smoothing"),
    ]
    for call, words in bad:
        with pytest.raises(RuntimeError, match=words):
            call()
