"""The operators of a policy update, as cases to measure: the log-probabilities of given
actions, the clipped policy loss with a KL term, the preference loss over paired lines of
play, and the AdamW step over many tensors.

A case is a dict of plain values.  `prepare` makes its inputs on the GPU from a seed,
`run` takes one pass: in plain torch operations where `own` is false, through
cugo_b200's entry points where it is true.  `exact` computes the same in 64 bits, mostly
through autograd, so that it shares no formula with the plain form's gradients."""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 256        # elements that share one scale of the 8-bit states
NEG = float("-inf")


# ---- the cases --------------------------------------------------------------------------

def _logp(name, rows, vocab, dtype, legal, back, pad=0):
    return {"name": name, "op": "logp", "rows": rows, "vocab": vocab, "dtype": dtype,
            "legal": legal, "back": back, "pad": pad}


def _policy(name, rows, vocab, dtype, legal, kl, weights, back, grad, pad=0):
    return {"name": name, "op": "policy", "rows": rows, "vocab": vocab, "dtype": dtype,
            "legal": legal, "kl": kl, "weights": weights, "back": back, "grad": grad, "pad": pad}


def _pairs(name, pairs, longest, vocab, dtype, legal, weights, pad=0):
    return {"name": name, "op": "preference", "pairs": pairs, "longest": longest, "vocab": vocab,
            "dtype": dtype, "legal": legal, "weights": weights, "pad": pad}


def _adamw(name, networks, hidden, blocks, param, bits, clip):
    return {"name": name, "op": "adamw", "networks": networks, "hidden": hidden,
            "blocks": blocks, "param": param, "bits": bits, "clip": clip}


def listed():
    return [
        # Scoring the decisions of one step of a few games: latency only.
        _logp("logp 64x179", 64, 179, "fp32", True, False, 1),
        # The log-probabilities of a self-play round under another policy (logp_old, ref_logp).
        _logp("logp 262144x179", 262144, 179, "fp32", True, False, 1),
        # A token policy trained on given actions with an entropy term, forward and backward.
        _logp("logp grad 8192x16384 bf16", 8192, 16384, "bf16", False, True),
        # The smallest training minibatch.
        _policy("policy 256x179", 256, 179, "fp32", True, "sampled", False, "fused", "bf16", 1),
        # The trainer's minibatch (32,768 decisions), held to a frozen actor by the full KL.
        _policy("policy 32768x179 full KL", 32768, 179, "fp32", True, "full", False, "fused", "bf16", 1),
        # The same minibatch's loss under autograd, with weights (padded rows have weight 0).
        _policy("policy autograd 65536x179", 65536, 179, "fp32", True, "sampled", True, "autograd", "fp32"),
        # A token policy over a large vocabulary, padded rows among them.
        _policy("policy 2048x131072 bf16", 2048, 131072, "bf16", False, "sampled", True, "fused", "bf16"),
        # Pairs of lines of play from duplicate deals, about 12 decisions each.
        _pairs("preference 128 pairs x179", 128, 24, 179, "fp32", True, False, 1),
        # Pairs of token sequences, prompts with weight 0.
        _pairs("preference 16 pairs x32768 bf16", 16, 1024, 32768, "bf16", False, True),
        # The trainer's two networks (3 x 512), states in 32 bits, gradients clipped by their norm.
        _adamw("adamw 2 nets 3x512", 2, 512, 3, "fp32", 32, True),
        # The larger networks (4 x 2048), states in 8 bits.
        _adamw("adamw8 2 nets 4x2048", 2, 2048, 4, "fp32", 8, True),
        # A network that fills the card's bandwidth, bf16 parameters, states in 8 bits.
        _adamw("adamw8 1 net 2x8192 bf16", 1, 8192, 2, "bf16", 8, False),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["logp", "policy", "preference", "adamw"])
    if op == "adamw":
        case = {"op": op, "networks": rng.randint(1, 2), "hidden": _between(rng, 48, 8192),
                "blocks": rng.randint(1, 4), "param": rng.choice(["fp32", "bf16"]),
                "bits": rng.choice([8, 32]), "clip": rng.random() < 0.5}
        while work(case)["bytes"] > 2e9:
            case["hidden"] = case["hidden"] * 3 // 4
        return case
    legal = rng.random() < 0.4
    vocab = rng.choice([179, _between(rng, 2, 1024)]) if legal else _between(rng, 2, 131072)
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    pad = rng.choice([0, 0, 1, 5, 8])
    most = (1 << 27) // (vocab + pad)  # logits of a case: half of the largest listed one's
    if op == "preference":
        pairs = _between(rng, 1, 256)
        longest = max(1, min(_between(rng, 1, 2048), most // (2 * pairs)))
        return {"op": op, "pairs": pairs, "longest": longest, "vocab": vocab, "dtype": dtype,
                "legal": legal, "weights": rng.random() < 0.5, "pad": pad}
    rows = _between(rng, 1, max(1, min(262144, most)))
    if op == "logp":
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "legal": legal,
                "back": rng.random() < 0.5, "pad": pad}
    back = rng.choice(["fused", "autograd", "none"])
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "legal": legal,
            "kl": rng.choice(["none", "sampled", "full"]), "weights": rng.random() < 0.5,
            "back": back, "grad": rng.choice([dtype, "bf16"]) if back == "fused" else dtype, "pad": pad}


def _shapes(case):
    """The parameters of the case's networks: 720 features in, 179 actions out."""
    h = case["hidden"]
    net = [(h, 720), (h,)] + [(h, h), (h,)] * (2 * case["blocks"]) + [(179, h), (179,)]
    return net * case["networks"]


def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        p = BYTES[case["param"]]
        state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
        # Parameter and states read and written, the gradient read; about 12 operations each.
        return {"bytes": n * (2 * p + p + state), "flops": 12 * n}
    if case["op"] == "preference":
        rows = sum(_lengths(case))
    else:
        rows = case["rows"]
    n, e = rows * case["vocab"], BYTES[case["dtype"]]
    total = n * e + rows * 16
    if case["legal"]:
        total += n
    if case["op"] == "policy":
        total += n * e if case["kl"] == "full" else 0
        total += n * BYTES[case["grad"]] if case["back"] != "none" else 0
    elif case["op"] == "preference" or case["back"]:
        total += n * e
    # An exponential, a few products and sums of every entry.
    return {"bytes": total, "flops": 8 * n}


# ---- the inputs -------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(case):
    """Rows of each of the 2 x pairs sequences, from 1 to the longest: the same for every
    seed, so that a case's work is known without its inputs."""
    k = 2 * case["pairs"]
    return [1 + (37 * i * i + 11 * i + 5) % case["longest"] for i in range(k)]


def _rows_of(logits_t, chunk=1 << 26):
    """Row ranges whose 64-bit copies stay small."""
    step = max(1, chunk // max(1, logits_t.shape[1]))
    return [(i, min(i + step, logits_t.shape[0])) for i in range(0, logits_t.shape[0], step)]


def _make_logits(g, rows, vocab, pad, dtype):
    wide = torch.empty((rows, vocab + pad), dtype=TYPES[dtype], device=DEV)
    wide.normal_(0.0, 2.0, generator=g)
    return wide[:, :vocab]


def _make_rows(case, rows, g):
    """Logits, legal actions (about a tenth, as in the game, at least one but in a few rows
    that have none) and taken actions, drawn from the logits' own distribution."""
    logits = _make_logits(g, rows, case["vocab"], case["pad"], case["dtype"])
    legal = None
    if case["legal"]:
        legal = torch.rand(logits.shape, device=DEV, generator=g) < 0.1
        some = torch.randint(case["vocab"], (rows, 1), device=DEV, generator=g)
        legal.scatter_(1, some, True)
        if rows >= 64:
            legal &= torch.rand((rows, 1), device=DEV, generator=g) > 0.002
    actions = torch.empty(rows, dtype=torch.int64, device=DEV)
    logp = torch.zeros(rows, dtype=torch.float64, device=DEV)
    for a, b in _rows_of(logits):
        x = logits[a:b].float()
        if legal is not None:
            x = x.masked_fill(~legal[a:b], NEG)
        noise = torch.empty_like(x).exponential_(generator=g)
        actions[a:b] = (x - noise.log()).argmax(1)
        del noise
        ok = torch.isfinite(x).any(1)
        y = torch.log_softmax(x.double(), 1).gather(1, actions[a:b, None])[:, 0]
        logp[a:b] = torch.where(ok, y, 0.0)
    return logits, legal, actions, logp


def _loss_scale(dtype, count):
    """Gradients in fp16 are taken of a loss scaled by about the number of its terms, as a
    trainer scales it: a mean over many rows lies below the type's range."""
    scale = 2.0 ** round(math.log2(count)) if dtype == "fp16" else 1.0
    return {"scale": scale, "d_loss": torch.tensor(scale, device=DEV)}


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "adamw":
        return _prepare_adamw(case, g, seed)
    if op == "preference":
        lengths = _lengths(case)
        rows = sum(lengths)
        logits, legal, actions, logp = _make_rows(case, rows, g)
        offsets = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(DEV)
        ref = (logp + 0.3 * torch.randn(rows, device=DEV, generator=g, dtype=torch.float64)).float()
        weight = None
        if case["weights"]:  # a prompt of weight 0 at the head of each sequence, a third of it
            at = torch.arange(rows, device=DEV)
            seq = torch.searchsorted(offsets, at, right=True) - 1
            start, length = offsets[seq], offsets[seq + 1] - offsets[seq]
            weight = ((at - start) * 3 >= length).float()
        return {"case": case, "logits": logits, "legal": legal, "actions": actions, "offsets": offsets,
                "ref_logp": ref, "weight": weight, "beta": 0.1, **_loss_scale(case["dtype"], case["pairs"])}
    logits, legal, actions, logp = _make_rows(case, case["rows"], g)
    rows = case["rows"]
    s = {"case": case, "logits": logits, "legal": legal, "actions": actions}
    if op == "logp":
        if case["back"]:
            s["d_logp"] = torch.randn(rows, device=DEV, generator=g)
            s["d_entropy"] = 0.1 * torch.randn(rows, device=DEV, generator=g)
        return s
    s |= _loss_scale(case["grad"], rows)
    # Log ratios after a few steps from the behaviour policy.  None lies within 1e-3 of where
    # the clip begins: there the gradient jumps, and the last bit of a sum decides.
    shift = 0.25 * torch.randn(rows, device=DEV, generator=g, dtype=torch.float64)
    for border in (math.log(1 - 0.2), math.log(1 + 0.28)):
        shift = torch.where((shift - border).abs() < 1e-3, border + 2e-3, shift)
    s["logp_old"] = (logp - shift).float()
    s["adv"] = torch.randn(rows, device=DEV, generator=g)
    s["weight"] = None
    if case["weights"]:
        s["weight"] = (torch.rand(rows, device=DEV, generator=g) < 0.8).float()
        s["weight"][0] = 1.0
    s["ref_logp"] = s["ref_logits"] = None
    if case["kl"] == "sampled":
        s["ref_logp"] = (logp + 0.2 * torch.randn(rows, device=DEV, generator=g, dtype=torch.float64)).float()
    elif case["kl"] == "full":
        ref = logits + 0.3 * torch.randn(logits.shape, device=DEV, generator=g).to(logits.dtype)
        s["ref_logits"] = ref
    return s


def _codes(x):
    """(e4m3 codes, e8m0 scales) of fp32 blocks [n, 256], rounded to nearest."""
    a = x.abs().amax(1)
    f, e = torch.frexp(a)
    k = torch.where(f <= 0.875, e - 9, e - 8)
    byte = torch.where(a > 0, k + 127, 27).clamp(27, 247)
    scale = torch.exp2((byte - 127).float())
    return (x / scale[:, None]).to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _prepare_adamw(case, g, seed):
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts = [0]
    for n in sizes:  # every tensor starts at a whole block of one buffer
        starts.append(starts[-1] + -(-n // BLOCK) * BLOCK)
    total = starts[-1]
    real = torch.zeros(total, dtype=torch.bool, device=DEV)
    for at, n in zip(starts, sizes):
        real[at:at + n] = True

    def views(flat):
        return [flat[a:a + n].view(s) for a, n, s in zip(starts, sizes, shapes)]

    def values(std, dtype=torch.float32):
        t = torch.empty(total, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=g)
        return t.mul_(real).to(dtype)

    p_type = TYPES[case["param"]]
    s = {"case": case, "sizes": sizes, "starts": starts, "p": values(0.03, p_type),
         "g": values(2e-3, p_type), "step": torch.full((1,), 41, dtype=torch.int64, device=DEV),
         "seed": seed & 0xFFFF, "views": views, "lr": 3e-4, "betas": (0.9, 0.999), "eps": 1e-8, "decay": 0.01,
         "clip": 1.0 if case["clip"] else None}
    m, v = values(6e-4), values(1e-3).square_()
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["m_scale"] = _codes(m.view(-1, BLOCK))
        s["v"], s["v_scale"] = _codes(v.view(-1, BLOCK))
        s["m"], s["v"] = s["m"].view(-1), s["v"].view(-1)
    s["params"], s["grads"] = views(s["p"]), views(s["g"])
    s["ms"], s["vs"] = views(s["m"]), views(s["v"])
    if case["bits"] == 8:
        cuts = [(a // BLOCK, -(-n // BLOCK)) for a, n in zip(starts, sizes)]
        s["m_scales"] = [s["m_scale"][a:a + n] for a, n in cuts]
        s["v_scales"] = [s["v_scale"][a:a + n] for a, n in cuts]
    return s


# ---- one pass ---------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"logp": _plain_logp, "policy": _plain_policy, "preference": _plain_preference,
            "adamw": _plain_adamw}[s["case"]["op"]](s)


def _own(s):
    from cugo_b200 import losses, optim
    case, op = s["case"], s["case"]["op"]
    if op == "adamw":
        norm = optim.adamw_step(
            s["params"], s["grads"], s["ms"], s["vs"], s["step"], lr=s["lr"], betas=s["betas"],
            eps=s["eps"], weight_decay=s["decay"], max_grad_norm=s["clip"], seed=s["seed"],
            exp_avg_scales=s.get("m_scales"), exp_avg_sq_scales=s.get("v_scales"))
        return _adamw_outputs(s, norm)
    if op == "logp":
        if not case["back"]:
            return losses.action_logp(s["logits"], s["actions"], s["legal"])
        x = s["logits"].detach().requires_grad_()
        logp, entropy = losses.action_logp(x, s["actions"], s["legal"])
        d, = torch.autograd.grad((logp, entropy), x, (s["d_logp"], s["d_entropy"]))
        return logp, entropy, d
    if op == "preference":
        x = s["logits"].detach().requires_grad_()
        out = losses.preference_loss(x, s["actions"], s["offsets"], s["ref_logp"], legal=s["legal"],
                                     weight=s["weight"], beta=s["beta"])
        d, = torch.autograd.grad(out.loss, x, s["d_loss"])
        return out.loss, out.margin, out.logp, d
    args = (s["actions"], s["logp_old"], s["adv"])
    more = dict(legal=s["legal"], weight=s["weight"], ref_logp=s["ref_logp"], ref_logits=s["ref_logits"],
                clip_low=0.2, clip_high=0.28, kl_coef=0.05, entropy_coef=0.01)
    if case["back"] == "fused":
        out, d = losses.policy_loss_grad(s["logits"], *args, **more, grad_dtype=TYPES[case["grad"]],
                                         grad_scale=s["scale"])
        return out.stats, out.logp, d
    x = s["logits"].detach()
    if case["back"] == "none":
        out = losses.policy_loss(x, *args, **more)
        return out.stats, out.logp
    x.requires_grad_()
    out = losses.policy_loss(x, *args, **more)
    d, = torch.autograd.grad(out.loss, x, s["d_loss"])
    return out.stats, out.logp, d


def _plain_rows(logits, legal, actions, weight=None):
    """Of every row, in 32 bits: whether it counts, log p of all entries (-inf where illegal),
    p, the log p of the taken action and the entropy (0 where the row does not count)."""
    x = logits.float()
    if legal is not None:
        x = x.masked_fill(~legal, NEG)
    top = x.amax(1, keepdim=True)
    a = actions.clamp(0, x.shape[1] - 1)[:, None]
    used = (top[:, 0] != NEG) & (actions >= 0) & (actions < x.shape[1])
    if legal is not None:
        used &= legal.gather(1, a)[:, 0]
    if weight is not None:
        used &= weight != 0
    x = x - torch.where(top == NEG, 0.0, top)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    lp = x - torch.log(total)
    p = e / total
    entropy = -torch.where(p == 0, 0.0, p * lp).sum(1)
    logp = lp.gather(1, a)[:, 0]
    return used, lp, p, torch.where(used, logp, 0.0), torch.where(used, entropy, 0.0)


def _hot_minus_p(p, actions):
    d = -p
    return d.scatter_add_(1, actions.clamp(0, p.shape[1] - 1)[:, None], torch.ones_like(p[:, :1]))


def _plain_logp(s):
    used, lp, p, logp, entropy = _plain_rows(s["logits"], s["legal"], s["actions"])
    if not s["case"]["back"]:
        return logp, entropy
    d = s["d_logp"][:, None] * _hot_minus_p(p, s["actions"])
    d -= torch.where(p == 0, 0.0, p * (lp + entropy[:, None])) * s["d_entropy"][:, None]
    return logp, entropy, torch.where(used[:, None], d, 0.0).to(s["logits"].dtype)


def _plain_policy(s):
    case = s["case"]
    used, lp, p, logp, entropy = _plain_rows(s["logits"], s["legal"], s["actions"], s["weight"])
    rows = used.numel()
    w = used.float() if s["weight"] is None else torch.where(used, s["weight"], 0.0)
    denominator = float(rows) if s["weight"] is None else s["weight"].double().sum().float()
    log_ratio = logp - s["logp_old"]
    ratio = torch.exp(log_ratio)
    bounded = ratio.clamp(1 - 0.2, 1 + 0.28)
    gain = torch.minimum(ratio * s["adv"], bounded * s["adv"])
    moves = (ratio * s["adv"] <= bounded * s["adv"])
    d_logp = torch.where(moves, -ratio * s["adv"], 0.0)
    kl = torch.zeros_like(logp)
    q_diff = None
    if case["kl"] == "sampled":
        diff = s["ref_logp"] - logp
        kl = torch.expm1(diff) - diff
        d_logp = d_logp - 0.05 * torch.expm1(diff)
    elif case["kl"] == "full":
        _, lq, _, _, _ = _plain_rows(s["ref_logits"], s["legal"], s["actions"])
        q_diff = torch.where(p == 0, 0.0, lp - lq)
        kl = (p * q_diff).sum(1)

    def mean(t):
        return (torch.where(used, t, 0.0).double() * w.double()).sum().float() / denominator

    policy, h, k = mean(-gain), mean(entropy), mean(kl)
    stats = torch.stack((policy - 0.01 * h + 0.05 * k, policy, h, k, mean(ratio - 1 - log_ratio),
                         mean(((ratio < 1 - 0.2) | (ratio > 1 + 0.28)).float()),
                         mean(torch.ones_like(ratio))))
    if case["back"] == "none":
        return stats, logp
    d = d_logp[:, None] * _hot_minus_p(p, s["actions"])
    d += torch.where(p == 0, 0.0, p * (lp + entropy[:, None])) * 0.01
    if q_diff is not None:
        d += p * (q_diff - kl[:, None]) * 0.05
    d *= (w * s["scale"] / denominator)[:, None]
    return stats, logp, torch.where(used[:, None], d, 0.0).to(TYPES[case["grad"]])


def _plain_preference(s):
    case = s["case"]
    used, _, p, logp, _ = _plain_rows(s["logits"], s["legal"], s["actions"], s["weight"])
    w = used.float() if s["weight"] is None else torch.where(used, s["weight"], 0.0)
    sums = torch.zeros(logp.numel() + 1, dtype=torch.float64, device=DEV)
    sums[1:] = (w * logp).double().cumsum(0)
    both = torch.zeros_like(sums)
    both[1:] = (w * (logp - s["ref_logp"])).double().cumsum(0)
    o = s["offsets"]
    seq_logp = (sums[o[1:]] - sums[o[:-1]]).float()
    score = both[o[1:]] - both[o[:-1]]
    margin = (s["beta"] * (score[0::2] - score[1::2])).float()
    loss = torch.log1p(torch.exp(-margin.abs())) + torch.clamp(-margin, min=0.0)
    slope = -s["beta"] * s["scale"] / margin.numel() * torch.sigmoid(-margin)
    each = torch.stack((slope, -slope), 1).reshape(-1)
    d_logp = torch.repeat_interleave(each, o[1:] - o[:-1], output_size=logp.numel()) * w
    d = d_logp[:, None] * _hot_minus_p(p, s["actions"])
    return loss.double().mean().float(), margin, seq_logp, torch.where(used[:, None], d, 0.0).to(TYPES[case["dtype"]])


def _mix(x):
    """A 32-bit mixer (xor-shifts and odd products), on whole numbers in 64 bits."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _round_e4m3(x, r):
    """x (at most 448) to e4m3, up or down by 16 random bits r; below 2^-6 the steps are 2^-9."""
    a = x.abs()
    low = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)
    bits = (a + low).view(torch.int32)
    bits = (bits + ((r << 4) + 8).int()) & ~0xFFFFF
    return torch.copysign(bits.view(torch.float32) - low, x)


def _plain_adamw(s):
    b1, b2 = s["betas"]
    t = s["step"].add_(1)
    total = s["p"].numel()
    grad = s["g"].float()
    norm = None
    if s["clip"] is not None:
        norm = grad.double().square_().sum().sqrt().float()
        grad = grad * torch.clamp(s["clip"] / (norm + 1e-6), max=1.0)
    eight = s["case"]["bits"] == 8
    if eight:
        m = _values(s["m"], s["m_scale"])
        v = _values(s["v"], s["v_scale"])
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + grad * (1 - b1)
    v = v * b2 + grad * grad * (1 - b2)
    bias1, bias2 = 1 - b1 ** t.double(), 1 - b2 ** t.double()
    p = s["p"].float() * (1 - s["lr"] * s["decay"])
    p -= (s["lr"] / bias1).float() * m / (torch.sqrt(v / bias2.float()) + s["eps"])
    if eight or s["p"].dtype != torch.float32:
        e = torch.arange(total, device=DEV)
        key = _mix((s["seed"] + t * 0x9E3779B9) & 0xFFFFFFFF)
        r = _mix((e & 0xFFFFFFFF) ^ ((key + (e >> 32) * 0x9E3779B9) & 0xFFFFFFFF))
    if s["p"].dtype == torch.float32:
        s["p"].copy_(p)
    else:  # up or down by 16 random bits: most updates are below half a step
        r_p = (r * 0x2C1B3C6D & 0xFFFFFFFF) >> 16
        s["p"].copy_(((p.view(torch.int32) + r_p.int()) & ~0xFFFF).view(torch.float32))
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return _adamw_outputs(s, norm)
    for name, x, random in (("m", m, r & 0xFFFF), ("v", v, r >> 16)):
        a = x.view(-1, BLOCK).abs().amax(1)
        f, ex = torch.frexp(a)
        byte = torch.where(a > 0, torch.where(f <= 0.875, ex - 9, ex - 8) + 127, 27).clamp(27, 247)
        inverse = torch.exp2((127 - byte).float())
        code = _round_e4m3((x.view(-1, BLOCK) * inverse[:, None]).view(-1), random)
        if name == "v":  # a second moment never becomes zero by rounding
            code = torch.where((x > 0) & (code == 0), 2.0 ** -9, code)
        s[name].copy_(code)
        s[name + "_scale"].copy_(byte)
    return _adamw_outputs(s, norm)


def _values(codes, scale):
    return (codes.float().view(-1, BLOCK) * torch.exp2(scale.float() - 127)[:, None]).view(-1)


def _adamw_outputs(s, norm):
    out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if s["case"]["bits"] == 8:
        out["m_scale"] = s["m_scale"].view(torch.float8_e8m0fnu)
        out["v_scale"] = s["v_scale"].view(torch.float8_e8m0fnu)
    if norm is not None:
        out["norm"] = norm
    return out


# ---- the same in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    return {"logp": _exact_logp, "policy": _exact_policy, "preference": _exact_preference}[case["op"]](s)


def _exact_rows(s, a, b):
    """(a leaf of rows a..b in 64 bits, its log-softmax over the legal entries with the rows
    that do not count replaced by a uniform one, whether each row counts)."""
    leaf = s["logits"][a:b].double().requires_grad_()
    ok = torch.ones(b - a, dtype=torch.bool, device=DEV)
    x = leaf
    if s["legal"] is not None:
        legal = s["legal"][a:b]
        ok &= legal.gather(1, s["actions"][a:b, None])[:, 0]
        x = torch.where(legal | ~ok[:, None], x, -1e300)
    if s.get("weight") is not None:
        ok &= s["weight"][a:b] != 0
    return leaf, torch.log_softmax(x, 1), ok


def _exact_logp(s):
    logps, entropies, grads = [], [], []
    for a, b in _rows_of(s["logits"], 1 << 25):
        leaf, lp, ok = _exact_rows(s, a, b)
        logp = torch.where(ok, lp.gather(1, s["actions"][a:b, None])[:, 0], 0.0)
        entropy = torch.where(ok, -(lp.exp() * lp).sum(1), 0.0)
        if s["case"]["back"]:
            total = (logp * s["d_logp"][a:b].double()).sum() + (entropy * s["d_entropy"][a:b].double()).sum()
            grads.append(torch.autograd.grad(total, leaf)[0])
        logps.append(logp.detach())
        entropies.append(entropy.detach())
    out = (torch.cat(logps), torch.cat(entropies))
    return out + (torch.cat(grads),) if s["case"]["back"] else out


def _exact_policy(s):
    case = s["case"]
    rows = case["rows"]
    weight = torch.ones(rows, dtype=torch.float64, device=DEV) if s["weight"] is None else s["weight"].double()
    denominator = weight.sum()
    sums, logps, grads = 0.0, [], []
    for a, b in _rows_of(s["logits"], 1 << 25):
        leaf, lp, ok = _exact_rows(s, a, b)
        w = torch.where(ok, weight[a:b], 0.0) / denominator
        logp = torch.where(ok, lp.gather(1, s["actions"][a:b, None])[:, 0], 0.0)
        old, adv = s["logp_old"][a:b].double(), s["adv"][a:b].double()
        ratio = (logp - old).exp()
        gain = torch.minimum(ratio * adv, ratio.clamp(0.8, 1.28) * adv)
        entropy = -(lp.exp() * lp).sum(1)
        kl = torch.zeros_like(logp)
        if case["kl"] == "sampled":
            d = s["ref_logp"][a:b].double() - logp
            kl = d.exp() - 1 - d
        elif case["kl"] == "full":
            y = s["ref_logits"][a:b].double()
            if s["legal"] is not None:
                y = torch.where(s["legal"][a:b] | ~ok[:, None], y, -1e300)
            kl = (lp.exp() * torch.where(lp < -1e200, 0.0, lp - torch.log_softmax(y, 1))).sum(1)
        parts = torch.stack((-gain, entropy, kl, ratio - 1 - (logp - old),
                             ((ratio < 0.8) | (ratio > 1.28)).double(), torch.ones_like(ratio)))
        parts = (torch.where(ok, parts, 0.0) * w).sum(1)
        total = parts[0] - 0.01 * parts[1] + 0.05 * parts[2]
        if case["back"] != "none":
            grads.append(torch.autograd.grad(total * s["scale"], leaf)[0])
        sums = sums + parts.detach()
        logps.append(logp.detach())
    loss = sums[0] - 0.01 * sums[1] + 0.05 * sums[2]
    out = (torch.cat((loss[None], sums)), torch.cat(logps))
    return out + (torch.cat(grads),) if case["back"] != "none" else out


def _exact_preference(s):
    rows, o = s["logits"].shape[0], s["offsets"].tolist()
    logps, keep = torch.zeros(rows, dtype=torch.float64, device=DEV), _rows_of(s["logits"], 1 << 25)
    used = torch.zeros(rows, dtype=torch.float64, device=DEV)
    for a, b in keep:
        with torch.no_grad():
            _, lp, ok = _exact_rows(s, a, b)
            logps[a:b] = torch.where(ok, lp.gather(1, s["actions"][a:b, None])[:, 0], 0.0)
            used[a:b] = ok.double()
    if s["weight"] is not None:
        used = used * s["weight"].double()
    leaf = logps.requires_grad_()
    seq = torch.stack([(leaf[i:j] * used[i:j]).sum() for i, j in zip(o, o[1:])])
    ref = torch.stack([(s["ref_logp"][i:j].double() * used[i:j]).sum() for i, j in zip(o, o[1:])])
    margin = s["beta"] * ((seq - ref)[0::2] - (seq - ref)[1::2])
    loss = -torch.nn.functional.logsigmoid(margin).mean()
    d_logp, = torch.autograd.grad(loss * s["scale"], leaf)
    grads = []
    for a, b in keep:
        x, lp, ok = _exact_rows(s, a, b)
        part = torch.where(ok, lp.gather(1, s["actions"][a:b, None])[:, 0], 0.0)
        grads.append(torch.autograd.grad((part * d_logp[a:b]).sum(), x)[0])
    return loss.detach(), margin.detach(), seq.detach(), torch.cat(grads)


def _exact_adamw(s):
    b1, b2 = s["betas"]
    t = int(s["step"]) + 1
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    if s["clip"] is not None:
        g = g * min(1.0, s["clip"] / (float(norm) + 1e-6))
    if s["case"]["bits"] == 8:
        def units(scale):
            return torch.exp2(scale.double() - 127).repeat_interleave(BLOCK)
        m, v = s["m"].double() * units(s["m_scale"]), s["v"].double() * units(s["v_scale"])
    else:
        m, v = s["m"].double(), s["v"].double()
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.square(), v, b2)
    p = s["p"].double()
    p = p - s["lr"] * (s["decay"] * p + (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + s["eps"]))
    out = {"p": p, "m": m, "v": v}
    if s["case"]["bits"] == 8:
        for name in ("m", "v"):
            a = out[name].view(-1, BLOCK).abs().amax(1)
            k = torch.where(a > 0, torch.ceil(torch.log2(a / 448)), -100.0).clamp(-100, 120)
            out[name] = (out[name].view(-1, BLOCK) * torch.exp2(-k)[:, None]).view(-1)
            out[name + "_scale"] = torch.exp2(k)
    if s["clip"] is not None:
        out["norm"] = norm
    return out
