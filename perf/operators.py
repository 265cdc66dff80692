"""Workloads of the sequence-model operators: the gated linear recurrence, the clipped policy loss
and the AdamW step over many tensors.

``run`` makes one pass through an operator: with ``own`` the framework's entry points, without it
the same mathematics in elementary torch operations.  ``exact`` is the definition in 64 bits.

    recurrence   a = sigmoid(f);  h_t = a_t h_{t-1} + (1 - a_t) z_t  (h_{t-1} = 0 where reset_t)
    policy       -min(rho A, clip(rho) A) + beta (exp(ref - lp) - (ref - lp) - 1), rho = exp(lp - old),
                 lp = log softmax(logits)[token]; mean over the unmasked tokens or the sequences
    adamw        decoupled weight decay; moments in 32 bits, or in 8 bits with one power of two per
                 256 entries and stochastic rounding from a counter
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}

LR, BETAS, EPS, DECAY, STEP = 1e-3, (0.9, 0.999), 1e-8, 0.01, 1000
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.04
BLOCK = 256  # entries that share one exponent in the 8-bit moments


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _recurrence(name, mode, dtype, b, l, d, packed=False, lengths=False, resets=False, carried=False):
    case = {"op": "recurrence", "mode": mode, "dtype": dtype, "b": b, "l": l, "d": d,
            "packed": packed, "lengths": lengths, "resets": resets, "carried": carried}
    return dict(case, name=name) if name else case


def _policy(name, mode, dtype, b, t, v, mask=True, kl=True, reduction="token"):
    case = {"op": "policy", "mode": mode, "dtype": dtype, "b": b, "t": t, "v": v, "mask": mask,
            "kl": kl, "reduction": reduction}
    return dict(case, name=name) if name else case


def _adamw(name, layout, width, count, dtype, states):
    case = {"op": "adamw", "layout": layout, "width": width, "count": count, "dtype": dtype,
            "states": states}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token for each of 64 running sequences: what a server does between two samples
        _recurrence("recurrence token", "step", "bfloat16", 64, 1, 2048),
        # the character model's training batch: 256 windows of 15 characters, 2 x 64 channels
        _recurrence("recurrence characters", "train", "float32", 256, 15, 128, packed=True),
        # an ordinary training batch, gates and candidates as two halves of one projection
        _recurrence("recurrence batch", "train", "bfloat16", 8, 2048, 2048, packed=True),
        # right-padded prompts read once before generation starts
        _recurrence("recurrence prompts", "read", "float16", 16, 1531, 1536, lengths=True, carried=True),
        # one very long sequence of packed documents: few channels, everything is in the length
        _recurrence("recurrence long", "train", "bfloat16", 1, 100003, 640, resets=True, carried=True),
        # the character vocabulary: short rows, the launches count
        _policy("policy characters", "train", "float32", 256, 15, 128, mask=False, reduction="token"),
        # log-probabilities of given answers under a frozen model
        _policy("policy score", "score", "bfloat16", 8, 511, 32000, kl=False),
        # an ordinary update: prompts and padding masked, an odd vocabulary
        _policy("policy batch", "train", "bfloat16", 16, 384, 50021, reduction="sequence"),
        # a large vocabulary, and the largest tensor of such a step
        _policy("policy large", "train", "bfloat16", 4, 1500, 131072),
        # the character network's five weight tensors
        _adamw("adamw characters", "layers", 250, 3, "float32", 32),
        # 32-bit states of an ordinary model
        _adamw("adamw blocks", "blocks", 1600, 4, "float32", 32),
        # 16-bit weights with 32-bit masters, moments in 8 bits, odd widths
        _adamw("adamw eight bits", "blocks", 2047, 6, "bfloat16", 8),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("recurrence", "policy", "adamw"))
    if op == "recurrence":
        mode, dtype = rng.choice(("step", "train", "train", "read")), rng.choice(sorted(DTYPES))
        packed, lengths, resets, carried = (rng.random() < 0.5 for _ in range(4))
        d = _log_uniform(rng, 1, 4096)
        if mode == "step":
            return _recurrence(None, mode, dtype, _log_uniform(rng, 1, 2048), 1, d)
        most = 120_000_000 // SIZE[dtype]
        l = min(_log_uniform(rng, 1, 131072), max(1, most // d))
        b = _log_uniform(rng, 1, max(1, min(512, most // (d * l))))
        return _recurrence(None, mode, dtype, b, l, d, packed, lengths, resets, carried)
    if op == "policy":
        v, dtype = _log_uniform(rng, 2, 200_000), rng.choice(sorted(DTYPES))
        rows = min(_log_uniform(rng, 1, 100_000), max(1, 1_500_000_000 // (v * SIZE[dtype])))
        b = _log_uniform(rng, 1, min(rows, 256))
        return _policy(None, rng.choice(("train", "train", "score")), dtype, b, max(1, rows // b), v,
                       rng.random() < 0.7, rng.random() < 0.7, rng.choice(("token", "sequence")))
    width, states = _log_uniform(rng, 3, 2047), rng.choice((8, 32))
    return _adamw(None, "blocks" if width > 400 else rng.choice(("blocks", "layers")), width,
                  rng.randint(1, 3 if width > 1000 else 6), rng.choice(sorted(DTYPES)), states)


def _numels(case):
    w, n = case["width"], case["count"]
    if case["layout"] == "layers":  # 16 characters in, n hidden layers, 128 out
        return [16 * w * 129] + n * [w * w * 5] + [w * 128 * 5]
    return n * [w * w, w, 4 * w * w, 4 * w, 4 * w * w, w]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def prepare(case, seed):
    return {"recurrence": _prepare_recurrence, "policy": _prepare_policy,
            "adamw": _prepare_adamw}[case["op"]](case, seed)


def _lengths(b, l):
    """Evenly spread from 0 to l, the longest first."""
    return [l - (l * i) // max(1, b - 1) if b > 1 else l for i in range(b)]


def _prepare_recurrence(case, seed):
    gen, dt = _generator(seed), DTYPES[case["dtype"]]
    b, l, d = case["b"], case["l"], case["d"]

    def normal(*shape, mean=0.0, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * std + mean).to(dtype)

    if case["mode"] == "step":
        return {"case": case, "z": normal(b, d), "f": normal(b, d, mean=2.0, std=1.5),
                "h": normal(b, d, dtype=torch.float32)}
    if case["packed"]:
        both = torch.cat([normal(b, l, d), normal(b, l, d, mean=2.0, std=1.5)], -1)
        z, f = both[..., :d], both[..., d:]
    else:
        z, f = normal(b, l, d), normal(b, l, d, mean=2.0, std=1.5)
    state = {"case": case, "z": z, "f": f, "h0": None, "lengths": None, "reset": None}
    if case["carried"]:
        state["h0"] = normal(b, d, dtype=torch.float32)
    if case["lengths"]:
        order = torch.randperm(b, generator=gen, device=DEVICE)
        state["lengths"] = torch.tensor(_lengths(b, l), device=DEVICE, dtype=torch.int32)[order]
    if case["resets"]:  # documents of a thousand tokens or so, back to back
        state["reset"] = torch.rand(b, l, generator=gen, device=DEVICE) < 1e-3
    if case["mode"] == "train":
        state["gy"] = normal(b, l, d)
        state["gh"] = normal(b, d, dtype=torch.float32)
        for name in ("z", "f", "h0"):
            if state[name] is not None:
                state[name] = state[name].detach().requires_grad_()
    return state


def _prepare_policy(case, seed):
    gen, dt = _generator(seed), DTYPES[case["dtype"]]
    b, t, v = case["b"], case["t"], case["v"]
    logits = torch.empty(b, t, v, device=DEVICE, dtype=dt)
    tokens = torch.empty(b, t, device=DEVICE, dtype=torch.int64)
    logp = torch.empty(b, t, device=DEVICE)
    for i in range(b):  # a sequence at a time: the whole in 32 bits is several times the logits
        logits[i] = (torch.randn(t, v, generator=gen, device=DEVICE) * 2.0).to(dt)
        x = logits[i].float()
        # sampled tokens: the largest of logits + Gumbel noise
        noise = -torch.log(-torch.log(torch.rand(t, v, generator=gen, device=DEVICE).clamp(1e-9, 1 - 1e-7)))
        tokens[i] = (x + noise).argmax(-1)
        logp[i] = torch.log_softmax(x, -1).gather(-1, tokens[i, :, None])[:, 0]
    mask = None
    if case["mask"]:  # a prompt in front and padding behind; the second of several sequences is empty
        at = torch.arange(t, device=DEVICE)
        first = torch.randint(0, t // 4 + 1, (b, 1), generator=gen, device=DEVICE)
        last = torch.randint(t // 2, t + 1, (b, 1), generator=gen, device=DEVICE)
        if b > 2:
            last[1] = first[1]
        mask = (at >= first) & (at < last)
        tokens = torch.where(mask, tokens, torch.full_like(tokens, -100))
    state = {"case": case, "logits": logits, "tokens": tokens, "mask": mask}
    if case["mode"] == "train":
        state["logits"] = logits.requires_grad_()
        state["old"] = logp + 0.2 * torch.randn(b, t, generator=gen, device=DEVICE)
        state["adv"] = torch.randn(b, t, generator=gen, device=DEVICE)
        state["ref"] = logp + 0.3 * torch.randn(b, t, generator=gen, device=DEVICE) if case["kl"] else None
    return state


def _prepare_adamw(case, seed):
    """Every tensor starts on a multiple of 256 entries of one buffer, so that a whole buffer is one
    output; the entries between two tensors are zeros and stay zeros."""
    gen, dt = _generator(seed), DTYPES[case["dtype"]]
    sizes = _numels(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    live = torch.zeros(total, device=DEVICE)
    for s, n in zip(starts, sizes):
        live[s:s + n] = 1.0

    def normal(std):
        return torch.randn(total, generator=gen, device=DEVICE).mul_(std).mul_(live)

    scale = torch.exp(normal(1.0))  # gradients of different weights differ in size
    state = {"case": case, "seed": seed & 0x7FFFFFFF, "starts": starts, "sizes": sizes}
    flat = {"master": normal(0.02), "g": normal(1e-3).mul_(scale).to(dt)}
    flat["p"] = flat["master"].to(dt) if case["dtype"] != "float32" else flat["master"]
    m = normal(3e-4).mul_(scale)
    v = normal(1e-3).mul_(scale).square_()
    if case["states"] == 8:
        word = _words(total, None, torch.zeros((), dtype=torch.int64, device=DEVICE))
        flat["m"], flat["m_exp"] = _encode(m, word[0], 14, True)
        flat["v"], flat["v_exp"] = _encode(v, word[1], 30, False)
    else:
        flat["m"], flat["v"] = m, v
    state["flat"] = flat
    state["parts"] = {}
    for name, x in flat.items():
        if name.endswith("_exp"):
            state["parts"][name] = [x[s // BLOCK:s // BLOCK + -(-n // BLOCK)] for s, n in zip(starts, sizes)]
        else:
            state["parts"][name] = [x[s:s + n] for s, n in zip(starts, sizes)]
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"recurrence": _own_recurrence, "policy": _own_policy, "adamw": _own_adamw}[op](state)
    return {"recurrence": _plain_recurrence, "policy": _plain_policy, "adamw": _plain_adamw}[op](state)


def _own_recurrence(s):
    from language_interpolation_amd import functional as PF
    if s["case"]["mode"] == "step":
        y = PF.gated_recurrence_step(s["z"], s["f"], s["h"])
        return {"y": y, "h": s["h"]}
    y, h = PF.gated_recurrence(s["z"], s["f"], h0=s["h0"], lengths=s["lengths"], reset=s["reset"])
    out = {"y": y, "h": h}
    if s["case"]["mode"] == "train":
        names = [n for n in ("z", "f", "h0") if s[n] is not None]
        grads = torch.autograd.grad((y, h), [s[n] for n in names], (s["gy"], s["gh"]))
        out.update({"g" + n: g for n, g in zip(names, grads)})
    return out


def _own_policy(s):
    from language_interpolation_amd import functional as PF
    if s["case"]["mode"] == "score":
        return PF.token_log_probs(s["logits"], s["tokens"], mask=s["mask"])
    loss, kl, clipped = PF.clipped_policy_loss(
        s["logits"], s["tokens"], s["old"], s["adv"], ref_logp=s["ref"], mask=s["mask"],
        clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL if s["ref"] is not None else 0.0,
        reduction=s["case"]["reduction"])
    (g,) = torch.autograd.grad(loss, s["logits"])
    return {"loss": loss, "kl": kl, "clipped": clipped, "g": g}


def _own_adamw(s):
    from language_interpolation_amd import functional as PF
    parts, eight = s["parts"], s["case"]["states"] == 8
    PF.adamw_step(parts["p"], parts["g"], parts["m"], parts["v"], STEP, lr=LR, betas=BETAS, eps=EPS,
                  weight_decay=DECAY, masters=parts["master"] if s["case"]["dtype"] != "float32" else None,
                  avg_exponents=parts["m_exp"] if eight else None,
                  sq_exponents=parts["v_exp"] if eight else None, seed=s["seed"])
    out = dict(s["flat"])
    if eight:
        out["m"] = PF.decode_moment(out["m"], out.pop("m_exp"), signed=True, dtype=torch.bfloat16)
        out["v"] = PF.decode_moment(out["v"], out.pop("v_exp"), signed=False, dtype=torch.bfloat16)
    del out["g"]
    return out


def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1: pairs of steps are joined, then pairs of pairs, ..."""
    k, l = 1, a.shape[1]
    while k < l:
        u = torch.cat([u[:, :k], u[:, k:] + a[:, k:] * u[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return u


def _plain_recurrence(s):
    case = s["case"]
    z, f = s["z"].detach().float(), s["f"].detach().float()
    a, rest = 1 / (1 + torch.exp(-f)), 1 / (1 + torch.exp(f))
    if case["mode"] == "step":
        s["h"].copy_(a * s["h"] + rest * z)
        return {"y": s["h"].to(s["z"].dtype), "h": s["h"]}
    b, l, d = z.shape
    h0 = s["h0"].detach() if s["h0"] is not None else torch.zeros(b, d, device=z.device)
    live = torch.ones(b, l, 1, dtype=torch.bool, device=z.device)
    if s["lengths"] is not None:
        live = (torch.arange(l, device=z.device) < s["lengths"][:, None])[..., None]
    keep = a if s["reset"] is None else torch.where(s["reset"][..., None], torch.zeros_like(a), a)
    # behind the end the state stays as it is
    keep = torch.where(live, keep, torch.ones_like(keep))
    u = torch.where(live, rest * z, torch.zeros_like(z))
    u[:, 0] += keep[:, 0] * h0
    h = _scan(keep, u)
    out = {"y": torch.where(live, h, torch.zeros_like(h)).to(s["z"].dtype), "h": h[:, -1]}
    if case["mode"] == "train":
        gy = torch.where(live, s["gy"].float(), torch.zeros_like(h))
        gy[:, -1] += s["gh"]
        follow = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)  # a_{t+1} carries e back
        e = _scan(follow.flip(1), gy.flip(1)).flip(1)
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        if s["reset"] is not None:
            before = torch.where(s["reset"][..., None], torch.zeros_like(before), before)
        zero = torch.zeros_like(e)
        out["gz"] = torch.where(live, e * rest, zero).to(s["z"].dtype)
        out["gf"] = torch.where(live, e * (a * rest) * (before - z), zero).to(s["z"].dtype)
        if s["h0"] is not None:
            out["gh0"] = keep[:, 0] * e[:, 0]
    return out


def _weights(mask, b, t, reduction, dtype):
    """The weight of each token in the mean; a batch without tokens has only zeros."""
    m = torch.ones(b, t, device=DEVICE, dtype=dtype) if mask is None else mask.to(dtype)
    if reduction == "token":
        return m / m.sum().clamp(min=1)
    count = m.sum(1, keepdim=True)
    return m / count.clamp(min=1) / (count > 0).sum().clamp(min=1)


def _plain_policy(s):
    case, mask = s["case"], s["mask"]
    x = s["logits"].detach().float()
    tokens = s["tokens"] if mask is None else torch.where(mask, s["tokens"], torch.zeros_like(s["tokens"]))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, dtype=torch.float64)
    at = (x.gather(-1, tokens[..., None]) - top)[..., 0]
    lp = at.double() - torch.log(total)  # whether a ratio is clipped is decided in 64 bits
    if case["mode"] == "score":
        lp = lp.float()
        return lp if mask is None else torch.where(mask, lp, torch.zeros_like(lp))
    adv, w = s["adv"], _weights(mask, case["b"], case["t"], case["reduction"], torch.float32)
    rho = torch.exp(lp - s["old"])
    clipped = torch.where(adv >= 0, rho > 1 + CLIP_HIGH, rho < 1 - CLIP_LOW)
    border = torch.where(adv >= 0, 1 + CLIP_HIGH, 1 - CLIP_LOW)
    term = -torch.where(clipped, border, rho).float() * adv
    coef = torch.where(clipped, torch.zeros_like(adv), -adv * rho.float())
    k = torch.zeros_like(adv)
    if s["ref"] is not None:
        delta = (s["ref"] - lp).float()
        k = torch.exp(delta) - delta - 1
        term, coef = term + KL * k, coef + KL * (1 - torch.exp(delta))
    zero = torch.zeros_like(adv)
    live = w > 0

    def mean(q):
        return torch.where(live, w * q, zero).sum()

    c = torch.where(live, w * coef, zero)[..., None]
    g = p.mul_((1 / total).float()[..., None]).mul_(-c)
    g.scatter_add_(-1, tokens[..., None], c)
    return {"loss": mean(term), "kl": mean(k), "clipped": mean(clipped.float()), "g": g.to(s["logits"].dtype)}


def _mix(x):
    """32 random-looking bits of a 32-bit counter (int64 holding unsigned values)."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B9) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xD1B54A33) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _words(total, state, key):
    """The two random bytes of each entry: bytes of two 32-bit words for every four entries."""
    at = torch.arange(total, device=DEVICE)
    if state is not None:  # entries are counted from the start of their tensor, each has a key
        starts = torch.tensor(state["starts"], device=DEVICE)
        which = torch.bucketize(at, starts, right=True) - 1
        at = at - starts[which]
        key = _mix((key + which) & 0xFFFFFFFF)
    word = ((at >> 2) * 2 + key) & 0xFFFFFFFF
    shift = (at & 3) * 8
    return [((_mix((word + i) & 0xFFFFFFFF) >> shift) & 255).int() for i in (0, 1)]


def _key(seed, step):
    at = torch.tensor([step & 0xFFFFFFFF], device=DEVICE)
    return _mix(_mix(at) ^ (seed & 0xFFFFFFFF))


def _encode(x, byte, top, signed):
    """8-bit codes and the block exponents: |x| is scaled by a power of two so that the block's
    largest has the exponent field `top`, three bits of mantissa stay, the rest is rounded up with
    the probability that it stands for; a positive second moment never becomes zero."""
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    exponent = size.view(-1, BLOCK).amax(1).view(torch.int32) >> 23
    power = torch.exp2((top - exponent).double()).repeat_interleave(BLOCK)
    bits = (size.double() * power).float().view(torch.int32)
    code = (bits + (byte << 12) + 2048) >> 20
    if signed:
        code = torch.where(torch.isfinite(x), code, 127) + torch.signbit(x).int() * 128
    else:
        code = torch.where(torch.isfinite(x), torch.maximum(code, (x > 0).int()), 255)
    return code.to(torch.uint8), exponent.to(torch.uint8)


def _decode(code, exponent, top, signed):
    code = code.int()
    size = ((code & 127 if signed else code) << 20).view(torch.float32).double()
    size = (size * torch.exp2((exponent.int() - top).double()).repeat_interleave(BLOCK)).float()
    size = torch.where((code & 127 if signed else code) == (127 if signed else 255), torch.nan, size)
    return torch.where(code > 127, -size, size) if signed else size


def _plain_adamw(s):
    flat, (b1, b2), eight = s["flat"], BETAS, s["case"]["states"] == 8
    g, p = flat["g"].float(), flat["master"]
    m = _decode(flat["m"], flat["m_exp"], 14, True) if eight else flat["m"]
    v = _decode(flat["v"], flat["v_exp"], 30, False) if eight else flat["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    denominator = torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** STEP)) + EPS
    p.copy_(p * (1 - LR * DECAY) - (m / denominator) * (LR / (1 - b1 ** STEP)))
    if s["case"]["dtype"] != "float32":
        flat["p"].copy_(p)
    if eight:
        word = _words(p.numel(), s, _key(s["seed"], STEP))
        for name, x, w, top, signed in (("m", m, word[0], 14, True), ("v", v, word[1], 30, False)):
            code, exponent = _encode(x, w, top, signed)
            flat[name].copy_(code)
            flat[name + "_exp"].copy_(exponent)
        m = _decode(flat["m"], flat["m_exp"], 14, True).to(torch.bfloat16)
        v = _decode(flat["v"], flat["v_exp"], 30, False).to(torch.bfloat16)
    else:
        flat["m"].copy_(m)
        flat["v"].copy_(v)
        m, v = flat["m"], flat["v"]
    return {"master": p, "p": flat["p"], "m": m, "v": v}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "recurrence":
        b, l, d, s = case["b"], case["l"], case["d"], SIZE[case["dtype"]]
        if case["mode"] == "step":
            return {"bytes": b * d * (3 * s + 8), "flops": 12 * b * d}
        n = d * (sum(_lengths(b, l)) if case["lengths"] else b * l)
        train = case["mode"] == "train"
        outputs = 3 if train else 1  # whole, zeros behind the ends too
        moved = n * s * (3 if train else 2) + outputs * b * l * d * s
        moved += b * d * 4 * (1 + case["carried"] + train * (1 + case["carried"]))
        moved += b * l * case["resets"] + 4 * b * case["lengths"]
        return {"bytes": moved, "flops": n * (30 if train else 12)}
    if case["op"] == "policy":
        rows, v, s = case["b"] * case["t"], case["v"], SIZE[case["dtype"]]
        train = case["mode"] == "train"
        moved = rows * v * s * (2 if train else 1) + rows * (8 + case["mask"])
        moved += rows * 4 * (2 + case["kl"] if train else 1)
        return {"bytes": moved, "flops": rows * v * (7 if train else 4)}
    n, s = sum(_numels(case)), SIZE[case["dtype"]]
    # the weights in 32 bits read and written, the gradient read, a 16-bit copy written
    moved = 8 + s + (s if case["dtype"] != "float32" else 0)
    # 8 bits: codes read and written, and the two moments returned as the values they stand for
    moved += 16 if case["states"] == 32 else 4 + 4
    return {"bytes": n * moved, "flops": n * 16}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "policy": _exact_policy,
                "adamw": _exact_adamw}[case["op"]](state)


def _walk(a, u, h):
    """h_t = a_t h_{t-1} + u_t along dim 1 from h, step by step: the length is cut into about
    sqrt(l) stretches that are walked side by side, then their ends are joined one after another."""
    b, l, d = a.shape
    k = max(1, math.isqrt(l))
    n = -(-l // k)
    pad = n * k - l
    a = torch.cat([a, a.new_ones(b, pad, d)], 1).view(b, n, k, d)
    u = torch.cat([u, u.new_zeros(b, pad, d)], 1).view(b, n, k, d)
    out, through = torch.empty_like(u), torch.empty_like(a)
    x, y = u.new_zeros(b, n, d), a.new_ones(b, n, d)
    for j in range(k):
        x, y = a[:, :, j] * x + u[:, :, j], a[:, :, j] * y
        out[:, :, j], through[:, :, j] = x, y
    for i in range(n):
        out[:, i] += through[:, i] * h[:, None]
        h = out[:, i, -1]
    return out.view(b, n * k, d)[:, :l]


def _exact_recurrence(s):
    case = s["case"]
    z, f = s["z"].double(), s["f"].double()
    a = torch.sigmoid(f)
    if case["mode"] == "step":
        h = z + a * (s["h"].double() - z)
        return {"y": h, "h": h}
    b, l, d = z.shape
    ends = s["lengths"].long() if s["lengths"] is not None else torch.full((b,), l, device=z.device)
    behind = torch.arange(l, device=z.device)[None] >= ends[:, None]
    h0 = s["h0"].double() if s["h0"] is not None else z.new_zeros(b, d)
    pass_on = a.clone()
    if s["reset"] is not None:
        pass_on[s["reset"]] = 0.0
    pass_on[behind] = 1.0
    u = z * torch.sigmoid(-f)
    u[behind] = 0.0
    h = _walk(pass_on, u, h0)
    y = h.clone()
    y[behind] = 0.0
    out = {"y": y, "h": h[:, -1].clone()}
    if case["mode"] == "train":
        back = s["gy"].double()
        back[behind] = 0.0
        # e_t = gy_t + pass_{t+1} e_{t+1}: walked from the last step with gh arriving there
        onward = torch.cat([pass_on[:, 1:], pass_on.new_ones(b, 1, d)], 1)
        e = _walk(onward.flip(1), back.flip(1), s["gh"].double()).flip(1)
        prior = torch.cat([h0[:, None], h[:, :-1]], 1)
        if s["reset"] is not None:
            prior[s["reset"]] = 0.0
        gz, gf = e * torch.sigmoid(-f), e * a * torch.sigmoid(-f) * (prior - z)
        gz[behind], gf[behind] = 0.0, 0.0
        out["gz"], out["gf"] = gz, gf
        if s["h0"] is not None:
            out["gh0"] = e[:, 0] * pass_on[:, 0]
    return out


def _exact_policy(s):
    case, mask = s["case"], s["mask"]
    b, t, v = s["logits"].shape
    lp = torch.zeros(b, t, dtype=torch.float64, device=DEVICE)
    w = _weights(mask, b, t, case["reduction"], torch.float64)
    chosen = s["tokens"].clamp(min=0)
    g = torch.zeros(b, t, v, dtype=torch.float64, device=DEVICE) if case["mode"] == "train" else None
    sums = torch.zeros(3, dtype=torch.float64, device=DEVICE)
    for i in range(b):  # a sequence at a time
        logs = torch.log_softmax(s["logits"][i].double(), -1)
        lp[i] = logs.gather(-1, chosen[i, :, None])[:, 0]
        if g is None:
            continue
        ratio, adv = torch.exp(lp[i] - s["old"][i].double()), s["adv"][i].double()
        free, held = ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
        value, slope = -torch.minimum(free, held), torch.where(free > held, 0.0, -free)
        kl = torch.zeros_like(value)
        if s["ref"] is not None:
            gap = s["ref"][i].double() - lp[i]
            kl = torch.expm1(gap) - gap
            value, slope = value + KL * kl, slope - KL * torch.expm1(gap)
        terms = torch.stack([value, kl, (free > held).double()])
        sums += torch.where(w[i] > 0, terms * w[i], 0.0).sum(1)
        c = torch.where(w[i] > 0, slope * w[i], 0.0)
        g[i] = -c[:, None] * torch.exp(logs)
        g[i].scatter_add_(-1, chosen[i, :, None], c[:, None])
    if g is None:
        return lp if mask is None else torch.where(mask, lp, 0.0)
    return {"loss": sums[0], "kl": sums[1], "clipped": sums[2], "g": g}


def _round_by_definition(x, byte, top, signed):
    """The value that the 8-bit code of x stands for, found on the grid of such values."""
    size = torch.where(torch.isfinite(x), x.abs(), 0.0)
    largest = size.view(-1, BLOCK).amax(1)
    e = torch.where(largest > 0, torch.frexp(largest)[1].double() + 126, 0.0).clamp(min=0).repeat_interleave(BLOCK)
    scaled = size * torch.exp2(top + 126 - e)  # in units of 2^-126
    power = torch.exp2(torch.floor(torch.log2(scaled.clamp(min=1.0))))
    grid = power / 8
    low = torch.floor(scaled / grid)
    rounded = torch.where(scaled / grid - low + (byte.double() + 0.5) / 256 >= 1, low + 1, low) * grid
    if not signed:
        rounded = torch.where((x > 0) & (rounded == 0), 1.0 / 8, rounded)
    return torch.sign(x) * rounded * 2.0 ** -126 * torch.exp2(e - top)


def _exact_adamw(s):
    flat, (b1, b2), eight = s["flat"], BETAS, s["case"]["states"] == 8
    m, v, g = flat["m"], flat["v"], flat["g"].double()
    if eight:
        m, v = _decode(m, flat["m_exp"], 14, True), _decode(v, flat["v_exp"], 30, False)
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g.square()
    step = (m / (1 - b1 ** STEP)) / (torch.sqrt(v / (1 - b2 ** STEP)) + EPS)
    p = flat["master"].double() * (1 - LR * DECAY) - LR * step
    if eight:
        word = _words(p.numel(), s, _key(s["seed"], STEP))
        m, v = _round_by_definition(m, word[0], 14, True), _round_by_definition(v, word[1], 30, False)
    return {"master": p, "p": p, "m": m, "v": v}
