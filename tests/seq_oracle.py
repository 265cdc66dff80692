"""Plain restatements of the sequence-model operators in 64 bits on the CPU, each with a bound on the
error of an fp32 implementation that follows from its roundings (test infrastructure).

U = 2^-24 is the relative error of one fp32 operation; a correctly rounded or 1-ulp elementary
function is counted as 2 U.  half(t) = eps(t)/2 is the error of one rounding to the type t."""
import numpy as np
import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the subnormals: the error of a rounding near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def recurrence(z, f, h0=None, lengths=None, reset=None, gy=None, gh=None):
    """dict of (value, bound) for y, h and, with gy, gz, gf, gh0.  A step computes two gates (exp, add,
    divide: 8 U relative each) and an fma, so it adds at most 16 U (|h| + |z|) to the error it passes
    on with the factor a; the joining of stretches (product of gates times the state) is of the same
    order a step, counted once more: 32 U."""
    dt = z.dtype
    b, l, d = z.shape
    z, f = z.double(), f.double()
    a, r = torch.sigmoid(f), torch.sigmoid(-f)
    n = torch.full((b,), l) if lengths is None else lengths.long().clamp(0, l)
    live = torch.arange(l)[None] < n[:, None]
    drop = torch.zeros(b, l, dtype=torch.bool) if reset is None else reset.bool()
    h = torch.zeros(b, d, dtype=torch.float64) if h0 is None else h0.double().clone()
    e = torch.zeros_like(h)
    y, prev = torch.zeros(b, l, d, dtype=torch.float64), torch.zeros(b, l, d, dtype=torch.float64)
    ey, eprev = torch.zeros_like(y), torch.zeros_like(y)
    for t in range(l):
        on = live[:, t, None]
        hp = torch.where(drop[:, t, None], 0.0, h)
        ep = torch.where(drop[:, t, None], 0.0, e)
        zt = torch.where(on, z[:, t], 0.0)
        at, rt = torch.where(on, a[:, t], 0.0), torch.where(on, r[:, t], 0.0)
        new = at * hp + rt * zt
        enew = at * ep + 32 * U * (at * hp.abs() + rt * zt.abs() + at * zt.abs())
        prev[:, t], eprev[:, t] = hp, ep
        h, e = torch.where(on, new, h), torch.where(on, enew, e)
        y[:, t], ey[:, t] = torch.where(on, new, 0.0), torch.where(on, enew, 0.0)
    out = {"y": (y, ey + half(dt) * y.abs() + tiny(dt)), "h": (h, e + 2.0 ** -140)}
    if gy is None:
        return out
    gz, gf = torch.zeros_like(y), torch.zeros_like(y)
    bz, bf = torch.zeros_like(y), torch.zeros_like(y)
    u = torch.zeros(b, d, dtype=torch.float64) if gh is None else gh.double().clone()
    eu = torch.zeros_like(u)
    for t in reversed(range(l)):
        on = live[:, t, None]
        gt = torch.where(on, gy[:, t].double(), 0.0)
        at, rt = torch.where(on, a[:, t], 0.0), torch.where(on, r[:, t], 0.0)
        zt = torch.where(on, z[:, t], 0.0)
        g = gt + u
        eg = eu + 4 * U * (gt.abs() + u.abs())
        gap = prev[:, t] - zt
        gz[:, t] = torch.where(on, g * rt, 0.0)
        gf[:, t] = torch.where(on, g * at * rt * gap, 0.0)
        bz[:, t] = rt * eg + 16 * U * (g * rt).abs()
        bf[:, t] = at * rt * (eg * gap.abs() + g.abs() * (eprev[:, t] + 4 * U * (prev[:, t].abs() + zt.abs()))) \
            + 32 * U * gf[:, t].abs()
        unew = torch.where(drop[:, t, None], 0.0, at * g)
        eunew = torch.where(drop[:, t, None], 0.0, at * eg + 32 * U * (at * g).abs())
        u, eu = torch.where(on, unew, u), torch.where(on, eunew, eu)
    out["gz"] = (gz, bz + half(dt) * gz.abs() + tiny(dt))
    out["gf"] = (gf, bf + half(dt) * gf.abs() + tiny(dt))
    out["gh0"] = (u, eu + 2.0 ** -140)
    return out


def policy(logits, tokens, old=None, adv=None, ref=None, mask=None, low=0.2, high=0.2, beta=0.0,
           reduction="token", gout=1.0, coef=None):
    """dict of (value, bound): lp; with old: loss, kl, clipped, grad; with coef: grad of sum coef lp.

    lp = (x - max) - log(sum exp(x - max)): the difference has U |x - max|, an exp 4 U relative and U
    |x - max| from its argument, a sum of v terms in lanes of at most v/64 and a tree 2^6 or more
    (v/64 + 16) U relative, the log 2 U of its size and the sum's relative error."""
    dt = logits.dtype
    b, t, v = logits.shape
    m = torch.ones(b, t, dtype=torch.bool) if mask is None else mask.bool()
    x = torch.where(m[..., None], logits.double(), 0.0)
    tok = torch.where(m, tokens.long(), 0)
    logs = torch.log_softmax(x, -1)
    lp = logs.gather(-1, tok[..., None])[..., 0]
    top = x.amax(-1)
    p = logs.exp()
    # error of exp weighted by its share: U sum p |x - max|
    spread = (p * (x - top[..., None]).abs().nan_to_num(posinf=0.0)).sum(-1)
    esum = (v / 64 + 24) * U + U * spread
    elp = U * 2 * (lp.abs() + (x.gather(-1, tok[..., None])[..., 0] - top).abs()) + esum + 4 * U
    out = {"lp": (torch.where(m, lp, 0.0), torch.where(m, elp, 0.0))}
    hit = torch.zeros(b, t, v, dtype=torch.float64).scatter_(-1, tok[..., None], 1.0)
    # (a share below the smallest normal number of fp32 may come out as a subnormal of fewer bits, or
    # as zero: an absolute error of up to 2^-126 in the share whatever its size)
    ep = p * (4 * U * ((x - top[..., None]).abs().nan_to_num(posinf=0.0) + 8) + esum[..., None]) + 2.0 ** -126
    if coef is not None:
        c = torch.where(m, coef.double(), 0.0)[..., None]
        g = c * (hit - p)
        out["grad"] = (g, c.abs() * (ep + 4 * U * (hit + p)) + half(dt) * g.abs() + tiny(dt))
    if old is None:
        return out
    adv = adv.double()[:, None].expand(b, t) if adv.dim() == 1 else adv.double()
    n = m.double().sum(1, keepdim=True)
    if reduction == "token":
        w = m.double() / max(float(m.sum()), 1.0)
    else:
        w = m.double() / n.clamp(min=1) / max(float((n > 0).sum()), 1.0)
    o = torch.where(m, old.double(), lp)
    rho = (lp - o).exp()
    free, held = rho * adv, rho.clamp(1 - low, 1 + high) * adv
    cut = free > held
    term, c = -torch.minimum(free, held), torch.where(cut, 0.0, -free)
    eterm = torch.where(cut, 4 * U * held.abs(), free.abs() * (elp + U * (lp - o).abs() * 2 + 8 * U))
    ec = torch.where(cut, 0.0, eterm)
    kl = torch.zeros_like(term)
    ekl = torch.zeros_like(term)
    if ref is not None:
        gap = torch.where(m, ref.double(), lp) - lp
        egap = elp + 2 * U * (ref.double().abs().nan_to_num() + lp.abs())
        kl = torch.expm1(gap) - gap
        ekl = torch.expm1(gap).abs() * egap + 8 * U * (gap.abs() + torch.expm1(gap).abs()) + egap ** 2
        term, eterm = term + beta * kl, eterm + beta * ekl
        c = c - beta * torch.expm1(gap)
        ec = ec + beta * (torch.exp(gap) * egap + 8 * U * torch.expm1(gap).abs())
    ok = w > 0

    def mean(q):
        return torch.where(ok, w * q, 0.0).sum()

    for name, q, e in (("loss", term, eterm), ("kl", kl, ekl), ("clipped", cut.double(), 0 * ekl)):
        # a weight and a product of fp32, a sum in 64 bits, one rounding
        out[name] = (mean(q), mean(e + 8 * U * q.abs()) + 2.0 ** -140)
    c = torch.where(ok, gout * w * c, 0.0)[..., None]
    ec = torch.where(ok, abs(gout) * w * ec, 0.0)[..., None]
    g = c * (hit - p)
    out["grad"] = (g, c.abs() * (ep + 8 * U * (hit + p)) + ec * (hit - p).abs() + half(dt) * g.abs() + tiny(dt))
    return out


def check(got, want, what):
    """got within the bound of want = (value, bound); where the value is no number, so is got."""
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: finite where the other is not"
    off = ((got - value).abs() - bound)[fine]
    if off.numel() and float(off.max()) > 0:
        at = (((got - value).abs() - bound).nan_to_num(nan=-1.0)).argmax()
        raise AssertionError(f"{what}: {got.flatten()[at]} instead of {value.flatten()[at]}, bound "
                             f"{bound.flatten()[at]}, at {int(at)} of {tuple(value.shape)}; "
                             f"{int((off > 0).sum())} entries")


# ---------------------------------------------------------------------------------------------
# AdamW in numpy fp32, operation by operation: the kernel has to give the same bits
# ---------------------------------------------------------------------------------------------
def mix(x):
    x = np.asarray(x, dtype=np.uint32).copy()
    x ^= x >> np.uint32(16)
    x *= np.uint32(0x9E3779B9)
    x ^= x >> np.uint32(15)
    x *= np.uint32(0xD1B54A33)
    return x ^ (x >> np.uint32(16))


def noise(n, seed, step, index):
    """The two random bytes of every entry."""
    with np.errstate(over="ignore"):
        key = mix(mix(mix(np.uint32(step)) ^ np.uint32(seed)) + np.uint32(index))
        e = np.arange(n, dtype=np.uint32)
        q = key + np.uint32(2) * (e >> np.uint32(2))
        shift = np.uint32(8) * (e & np.uint32(3))
        return [(mix(q + np.uint32(i)) >> shift) & np.uint32(255) for i in (0, 1)]


def _blocks(x):
    return np.repeat(x, 256)


def encode(x, byte, top, signed):
    n = x.size
    size = np.where(np.isfinite(x), np.abs(x), np.float32(0)).astype(np.float32)
    padded = np.concatenate([size, np.zeros(-n % 256, np.float32)]).reshape(-1, 256)
    exponent = (padded.max(1).view(np.uint32) >> np.uint32(23)).astype(np.int64)
    t = np.ldexp(size.astype(np.float64), top - _blocks(exponent)[:n]).astype(np.float32)
    code = (t.view(np.uint32) + (byte << np.uint32(12)) + np.uint32(2048)) >> np.uint32(20)
    if signed:
        code = np.where(np.isfinite(x), code, 127) | np.where(np.signbit(x), 128, 0)
    else:
        code = np.where(np.isfinite(x), np.maximum(code, x > 0), 255)
    return code.astype(np.uint8), exponent.astype(np.uint8)


def decode(code, exponent, top, signed):
    mag = (code & 127 if signed else code).astype(np.uint32)
    t = (mag << np.uint32(20)).view(np.float32).astype(np.float64)
    x = np.ldexp(t, _blocks(exponent.astype(np.int64))[:code.size] - top).astype(np.float32)
    x = np.where(mag == (127 if signed else 255), np.float32(np.nan), x)
    return np.where(code > 127, -x, x).astype(np.float32) if signed else x


def adamw(w, g, m, v, step, lr, betas, eps, wd, scale=1.0):
    """New (w, m, v), fp32 arrays."""
    f = np.float32
    b1, b2 = betas
    with np.errstate(all="ignore"):
        g = g * f(scale)
        m = m * f(b1) + g * f(1 - b1)
        v = v * f(b2) + (g * g) * f(1 - b2)
        c1, c2 = f(lr / (1 - b1 ** step)), f(1 / np.sqrt(1 - b2 ** step))
        w = w * f(1 - lr * wd) - (m / (np.sqrt(v) * c2 + f(eps))) * c1
    return w.astype(f), m.astype(f), v.astype(f)
