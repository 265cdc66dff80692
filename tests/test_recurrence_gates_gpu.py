"""The gated recurrence with gates near 1 from an empty state: what the input adds, (1 - a) z, is all there is of the state,
so its digits are those of 1 - a."""
import pytest
import torch

import seq_oracle as so
from language_interpolation_amd import functional as PF

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = so.U


def _walk(z, f, h0=None, gy=None, gh=None):
    """{name: (value, bound)} in 64 bits.  a and r = 1 - a are computed with at most 8 U of each its own size (an exponential
    2 U, an addition U, a reciprocal 2 U, for r a product U more), their products with the state and the input are rounded
    once: a step adds 16 U (a |h| + r |z|) to the error that it passes on with the factor a.  The joining of stretches
    (product of gates times the state) is of the same order, counted once more: 32 U."""
    dt = z.dtype
    z, f = z.double(), f.double()
    a, r = torch.sigmoid(f), torch.sigmoid(-f)
    b, l, d = z.shape
    h = torch.zeros(b, d, dtype=torch.float64) if h0 is None else h0.double().clone()
    e = torch.zeros_like(h)
    y, ey, before, ebefore = (torch.zeros_like(z) for _ in range(4))
    for t in range(l):
        before[:, t], ebefore[:, t] = h, e
        e = a[:, t] * e + 32 * U * (a[:, t] * h.abs() + r[:, t] * z[:, t].abs())
        h = a[:, t] * h + r[:, t] * z[:, t]
        y[:, t], ey[:, t] = h, e
    out = {"y": (y, ey + so.half(dt) * y.abs() + so.tiny(dt)), "h": (h, e + 2.0 ** -140)}
    if gy is None:
        return out
    gy = gy.double()
    u, eu = gh.double().clone(), torch.zeros_like(h)
    gz, gf, bz, bf = (torch.zeros_like(z) for _ in range(4))
    for t in reversed(range(l)):
        at, rt, gap = a[:, t], r[:, t], before[:, t] - z[:, t]
        g, eg = gy[:, t] + u, eu + 4 * U * (gy[:, t].abs() + u.abs())
        gz[:, t], bz[:, t] = g * rt, rt * eg + 16 * U * (g * rt).abs()
        gf[:, t] = g * at * rt * gap
        egap = ebefore[:, t] + 4 * U * (before[:, t].abs() + z[:, t].abs())
        bf[:, t] = at * rt * (eg * gap.abs() + g.abs() * egap) + 32 * U * gf[:, t].abs()
        u, eu = at * g, at * eg + 32 * U * (at * g).abs()
    out["gz"] = (gz, bz + so.half(dt) * gz.abs() + so.tiny(dt))
    out["gf"] = (gf, bf + so.half(dt) * gf.abs() + so.tiny(dt))
    out["gh0"] = (u, eu + 2.0 ** -140)
    return out


def _inputs(b, l, d, dtype, low, high, seed):
    """Gates that stay the same along a channel, so that errors of one sign add up; inputs of one sign."""
    g = torch.Generator().manual_seed(seed)
    z = (torch.rand(b, l, d, generator=g) + 0.5).to(dtype)
    f = (low + (high - low) * torch.rand(b, 1, d, generator=g)).expand(b, l, d).to(dtype)
    return z, f, torch.randn(b, l, d, generator=g).to(dtype), torch.randn(b, d, generator=g)


# a wave a row; two channels a lane in 16 bits; rows that share waves; several chunks of one row
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("low,high", [(8.0, 20.0), (-20.0, -8.0), (-4.0, 4.0)])
@pytest.mark.parametrize("b,l,d", [(2, 600, 33), (70, 300, 130), (450, 304, 3), (1, 2500, 64)])
def test_states_that_gather_slowly(b, l, d, low, high, dtype):
    z, f, gy, gh = _inputs(b, l, d, dtype, low, high, seed=l + d)
    want = _walk(z, f, None, gy, gh)
    zd, fd, h0 = z.cuda().requires_grad_(), f.contiguous().cuda().requires_grad_(), torch.zeros(b, d, device="cuda", requires_grad=True)
    y, h = PF.gated_recurrence(zd, fd, h0)
    grads = torch.autograd.grad((y, h), (zd, fd, h0), (gy.cuda(), gh.cuda()))
    for name, x in zip(("y", "h", "gz", "gf", "gh0"), (y, h) + grads):
        so.check(x, want[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("low,high", [(8.0, 20.0), (-20.0, -8.0)])
@pytest.mark.parametrize("d", [33, 64])
def test_states_that_gather_token_by_token(d, low, high, dtype):
    z, f, _, _ = _inputs(3, 200, d, dtype, low, high, seed=d)
    want = _walk(z, f)
    zd, fd, h = z.cuda(), f.contiguous().cuda(), torch.zeros(3, d, device="cuda")
    for t in range(200):
        y = PF.gated_recurrence_step(zd[:, t], fd[:, t], h)
        so.check(y, tuple(x[:, t] for x in want["y"]), f"token {t}")
    so.check(h, want["h"], "state")


def test_an_input_far_larger_than_the_state():
    """A single large input through a gate near 1 leaves (1 - a) z of itself, and what was there stays."""
    z = torch.zeros(1, 40, 4)
    z[0, 0], z[0, 20] = 1.0, 1e5
    f = torch.full((1, 40, 4), 15.0)
    f[0, 0] = -3.0
    want = _walk(z, f)
    y, h = PF.gated_recurrence(z.cuda(), f.cuda())
    so.check(y, want["y"], "y")
    so.check(h, want["h"], "h")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_numbers_go_where_the_formula_lets_them(dtype):
    """NaN in a gate or an input reaches the later steps of its channel; an infinite input is an infinite state, until a
    reset; a gate that is closed to the last (f = -inf) drops whatever was finite."""
    inf, nan = float("inf"), float("nan")
    z, f = torch.ones(1, 40, 6), torch.zeros(1, 40, 6)
    f[0, 7, 0], z[0, 7, 1], z[0, 7, 2], z[0, 7, 3] = nan, nan, inf, -inf
    f[0, 9, 4] = -inf
    f[0, 11, 5] = 300.0
    reset = torch.zeros(1, 40, dtype=torch.bool)
    reset[0, 30] = True
    y, h = PF.gated_recurrence(z.to(dtype).cuda(), f.to(dtype).cuda(), reset=reset.cuda())
    y = y[0].float().cpu()
    assert bool(torch.isfinite(y[:7]).all()) and bool(torch.isfinite(y[30:]).all()) and bool(torch.isfinite(h).all())
    assert bool(torch.isnan(y[7:30, :2]).all())
    assert bool((y[7:30, 2] == inf).all()) and bool((y[7:30, 3] == -inf).all())
    assert bool(torch.isfinite(y[:, 4:]).all()) and float(y[9, 4]) == 1.0 and torch.equal(y[11, 5], y[10, 5])
    state = torch.zeros(1, 6, device="cuda")
    for t in range(9):
        out = PF.gated_recurrence_step(z[:, t].to(dtype).cuda(), f[:, t].to(dtype).cuda(), state)[0].float().cpu()
    assert bool(torch.isnan(out[:2]).all()) and float(out[2]) == inf and float(out[3]) == -inf
    assert bool(torch.isfinite(out[4:]).all())
