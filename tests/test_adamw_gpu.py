"""AdamW over many tensors: the same bits as the rule in numpy fp32, operation by operation."""
import numpy as np
import pytest
import torch

import seq_oracle as so

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
# around the vector width, the 256 entries of an exponent and a workgroup's share; > 32 tensors: two launches
SIZES = [1, 2, 3, 4, 5, 255, 256, 257, 1000, 1023, 1024, 1025, 4095, 4099, 8191, 8192, 8193, 20011]
MANY = SIZES + [7 + 13 * i for i in range(30)]


def _tensors(sizes, dtype, bits, seed, off=0):
    """Device lists and their numpy copies; off: elements by which every tensor misses 256 bytes."""
    rng = np.random.default_rng(seed)
    host, dev = [], {k: [] for k in ("w", "p", "g", "m", "v", "me", "ve")}

    def put(x, kind):
        buf = torch.empty(x.size + off, dtype=kind, device="cuda")[off:]
        return buf.copy_(torch.from_numpy(np.ascontiguousarray(x)))
    for n in sizes:
        w = rng.normal(size=n).astype(np.float32)
        g = rng.normal(size=n).astype(np.float32) * np.exp(rng.normal(size=n) * 3).astype(np.float32)
        g[rng.random(n) < 0.1] = 0.0
        g = torch.from_numpy(g).to(dtype).float().numpy()
        m = (rng.normal(size=n) * np.exp(rng.normal(size=n) * 2)).astype(np.float32)
        v = np.square(rng.normal(size=n) * np.exp(rng.normal(size=n) * 2)).astype(np.float32)
        h = {"w": w, "g": g}
        if bits == 8:
            h["m"], h["me"] = so.encode(m, np.zeros(n, np.uint32) + 128, 14, True)
            h["v"], h["ve"] = so.encode(v, np.zeros(n, np.uint32) + 128, 30, False)
        else:
            h["m"], h["v"] = m, v
        host.append(h)
        dev["g"].append(put(g, dtype))
        dev["w"].append(put(w, F32))
        dev["p"].append(dev["w"][-1] if dtype == F32 else put(w, dtype))
        for k in ("m", "v"):
            dev[k].append(put(h[k], torch.uint8 if bits == 8 else F32))
            if bits == 8:
                dev[k + "e"].append(torch.from_numpy(h[k + "e"]).cuda())
    return host, dev


def _step(dev, dtype, bits, step, **kw):
    from language_interpolation_amd import functional as PF
    args = dict(HYPER, **kw)
    PF.adamw_step(dev["p"], dev["g"], dev["m"], dev["v"], step, masters=None if dtype == F32 else dev["w"],
                  avg_exponents=dev["me"] if bits == 8 else None, sq_exponents=dev["ve"] if bits == 8 else None, **args)


def _host_step(host, bits, step, seed=0, scale=1.0):
    for i, h in enumerate(host):
        n = h["w"].size
        m = so.decode(h["m"], h["me"], 14, True) if bits == 8 else h["m"]
        v = so.decode(h["v"], h["ve"], 30, False) if bits == 8 else h["v"]
        h["w"], m, v = so.adamw(h["w"], h["g"], m, v, step, HYPER["lr"], HYPER["betas"], HYPER["eps"],
                                HYPER["weight_decay"], scale)
        if bits == 8:
            # (the numbering of the random bits goes through the launches)
            a, b = so.noise(n, seed, step, i)
            h["m"], h["me"] = so.encode(m, a, 14, True)
            h["v"], h["ve"] = so.encode(v, b, 30, False)
        else:
            h["m"], h["v"] = m, v


def _same(x, y):
    x = x.cpu().numpy()
    return x.dtype == y.dtype and np.array_equal(x, y, equal_nan=x.dtype.kind == "f")


def _compare(host, dev, dtype, bits):
    for i, h in enumerate(host):
        what = (i, h["w"].size)
        assert _same(dev["w"][i], h["w"]), what
        assert _same(dev["p"][i].float(), torch.from_numpy(h["w"]).to(dtype).float().numpy()), what
        for k in ("m", "v") + (("me", "ve") if bits == 8 else ()):
            assert _same(dev[k][i], h[k]), (k,) + what


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("off", [0, 1, 2])
def test_the_same_bits_as_the_rule(dtype, bits, off):
    host, dev = _tensors(MANY, dtype, bits, seed=off, off=off)
    for step in (1, 2, 1000):
        _step(dev, dtype, bits, step, seed=99)
        _host_step(host, bits, step, seed=99)
        _compare(host, dev, dtype, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_scaled_gradients_and_device_counters(bits):
    host, dev = _tensors(SIZES, F32, bits, seed=5)
    scale = torch.tensor(0.37, device="cuda")
    counters = [torch.full((), 6, dtype=torch.int64, device="cuda") for _ in SIZES]
    counters[3] = counters[0]  # shared: advanced once a call
    for step in (7, 8):
        _step(dev, F32, bits, counters, seed=3, grad_scale=scale)
        _host_step(host, bits, step, seed=3, scale=0.37)
        assert all(int(c) == step for c in counters)
    _compare(host, dev, F32, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_large_tensor(bits):
    """Entries behind 2^24, odd size: every workgroup of a long launch, and what lies behind the end."""
    n = (1 << 24) + 12345
    g = torch.Generator(device="cuda").manual_seed(1)
    guard = 64
    flat = {k: torch.randn(n + guard, device="cuda", generator=g) for k in ("p", "g")}
    if bits == 8:
        for k in ("m", "v"):
            flat[k] = torch.randint(0, 100, (n + guard,), device="cuda", generator=g).to(torch.uint8)
        exps = {k: torch.full(((n + 255) // 256 + 1,), 120, dtype=torch.uint8, device="cuda") for k in ("me", "ve")}
    else:
        flat["m"], flat["v"] = flat["p"] * 0.1, flat["g"].square()
    before = {k: x.clone() for k, x in flat.items()}
    dev = {k: [x[:n]] for k, x in flat.items()}
    if bits == 8:
        dev.update({k: [x[:-1]] for k, x in exps.items()})
    _step(dev, F32, bits, 10, seed=1)
    for k, x in flat.items():
        assert torch.equal(x[n:], before[k][n:]), k
    if bits == 8:
        assert all(int(x[-1]) == 120 for x in exps.values())
    for lo in (0, 1 << 20, n - 5000 - n % 256):
        lo -= lo % 256
        hi = min(n, lo + 5120)
        cut = {k: x[lo:hi].cpu().numpy() for k, x in before.items()}
        e = np.full((hi - lo + 255) // 256, 120, np.uint8)
        m = so.decode(cut["m"], e, 14, True) if bits == 8 else cut["m"]
        v = so.decode(cut["v"], e, 30, False) if bits == 8 else cut["v"]
        w, m, v = so.adamw(cut["p"], cut["g"], m, v, 10, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
        assert _same(flat["p"][lo:hi], w)
        if bits == 8:
            a, b = (x[lo:hi] for x in so.noise(hi, 1, 10, 0))
            assert _same(flat["m"][lo:hi], so.encode(m, a, 14, True)[0])
            assert _same(flat["v"][lo:hi], so.encode(v, b, 30, False)[0])
        else:
            assert _same(flat["m"][lo:hi], m) and _same(flat["v"][lo:hi], v)


def test_values_that_are_no_numbers_and_extremes():
    """A gradient that is not finite spoils its own entry, not its block; denormals and the largest."""
    for bits in (32, 8):
        host, dev = _tensors([1000], F32, bits, seed=6)
        bad = {3: np.nan, 260: np.inf, 261: -np.inf, 500: 3e38, 501: 1e-44, 700: -1e-38}
        for at, x in bad.items():
            host[0]["g"][at] = x
            dev["g"][0][at] = float(x)
        _step(dev, F32, bits, 5, seed=2)
        _host_step(host, bits, 5, seed=2)
        if bits == 8:
            _compare(host, dev, F32, bits)
        else:
            assert _same(dev["w"][0], host[0]["w"])
        fine = torch.ones(1000, dtype=torch.bool, device="cuda")
        fine[[3, 260, 261, 500]] = False
        assert bool(torch.isfinite(dev["w"][0][fine]).all())


def test_decoded_moments():
    from language_interpolation_amd import functional as PF
    codes = torch.arange(256, dtype=torch.uint8).repeat(40)[:10001].contiguous()
    exps = torch.randint(0, 255, (40,), generator=torch.Generator().manual_seed(1)).to(torch.uint8)
    for signed, top in ((True, 14), (False, 30)):
        want = so.decode(codes.numpy(), exps.numpy(), top, signed)
        got = PF.decode_moment(codes.cuda(), exps.cuda(), signed)
        assert _same(got, want)
        odd = torch.empty(10009, dtype=torch.uint8, device="cuda")[3:10004].copy_(codes)  # no multiple of 8
        assert _same(PF.decode_moment(odd, exps.cuda(), signed), want)
        for dt in (BF16, F16):
            assert torch.equal(PF.decode_moment(codes.cuda(), exps.cuda(), signed, dt).cpu().nan_to_num(7.0),
                               torch.from_numpy(want).to(dt).nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_eight_bit_blocks_of_every_size(dtype):
    """Blocks from the smallest to the largest exponent, codes of every value (no numbers among them), gradients
    from none to large: v is 0, below 2^-96 or infinite in some waves and ordinary in others."""
    n, rng = 4000 * 256 - 77, np.random.default_rng(12)
    blocks = -(-n // 256)
    host, dev = _tensors([n], dtype, 8, seed=12)
    h = host[0]
    g = rng.normal(size=n) * np.exp2(np.repeat(rng.integers(-70, 30, blocks), 256)[:n])
    g[np.repeat(rng.random(blocks) < 0.3, 256)[:n]] = 0.0
    h["g"] = torch.from_numpy(g.astype(np.float32)).to(dtype).float().numpy()
    for k, none in (("m", 127), ("v", 255)):
        h[k] = rng.integers(0, 256, n).astype(np.uint8)
        every = np.repeat(rng.random(blocks) < 0.8, 256)[:n]  # the other blocks have codes that are no numbers
        h[k][every & ((h[k] & none) == none)] = 5
        h[k + "e"] = rng.integers(0, 255, blocks).astype(np.uint8)
        dev[k][0].copy_(torch.from_numpy(h[k]))
        dev[k + "e"][0].copy_(torch.from_numpy(h[k + "e"]))
    dev["g"][0].copy_(torch.from_numpy(h["g"]))
    for step in (3, 4):
        _step(dev, dtype, 8, step, seed=8)
        with np.errstate(all="ignore"):
            _host_step(host, 8, step, seed=8)
        assert _same(dev["w"][0], h["w"])
        for k, none in (("m", 127), ("v", 255)):  # (the sign of what is no number is not specified)
            got, want = dev[k][0].cpu().numpy(), h[k]
            odd = (want & none) == none
            assert np.array_equal((got & none) == none, odd) and np.array_equal(got[~odd], want[~odd]), k
            assert _same(dev[k + "e"][0], h[k + "e"]), k


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_many_decoded_moments(dt):
    """Enough of them for several turns a thread; the end inside a turn, aligned and not."""
    from language_interpolation_amd import functional as PF
    n = (1 << 23) + 5 * 512 + 13
    g = torch.Generator().manual_seed(2)
    codes = torch.randint(0, 256, (n,), generator=g).to(torch.uint8)
    exps = torch.randint(100, 140, (-(-n // 256),), generator=g).to(torch.uint8)
    odd = torch.empty(n + 3, dtype=torch.uint8, device="cuda")[3:].copy_(codes)
    for signed, top in ((True, 14), (False, 30)):
        want = torch.from_numpy(so.decode(codes.numpy(), exps.numpy(), top, signed)).to(dt).nan_to_num(7.0)
        for c in (codes.cuda(), odd):
            assert torch.equal(PF.decode_moment(c, exps.cuda(), signed, dt).cpu().nan_to_num(7.0), want)


def test_eight_bits_follow_thirty_two():
    """200 steps with drifting gradients: a moment kept in 8 bits has the expected value of the exact
    one, where rounding to nearest would not let v move at all.  Mean over 50 000 entries; an entry's
    error is a sum of roundings of at most 2^-3 of it, remembered for 1/(1-b2) = 1000 steps, so its
    standard deviation is under 2^-3 sqrt(200) < 1.8 of v and that of the mean under 0.8 %: 4 % is
    5 deviations."""
    from language_interpolation_amd import functional as PF
    n, betas = 50_000, (0.9, 0.999)
    gen = torch.Generator(device="cuda").manual_seed(3)
    p = torch.zeros(n, device="cuda")
    m, v = torch.zeros(2, n, dtype=torch.uint8, device="cuda")
    me, ve = torch.zeros(2, PF.moment_blocks(n), dtype=torch.uint8, device="cuda")
    m32, v32 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for step in range(1, 201):
        g = torch.randn(n, device="cuda", generator=gen) * (1.0 if step < 60 else 0.05) + 0.02
        PF.adamw_step([p], [g], [m], [v], step, lr=0.0, betas=betas, avg_exponents=[me], sq_exponents=[ve], seed=11)
        m32.mul_(0.9).add_(g, alpha=0.1)
        v32.mul_(0.999).add_(g * g, alpha=1e-3)
    got = PF.decode_moment(v, ve, signed=False)
    assert bool((got > 0).all())
    assert abs(float(got.mean() / v32.mean()) - 1) < 0.04
    assert abs(float((PF.decode_moment(m, me, signed=True) - m32).mean())) < 0.04 * float(m32.abs().mean())


def test_optimizer_against_torch_in_64_bits():
    """train.AdamW on permuted leaves, groups, a missing gradient; state_dict there and back."""
    from language_interpolation_amd.train import AdamW
    torch.manual_seed(0)
    shapes = [(5, 7, 9), (130, 70), (17,), ()]
    base = [torch.randn(s) for s in shapes]
    ps = [b.clone().cuda().requires_grad_() for b in base]
    ps[0] = base[0].permute(1, 2, 0).contiguous().cuda().permute(2, 0, 1).requires_grad_()
    qs = [b.clone().double().requires_grad_() for b in base]
    mine = AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 1e-2, "weight_decay": 0.0}], lr=3e-3)
    ref = torch.optim.AdamW([{"params": qs[:2]}, {"params": qs[2:], "lr": 1e-2, "weight_decay": 0.0}], lr=3e-3)
    for step in range(6):
        for p, q in zip(ps, qs):
            g = torch.randn(q.shape, generator=torch.Generator().manual_seed(step * 10 + q.dim()))
            p.grad, q.grad = g.cuda(), g.double()
        if step == 2:
            ps[2].grad = qs[2].grad = None
        mine.step()
        ref.step()
        if step == 3:  # go on in a new optimizer
            state = mine.state_dict()
            mine = AdamW([{"params": ps[:2]}, {"params": ps[2:]}], lr=1.0)
            mine.load_state_dict(state)
    for p, q in zip(ps, qs):
        # a step moves a weight by lr (1 + wd) at most and rounds a few times, its ratio m / sqrt(v)
        # is off by some 8 U after 6 steps of 4 roundings: 6 steps x (U |p| + 32 U lr)
        bound = 6 * (2 * so.U * (q.abs().max() + 1) + 64 * so.U * 1e-2)
        assert float((p.detach().cpu().double() - q.detach()).abs().max()) < bound


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_optimizer_keeps_its_types_through_a_checkpoint(dtype, tmp_path):
    from language_interpolation_amd.train import AdamW

    def make():
        g = torch.Generator().manual_seed(1)
        return [torch.randn(s, generator=g).to(dtype).cuda().requires_grad_() for s in ((70, 90), (33,))]

    def grads(ps, step):
        g = torch.Generator().manual_seed(step)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(dtype).cuda()

    a = make()
    opt = AdamW(a, lr=1e-2, moment_bits=8, seed=4)
    for step in range(3):
        grads(a, step)
        opt.step()
    torch.save({"p": a, "opt": opt.state_dict()}, tmp_path / "c.pt")
    grads(a, 3)
    opt.step()
    saved = torch.load(tmp_path / "c.pt", weights_only=True)
    b = [p.detach().clone().requires_grad_() for p in saved["p"]]
    again = AdamW(b, lr=5.0, capturable=False)
    again.load_state_dict(saved["opt"])
    st = again.state[b[0]]
    assert st["exp_avg"].dtype == torch.uint8 and st["exp_avg_exponent"].dtype == torch.uint8
    assert again.state[b[1]]["exp_avg"].dtype == F32  # a small tensor keeps 32 bits
    if dtype != F32:
        assert st["master"].dtype == F32
    grads(b, 3)
    again.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_checkpoint_of_torch_goes_on(dtype):
    """Moments of torch.optim.AdamW (there in the weights' type), then a step here and there in 64 bits."""
    from language_interpolation_amd.train import AdamW
    gen = torch.Generator().manual_seed(7)
    base = torch.randn(60, 30, generator=gen).to(dtype)
    grads = [torch.randn(60, 30, generator=gen).to(dtype) for _ in range(3)]
    p = base.clone().cuda().requires_grad_()
    opt = torch.optim.AdamW([p], lr=1e-2)
    for g in grads[:2]:
        p.grad = g.cuda()
        opt.step()
    state = opt.state_dict()
    mine = AdamW([p], lr=1.0)
    mine.load_state_dict(state)
    st = mine.state[p]
    w, m, v = (x.detach().float().cpu().numpy().ravel() for x in (p, st["exp_avg"], st["exp_avg_sq"]))
    assert st["step"] == 2 and st["exp_avg"].dtype == F32 and ("master" in st) == (dtype != F32)
    p.grad = grads[2].cuda()
    mine.step()
    want = so.adamw(w, grads[2].float().numpy().ravel(), m, v, 3, 1e-2, (0.9, 0.999), 1e-8, 1e-2)[0]
    assert _same(p.detach().float().view(-1), torch.from_numpy(want).to(dtype).float().numpy())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_step(dtype, bits):
    """A captured step counts its replays and gives the bits of the eager ones."""
    from language_interpolation_amd.train import AdamW
    gen = torch.Generator().manual_seed(2)
    base = [torch.randn(s, generator=gen).to(dtype) for s in ((300, 50), (77,))]
    grads = [[torch.randn(b.shape, generator=gen).to(dtype).cuda() for b in base] for _ in range(5)]
    ps = [[b.clone().cuda().requires_grad_() for b in base] for _ in range(2)]
    eager, opt = AdamW(ps[0], lr=1e-2, moment_bits=bits), AdamW(ps[1], lr=1e-2, moment_bits=bits, capturable=True)
    for p, g in zip(ps[1], grads[0]):
        p.grad = g.clone()
    opt.step()  # the state exists before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(5):
        for p, g in zip(ps[0], grads[i]):
            p.grad = g
        eager.step()
        if i:
            for p, g in zip(ps[1], grads[i]):
                p.grad.copy_(g)
            graph.replay()
            torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(*ps)), i
        torch.randn(1000, device="cuda").sum().item()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            eager.step()
    fresh = AdamW(ps[1], lr=1e-2, moment_bits=bits, capturable=True)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.step()


def test_side_stream():
    host, dev = _tensors(SIZES, F32, 8, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(dev, F32, 8, 4, seed=5)
    torch.cuda.synchronize()
    _host_step(host, 8, 4, seed=5)
    _compare(host, dev, F32, 8)


def test_refusals():
    from language_interpolation_amd import functional as PF
    from language_interpolation_amd.train import AdamW
    p, g, m, v = (torch.zeros(8, 4, device="cuda") for _ in range(4))
    ok = dict(lr=1e-3)
    with pytest.raises(ValueError):
        PF.adamw_step([p], [g], [m], [v], 0, **ok)
    with pytest.raises(ValueError):
        PF.adamw_step([p, p], [g, g], [m, m], [v, v], 1, **ok)
    with pytest.raises(ValueError):
        PF.adamw_step([p], [g.t().contiguous().t()], [m], [v], 1, **ok)
    with pytest.raises(ValueError):
        PF.adamw_step([p[:, :2]], [g[:, :2]], [m[:, :2]], [v[:, :2]], 1, **ok)
    with pytest.raises(ValueError):
        PF.adamw_step([p.half()], [g.half()], [m], [v], 1, **ok)
    with pytest.raises(ValueError):
        PF.adamw_step([p], [g], [m], [v], 1, masters=[p], **ok)
    with pytest.raises(ValueError):
        PF.adamw_step([p], [g], [m.byte()], [v.byte()], 1, avg_exponents=[torch.zeros(2, dtype=torch.uint8, device="cuda")],
                      sq_exponents=[torch.zeros(1, dtype=torch.uint8, device="cuda")], **ok)
    with pytest.raises(ValueError):
        PF.adamw_step([p], [g], [m], [v], 1, betas=(1.0, 0.9), lr=1e-3)
    with pytest.raises(ValueError):
        PF.adamw_step([p], [g, g], [m], [v], 1, **ok)
    with pytest.raises(ValueError):
        AdamW([p], moment_bits=4)
    PF.adamw_step([], [], [], [], 1, **ok)
    e = torch.zeros(0, device="cuda")
    PF.adamw_step([e], [e], [e], [e], 1, **ok)
