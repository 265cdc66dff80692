"""Gated linear recurrence (functional.gated_recurrence / _step) against the 64-bit restatement."""
import pytest
import torch

import seq_oracle as so

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _inputs(b, l, d, dtype, seed, slow=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(b, l, d, generator=g).to(dtype)
    f = (torch.randn(b, l, d, generator=g) * 1.5 + slow).to(dtype)
    gy = torch.randn(b, l, d, generator=g).to(dtype)
    h0, gh = torch.randn(b, d, generator=g), torch.randn(b, d, generator=g)
    return z, f, gy, h0, gh


def _run(z, f, gy, h0=None, gh=None, lengths=None, reset=None, packed=False):
    from language_interpolation_amd import functional as PF
    if packed:  # halves of one projection
        both = torch.cat([z, f], -1).cuda()
        zd, fd = both[..., :z.shape[-1]].detach(), both[..., z.shape[-1]:].detach()
        assert z.shape[-1] == 0 or both.numel() == 0 or not zd.is_contiguous() or z.shape[0] * z.shape[1] == 1
    else:
        zd, fd = z.cuda(), f.cuda()
    leaves = [zd.requires_grad_(), fd.requires_grad_()]
    hd = None
    if h0 is not None:
        hd = h0.cuda().requires_grad_()
        leaves.append(hd)
    cuda = lambda x: None if x is None else x.cuda()  # noqa: E731
    y, h = PF.gated_recurrence(zd, fd, h0=hd, lengths=cuda(lengths), reset=cuda(reset))
    gh = torch.zeros_like(h) if gh is None else gh.cuda()
    grads = torch.autograd.grad((y, h), leaves, (gy.cuda(), gh))
    return dict(zip(("y", "h", "gz", "gf", "gh0"), (y, h) + grads))


def _compare(got, want):
    for name, x in got.items():
        so.check(x, want[name], name)


SHAPES = [(1, 1, 1), (1, 1, 64), (3, 2, 5), (2, 15, 128), (2, 16, 65), (1, 17, 130), (2, 31, 256),
          (1, 33, 257), (1, 100, 96), (1, 513, 40), (1, 1025, 66), (2, 300, 1), (1, 3, 1031)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dtype):
    b, l, d = shape
    z, f, gy, h0, gh = _inputs(b, l, d, dtype, seed=b * 1000 + l + d)
    for packed in (False, True):
        _compare(_run(z, f, gy, h0, gh, packed=packed), so.recurrence(z, f, h0, gy=gy, gh=gh))
    _compare(_run(z, f, gy), so.recurrence(z, f, gy=gy))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("l", [1, 16, 40, 257, 700])
def test_lengths_and_resets(dtype, l):
    b, d = 5, 70
    z, f, gy, h0, gh = _inputs(b, l, d, dtype, seed=l)
    lengths = torch.tensor([l, 0, l // 2, 1, -3], dtype=torch.int32)  # below 0 counts as 0
    g = torch.Generator().manual_seed(l)
    reset = torch.rand(b, l, generator=g) < 0.1
    reset[0, 0] = True
    # what lies behind the end is not read
    for i, n in enumerate(lengths.clamp(min=0).tolist()):
        for x in (z, f, gy):
            x[i, n:] = float("nan")
    for lens, res in ((lengths, None), (lengths, reset), (lengths.long(), reset.to(torch.uint8))):
        _compare(_run(z, f, gy, h0, gh, lens, res), so.recurrence(z, f, h0, lens, res, gy, gh))
    z, f, gy, h0, gh = _inputs(b, l, d, dtype, seed=l + 1)
    _compare(_run(z, f, gy, h0, gh, None, reset), so.recurrence(z, f, h0, None, reset, gy, gh))
    every = torch.ones(b, l, dtype=torch.bool)
    _compare(_run(z, f, gy, h0, gh, None, every), so.recurrence(z, f, h0, None, every, gy, gh))


@pytest.mark.parametrize("slow", [-6.0, 6.0, 12.0])
def test_gates_near_zero_and_one(slow):
    """Memory of one step, and of more steps than there are."""
    z, f, gy, h0, gh = _inputs(2, 600, 33, F32, seed=7, slow=slow)
    _compare(_run(z, f, gy, h0, gh), so.recurrence(z, f, h0, gy=gy, gh=gh))


def test_closed_and_open_gates():
    """f at the ends of the type and at infinity: the gate is 0 or 1, nothing becomes NaN."""
    z, f, gy, h0, gh = _inputs(2, 50, 40, F16, seed=8)
    f[:, ::5] = torch.finfo(F16).min
    f[:, 1::5] = torch.finfo(F16).max
    f[:, 2::10] = float("-inf")
    f[:, 3::10] = float("inf")
    _compare(_run(z, f, gy, h0, gh), so.recurrence(z, f, h0, gy=gy, gh=gh))


def test_strides_broadcasts_and_transposed_inputs():
    from language_interpolation_amd import functional as PF
    z, f, gy, h0, gh = _inputs(3, 50, 24, F32, seed=9)
    # time-major storage, read in place
    zt, ft = z.transpose(0, 1).contiguous().cuda().transpose(0, 1), f.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    want = so.recurrence(z, f, h0)
    so.check(PF.gated_recurrence(zt, ft, h0.cuda())[0], want["y"], "time-major")
    # channels not contiguous, and an address that is no multiple of 16
    zc = z.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    off = torch.empty(f.numel() + 1, device="cuda")[1:].view(f.shape).copy_(f)
    so.check(PF.gated_recurrence(zc, off, h0.cuda())[0], want["y"], "channels strided")
    # one gate row for the batch: its gradient is the sum
    f1 = f[:1].cuda().requires_grad_()
    y, _ = PF.gated_recurrence(z.cuda(), f1.expand(3, 50, 24), h0.cuda())
    (g1,) = torch.autograd.grad(y, f1, gy.cuda())
    ref = so.recurrence(z, f[:1].expand(3, 50, 24), h0, gy=gy)["gf"]
    so.check(g1, (ref[0].sum(0, keepdim=True), ref[1].sum(0, keepdim=True) + 4 * so.U * ref[0].abs().sum(0, keepdim=True)),
             "shared gate")
    # a gradient without strides (of a sum), and none for one of the two outputs
    zz, ff = z.cuda().requires_grad_(), f.cuda().requires_grad_()
    y, h = PF.gated_recurrence(zz, ff)
    gz, gf = torch.autograd.grad(y.sum(), (zz, ff), retain_graph=True)
    ref = so.recurrence(z, f, gy=torch.ones_like(z))
    so.check(gz, ref["gz"], "gz of a sum")
    so.check(gf, ref["gf"], "gf of a sum")
    gz, gf = torch.autograd.grad(h, (zz, ff), gh.cuda())
    ref = so.recurrence(z, f, gy=torch.zeros_like(z), gh=gh)
    so.check(gz, ref["gz"], "gz of the state")
    so.check(gf, ref["gf"], "gf of the state")


# few and many (stretches of 16 steps) x (64 channels): one and two channels a lane in 16-bit types; narrow rows
# that share a wave
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(3, 300, 1), (3, 300, 2), (3, 300, 127), (120, 300, 129), (70, 300, 255), (65, 1025, 66),
                                   (260, 16, 1031), (33, 257, 512), (6500, 64, 1), (450, 304, 3), (4200, 16, 7),
                                   (131, 513, 32), (5, 14000, 5)])
def test_rows_at_any_element(dtype, shape):
    """16-bit rows of odd strides and addresses, cut and reset: pairs of channels start at any element."""
    from language_interpolation_amd import functional as PF
    b, l, d = shape
    z, f, gy, h0, gh = _inputs(b, l, d, dtype, seed=d)
    g = torch.Generator().manual_seed(d)
    lengths = torch.randint(0, l + 1, (b,), generator=g, dtype=torch.int32)
    lengths[0], lengths[-1] = l, 0
    reset = torch.rand(b, l, generator=g) < 0.02
    stride = d + 2 + (d + 1) % 2  # odd
    rows = []
    for x in (z, f, gy):
        wide = torch.full((b, l, stride), float("nan"), dtype=dtype, device="cuda")
        rows.append(wide[..., 1:1 + d].copy_(x.cuda()))
    zd, fd, hd = rows[0].requires_grad_(), rows[1].requires_grad_(), h0.cuda().requires_grad_()
    y, h = PF.gated_recurrence(zd, fd, h0=hd, lengths=lengths.cuda(), reset=reset.cuda())
    grads = torch.autograd.grad((y, h), (zd, fd, hd), (rows[2], gh.cuda()))
    _compare(dict(zip(("y", "h", "gz", "gf", "gh0"), (y, h) + grads)),
             so.recurrence(z, f, h0, lengths, reset, gy, gh))
    _compare(_run(z, f, gy, h0, gh), so.recurrence(z, f, h0, gy=gy, gh=gh))


def test_gradient_against_differences():
    z, f, gy, h0, gh = (x.double() for x in _inputs(2, 37, 3, F32, seed=10))
    got = _run(z.float(), f.float(), gy.float(), h0.float(), gh.float())
    g = torch.Generator().manual_seed(11)
    direction = {"gz": torch.randn(z.shape, generator=g).double(), "gf": torch.randn(z.shape, generator=g).double(),
                 "gh0": torch.randn(h0.shape, generator=g).double()}
    for name, v in direction.items():
        def loss(s):
            o = so.recurrence(z + s * v if name == "gz" else z, f + s * v if name == "gf" else f,
                              h0 + s * v if name == "gh0" else h0)
            return float((o["y"][0] * gy).sum() + (o["h"][0] * gh).sum())
        numeric = (loss(1e-4) - loss(-1e-4)) / 2e-4
        formula = float((got[name].cpu().double() * v).sum())
        # a central difference at 1e-4 is off by 1e-8 times a third derivative of order 10^2
        assert abs(numeric - formula) < 1e-5 * (1 + abs(numeric)) * 10


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("b,d", [(1, 1), (3, 64), (64, 130), (2, 2048), (70, 1031)])
def test_single_token(b, d, dtype):
    from language_interpolation_amd import functional as PF
    z, f, _, h0, _ = _inputs(b, 3, d, dtype, seed=b + d)
    want = so.recurrence(z, f, h0)
    h = h0.cuda()
    for t in range(3):  # token by token, z and f as rows of a longer tensor
        version = h._version
        y = PF.gated_recurrence_step(z.cuda()[:, t], f.cuda()[:, t], h)
        assert h._version > version and y.dtype == dtype
        so.check(y, tuple(x[:, t] for x in want["y"]), f"token {t}")
    so.check(h, want["h"], "state")
    # a state inside a larger buffer: its neighbours stay
    pool = torch.full((b, d + 3), 7.0, device="cuda")
    pool[:, :d] = h0.cuda()
    PF.gated_recurrence_step(z[:, 0].cuda(), f[:, 0].cuda(), pool[:, :d])
    assert bool((pool[:, d:] == 7).all())
    so.check(pool[:, :d], so.recurrence(z[:, :1], f[:, :1], h0)["h"], "state in a pool")


def test_inference_mode():
    """As a server calls it: states made inside and outside of inference mode."""
    from language_interpolation_amd import functional as PF
    z, f, _, h0, _ = _inputs(3, 20, 40, BF16, seed=14)
    want = so.recurrence(z, f, h0)
    outside = h0.cuda()
    with torch.inference_mode():
        inside = h0.cuda()
        for h in (inside, outside):
            for t in range(20):
                PF.gated_recurrence_step(z.cuda()[:, t], f.cuda()[:, t], h)
            so.check(h, want["h"], "state")
        y, h = PF.gated_recurrence(z.cuda(), f.cuda(), h0.cuda())
    so.check(y, want["y"], "y")


def test_pieces_make_the_whole():
    """A long row in pieces with the state handed on, then token by token, is the row at once."""
    from language_interpolation_amd import functional as PF
    z, f, _, h0, _ = _inputs(2, 300, 40, F32, seed=12)
    want = so.recurrence(z, f, h0)
    zd, fd, h = z.cuda(), f.cuda(), h0.cuda()
    parts = []
    for lo, hi in ((0, 100), (100, 101), (101, 290)):
        y, h = PF.gated_recurrence(zd[:, lo:hi], fd[:, lo:hi], h)
        parts.append(y)
    for t in range(290, 300):
        parts.append(PF.gated_recurrence_step(zd[:, t], fd[:, t], h)[:, None])
    so.check(torch.cat(parts, 1), want["y"], "pieces")
    so.check(h, want["h"], "state")


def test_empty_and_repeated():
    from language_interpolation_amd import functional as PF
    e = torch.empty(2, 0, 8, device="cuda", requires_grad=True)
    h0 = torch.randn(2, 8, device="cuda", requires_grad=True)
    y, h = PF.gated_recurrence(e, e, h0)
    assert y.shape == (2, 0, 8) and torch.equal(h, h0)
    gh = torch.randn(2, 8, device="cuda")
    assert torch.equal(torch.autograd.grad(h, h0, gh)[0], gh)
    assert PF.gated_recurrence(torch.empty(0, 3, 8, device="cuda"), torch.empty(0, 3, 8, device="cuda"))[1].shape == (0, 8)
    z, f, gy, h0, gh = _inputs(2, 900, 200, BF16, seed=13)
    first = _run(z, f, gy, h0, gh)
    again = _run(z, f, gy, h0, gh)
    assert all(torch.equal(first[k], again[k]) for k in first)  # the same bits


def test_streams_and_graph_replays():
    """Two calls at once on two streams, and a captured forward + backward replayed on new inputs."""
    from language_interpolation_amd import functional as PF
    ins = [_inputs(2, 1200, 192, BF16, seed=20 + i) for i in range(4)]
    dev = [[x.cuda() for x in s] for s in ins]
    plain = [_run(*s) for s in ins]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]), torch.no_grad():
            z, f, _, h0, _ = dev[i]
            outs.append(PF.gated_recurrence(z, f, h0))
    torch.cuda.synchronize()
    for i in range(4):
        assert torch.equal(outs[i][0], plain[i]["y"]) and torch.equal(outs[i][1], plain[i]["h"])
    del outs

    static = [torch.empty_like(x) for x in dev[0]]
    z, f = static[0].requires_grad_(), static[1].requires_grad_()
    h0 = static[3].requires_grad_()

    def body():
        y, h = PF.gated_recurrence(z, f, h0)
        return (y, h) + torch.autograd.grad((y, h), (z, f, h0), (static[2], static[4]))

    def load(i):
        with torch.no_grad():
            for s, x in zip(static, dev[i]):
                s.copy_(x)

    load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, as a program with two batch shapes holds them
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = body()
        graphs.append((graph, out))
    for i in (1, 2, 3, 0, 1):
        load(i)
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        for name, x in zip(("y", "h", "gz", "gf", "gh0"), out):
            assert torch.equal(x, plain[i][name]), (i, name)
        torch.randn(1000, device="cuda").sum().item()  # eager work between the replays


def test_refusals():
    from language_interpolation_amd import functional as PF
    z = torch.randn(2, 5, 8, device="cuda")
    with pytest.raises(TypeError):
        PF.gated_recurrence(z, z.half())
    with pytest.raises(TypeError):
        PF.gated_recurrence(z.double(), z.double())
    with pytest.raises(ValueError):
        PF.gated_recurrence(z, z[:, :4])
    with pytest.raises(TypeError):
        PF.gated_recurrence(z, z, h0=torch.zeros(2, 8, device="cuda", dtype=BF16))
    with pytest.raises(ValueError):
        PF.gated_recurrence(z, z, lengths=torch.zeros(3, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError):
        PF.gated_recurrence(z, z, reset=torch.zeros(2, 5, dtype=torch.bool))
    with pytest.raises(RuntimeError):
        PF.gated_recurrence_step(z[:, 0].requires_grad_(), z[:, 0], torch.zeros(2, 8, device="cuda"))
    with pytest.raises(ValueError):  # two sequences, one state
        PF.gated_recurrence_step(z[:, 0], z[:, 0], torch.zeros(1, 8, device="cuda").expand(2, 8))
    zz = z.clone().requires_grad_()
    y, _ = PF.gated_recurrence(zz, z)
    (g,) = torch.autograd.grad(y.sum(), zz, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative, and no silent zero in its place
        torch.autograd.grad(g.sum(), zz)
