"""Token log-probabilities and the clipped policy loss against the 64-bit restatement."""
import pytest
import torch

import seq_oracle as so

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LOW, HIGH, BETA = 0.2, 0.28, 0.04


def _inputs(b, t, v, dtype, seed, mask=True, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b, t, v, generator=g) * spread).to(dtype)
    tokens = torch.randint(0, v, (b, t), generator=g)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, tokens[..., None])[..., 0]
    # ratios on both sides of both borders (log 0.8 = -0.223, log 1.28 = 0.247), none within 0.02
    steps = torch.tensor([-0.6, -0.35, -0.1, 0.0, 0.1, 0.35, 0.6])
    gap = steps[torch.randint(0, 7, (b, t), generator=g)] + 0.04 * (torch.rand(b, t, generator=g) - 0.5)
    old = (lp - gap).float()
    adv = torch.randn(b, t, generator=g)
    ref = (lp + 0.3 * torch.randn(b, t, generator=g)).float()
    m = None
    if mask:
        m = torch.rand(b, t, generator=g) < 0.7
        m[0] = False  # a sequence without tokens
        if b * t > 1:
            m[-1, -1] = True
        tokens = torch.where(m, tokens, -100)
    return logits, tokens, old, adv, ref, m


def _cuda(x):
    return None if x is None else x.cuda()


def _loss(logits, tokens, old, adv, ref, m, reduction="token", gout=1.0, beta=BETA):
    from language_interpolation_amd import functional as PF
    x = logits if logits.is_cuda else logits.cuda()
    x = x.detach().requires_grad_()
    loss, kl, cut = PF.clipped_policy_loss(x, tokens.cuda(), old.cuda(), adv.cuda(), _cuda(ref), _cuda(m),
                                           clip_low=LOW, clip_high=HIGH, kl_coef=beta if ref is not None else 0.0,
                                           reduction=reduction)
    (g,) = torch.autograd.grad(loss, x, torch.tensor(gout, device="cuda"))
    return {"loss": loss, "kl": kl, "clipped": cut, "grad": g}


def _want(logits, tokens, old, adv, ref, m, reduction="token", gout=1.0, beta=BETA):
    w = so.policy(logits, tokens, old, adv, ref, m, LOW, HIGH, beta if ref is not None else 0.0, reduction, gout)
    w.pop("lp")
    return w


def _compare(got, want):
    for name, x in want.items():
        so.check(got[name], x, name)


# around the widths at which another number of lanes or registers holds a row, odd and even
WIDTHS = [1, 2, 3, 7, 64, 127, 128, 129, 500, 512, 1000, 1024, 1025, 2048, 2049, 4096, 4099, 8191, 8192,
          9001, 16384, 16391, 32768, 33001, 65536, 65543, 131072, 131077, 200003]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", WIDTHS)
def test_loss_and_gradient(v, dtype):
    b, t = (4, 9) if v <= 4096 else (2, 3)
    s = _inputs(b, t, v, dtype, seed=v)
    _compare(_loss(*s), _want(*s))
    s = _inputs(b, t, v, dtype, seed=v + 1, mask=False)
    _compare(_loss(*s, reduction="sequence", gout=-0.37), _want(*s, reduction="sequence", gout=-0.37))


@pytest.mark.parametrize("b,t,v", [(1, 1, 5), (256, 15, 128), (3, 700, 40), (1, 2500, 33), (300, 1, 260), (2, 5000, 2)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_batches(b, t, v, reduction):
    for mask in (True, False):
        s = _inputs(b, t, v, F32, seed=b + t, mask=mask)
        _compare(_loss(*s, reduction=reduction), _want(*s, reduction=reduction))
    logits, tokens, old, adv, ref, m = _inputs(b, t, v, BF16, seed=b)
    per_row = adv[:, 0].contiguous()  # one advantage a sequence
    got = _loss(logits, tokens, old, per_row, None, m, reduction)
    _compare(got, _want(logits, tokens, old, per_row, None, m, reduction))
    assert float(got["kl"]) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [1, 5, 128, 3001, 8192, 50021, 131073])
def test_log_probs_and_their_gradient(v, dtype):
    from language_interpolation_amd import functional as PF
    logits, tokens, _, _, _, m = _inputs(3, 4, v, dtype, seed=v + 2)
    coef = torch.randn(3, 4, generator=torch.Generator().manual_seed(v))
    want = so.policy(logits, tokens, mask=m, coef=coef)
    x = logits.cuda().requires_grad_()
    lp = PF.token_log_probs(x, tokens.cuda(), mask=m.cuda())
    (g,) = torch.autograd.grad(lp, x, coef.cuda())
    so.check(lp, want["lp"], "lp")
    so.check(g, want["grad"], "grad")
    with torch.no_grad():
        flat = PF.token_log_probs(logits.cuda().view(12, v), tokens.cuda().view(12).int(), m.cuda().view(12))
    assert torch.equal(flat.view(3, 4), lp)


@pytest.mark.parametrize("v", [128, 5000, 40000])
def test_what_is_masked_is_not_read(v):
    logits, tokens, old, adv, ref, m = _inputs(3, 6, v, F32, seed=30)
    want = _want(logits, tokens, old, adv, ref, m)
    for junk in (float("nan"), float("inf"), torch.finfo(F32).min):
        spoilt = [torch.where(m, x, torch.full_like(x, junk)) for x in (old, adv, ref)]
        x = torch.where(m[..., None], logits, torch.full_like(logits, junk))
        got = _loss(x, torch.where(m, tokens, 1 << 40), *spoilt, m)
        _compare(got, want)
        assert bool((got["grad"][~m.cuda()] == 0).all())


def test_nothing_counts():
    logits, tokens, old, adv, ref, m = _inputs(2, 5, 77, BF16, seed=31)
    for reduction in ("token", "sequence"):
        got = _loss(logits, tokens, old, adv, ref, torch.zeros_like(m), reduction)
        assert all(bool((x == 0).all()) for x in got.values())


@pytest.mark.parametrize("v", [100, 3000, 20001])
def test_classes_that_are_ruled_out(v):
    """Logits of -inf and of the type's lowest value have no share and no gradient."""
    for junk, dtype in ((float("-inf"), F32), (torch.finfo(BF16).min, BF16), (float("-inf"), F16)):
        logits, tokens, old, adv, ref, m = _inputs(2, 6, v, dtype, seed=32, mask=False)
        out = torch.rand(2, 6, v, generator=torch.Generator().manual_seed(v)) < 0.5
        out.scatter_(-1, tokens[..., None], False)
        logits = torch.where(out, torch.full_like(logits, junk), logits)
        lp = torch.log_softmax(logits.double(), -1).gather(-1, tokens[..., None])[..., 0]
        s = (logits, tokens, (lp - 0.1).float(), adv, (lp + 0.1).float(), None)
        got = _loss(*s)
        _compare(got, _want(*s))
        assert bool((got["grad"][out.cuda()] == 0).all())


def test_large_logits_and_a_certain_token():
    """Rows far from zero, and rows where one class has all: lp near 0 keeps its digits."""
    logits, tokens, old, adv, ref, m = _inputs(3, 4, 900, F32, seed=33, mask=False, spread=30.0)
    logits = logits + 4000.0
    logits.scatter_(-1, tokens[..., None], 4100.0)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, tokens[..., None])[..., 0]
    s = (logits, tokens, (lp - 0.05).float(), adv, (lp + 0.05).float(), None)
    _compare(_loss(*s), _want(*s))


def test_no_such_class_is_loud():
    logits, tokens, old, adv, ref, _ = _inputs(2, 3, 50, F32, seed=34, mask=False)
    from language_interpolation_amd import functional as PF
    for bad in (-1, 50, 1 << 40, -(1 << 40)):
        tokens[1, 1] = bad
        lp = PF.token_log_probs(logits.cuda(), tokens.cuda())
        assert torch.isnan(lp).sum() == 1 and bool(torch.isnan(lp[1, 1]))
        assert bool(torch.isnan(_loss(logits, tokens, old, adv, ref, None)["loss"]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [65, 128, 5001])
def test_slices_and_padded_vocabularies(v, dtype):
    """Next-token logits as a slice over time, classes as a slice of a padded table, a base address
    that is no multiple of 16: read in place, the gradient belongs to the slice."""
    from language_interpolation_amd import functional as PF
    s = _inputs(3, 6, v, dtype, seed=35)
    logits, rest = s[0], s[1:]
    want = _want(*s)
    wide = torch.full((3, 8, v + 7), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:7, 3:v + 3] = logits.cuda()
    got = _loss(wide[:, 1:7, 3:v + 3], *rest)
    _compare(got, want)
    # rows at the offsets of the logits' rows within 16 bytes, and no more memory than that takes
    vec = 16 // logits.element_size()
    assert got["grad"].data_ptr() % 16 == wide[:, 1:7, 3:].data_ptr() % 16
    assert (got["grad"].stride(1) - wide.stride(1)) % vec == 0
    assert got["grad"].untyped_storage().nbytes() <= (3 * (6 * (v + vec) + vec) + vec) * logits.element_size()
    turned = logits.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    _compare(_loss(turned, *rest), want)
    classes_first = logits.cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0)
    _compare(_loss(classes_first, *rest), want)
    # through the slice into the whole
    whole = torch.zeros(3, 7, v, dtype=dtype, device="cuda")
    whole[:, :6] = logits.cuda()
    whole.requires_grad_()
    loss, _, _ = PF.clipped_policy_loss(whole[:, :-1], rest[0].cuda(), rest[1].cuda(), rest[2].cuda(), rest[3].cuda(),
                                        rest[4].cuda(), clip_low=LOW, clip_high=HIGH, kl_coef=BETA)
    loss.backward()
    so.check(whole.grad[:, :6], want["grad"], "whole")
    assert bool((whole.grad[:, 6] == 0).all())
    # the last position of every sequence only
    last = _loss(wide[:, 6:7, 3:v + 3], *(x[:, 5:] for x in rest))
    _compare(last, _want(logits[:, 5:], *(x[:, 5:] for x in rest)))
    assert last["grad"].untyped_storage().nbytes() <= (3 * (v + 2 * vec) + vec) * logits.element_size()
    # one row of logits for all tokens
    one = logits[:1, :1].cuda().expand(3, 6, v)
    shared = logits[:1, :1].expand(3, 6, v)
    so.check(PF.token_log_probs(one, rest[0].cuda(), rest[4].cuda()), so.policy(shared, rest[0], mask=rest[4])["lp"], "shared")


def test_repeated_backward_and_loss_scale():
    from language_interpolation_amd import functional as PF
    for v in (96, 6000):
        s = _inputs(2, 5, v, F16, seed=36)
        x = s[0].cuda().requires_grad_()
        loss, _, _ = PF.clipped_policy_loss(x, *(t.cuda() for t in s[1:5]), mask=s[5].cuda(), clip_low=LOW,
                                            clip_high=HIGH, kl_coef=BETA)
        for scale in (1.0, 1.0, 65536.0, 1.0, 3.0):  # at 1 much of it underflows in fp16
            (g,) = torch.autograd.grad(loss, x, torch.tensor(scale, device="cuda"), retain_graph=True)
            so.check(g, _want(*s, gout=scale)["grad"], f"scale {scale}")
        first, again = _loss(*s), _loss(*s)
        assert all(torch.equal(first[k], again[k]) for k in first)
        with torch.no_grad():  # without a gradient: the same numbers
            plain = PF.clipped_policy_loss(x, *(t.cuda() for t in s[1:5]), mask=s[5].cuda(), clip_low=LOW,
                                           clip_high=HIGH, kl_coef=BETA)
        assert all(torch.equal(p, first[k]) for p, k in zip(plain, ("loss", "kl", "clipped")))


def test_results_changed_in_place():
    """Each of the three is a tensor of its own: the loss is divided (accumulated steps), figures are summed."""
    from language_interpolation_amd import functional as PF
    inputs = _inputs(2, 6, 40, F32, 77)
    logits, tokens, old, adv, ref, m = (_cuda(x) for x in inputs)
    whole = _loss(*inputs)
    x = logits.requires_grad_()
    loss, kl, cut = PF.clipped_policy_loss(x, tokens, old, adv, ref, m, LOW, HIGH, BETA)
    assert not any(r._is_view() for r in (loss, kl, cut))
    kl += 1.0
    cut.zero_()
    loss /= 4
    loss.backward()
    assert torch.equal(loss, whole["loss"] / 4)
    assert torch.equal(kl, whole["kl"] + 1.0)
    so.check(x.grad, _want(*inputs, gout=0.25)["grad"], "grad")


def test_no_gradient_is_made_where_none_can_follow():
    from language_interpolation_amd import functional as PF
    s = _inputs(4, 64, 20000, BF16, seed=36)
    x = s[0].cuda().requires_grad_()
    rest = [t.cuda() for t in s[1:5]]
    with torch.no_grad():
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        PF.clipped_policy_loss(x, *rest, mask=s[5].cuda(), kl_coef=BETA)
        assert torch.cuda.max_memory_allocated() - before < x.numel()  # bytes: half of a gradient


def test_changed_logits_are_noticed():
    """The backward may need the logits again: changed in place, it refuses."""
    from language_interpolation_amd import functional as PF
    s = _inputs(2, 5, 96, F32, seed=37)
    x = s[0].cuda().requires_grad_()
    y = x * 1.0
    loss, _, _ = PF.clipped_policy_loss(y, *(t.cuda() for t in s[1:5]), mask=s[5].cuda(), kl_coef=BETA)
    y.mul_(2.0)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_gradient_against_differences():
    logits, tokens, old, adv, ref, m = _inputs(2, 6, 41, F32, seed=38)
    got = _loss(logits, tokens, old, adv, ref, m)["grad"].cpu().double()
    d = torch.randn(logits.shape, generator=torch.Generator().manual_seed(39)).double()

    def value(s):
        return float(so.policy(logits.double() + s * d, tokens, old, adv, ref, m, LOW, HIGH, BETA)["loss"][0])
    numeric, formula = (value(1e-5) - value(-1e-5)) / 2e-5, float((got * d).sum())
    # no ratio comes near a border within 1e-5; the difference is off by some 1e-10 of third derivatives
    assert abs(numeric - formula) < 1e-5 * (1 + abs(numeric))


def test_streams_and_graph_replays():
    from language_interpolation_amd import functional as PF
    ins = [_inputs(4, 30, 2500, BF16, seed=40 + i) for i in range(4)]
    dev = [[x.cuda() for x in s] for s in ins]
    plain = [_loss(*s) for s in ins]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(_loss_on(dev[i]))
    torch.cuda.synchronize()
    for i in range(4):
        assert all(torch.equal(outs[i][k], plain[i][k]) for k in plain[i])
    del outs
    static = [x.clone() for x in dev[0]]
    static[0].requires_grad_()

    def body(scale):
        loss, kl, cut = PF.clipped_policy_loss(static[0], *static[1:5], mask=static[5], clip_low=LOW, clip_high=HIGH,
                                               kl_coef=BETA)
        return {"loss": loss, "kl": kl, "clipped": cut,
                "grad": torch.autograd.grad(loss, static[0], scale)[0]}

    scale = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(scale)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body(scale)
    for i, s in ((1, 1.0), (2, 1.0), (3, 2.0), (0, 1.0), (1, 0.5)):
        with torch.no_grad():
            for x, y in zip(static, dev[i]):
                x.copy_(y)
        scale.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        want = plain[i] if s == 1.0 else _loss(*ins[i], gout=s)
        for k in want:
            assert torch.equal(out[k], want[k]), (i, s, k)
        torch.randn(1000, device="cuda").sum().item()


def _loss_on(s):
    return _loss(*s)


def test_refusals():
    from language_interpolation_amd import functional as PF
    x = torch.randn(2, 3, 8, device="cuda")
    tok, f = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, device="cuda")
    with pytest.raises(TypeError):
        PF.token_log_probs(x.double(), tok)
    with pytest.raises(ValueError):
        PF.token_log_probs(x, tok[:, :2])
    with pytest.raises(TypeError):
        PF.token_log_probs(x, tok.float())
    with pytest.raises(RuntimeError):
        PF.token_log_probs(x, tok, mask=torch.ones(2, 3, dtype=torch.bool))
    with pytest.raises(ValueError):
        PF.clipped_policy_loss(x, tok, f, f, reduction="sum")
    with pytest.raises(ValueError):
        PF.clipped_policy_loss(x, tok, f, f, kl_coef=0.1)
    with pytest.raises(ValueError):
        PF.clipped_policy_loss(x, tok, f, f, clip_low=-0.1)
    with pytest.raises(TypeError):
        PF.clipped_policy_loss(x, tok, f.half(), f)
    with pytest.raises(ValueError):
        PF.clipped_policy_loss(x, tok, f, torch.zeros(3, device="cuda"))
    empty = PF.clipped_policy_loss(x[:0], tok[:0], f[:0], f[:0])
    assert [float(e) for e in empty] == [0.0, 0.0, 0.0]
