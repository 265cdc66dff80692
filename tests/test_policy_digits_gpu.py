"""Digits of the token log-probabilities, the policy loss and their gradients that a bound over whole sums does not see."""
import math

import numpy as np
import pytest
import torch

import seq_oracle as so
from language_interpolation_amd import functional as PF

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = so.U


@pytest.mark.parametrize("v", [3, 129, 1000, 5003, 40001, 131071, 199999])
def test_the_share_of_equal_classes(v):
    """Equal logits: every exponential is 1 and their sum is v, so a gradient is c / v to a division and a product
    (4 U counted), in the backward of its own as in the loss's."""
    c = torch.tensor([[0.7, -1.3, 5.0]])
    x = torch.full((1, 3, v), -2.5, device="cuda", requires_grad=True)
    tokens = torch.full((1, 3), v - 1, device="cuda")
    lp = PF.token_log_probs(x, tokens)
    (g,) = torch.autograd.grad(lp, x, c.cuda())
    want = -c.double() / v
    assert bool(((g[..., :-1].cpu().double() - want[..., None]).abs() <= 4 * U * want[..., None].abs()).all())
    rows = torch.full((1, 3), -math.log(v), device="cuda")
    loss = PF.clipped_policy_loss(x, tokens, rows, c.cuda())[0]
    (one,) = torch.autograd.grad(loss, x, retain_graph=True)
    (two,) = torch.autograd.grad(loss, x, torch.tensor(2.0, device="cuda"))  # made anew from what was kept
    assert bool(((two - 2 * one)[..., :-1].abs() <= 8 * U * two[..., :-1].abs()).all())


@pytest.mark.parametrize("v", [5, 130, 3001, 40001, 70001])
@pytest.mark.parametrize("anew", [False, True])
def test_shares_of_unlikely_classes(v, anew):
    """fp32: two classes' gradients are to each other as exp of their logits' difference, however unlikely.  An exponential
    2 U, a product U on either side: 8 U counted, and the exact quotient's own rounding."""
    g = torch.Generator().manual_seed(v)
    x = -80.0 * torch.rand(1, 4, v, generator=g)
    x[..., 0], tokens = 0.0, torch.full((1, 4), v - 1)
    xd = x.cuda().requires_grad_()
    if anew:
        (got,) = torch.autograd.grad(PF.token_log_probs(xd, tokens.cuda()).sum(), xd)
    else:
        rows = torch.full((1, 4), -40.0, device="cuda")
        ref = rows + 0.5
        loss = PF.clipped_policy_loss(xd, tokens.cuda(), rows, torch.zeros(1, 4, device="cuda"), ref, kl_coef=0.5)[0]
        (got,) = torch.autograd.grad(loss, xd)
    got = got.cpu().double()[..., :-1]
    ratio, want = got / got[..., :1], x.double()[..., :-1].exp()
    # (a gradient of fp32's subnormals has fewer bits)
    fine = got.abs() > 2.0 ** -120
    assert float(fine.double().mean()) > 0.5
    assert bool(((ratio - want).abs() <= 8 * U * want)[fine].all()), float(((ratio / want - 1).abs()[fine]).max() / U)


@pytest.mark.parametrize("below", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ratios_next_to_a_border(dtype, below):
    """Two equal logits, lp = -log 2: borders one fp32 step apart on both sides of a ratio.  lp comes from a sum of 2 exactly, so
    it is as exact as the logarithm (2^-27 counted); a ratio further than that from the border is clipped or not."""
    f = np.float32
    cases = []
    for old in np.linspace(-1.1, -0.8, 40).astype(f) if not below else np.linspace(-0.6, -0.3, 40).astype(f):
        d = -math.log(2.0) - float(old)
        exact = abs(math.expm1(d))
        for clip in (f(exact), np.nextafter(f(exact), f(0)), np.nextafter(f(exact), f(1))):
            gap = d - math.log1p(-float(clip) if below else float(clip))
            if abs(gap) > 2.0 ** -27:
                cases.append((old, float(clip), gap < 0 if below else gap > 0))
    assert len(cases) > 60 and 10 < sum(c for _, _, c in cases) < len(cases) - 10
    # (an fp32 ratio falls on the border itself in some of them: those are what this is about)
    x = torch.zeros(1, 1, 2, dtype=dtype, device="cuda", requires_grad=True)
    token, adv = torch.zeros(1, 1, dtype=torch.int64, device="cuda"), torch.full((1, 1), -1.0 if below else 1.0, device="cuda")
    for old, clip, cut in cases:
        kw = {"clip_low": clip} if below else {"clip_high": clip}
        loss, _, clipped = PF.clipped_policy_loss(x, token, torch.full((1, 1), float(old), device="cuda"), adv, **kw)
        (g,) = torch.autograd.grad(loss, x)
        assert bool(clipped == 1.0) == cut and bool((g == 0).all()) == cut, (old, clip)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_a_certain_token_is_not_more_than_certain(dtype):
    """Sums of 1 and just above: log-probabilities are 0 or below, 0 where nothing but the token has a share."""
    one = torch.tensor([[[3.5]]], dtype=dtype, device="cuda")
    zero = torch.zeros(1, 1, dtype=torch.int64, device="cuda")
    assert float(PF.token_log_probs(one, zero)) == 0.0
    for v in (2, 64, 300, 5000, 150000):
        x = torch.full((1, 1, v), -60000.0 if dtype != F16 else -300.0, dtype=dtype, device="cuda")
        x[..., v - 1] = 0.0
        assert float(PF.token_log_probs(x, zero + v - 1)) == 0.0
        # another class behind a distance of n: 1 + e^-n, its log e^-n to first order.  The sum of a lane is fp32 (U), that
        # of a row 16 such (16 U), the log of a number near 1 is off by a unit of itself
        for n in (6, 9, 12, 15, 18, 25):
            x[..., 0] = -float(n)
            lp = float(PF.token_log_probs(x, zero + v - 1))
            want = -math.log1p(math.exp(-n))
            assert lp <= 0.0 and abs(lp - want) <= 17 * U * 2, (v, n)


def test_the_log_of_a_sum_near_one_keeps_its_digits():
    """The share of the likeliest class comes in a lane of another wave than the second's, whose sum is exact: nothing but
    the logarithm rounds, to 2 U of itself (4 U with the exponential and 3 U of the fp32 result: 12 U counted)."""
    v = 4096  # 1024 vectors of 4 in 256 threads
    for n in (5.0, 9.0, 13.0, 17.0, 21.0):
        x = torch.full((1, 1, v), float("-inf"), device="cuda")
        x[..., 0], x[..., 64 * 4 * 3] = 0.0, -n
        lp = float(PF.token_log_probs(x, torch.zeros(1, 1, dtype=torch.int64, device="cuda")))
        want = -math.log1p(math.exp(-n))
        assert abs(lp - want) <= (12 + n) * U * abs(want), n


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [128, 1001, 5001, 50021])
def test_errors_of_the_sums_do_not_add_up(dtype, v):
    """Ratios far from the borders, all advantages 1: the loss is the mean ratio, so an error of one sign in the sums of a
    vocabulary is the loss's.  What is left is rounding: a loss is rounded by at most U of itself and by chance (a
    deviation of U / sqrt 3), so the mean over 100 losses has one of 0.06 U: 5 of those, and as much for ratios and sums of
    512 tokens, whose own roundings (under 16 U) have a mean deviation below 16 U / sqrt(51200) = 0.07 U."""
    g = torch.Generator(device="cuda").manual_seed(v)
    n = 512 if v < 10000 else 128
    tokens = torch.randint(0, v, (1, n), generator=g, device="cuda")
    off = []
    for _ in range(100):
        x = (torch.randn(1, n, v, generator=g, device="cuda") * 2.0).to(dtype)
        lp = torch.cat([torch.log_softmax(part.double(), -1) for part in x.split(64, 1)], 1).gather(-1, tokens[..., None])[..., 0]
        old = (lp - 0.3 - 0.2 * torch.rand(1, n, generator=g, device="cuda")).float()
        loss = PF.clipped_policy_loss(x, tokens, old, torch.ones(1, n, device="cuda"), clip_high=10.0)[0]
        off.append(float(loss) / -float(torch.exp(lp - old.double()).mean()) - 1)
    bound = 5 * U * (1 / math.sqrt(3 * 100) + 16 / math.sqrt(100 * n))
    assert abs(sum(off) / len(off)) <= bound, (sum(off) / len(off) / U, bound / U)


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_a_border_is_not_rounded_for_all_tokens_alike(reduction):
    """Every token clipped, half at either border, so that the loss nearly cancels.  A term is rounded to fp32 once, by chance
    (a deviation of U / sqrt 3 of itself), so the mean of n is off by U rms / sqrt(3 n): 6 of those, and the result's rounding."""
    g = torch.Generator().manual_seed(2)
    b, t, high, low = 256, 256, float(np.float32(0.28)), float(np.float32(0.2))
    up = torch.rand(b, t // 2, generator=g)
    adv = torch.cat([up, -1.6 * up], 1)
    old = torch.cat([torch.full((b, t // 2), math.log(0.5) - 1.0), torch.full((b, t // 2), math.log(0.5) + 1.0)], 1)
    up64 = torch.ones(b, t, dtype=torch.float64)
    terms = -torch.where(adv >= 0, (1 + high) * up64, (1 - low) * up64) * adv.double()
    loss, _, clipped = PF.clipped_policy_loss(torch.zeros(b, t, 2, device="cuda"), torch.zeros(b, t, dtype=torch.int64, device="cuda"),
                                              old.cuda(), adv.cuda(), mask=torch.ones(b, t, dtype=torch.bool, device="cuda"),
                                              clip_high=high, clip_low=low, reduction=reduction)
    want = float(terms.mean())
    assert float(clipped) == 1.0 and abs(want) < 1e-6
    bound = 6 * U * float(terms.square().mean().sqrt()) / math.sqrt(3 * b * t) + U * abs(want)
    assert abs(float(loss) - want) <= bound, (float(loss) - want, bound)
