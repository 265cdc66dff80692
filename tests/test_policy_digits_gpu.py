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
