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
