"""What the sequence-model operators hand to the library, without a GPU: the entries are replaced, tensors take the
place of addresses."""
import contextlib

import pytest
import torch

from language_interpolation_amd import functional as PF

F32 = torch.float32


@pytest.fixture
def calls(monkeypatch):
    """The calls made of the library: (entry, arguments with tensors for addresses)."""
    made = []
    monkeypatch.setattr(PF, "_at", lambda t: t)
    monkeypatch.setattr(PF, "_launch", lambda name, device, *args: made.append((name, args)))
    return made


@contextlib.contextmanager
def default_dtype(dtype):
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        yield
    finally:
        torch.set_default_dtype(before)


def _recurrence(b=2, l=40, d=3, dtype=F32, h0=True):
    z, f = (torch.randn(b, l, d, dtype=F32).to(dtype).requires_grad_() for _ in range(2))
    h0 = torch.zeros(b, d, dtype=F32, requires_grad=True) if h0 else None
    y, h = PF.GatedRecurrenceFunction.apply(z, f, h0, None, None, True)
    grads = torch.autograd.grad((y, h), [x for x in (z, f, h0) if x is not None],
                                (torch.zeros_like(y), torch.zeros_like(h)))
    return y, h, grads


@pytest.mark.parametrize("default", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_buffers_of_floats_are_floats(calls, default):
    """The kernels write 4-byte floats whatever the program's default dtype."""
    b, l, d, t, v = 2, 40, 3, 5, 11
    with default_dtype(default):
        y, h, grads = _recurrence(b, l, d)
        assert h.dtype == F32 and grads[2].dtype == F32
        empty = PF.GatedRecurrenceFunction.apply(torch.zeros(b, 0, d, dtype=F32), torch.zeros(b, 0, d, dtype=F32), None, None,
                                                 None, False)
        assert empty[1].dtype == F32
        x = torch.randn(b, t, v, dtype=F32, requires_grad=True)
        tokens = torch.zeros(b, t, dtype=torch.int64)
        lp = PF.TokenLogProbsFunction.apply(x, tokens, None, True)
        torch.autograd.grad(lp, x, torch.zeros_like(lp))
        old, adv = torch.zeros(b, t, dtype=F32), torch.zeros(b, t, dtype=F32)
        loss, _, _ = PF.ClippedPolicyLossFunction.apply(x, tokens, None, old, adv, None, 0.2, 0.2, 0.0, 0, True)
        torch.autograd.grad(loss, x, torch.ones((), dtype=F32))
    steps = -(-l // 16)
    floats = {"pp_gated_recurrence_fwd": {11: b * d, 12: b * steps * d},
              "pp_gated_recurrence_bwd": {9: b * steps * d, 13: b * d, 16: b * d},
              "pp_token_log_probs_fwd": {6: b * t, 7: b * t * 2},
              "pp_token_log_probs_bwd": {6: b * t * 2, 7: b * t},
              "pp_clipped_policy_loss_fwd": {15: 3, 16: b * t * 2, 17: b * t}}
    assert {name for name, _ in calls} == set(floats)
    for name, args in calls:
        for at, count in floats[name].items():
            if args[at] is not None:
                assert args[at].dtype == F32 and args[at].numel() == count and args[at].is_contiguous(), (name, at)


def _inside(t, strides, shape):
    """Elements shape[0] x shape[1] rows of shape[2] at these strides lie inside the storage of t."""
    last = t.storage_offset() + sum((n - 1) * s for n, s in zip(shape, (*strides, 1)))
    return last < t.untyped_storage().nbytes() // t.element_size()


@pytest.mark.parametrize("policy", [False, True])
def test_logits_laid_out_anew_by_a_hook(calls, policy):
    """Hooks on saved tensors (save_on_cpu, compression) bring a slice of the logits back as a tensor of its own: the
    backward goes by the strides of what it is given."""
    b, t, v = 3, 6, 65
    wide = torch.randn(b, t + 2, v + 7, dtype=F32, requires_grad=True)
    tokens = torch.zeros(b, t, dtype=torch.int64)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x.contiguous().clone(), lambda x: x):
        x = wide[:, 1:t + 1, 3:v + 3]
        if policy:
            rows = torch.zeros(b, t)
            out, _, _ = PF.ClippedPolicyLossFunction.apply(x, tokens, None, rows, rows, None, 0.2, 0.2, 0.0, 0, True)
        else:
            out = PF.TokenLogProbsFunction.apply(x, tokens, None, True)
    for _ in range(2):
        torch.autograd.grad(out, wide, torch.zeros_like(out), retain_graph=True)
    backward = [args for name, args in calls if name == "pp_token_log_probs_bwd"]
    assert len(backward) == 2
    for a in backward:
        assert a[0].shape == (b, t, v) and _inside(a[0], a[1:3], (b, t, v)) and a[0].stride() == (*a[1:3], 1)
        grad, gb, gt = a[10:13]
        vec = 16 // 4
        assert _inside(grad, (gb, gt), (b, t, v)) and gt >= v and gb >= (t - 1) * gt + v
        assert (gb - a[1]) % vec == 0 and (gt - a[2]) % vec == 0 and (grad.data_ptr() - a[0].data_ptr()) % 16 == 0


def _policy(x, tokens):
    rows = torch.zeros(tokens.shape)
    return PF.ClippedPolicyLossFunction.apply(x, tokens, None, rows, rows, None, 0.2, 0.2, 0.0, 0, True)[0]


def test_the_gradient_made_in_the_forward_is_a_saved_tensor(calls):
    """Hooks see it (offloading moves it off the card), and the node holds no tensor beside what it saved."""
    packed = []
    tokens = torch.zeros(2, 5, dtype=torch.int64)
    x = torch.randn(2, 5, 33, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or len(packed) - 1,
                                                  lambda i: packed[i].clone()):
        loss = _policy(x, tokens)
    made = calls[0][1][18]
    assert made.shape == x.shape and any(t.data_ptr() == made.data_ptr() for t in packed)
    held = [v for value in vars(loss.grad_fn).values() for v in (value if isinstance(value, (tuple, list)) else [value])]
    assert not any(isinstance(v, torch.Tensor) for v in held)


def test_checkpointed_loss_hands_out_the_gradient_of_the_second_forward(calls):
    from torch.utils.checkpoint import checkpoint
    tokens = torch.zeros(2, 5, dtype=torch.int64)
    x = torch.randn(2, 5, 33, requires_grad=True)
    (g,) = torch.autograd.grad(checkpoint(_policy, x, tokens, use_reentrant=False), x)
    forward = [a for name, a in calls if name == "pp_clipped_policy_loss_fwd"]
    (back,) = [a for name, a in calls if name == "pp_token_log_probs_bwd"]
    assert len(forward) == 2 and back[9] == 1  # done if the upstream gradient is 1
    assert back[10].data_ptr() == forward[1][18].data_ptr() == g.data_ptr()


def test_a_gradient_is_handed_out_once(calls):
    """What was handed out belongs to the program, which may change it before it asks again."""
    tokens = torch.zeros(2, 5, dtype=torch.int64)
    x = torch.randn(2, 5, 33, requires_grad=True)
    loss = _policy(x, tokens)
    (first,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert first.data_ptr() == calls[0][1][18].data_ptr()
    first.zero_()
    for _ in range(2):
        (again,) = torch.autograd.grad(loss, x, retain_graph=True)
        assert again.data_ptr() != first.data_ptr()
    assert [a[9] for name, a in calls if name == "pp_token_log_probs_bwd"] == [1, 0, 0]
