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


def test_many_rows_are_taken_in_slices(calls):
    """A launch takes 65535 rows: more are several launches over the rows' own parts of every tensor."""
    b, l, d = 150001, 2, 1
    z, f = (torch.randn(b, l, 2 * d)[..., :d].requires_grad_() for _ in range(2))
    h0 = torch.randn(b, d, requires_grad=True)
    lengths, reset = torch.ones(b, dtype=torch.int32), torch.zeros(b, l, dtype=torch.uint8)
    y, h = PF.GatedRecurrenceFunction.apply(z, f, h0, lengths, reset, True)
    gz, gf, gh0 = torch.autograd.grad((y, h), (z, f, h0), (torch.zeros(b, l, d), torch.zeros(b, d)))
    fwd = [a for name, a in calls if name.endswith("_fwd")]
    bwd = [a for name, a in calls if name.endswith("_bwd")]
    for made, whole in ((fwd, {0: z, 3: f, 7: h0, 8: lengths, 9: reset, 10: y, 11: h, 12: None}),
                        (bwd, {0: z, 3: f, 7: lengths, 8: reset, 9: None, 10: None, 13: None, 14: gz, 15: gf, 16: gh0})):
        rows = [a[-3] for a in made]
        assert len(rows) == 3 and sum(rows) == b and max(rows) <= 65535 and max(rows) - min(rows) < 3
        first = 0
        for a in made:
            assert a[-2:] == (l, d)
            for at, t in whole.items():
                part = a[at]
                assert part.shape[0] == a[-3]
                if t is not None:
                    assert part.data_ptr() == t[first:].data_ptr() and part.stride() == t.stride()
            first += a[-3]
    assert [a[12].data_ptr() for a in fwd] == [a[9].data_ptr() for a in bwd]  # the kept states
    assert fwd[1][12].data_ptr() - fwd[0][12].data_ptr() == 4 * fwd[0][-3] * d


def test_rows_of_a_launch_are_what_the_entry_takes():
    """The entries say so themselves, before they look at addresses (an odd one here) or launch anything."""
    import ctypes
    from language_interpolation_amd import _lib
    lib, odd = _lib.load(), ctypes.c_void_p(4097)

    def entry(b, l, d):
        return lib.pp_gated_recurrence_fwd(odd, 1, 1, odd, 1, 1, 0, None, None, None, odd, odd, None, None, 0, b, l, d, None)
    for l in (1, 16, 17, 256, 257, 5000, 32767, 131072, 1 << 24):
        for d in (1, 64, 65, 2048, 1 << 20):
            most = PF._rows_of_a_launch(l, d)
            assert most >= 1
            if most > 1:
                assert entry(most, l, d) == -3, (l, d)  # only the address is wrong
                assert entry(most + 1, l, d) in (-2, -6), (l, d)


def test_the_workspace_of_shared_rows_is_what_they_use():
    """Rows of up to 32 channels that share waves: 12 bytes for each of a chunk's lanes, not for 128 channels a row."""
    from language_interpolation_amd import _lib
    need = _lib.load().pp_gated_recurrence_workspace_bytes
    chunks = -(-131072 // 256)
    assert need(457, 131072, 1) == 16 + 12 * 64 * -(-457 // 64) * chunks
    assert need(450, 304, 3) == 16 + 12 * 64 * -(-1350 // 64) * 2
    assert need(131, 513, 32) == 16 + 12 * 64 * -(-131 * 32 // 64) * 3
    # a wave or more a row: one or two channels a lane, whichever the type takes
    assert need(1, 1000, 64) >= 16 + 12 * 64 * 4 and need(8, 2048, 2048) == 16 + 12 * 8 * 2048 * 8
    assert need(3, 256, 40) == 0


def test_saved_tensors_that_come_back_turned(calls):
    """A hook may keep a tensor in another order of its elements: what the entries take as contiguous is made so."""
    def turned(x):
        return x.transpose(0, -1).contiguous().transpose(0, -1) if x.dim() > 1 else x
    b, l, d, t, v = 3, 40, 5, 6, 17
    with torch.autograd.graph.saved_tensors_hooks(turned, lambda x: x):
        z, f = (torch.randn(b, l, d, requires_grad=True) for _ in range(2))
        lengths, reset = torch.ones(b, dtype=torch.int32), torch.zeros(b, l, dtype=torch.uint8)
        y, h = PF.GatedRecurrenceFunction.apply(z, f, None, lengths, reset, True)
        x, tokens, mask = torch.randn(b, t, v, requires_grad=True), torch.zeros(b, t, dtype=torch.int64), torch.ones(b, t, dtype=torch.uint8)
        lp = PF.TokenLogProbsFunction.apply(x, tokens, mask, True)
        rows = torch.zeros(b, t)
        loss = PF.ClippedPolicyLossFunction.apply(x, tokens, mask, rows, rows, None, 0.2, 0.2, 0.0, 0, True)[0]
    torch.autograd.grad((y, h), (z, f), (torch.zeros(b, l, d), torch.zeros(b, d)))
    torch.autograd.grad(lp, x, torch.zeros(b, t))
    torch.autograd.grad(loss, x)
    (rec,) = [a for name, a in calls if name == "pp_gated_recurrence_bwd"]
    assert rec[0].stride() == (rec[1], rec[2], 1) and rec[3].stride() == (rec[4], rec[5], 1)
    assert all(rec[i].is_contiguous() for i in (7, 8, 9))
    classes = [a for name, a in calls if name == "pp_token_log_probs_bwd"]
    assert len(classes) == 2
    for a in classes:
        assert a[0].stride() == (a[1], a[2], 1) and a[10].stride() == (a[11], a[12], 1)
        assert all(a[i].is_contiguous() for i in (4, 5, 6, 7))


def test_empty_batches_have_empty_gradients(calls):
    for b, t in ((0, 5), (3, 0)):
        x = torch.zeros(b, t, 9, requires_grad=True)
        tokens, rows = torch.zeros(b, t, dtype=torch.int64), torch.zeros(b, t)
        lp = PF.TokenLogProbsFunction.apply(x, tokens, None, True)
        assert torch.autograd.grad(lp, x, rows)[0].shape == x.shape
        loss = PF.ClippedPolicyLossFunction.apply(x, tokens, None, rows, rows, None, 0.2, 0.2, 0.0, 0, True)[0]
        for _ in range(2):
            assert torch.autograd.grad(loss, x, retain_graph=True)[0].shape == x.shape
    assert not calls
