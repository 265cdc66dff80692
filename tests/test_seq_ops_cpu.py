"""Sequence-model operators without a GPU: refusals of the C entries and of the Python ones, and the
restatements the GPU tests compare with."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import seq_oracle as so
from language_interpolation_amd import _lib
from language_interpolation_amd import functional as PF

NULL, OK, BAD, ODD = None, ctypes.c_void_p(4096), ctypes.c_void_p(4098), ctypes.c_void_p(4097)
E_NULL, E_SHAPE, E_ALIGN, E_WS, E_METHOD, E_RANGE = -1, -2, -3, -4, -5, -6


def _rec(z=OK, f=OK, y=OK, h=OK, dtype=0, b=2, l=5, d=8, starts=NULL, h0=NULL):
    lib = _lib.load()
    return lib.pp_gated_recurrence_fwd(z, l * d, d, f, l * d, d, dtype, h0, NULL, NULL, y, h, starts, NULL, 0, b, l,
                                       d, NULL)


def test_recurrence_entry_refuses():
    lib = _lib.load()
    for kw in (dict(z=NULL), dict(f=NULL), dict(y=NULL), dict(h=NULL)):
        assert _rec(**kw) == E_NULL
    for kw in (dict(b=0), dict(l=0), dict(d=0), dict(d=-4), dict(b=65536)):
        assert _rec(**kw) == E_SHAPE
    assert _rec(dtype=3) == E_METHOD and _rec(dtype=-1) == E_METHOD
    assert _rec(z=BAD) == E_ALIGN and _rec(f=ODD, dtype=1) == E_ALIGN
    assert _rec(h0=BAD) == E_ALIGN and _rec(starts=BAD) == E_ALIGN
    assert _rec(l=2 ** 31 - 1) == E_RANGE
    assert _rec(b=65535, l=32767, d=1) == E_RANGE  # more than 2^32 threads
    assert lib.pp_gated_recurrence_step(OK, 8, OK, 8, 0, OK, 1 << 20, OK, 65535, 1 << 20, NULL) == E_RANGE
    assert lib.pp_gated_recurrence_step(OK, 8, OK, 8, 0, OK, 7, OK, 2, 8, NULL) == E_SHAPE
    assert lib.pp_gated_recurrence_step(OK, 8, OK, 8, 0, NULL, 8, OK, 2, 8, NULL) == E_NULL
    assert lib.pp_gated_recurrence_bwd(OK, 8, 8, OK, 8, 8, 0, NULL, NULL, NULL, OK, 8, 8, NULL, OK, OK, NULL, NULL, 0,
                                       1, 1, 8, NULL) == E_NULL  # no kept states
    steps = 16
    assert [lib.pp_gated_recurrence_starts(l) for l in (0, 1, steps, steps + 1)] == [0, 1, 1, 2]
    need = lib.pp_gated_recurrence_workspace_bytes(1, 100000, 64)
    if need:
        assert lib.pp_gated_recurrence_fwd(OK, 1, 1, OK, 1, 1, 0, NULL, NULL, NULL, OK, OK, NULL, OK, need - 1, 1,
                                           100000, 64, NULL) == E_WS


def _pol(logits=OK, tokens=OK, old=OK, adv=OK, out=OK, stats=NULL, coef=NULL, grad=NULL, gb=None, gt=None, ws=OK,
         nbytes=1 << 20, dtype=0, low=0.2, high=0.2, b=2, t=3, v=8):
    return _lib.load().pp_clipped_policy_loss_fwd(logits, t * v, v, dtype, tokens, NULL, old, adv, t, 1, NULL, low, high,
                                                  0.0, 0, out, stats, coef, grad, t * v if gb is None else gb,
                                                  v if gt is None else gt, ws, nbytes, b, t, v, NULL)


def test_policy_entry_refuses():
    lib = _lib.load()
    for kw in (dict(logits=NULL), dict(tokens=NULL), dict(old=NULL), dict(adv=NULL), dict(out=NULL), dict(grad=OK),
               dict(grad=OK, stats=OK), dict(grad=OK, coef=OK)):
        assert _pol(**kw) == E_NULL
    for kw in (dict(b=0), dict(t=0), dict(v=0), dict(low=-0.1), dict(high=float("nan"))):
        assert _pol(**kw) == E_SHAPE
    assert _pol(dtype=7) == E_METHOD
    assert _pol(logits=BAD) == E_ALIGN
    full = dict(grad=OK, stats=OK, coef=OK)
    assert _pol(**dict(full, grad=ctypes.c_void_p(4104))) == E_ALIGN  # another offset in 16 bytes
    assert _pol(**full, gt=9, gb=28) == E_ALIGN and _pol(**full, gb=26) == E_ALIGN
    assert _pol(**full, gt=4) == E_SHAPE and _pol(**full, gb=20) == E_SHAPE  # rows that overlap
    assert _pol(ws=NULL) == E_WS and _pol(nbytes=8) == E_WS
    assert _pol(b=1 << 20, t=1 << 20) == E_RANGE
    assert lib.pp_token_log_probs_fwd(OK, 8, 8, 0, OK, NULL, NULL, NULL, 1, 1, 8, NULL) == E_NULL
    assert lib.pp_token_log_probs_fwd(OK, 8, 8, 0, ctypes.c_void_p(4100), NULL, OK, NULL, 1, 1, 8, NULL) == E_ALIGN
    assert lib.pp_token_log_probs_bwd(OK, 8, 8, 0, OK, NULL, NULL, OK, NULL, 0, OK, 8, 8, 1, 1, 8, NULL) == E_NULL


def _adam(count=1, dtype=0, bits=32, p=4096, g=4096, m=4096, v=4096, w=None, e=None, n=8, step=1, b1=0.9, b2=0.99):
    def arr(x):
        return None if x is None else (ctypes.c_void_p * max(count, 1))(*[x] * max(count, 1))
    k = max(count, 1)
    return _lib.load().pp_adamw_step(count, dtype, bits, arr(p), arr(g), arr(w), arr(m), arr(v), arr(e), arr(e),
                                     (ctypes.c_int64 * k)(*[n] * k), (ctypes.c_int64 * k)(*[step] * k), None, 1e-3, b1,
                                     b2, 1e-8, 0.0, None, 0, 0, None)


def test_adamw_entry_refuses():
    lib = _lib.load()
    assert _adam(count=0) == E_SHAPE and _adam(count=33) == E_SHAPE
    assert _adam(dtype=5) == E_METHOD and _adam(bits=16) == E_METHOD
    assert _adam(p=0) == E_NULL and _adam(dtype=1) == E_NULL and _adam(bits=8) == E_NULL
    assert _adam(n=0) == E_SHAPE and _adam(step=0) == E_SHAPE and _adam(b1=1.0) == E_SHAPE and _adam(b2=-0.1) == E_SHAPE
    assert _adam(b1=float("nan")) == E_SHAPE
    assert _adam(n=1 << 40) == E_RANGE and _adam(n=1 << 34) == E_RANGE
    assert _adam(g=4098) == E_ALIGN and _adam(dtype=2, w=4096, p=4097) == E_ALIGN
    two = (ctypes.c_void_p * 2)(4096, 4096)
    assert lib.pp_count_step(2, two, None) == E_SHAPE  # the same counter twice
    assert lib.pp_count_step(1, (ctypes.c_void_p * 1)(4100), None) == E_ALIGN
    assert [lib.pp_moment_blocks(n) for n in (0, 1, 256, 257)] == [0, 1, 1, 2]
    assert lib.pp_decode_moment(OK, OK, OK, 0, 1, 0, None) == E_SHAPE
    assert lib.pp_decode_moment(OK, NULL, OK, 0, 1, 5, None) == E_NULL


def test_there_is_no_cpu_path():
    z = torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        PF.gated_recurrence(z, z)
    with pytest.raises(RuntimeError, match="no CPU path"):
        PF.gated_recurrence_step(z[0], z[0], z[0])
    with pytest.raises(RuntimeError, match="no CPU path"):
        PF.token_log_probs(z, torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        PF.clipped_policy_loss(z, torch.zeros(2, 3, dtype=torch.int64), z[..., 0], z[..., 0])
    with pytest.raises(RuntimeError, match="no CPU path"):
        PF.adamw_step([z], [z], [z], [z], 1, lr=1e-3)
    from language_interpolation_amd.train import AdamW
    p = torch.zeros(3, requires_grad=True)
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="MI355X"):
        AdamW([p]).step()


def test_configured_optimizers():
    import os

    from language_interpolation_amd import train as T
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "configs",
                        "high_order_interpolation.yaml")
    for name, bits in (("adamw", 32), ("adamw_8bit", 8)):
        net = T.prediction_net(T.load_config(root, [f"optimizer={name}", "optimizer.lr=2e-4"]), device="cpu")
        opt = net.configure_optimizers(capturable=True)
        group = opt.param_groups[0]
        assert isinstance(opt, T.AdamW) and group["moment_bits"] == bits and group["lr"] == 2e-4
        assert group["weight_decay"] == 1e-2 and group["capturable"]


def test_restated_recurrence_is_the_formula_and_its_gradient():
    g = torch.Generator().manual_seed(0)
    z, f = (torch.randn(2, 9, 3, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    h0 = torch.randn(2, 3, generator=g, dtype=torch.float64, requires_grad=True)
    gy, gh = torch.randn(2, 9, 3, generator=g).double(), torch.randn(2, 3, generator=g).double()
    lengths = torch.tensor([9, 4])
    reset = torch.zeros(2, 9, dtype=torch.bool)
    reset[0, 5] = reset[1, 0] = True
    rows, last = [], []
    for i in range(2):
        h, out = h0[i], []
        for t in range(9):
            if t < lengths[i]:
                a = torch.sigmoid(f[i, t])
                h = a * (0.0 if reset[i, t] else h) + (1 - a) * z[i, t]
                out.append(h)
            else:
                out.append(torch.zeros_like(h))
        rows.append(torch.stack(out))
        last.append(h)
    y, h = torch.stack(rows), torch.stack(last)
    grads = torch.autograd.grad((y, h), (z, f, h0), (gy, gh))
    got = so.recurrence(z.detach(), f.detach(), h0.detach(), lengths, reset, gy, gh)
    for name, want in zip(("y", "h", "gz", "gf", "gh0"), (y, h) + grads):
        assert torch.allclose(got[name][0], want.detach(), rtol=1e-12, atol=1e-12), name
        assert bool((got[name][1] < 1e-4).all())


def test_restated_policy_is_the_formula_and_its_gradient():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 4, 6, generator=g, dtype=torch.float64, requires_grad=True)
    tokens = torch.randint(0, 6, (3, 4), generator=g)
    old, adv, ref = (torch.randn(3, 4, generator=g) * s for s in (0.3, 1.0, 0.3))
    m = torch.tensor([[1, 1, 0, 1], [0, 0, 0, 0], [1, 0, 0, 0]], dtype=torch.bool)
    lp = torch.log_softmax(x, -1).gather(-1, tokens[..., None])[..., 0]
    old = (lp.detach() + old).float()
    rho = torch.exp(lp - old)
    k = torch.exp(ref - lp) - (ref - lp) - 1
    term = -torch.minimum(rho * adv, rho.clamp(0.8, 1.28) * adv) + 0.1 * k
    for reduction, want in (("token", term[m].mean()),
                            ("sequence", (term[0][m[0]].mean() + term[2][m[2]].mean()) / 2)):
        got = so.policy(x.detach(), tokens, old, adv, ref, m, 0.2, 0.28, 0.1, reduction)
        (grad,) = torch.autograd.grad(want, x, retain_graph=True)
        assert abs(float(got["loss"][0]) - float(want.detach())) < 1e-12
        assert torch.allclose(got["grad"][0], grad, atol=1e-12)


def test_codes_are_unbiased_and_ordered():
    rng = np.random.default_rng(0)
    x = np.square(rng.normal(size=256 * 400)).astype(np.float32)
    mean, count = np.zeros(x.size), 64
    # the subnormal codes are 2^-32 of the block's largest apart (exponent fields 30 to 1, 3 bits)
    floor = np.repeat(x.reshape(-1, 256).max(1), 256) * 2.0 ** -32
    for step in range(count):
        a, b = so.noise(x.size, 7, step + 1, 0)
        code, e = so.encode(x, b, 30, False)
        y = so.decode(code, e, 30, False)
        # three bits of mantissa: never further than 2^-3 of the value
        assert np.all(np.abs(y - x) <= x * 0.125 + floor)
        mean += y / count
    # an entry's mean of 64 has a deviation of at most 2^-4 / 8 of it; the bias over all is far smaller
    big = x > floor * 16
    assert big.mean() > 0.99
    assert abs(float((mean / x - 1)[big].mean())) < 6 * 2.0 ** -7 / np.sqrt(big.sum())
    m = rng.normal(size=2560).astype(np.float32)
    code, e = so.encode(m, so.noise(m.size, 7, 1, 0)[0], 14, True)
    y = so.decode(code, e, 14, True)
    assert np.all(np.sign(y) * np.sign(m) >= 0) and np.all(np.abs(y - m) <= np.abs(m) * 0.125 + np.abs(m).max() * 2.0 ** -16)
    bits = np.concatenate([so.noise(1 << 16, s, s + 1, s)[i] for s in range(4) for i in (0, 1)])
    counts = np.bincount(bits, minlength=256)
    # 2^19 draws in 256 bins: mean 2048, deviation 45
    assert counts.min() > 2048 - 6 * 45 and counts.max() < 2048 + 6 * 45


def test_no_packed_fp32_instruction_in_the_sequence_operators(tmp_path):
    """Some packed-fp32 forms have given wrong results on this chip; the units are compiled without."""
    csrc = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")
    subprocess.run(["make", "-C", csrc, "asm-seq", f"ASMDIR={tmp_path}", "-j", "3"], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    for unit in ("pp_recurrence", "pp_policy", "pp_adamw"):
        text = (tmp_path / f"{unit}.s").read_text()
        assert text.count(".amdhsa_kernel") >= 4
        assert not re.findall(r"v_pk_(?:mul|add|fma)_f32", text), unit
        # nothing spills: a row, or a stretch, is held in registers by design
        assert not re.findall(r"\.vgpr_spill_count:\s+[1-9]", text), unit
