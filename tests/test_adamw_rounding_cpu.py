"""What the 8 random bits of an 8-bit moment's rounding can carry, and the betas that are refused because they cannot."""
import ctypes

import numpy as np
import pytest
import torch

import seq_oracle as so
from language_interpolation_amd import _lib
from language_interpolation_amd import functional as PF
from language_interpolation_amd.train import AdamW


def _decay(b2, steps):
    """A second moment without gradients: its mean after the steps, in units of its mean before, and the share that moved."""
    rng = np.random.default_rng(0)
    x = np.square(rng.normal(size=256 * 100)).astype(np.float32)
    first = v = so.decode(*so.encode(x, so.noise(x.size, 1, 1, 0)[1], 30, False), 30, False)
    for s in range(steps):
        v = so.decode(*so.encode(v * np.float32(b2), so.noise(v.size, 1, s + 2, 0)[1], 30, False), 30, False)
    big = first > first.max() * 1e-3
    return float(v[big].mean() / first[big].mean()), float((v != first)[big].mean())


def test_moments_follow_the_betas_in_use():
    """b^n to a few per cent: a code step is rounded up or down by 256ths of it."""
    for b2, steps, within in ((0.99, 20, 0.01), (0.999, 200, 0.02), (0.9995, 400, 0.03)):
        mean, _ = _decay(b2, steps)
        assert abs(mean / b2 ** steps - 1) < within


def test_betas_too_near_one_would_stand_still_and_are_refused():
    assert _decay(0.9999, 300) == (1.0, 0.0)  # every entry keeps its code for ever
    most = 1 - 2.0 ** -12
    p = torch.zeros(5000, requires_grad=True)
    for betas in ((0.9, 0.9999), (0.9, np.nextafter(most, 1.0)), (0.9999, 0.99)):
        with pytest.raises(ValueError, match="8-bit"):
            AdamW([p], betas=betas, moment_bits=8)
        with pytest.raises(ValueError, match="8-bit"):
            PF.adamw_step([p], [p], [p], [p], 1, lr=1e-3, betas=betas, avg_exponents=[p], sq_exponents=[p])
        AdamW([p], betas=betas)
    AdamW([p], betas=(0.9, most), moment_bits=8)
    # the groups' own numbers count
    with pytest.raises(ValueError, match="8-bit"):
        AdamW([{"params": [p], "betas": (0.9, 0.9999)}], moment_bits=8)
    with pytest.raises(ValueError, match="8-bit"):
        AdamW([{"params": [p], "moment_bits": 8}], betas=(0.9, 0.9999))


def test_the_entry_refuses_them():
    def entry(bits, b1, b2):
        a = (ctypes.c_void_p * 1)(4097)  # (an odd address: nothing is launched whatever the betas)
        one = (ctypes.c_int64 * 1)(1)
        return _lib.load().pp_adamw_step(1, 0, bits, a, a, None, a, a, a, a, (ctypes.c_int64 * 1)(8), one, None, 1e-3, b1, b2,
                                         1e-8, 0.0, None, 0, 0, None)
    most = 1 - 2.0 ** -12
    assert entry(8, 0.9, 0.9999) == -6 and entry(8, 0.9999, 0.9) == -6
    assert entry(8, 0.9, most) == -3 and entry(32, 0.9999, 0.9999) == -3
