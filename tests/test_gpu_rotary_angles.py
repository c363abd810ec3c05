"""Cosines and sines as the rotary layer makes them, one pair at a time, against 80-bit arithmetic: near and far positions, frequencies below
and above one."""
import numpy as np
import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu


def _angles(positions, frequency):
    """cos and sin of the exact product: of 31 by 24 bits and of 31 by 29 bits, each of which 64 bits hold."""
    p = positions.astype(np.longdouble)
    coarse = np.float64(np.float32(frequency))
    a, b = p * np.longdouble(coarse), p * np.longdouble(np.float64(frequency) - coarse)
    return np.cos(a) * np.cos(b) - np.sin(a) * np.sin(b), np.sin(a) * np.cos(b) + np.cos(a) * np.sin(b)


@pytest.mark.parametrize("most", [5000, 1 << 20, (1 << 31) - 1], ids=["near", "2^20", "2^31"])
@pytest.mark.parametrize("pairing", ["HALVES", "NEIGHBOURS"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_unit_vectors(most, pairing, dtype):
    """The vector (1, 0) becomes (cos, sin).  Sine and cosine are off by two steps of theirs at most (a step of numbers in [1/2, 1) is U), what is added
    for the part of the angle that 32 bits do not hold is rounded once more: 3 U, and half a step of the type."""
    from dihydrogen_amd.tokens import RotaryPairing, RotaryPositions
    assert np.finfo(np.longdouble).nmant >= 63
    frequencies = torch.tensor([1.0, 0.7498942093324559, 10000.0 ** (-5 / 16), 3.0001], dtype=torch.float64)
    layer = RotaryPositions(16, [4], pairing=RotaryPairing[pairing])
    layer.frequencies = frequencies
    rng = np.random.default_rng(1)
    positions = rng.integers(-most, most, 20000)
    positions[:3] = most, -most, 0
    x = torch.zeros(1, 20000, 1, 16, dtype=dtype, device="cuda")
    first, second = (slice(0, 4), slice(4, 8)) if pairing == "HALVES" else (slice(0, 8, 2), slice(1, 8, 2))
    x[..., first] = 1
    y = torch.empty_like(x)
    layer.forward(x, torch.tensor(positions, dtype=torch.int32, device="cuda")[None], y)
    for i, f in enumerate(frequencies.tolist()):
        for got, want in zip((y[0, :, 0, first][:, i], y[0, :, 0, second][:, i]), _angles(positions, f)):
            want = torch.tensor(want.astype(np.float64), device="cuda")
            half = 0.0 if dtype == torch.float32 else ref.half_step(dtype)
            ref.check(got, want, 3 * ref.U + half * want.abs(), f"frequency {f}")
