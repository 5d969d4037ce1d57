"""The 4-bit format's restatement (oracle/mla_fp4_ref.py) against independent definitions."""
from fractions import Fraction

import numpy as np
import torch

from oracle import mla_fp4_ref as F4

VALUES = [Fraction(v) / 2 for v in (0, 1, 2, 3, 4, 6, 8, 12)]


def test_decode_table():
    want = [float(v) for v in VALUES] + [-float(v) for v in VALUES]
    assert F4.e2m1_decode(np.arange(16)).tolist() == want


def test_encode_is_nearest_ties_to_even():
    xs = [i / 64 for i in range(0, 64 * 7)] + [0.25 + 2 ** -40, 5 - 2 ** -40, 5 + 2 ** -40, 1e-30]
    for x in xs:
        f = min(Fraction(x), Fraction(6))
        best = min(range(8), key=lambda c: (abs(VALUES[c] - f), c & 1))
        assert F4.e2m1_encode(np.array([x]))[0] == best, x
        assert F4.e2m1_encode(np.array([-x]))[0] == best | 8, x


def test_scale_is_the_smallest_power_of_two():
    amax = torch.tensor([0.0, 6.0, 6.03125, 5.9, 3.0, 3.02, 1e-38, 2.0 ** -133, 3.3e38, 448.0, 0.75]).to(torch.bfloat16)
    for a in amax.tolist():
        want = 0 if a == 0 else next(k for k in range(-126, 128) if Fraction(a) <= 6 * Fraction(2) ** k)
        assert F4.scale_byte(np.array([a]))[0] == want + 127, a
    assert F4.scale_byte(np.array([np.inf, np.nan])).tolist() == [255, 255]


def test_round_trip_is_exact_on_the_grid():
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 256, (40, 256), generator=g, dtype=torch.uint8).numpy()
    codes[:, ::16] |= 7  # every block holds a 6: its scale is the one it was made with
    byte = torch.randint(20, 230, (40, 16), generator=g, dtype=torch.uint8).numpy()
    v = F4.dequantize_latent(codes, byte)
    assert np.array_equal(v, torch.from_numpy(v).to(torch.bfloat16).double().numpy())  # fits bf16
    c2, b2 = F4.quantize_latent(torch.from_numpy(v).to(torch.bfloat16))
    assert np.array_equal(b2, byte) and np.array_equal(c2, codes)


def test_bad_blocks_are_marked():
    x = torch.ones(3, 512)
    x[0, 40], x[1, 511] = float("nan"), float("-inf")
    codes, byte = F4.quantize_latent(x)
    v = F4.dequantize_latent(codes, byte)
    assert np.isnan(v[0, 32:64]).all() and np.isnan(v[1, 480:]).all() and np.isnan(v).sum() == 64


def test_values_past_the_largest_are_stored_as_it():
    top = torch.finfo(torch.bfloat16).max
    x = torch.zeros(4, 512)
    x[0, :4] = torch.tensor([top, -top, 1.75 * 2.0 ** 127, 2.5 * 2.0 ** 126])
    x[1, 32:34] = torch.tensor([1.5 * 2.0 ** 127, -1.5 * 2.0 ** 127])
    x[2, 0] = -top
    codes, byte = F4.quantize_latent(x)
    v = F4.dequantize_latent(codes, byte)
    assert v[0, :4].tolist() == [1.5 * 2.0 ** 127, -1.5 * 2.0 ** 127, 1.5 * 2.0 ** 127, 2.0 ** 127]  # the tie to the even code
    assert v[1, 32:34].tolist() == [1.5 * 2.0 ** 127, -1.5 * 2.0 ** 127] and byte[1, 1] == 125 + 127
    assert np.isfinite(torch.from_numpy(v).to(torch.bfloat16).float().numpy()).all() and byte[0, 0] == 126 + 127
