"""The 8-bit oracle's quotients: its codes of 16-bit rows are those of the exact rational quotient, next to ties too."""
import numpy as np
import pytest

from oracle import w8a8 as o8


def exact_code(a, b, f):
    """round_half_even(127 a / (b 2^f)) in whole numbers."""
    q, r = np.divmod(254 * a, b << (f + 1))  # 254 a / (b 2^(f+1))
    twice = 2 * r - (b << (f + 1))
    return q + ((twice > 0) | ((twice == 0) & (q % 2 == 1)))


@pytest.mark.parametrize("bits", [8, 11])  # bf16, fp16
def test_codes_of_16_bit_values_are_exact(bits):
    lo, hi = 1 << (bits - 1), 1 << bits
    a = np.arange(lo, hi, dtype=np.int64)
    nearest = 1.0
    for f in range(0, 9):
        for b in np.arange(lo, hi, max(1, (hi - lo) // 256), dtype=np.int64):
            v = a[a <= b << f] if f == 0 else a
            if not len(v):
                continue
            row = np.concatenate(([np.float32(b) * np.float32(2.0**f)], v.astype(np.float32)))
            codes, most = o8.codes(row[None])
            assert most[0] == b * 2.0**f and codes[0, 0] == 127
            assert np.array_equal(codes[0, 1:], exact_code(v, b, f)), (b, f)
            twice = 254 * v  # the quotient is twice / (b 2^(f+1)); ties are odd multiples of b 2^f
            odd = 2 * (twice // (2 * (b << f))) + 1
            off = np.abs(twice - odd * (b << f)) / twice
            if (off > 0).any():
                nearest = min(nearest, off[off > 0].min())
    assert 1 / (254 * hi) <= nearest < 2.0**-15  # the bound, and that the rows come near it


def test_the_nearest_to_a_tie():
    codes, _ = o8.codes(np.array([[2031 * 256, 2047]], dtype=np.float32))  # 127 * 2047 / (2031 * 256) = 0.50000192
    assert codes.tolist() == [[127, 1]]
