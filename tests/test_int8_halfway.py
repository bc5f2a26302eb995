"""The codes of 16-bit values next to the half way points: every pair of mantissas, in the arithmetic of csrc/quantize_int8.cu (fast_codes, COARSE), which
decides them by rounding the quotient to eight units of its last place."""
import numpy as np
import pytest


def snapped(u, a):
    """That kernel's code of u in a row whose largest magnitude is a, in 32 bits as it computes them"""
    inv = np.float32(127) / a
    bits = (u * inv).astype(np.float32).view(np.uint32)
    m = ((bits + np.uint32(4)) & np.uint32(0xFFFFFFF8)).view(np.float32) + np.float32(12582912)
    return m.view(np.uint32).astype(np.uint8).view(np.int8)


def pairs(bits, low_a=0):
    """(a as a column, all u with |u| <= a as a row) for mantissas of `bits` bits, u's exponent 0 to 11 below a's"""
    m = np.arange(1 << (bits - 1), 1 << bits, dtype=np.float32) * np.float32(2.0 ** (1 - bits))
    return m[:, None], np.concatenate([m * np.float32(2.0 ** -e) for e in range(12)])[None, :]


@pytest.mark.parametrize("bits", [8, 11])
@pytest.mark.parametrize("binade", [-100, 0, 3, 100])
def test_every_pair_of_mantissas(bits, binade):
    a, u = pairs(bits)
    two = np.float32(2.0 ** binade)
    for i in range(0, len(a), 128):
        part = a[i:i + 128]
        for sign in (1, -1):
            exact = np.rint(127 * u.astype(np.float64) / part.astype(np.float64))          # (a quotient off a half way point is 2^-20 from it, relative)
            ok = u <= part
            got = snapped(sign * u * two, part * two)
            assert (got == sign * exact)[ok].all()


def test_half_way_points_are_among_them():
    a, u = pairs(11)
    twice = 254 * u.astype(np.float64) / a.astype(np.float64)
    half = (twice == np.rint(twice)) & (twice % 2 == 1) & (u <= a)
    # a / 2 is half way for every a.  Others are where a's mantissa is j times 127, j = 9 .. 16: the j k / 2 that have 11 bits, k odd, for j = 15 those up
    # to k = 136
    assert (half.sum(1) >= 1).all() and (half.sum(1) > 1).sum() == 8 and half.sum(1).max() > half.sum(1)[127 * 15 - 1024] == 68
