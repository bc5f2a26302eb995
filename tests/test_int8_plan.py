"""How products of codes are cut (csrc/linear_int8.cuh, li_choose): the plan taken for the products whose plans were timed is the fastest of them."""
import ctypes
import itertools

import pytest

from wg2x2._lib import lib

B200 = (74, 33, 15)          # clusters of 2, 4 and 8 CTAs that run at once


def plan(rows, C, K, nchw=False, at_once=B200):
    out = (ctypes.c_int * 3)()
    assert lib.wg2x2_test_linear_int8_plan(rows, C, K, int(nchw), (ctypes.c_int * 3)(*at_once), out) == 0
    return tuple(out)


# rows, C, K (pixels of an NCHW result): us in a graph, weights from memory in turn, of the plans (columns, CTAs that share a tile, pairs of SMs)
TIMED = [
    ((24, 2048, 8191), {(32, 1, 0): 7.17, (16, 1, 0): 7.61, (32, 2, 0): 9.22}),
    ((32, 2048, 8191), {(32, 1, 0): 7.17, (16, 1, 0): 7.61, (32, 2, 0): 9.22}),
    ((64, 4096, 8192), {(32, 1, 0): 10.83, (64, 1, 0): 11.11, (64, 2, 0): 14.63, (16, 1, 0): 17.27}),
    ((64, 512, 8000), {(64, 1, 0): 4.10, (32, 1, 0): 4.48, (16, 1, 0): 5.88, (64, 2, 0): 7.42}),
    ((16, 8192, 1024), {(16, 8, 0): 7.17, (16, 4, 0): 8.58, (16, 2, 0): 11.65, (16, 1, 0): 16.00}),
    ((32, 8192, 4096), {(32, 4, 0): 12.00, (16, 2, 0): 13.45, (32, 2, 0): 14.04, (32, 1, 0): 16.68}),
    ((100, 8192, 1024), {(32, 4, 0): 9.73, (128, 8, 0): 10.50, (64, 4, 0): 10.75, (16, 2, 0): 12.03}),
    ((256, 4096, 4096), {(64, 1, 0): 10.39, (128, 1, 0): 11.41, (128, 1, 1): 13.75, (256, 1, 0): 15.07}),
    ((256, 512, 1000), {(32, 1, 0): 4.35, (16, 1, 0): 4.48, (64, 1, 0): 4.48, (128, 1, 0): 4.99}),
    ((2000, 2048, 2048), {(256, 1, 0): 10.11, (256, 1, 1): 11.52, (128, 1, 0): 11.77, (128, 1, 1): 14.21}),
    ((8192, 1024, 1024), {(256, 1, 0): 10.75, (256, 1, 1): 12.29, (128, 1, 0): 13.19, (128, 1, 1): 15.75}),
    ((16384, 512, 2048), {(256, 1, 0): 22.40, (256, 1, 1): 26.24, (128, 1, 0): 27.39, (128, 1, 1): 32.13}),
    ((8192, 4096, 4096), {(256, 1, 1): 89.23, (256, 1, 0): 95.95, (128, 1, 0): 120.67, (128, 1, 1): 126.32}),
    ((700, 4100, 9000), {(256, 1, 1): 35.16, (128, 1, 1): 38.91, (128, 1, 0): 44.71, (256, 1, 0): 45.05}),
    ((17 * 784, 1024, 513, True), {(128, 1, 0): 14.21, (128, 1, 1): 16.00, (256, 1, 0): 16.13, (256, 1, 1): 16.51}),
    ((64 * 3136, 64, 64, True), {(64, 1, 0): 15.62, (32, 1, 0): 18.05, (16, 1, 0): 35.58}),
]


@pytest.mark.parametrize("size,times", TIMED, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else "")
def test_takes_the_fastest_plan(size, times):
    assert plan(*size) == min(times, key=times.get)


def test_plans_can_be_run():
    """Every plan: a power of two of columns, shares with a piece of the contraction each, no more clusters than run at once"""
    for rows, C, K, nchw in itertools.product((1, 5, 17, 33, 100, 257, 1000, 5000, 33333, 2 ** 31 - 300), (1, 100, 129, 1000, 8192, 131071), (1, 16, 100, 1000, 9000), (False, True)):
        for at_once in (B200, (0, 0, 0), (70, 20, 0)):
            N, S, pairs = plan(rows, C, K, nchw, at_once)
            assert N in (16, 32, 64, 128, 256) and S in (1, 2, 4, 8) and S <= -(-C // 128) and pairs in (0, 1)
            lanes, cols = (rows, K) if nchw else (K, rows)
            if S > 1:
                assert N <= 128 and not pairs and -(-lanes // 128) * -(-cols // N) <= at_once[(2, 4, 8).index(S)]
            if pairs:
                assert N == 256 and at_once[0]


def test_refuses():
    at_once, out = (ctypes.c_int * 3)(*B200), (ctypes.c_int * 3)()
    for bad in ((0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1, 131072, 1, 0), (2 ** 31, 1, 1, 0), (1, 1, 1, 2)):
        assert lib.wg2x2_test_linear_int8_plan(*bad, at_once, out) == -1
    assert lib.wg2x2_test_linear_int8_plan(1, 1, 1, 0, None, out) == -1 and lib.wg2x2_test_linear_int8_plan(1, 1, 1, 0, at_once, None) == -1
