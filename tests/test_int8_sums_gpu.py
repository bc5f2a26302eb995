"""The norm's sum of squares: held to the number of additions that follow one another in the kernel that a row takes, with rows that lose
half a step in nearly every one of them."""
import pytest
import torch

import wg2x2

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _chain(layout, C, dtype):
    """Additions one after another, at most: of a thread's values, then over lanes and warps"""
    if layout == "NCHW":
        own = 64 if C <= 1024 else -(-C // 32) + 4 if C <= 6000 else -(-C // 512)         # (four sums a thread, of eight warps)
    else:
        own = 64 if C <= (16384 if dtype == torch.float32 else 32768) else -(-C // 512)
    return own + 16


def _rows(kind, rows, C, dtype, layout):
    if kind == "random":
        return torch.randn((rows, C), generator=torch.Generator(device="cuda").manual_seed(C), device="cuda").to(dtype)
    if kind == "even":
        return (torch.arange(rows, device="cuda")[:, None] * 0.0371 + 1.0).expand(rows, C).to(dtype).contiguous()
    # a one in front of a thread's values, each of which is just too small to move it: in front of every 32 channels' first four (warps of
    # images), or of the first thousand channels
    small = 2.0 ** -12 * (0.995 if dtype == torch.float32 else 0.99)
    x = torch.full((rows, C), small, device="cuda")
    x[:, :32:4 if layout == "NCHW" else 1] = 1
    return x.to(dtype)


@pytest.mark.parametrize("kind", ["random", "even", "lost"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout,C", [("NCHW", 700), ("NCHW", 1500), ("NCHW", 2500), ("NCHW", 6000), ("NCHW", 9000), ("NHWC", 100), ("NHWC", 1001), ("NHWC", 4096),
                                      ("NHWC", 16384), ("NHWC", 40000), ("NHWC", 200001)])
def test_sum_of_squares(layout, C, dtype, kind):
    x, eps = _rows(kind, 40, C, dtype, layout), 1e-6
    w = torch.ones(C, device="cuda")
    q, s = wg2x2.rms_norm_int8(x if layout == "NHWC" else x.view(40, C, 1, 1), w, eps=eps, layout=layout)
    h = x.double()
    want = h.abs().amax(1) / 127 / torch.sqrt(h.square().mean(1) + eps)
    # a square and the additions, of which the root halves the error, as it does of the mean's division and of eps; the root, a / 127, the quotient
    tol = 1.01 * (0.5 * (1 + _chain(layout, C, dtype) + 2) + 3) * U
    off = ((s.flatten().double() - want).abs() / want).max().item()
    assert off <= tol, (off / U, tol / U)


@pytest.mark.parametrize("layout,C", [("NHWC", 64), ("NHWC", 1001), ("NHWC", 40000), ("NCHW", 64), ("NCHW", 2500), ("NCHW", 9000)])
def test_large_eps_counts(layout, C):
    """eps next to a mean square of its size, where their sum leaves 32 bits and where the sum of the squares alone does"""
    for size, eps in ((1.0, 1e38), (1e18, 1e36), (1.7e19, 3e38), (1.8e19, 3.4e38), (1e19, 3.4e38), (1e20, 3.4e38), (1e18, 3.4e38)):
        x = (1 + torch.rand((40, C), generator=torch.Generator(device="cuda").manual_seed(C), device="cuda")) * size
        q, s = wg2x2.rms_norm_int8(x if layout == "NHWC" else x.view(40, C, 1, 1), torch.ones(C, device="cuda"), eps=eps, layout=layout)
        h = x.double()
        want = h.amax(1) / 127 / torch.sqrt(h.square().mean(1) + float(torch.tensor(eps, dtype=torch.float32)))
        tol = 1.01 * (0.5 * (1 + _chain(layout, C, torch.float32) + 2) + 3) * U
        assert ((s.flatten().double() - want).abs() <= tol * want + 2.0 ** -149).all(), (size, eps)
