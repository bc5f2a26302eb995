"""Every pair of 16-bit mantissas through the quantiser's kernels (the arithmetic by itself: test_int8_halfway.py)"""
import pytest
import torch

import wg2x2

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bits", [(torch.float16, 11), (torch.bfloat16, 8)])
@pytest.mark.parametrize("layout", ["NHWC", "NCHW"])
def test_every_pair_of_mantissas(dtype, bits, layout):
    m = torch.arange(1 << (bits - 1), 1 << bits, device="cuda", dtype=torch.float64) * 2.0 ** (1 - bits)
    for binade in ((-2, 14) if dtype == torch.float16 else (-100, 0, 100)):
        below = range(12) if binade > 0 or dtype == torch.bfloat16 else range(10)          # (half's own denormal numbers have fewer bits)
        u = torch.cat([m * 2.0 ** (binade - e) for e in below])
        u = torch.cat([u, -u])
        for parts in (1, 3, 30):                                                           # long rows, shorter ones, and rows of a few hundred values
            for k in range(0, parts, max(1, parts // 3)):
                mine = u[k::parts]
                a = (m * 2.0 ** binade)[:, None]
                x = torch.cat([a, torch.where(mine.abs() <= a, mine, 0.0)], 1).to(dtype)
                assert torch.equal(x.double()[:, 0], a[:, 0])
                want = torch.round(127 * x.double() / a).to(torch.int8)
                xin = x if layout == "NHWC" else x.view(len(x), -1, 1, 1)
                q, s = wg2x2.quantize_int8(xin, layout=layout)
                assert torch.equal(q.reshape(want.shape), want) and torch.equal(s.flatten(), (a[:, 0] / 127).float())
                if layout == "NHWC":
                    odd = torch.cat([x, x], 1)[:, 1:x.shape[1] + 1]                         # (the same values turned by one, rows off 16 bytes)
                    assert torch.equal(wg2x2.quantize_int8(odd)[0], torch.cat([want, want], 1)[:, 1:x.shape[1] + 1])
