"""Products in 8 bits one behind the other and between other kernels with tensor memory, launched without a graph, so that each next one comes in
while the one before still runs."""
import pytest
import torch

import wg2x2

pytestmark = pytest.mark.gpu


def test_products_between_kernels_with_tensor_memory():
    g = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    calls = []
    # clusters that share a tile; a tile an SM, of few and of many; pairs of SMs; small products
    for rows, C, K in ((9, 8192, 256), (24, 2048, 8191), (64, 8192, 1000), (256, 512, 1000), (300, 384, 4000), (2600, 2000, 3000), (4, 256, 100)):
        q, w = wg2x2.quantize_int8(rnd(rows, C)), wg2x2.quantize_int8(rnd(K, C))
        calls.append(lambda q=q, w=w: wg2x2.linear_int8(*q, *w, dtype=torch.bfloat16))
    x, w1 = rnd(2, 128, 14, 14), wg2x2.round_tf32(rnd(256, 128, 1, 1))
    calls.append(lambda: wg2x2.conv1x1(x, w1))
    for B, H, C, layout in ((1, 14, 256, "NCHW"), (2, 28, 128, "NCHW"), (4, 56, 64, "NCHW"), (2, 14, 256, "NHWC")):
        xl = rnd(B, C, H, H) if layout == "NCHW" else rnd(B, H, H, C)
        prepared = wg2x2.prepare_weights(rnd(16, C, C) / C ** 0.5)
        calls.append(lambda xl=xl, prepared=prepared, C=C, layout=layout: wg2x2.layer_fwd_prepared(xl, prepared, C, layout=layout))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    order = torch.randint(len(calls), (1500,), generator=torch.Generator().manual_seed(1)).tolist()
    for part in range(0, len(order), 100):
        got = [(i, calls[i]()) for i in order[part:part + 100]]
        assert all(torch.equal(y, want[i]) for i, y in got)
    assert wg2x2.last_device_status()[0] == 0


@pytest.mark.parametrize("rows,C,K", [(1, 4096, 300), (4, 256, 100), (32, 512, 1000)])
def test_dropped_load_is_of_the_next_product(rows, C, K):
    """The hook that makes a wait run out is used up by the next product, also by a small one, which waits for nothing"""
    from wg2x2._lib import lib
    q, w = wg2x2.quantize_int8(torch.randn((rows, C), device="cuda")), wg2x2.quantize_int8(torch.randn((K, C), device="cuda"))
    want = wg2x2.linear_int8(*q, *w)
    x, w1 = torch.randn((2, 64, 14, 14), device="cuda"), wg2x2.round_tf32(torch.randn((64, 64, 1, 1), device="cuda"))
    other = wg2x2.conv1x1(x, w1)
    assert wg2x2.last_device_status()[0] == 0
    assert lib.wg2x2_set_wait_limit(20000) == 0 and lib.wg2x2_test_drop_load(0) == 0
    try:
        assert torch.equal(wg2x2.linear_int8(*q, *w), want)
        torch.cuda.synchronize()
        assert torch.equal(wg2x2.conv1x1(x, w1), other) and wg2x2.last_device_status()[0] == 0
    finally:
        lib.wg2x2_set_wait_limit(0)
        lib.wg2x2_test_drop_load(-1)
        wg2x2.last_device_status()
