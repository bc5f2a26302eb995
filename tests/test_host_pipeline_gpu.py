"""HostLayerPipeline and weights that change from batch to batch."""
import pytest
import torch

import wg2x2

pytestmark = pytest.mark.gpu


def _batch(pipe, x, Wt):
    y = torch.empty_like(x).pin_memory()
    pipe.submit(x, Wt, y).synchronize()
    return y


@pytest.mark.parametrize("how", ["fresh", "written", "data", "inference"])
def test_weights_of_each_batch(how):
    """A tensor of each batch's own (whose memory has the address of the one before, that was freed), one written to in place, the data of a
    parameter (which counts its own writes), and a tensor whose writes torch does not count"""
    B, H, W, C = 2, 8, 8, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((B, H, W, C)).pin_memory()
    pipe = wg2x2.HostLayerPipeline(B, H, W, C, C, layout="NHWC", math="tf32", chunks=1)
    values = [torch.randn((16, C, C), generator=g, device="cuda") for _ in range(4)]
    want = [wg2x2.layer_fwd_prepared(x.cuda(), wg2x2.prepare_weights(v), C, layout="NHWC").cpu() for v in values]
    with torch.inference_mode(how == "inference"):
        kept = torch.nn.Parameter(torch.zeros((16, C, C), device="cuda"), requires_grad=False)
    places = set()
    for v, y in zip(values, want):
        if how == "fresh":
            Wt = torch.empty_like(v).copy_(v)
        elif how == "data":
            kept.data.copy_(v)
            Wt = kept.data
        else:
            with torch.inference_mode():
                kept.copy_(v)
            Wt = kept
        places.add(Wt.data_ptr())
        assert torch.equal(_batch(pipe, x, Wt), y)
        assert torch.equal(_batch(pipe, x, Wt), y)
        del Wt


@pytest.mark.parametrize("math", ["tf32", "fp32"])
def test_weights_let_go_while_they_are_queued(math):
    B, H, W, C = 2, 8, 8, 32
    x = torch.randn((B, H, W, C)).pin_memory()
    pipe = wg2x2.HostLayerPipeline(B, H, W, C, C, layout="NHWC", math=math, chunks=1)
    value = torch.randn((16, C, C), device="cuda")
    want = _batch(pipe, x, value)
    y = torch.empty_like(x).pin_memory()
    Wt, other = value.clone(), torch.randn((16, C, C), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(pipe.s_run):
        torch.cuda._sleep(40_000_000)
    done = pipe.submit(x, Wt, y)
    del Wt
    pipe._weights(other)                                                          # (what the next batch would do)
    junk = [torch.full((16, C, C), 1e9, device="cuda") for _ in range(50)]        # memory that was given back, on the caller's stream
    done.synchronize()
    assert torch.equal(y, want) and len(junk) == 50
