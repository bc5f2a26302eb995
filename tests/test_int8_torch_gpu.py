"""The 8-bit calls and what torch knows of tensors: counted writes, views that stand for other values than their memory's."""
import pytest
import torch

import wg2x2

pytestmark = pytest.mark.gpu


def test_outputs_count_as_written():
    """A tensor that a backward pass needs and a call writes over: torch refuses that pass"""
    x, one = torch.randn((6, 32), device="cuda"), torch.ones(32, device="cuda")
    q, s = wg2x2.quantize_int8(x)
    w = torch.randn((6, 32), device="cuda", requires_grad=True)

    def refused(t, write):
        loss = (w[:, :1] * t.float().reshape(6, -1)[:, :1] * 2).sum() if t.dtype == torch.int8 else (w.flatten()[:t.numel()] * t.flatten()).sum()
        before = t._version
        write()
        assert t._version > before
        if t.dtype != torch.int8:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
    refused(q, lambda: wg2x2.quantize_int8(x, out=q, scale_out=torch.empty_like(s)))
    refused(s, lambda: wg2x2.quantize_int8(x, scale_out=s))
    refused(s, lambda: wg2x2.rms_norm_int8(x, one, scale_out=s))
    refused(q, lambda: wg2x2.rms_norm_int8(x, one, out=q))
    h = torch.randn_like(x)
    refused(h, lambda: wg2x2.rms_norm_int8(x, one, residual=h, residual_out=h))
    y = torch.randn((6, 6), device="cuda")
    refused(y, lambda: wg2x2.linear_int8(q, s, q.clone(), s.clone(), out=y))
    with torch.inference_mode():
        s2 = torch.empty_like(s)
        wg2x2.quantize_int8(x, scale_out=s2)
    wg2x2.quantize_int8(x, scale_out=s2)
    assert torch.equal(s2, wg2x2.quantize_int8(x)[1])


def test_negated_views_are_refused():
    """The imaginary part of a conjugate: a view whose values are the negatives of its memory's"""
    x = torch.randn((5, 1), dtype=torch.complex64, device="cuda").conj().imag
    assert x.is_neg()
    with pytest.raises(ValueError, match="negated"):
        wg2x2.quantize_int8(x)
    with pytest.raises(ValueError, match="negated"):
        wg2x2.rms_norm_int8(x.resolve_neg(), torch.ones(1, device="cuda"), residual=x)
    q, s = wg2x2.quantize_int8(x.resolve_neg())
    assert torch.equal(q.float().flatten() * s, x.flatten().sign() * 127 * s)
