"""The 8-bit per-pixel products: refusals of the C ABI (checked before any CUDA call; the pointers are fake) and of the Python calls that
need no GPU."""
import ctypes
import math

import pytest

import wg2x2
from wg2x2._lib import lib

OK, BAD, UNSUPPORTED = 0, -1, -5
F32, F16, BF16 = 0, 1, 2
A = 1 << 20          # fake addresses, far apart


def quantize(X=A, type=F32, ldx=64, Q=2 * A, ldq=64, scale=3 * A, B=10, HW=1, C=64, layout=0, relu=0):
    return lib.wg2x2_quantize_int8(X, type, ldx, Q, ldq, scale, B, HW, C, layout, relu, None)


def norm(X=A, ldx=64, residual=4 * A, ldr=64, residual_out=5 * A, ldo=64, weight=6 * A, weight_f32=0, eps=1e-6, type=BF16, Q=2 * A, ldq=64, scale=3 * A,
         B=10, HW=1, C=64, layout=0):
    return lib.wg2x2_rms_norm_int8(X, ldx, residual, ldr, residual_out, ldo, weight, weight_f32, eps, type, Q, ldq, scale, B, HW, C, layout, None)


def linear(Q=A, ldq=64, q_scale=2 * A, W=3 * A, ldw=64, w_scale=4 * A, bias=5 * A, relu=0, Y=6 * A, type=F32, ldy=32, B=10, HW=1, C=64, K=32, layout=0):
    return lib.wg2x2_linear_int8(Q, ldq, q_scale, W, ldw, w_scale, bias, relu, Y, type, ldy, B, HW, C, K, layout, None)


def test_no_rows_is_no_work():
    assert quantize(B=0) == OK and norm(B=0) == OK and linear(B=0) == OK
    assert quantize(B=0, X=None, Q=None, scale=None) == OK and linear(B=0, Q=None, q_scale=None, Y=None) == OK


@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(layout=2), dict(B=-1), dict(HW=0), dict(C=0), dict(X=None), dict(Q=None), dict(scale=None),
                                 dict(ldx=63), dict(ldq=63), dict(X=A + 2), dict(scale=3 * A + 2), dict(Q=A + 256), dict(scale=A + 256), dict(scale=2 * A + 4),
                                 dict(B=1 << 60, HW=1 << 20)])
def test_quantize_refuses(bad):
    assert quantize(**bad) == BAD


@pytest.mark.parametrize("bad", [dict(type=3), dict(layout=-1), dict(C=-4), dict(weight=None), dict(residual=None), dict(residual_out=None), dict(eps=0.0), dict(eps=-1.0),
                                 dict(eps=math.nan), dict(eps=math.inf), dict(eps=1e-31), dict(ldr=63), dict(ldo=63), dict(residual=4 * A + 1), dict(residual_out=5 * A + 1),
                                 dict(weight=6 * A + 1), dict(weight=6 * A + 2, weight_f32=1), dict(residual_out=A + 2), dict(residual_out=4 * A + 128),
                                 dict(residual_out=A, ldo=128), dict(Q=4 * A), dict(Q=5 * A + 64), dict(scale=5 * A), dict(Q=6 * A), dict(residual_out=6 * A)])
def test_norm_refuses(bad):
    assert norm(**bad) == BAD


@pytest.mark.parametrize("bad", [dict(type=5), dict(layout=3), dict(B=-2), dict(HW=-1), dict(C=0), dict(K=0), dict(Q=None), dict(q_scale=None), dict(W=None), dict(w_scale=None),
                                 dict(Y=None), dict(ldq=48), dict(ldw=63), dict(ldy=31), dict(Q=A + 8), dict(W=3 * A + 1), dict(ldq=72), dict(ldw=68), dict(q_scale=2 * A + 1),
                                 dict(bias=5 * A + 2), dict(Y=6 * A + 2), dict(Y=6 * A + 1, type=F16), dict(Y=A), dict(Y=3 * A + 4), dict(Y=2 * A), dict(Y=4 * A), dict(Y=5 * A)])
def test_linear_refuses(bad):
    assert linear(**bad) == BAD


def test_quantize_limits():
    far = dict(X=1 << 50, Q=1 << 52, scale=1 << 54)
    assert quantize(C=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31, **far) == UNSUPPORTED
    assert quantize(B=1 << 31, **far) == UNSUPPORTED
    assert quantize(B=1 << 37, **far) == UNSUPPORTED and quantize(ldx=1 << 40, **far) == UNSUPPORTED
    assert quantize(B=1 << 37, layout=1, C=1, **far) == UNSUPPORTED


def test_linear_limits():
    assert linear(C=131072, ldq=131072, ldw=131072, W=1 << 32, Y=1 << 40, w_scale=1 << 41, q_scale=1 << 42, bias=1 << 43) == UNSUPPORTED
    assert linear(B=1 << 30, K=1 << 30, Q=1 << 45, Y=1 << 50, q_scale=1 << 48, w_scale=1 << 47, bias=1 << 46, ldy=1 << 30) == UNSUPPORTED
    assert linear(B=1 << 31, Q=1 << 45, Y=1 << 50, q_scale=1 << 48, ldq=64) == UNSUPPORTED


def test_python_calls_want_cuda_tensors():
    import torch
    x = torch.zeros(4, 16)
    for call in (lambda: wg2x2.quantize_int8(x), lambda: wg2x2.rms_norm_int8(x, x[0]), lambda: wg2x2.quantize_int8(None), lambda: wg2x2.quantize_int8([1.0]),
                 lambda: wg2x2.linear_int8(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0])):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(KeyError):
        wg2x2.quantize_int8(x, layout="NHCW")
