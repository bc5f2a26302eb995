"""The 8-bit per-pixel products against their definitions in 64 bits.  Codes are whole numbers and have to be equal; sums of the product are
exact; the tolerances of the rest count roundings of half a step."""
import math
import threading

import pytest
import torch

import wg2x2

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = 2.0 ** -119
U = 2.0 ** -24             # half a step of 32 bits, relative


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(sum((i + 1) * ord(c) for i, c in enumerate(str(key))))


def _codes(u):
    """(q, scale of u in 64 bits, a) of rows u (..., C) in 64 bits whose values 32 bits hold"""
    a = u.abs().amax(-1)
    a = torch.where(u.isnan().any(-1), math.nan, a)
    dead, bad = a < TINY, ~a.isfinite()
    q = torch.round(127 * u / torch.where(dead | bad, 1.0, a)[..., None])         # (127 u is exact; a quotient that is not half way is 2^-33 from it)
    q = torch.where((dead | bad)[..., None], 0.0, q)
    scale = torch.where(dead, 0.0, torch.where(bad, math.nan, a / 127))
    return q.to(torch.int8), scale


def _special(x):
    """Rows where it can go wrong, in place of some of x's (rows, C)"""
    rows, C = x.shape
    put = [lambda r: r.zero_(), lambda r: r.fill_(TINY / 2), lambda r: r[C // 2].fill_(math.nan), lambda r: r[C - 1].fill_(-math.inf),
           lambda r: r.copy_(torch.arange(C, device=r.device) % 7 * 0.5 - 1.5),                    # halves of the largest: 63.5 steps
           lambda r: r.mul_(0).add_((torch.arange(C, device=r.device) % 255 - 127) / 2).clamp_(-63.5, 63.5),     # half way between codes
           lambda r: (r.zero_(), r[0].fill_(-3.0)), lambda r: r.mul_(1e-7 if x.dtype == torch.float16 else 1e-30),
           lambda r: r.fill_(torch.finfo(x.dtype).max), lambda r: r.fill_(TINY if x.dtype != torch.float16 else 6e-8)]
    for i, f in enumerate(put):
        if 2 * i + 1 < rows:
            f(x[2 * i + 1])
    return x


def _placed(x, pitch, offset):
    """x (rows, C) as a view with that row pitch, that many elements into a buffer of its own"""
    rows, C = x.shape
    buf = torch.zeros(offset + rows * pitch + 64, dtype=x.dtype, device=x.device)
    v = buf[offset:offset + rows * pitch].view(rows, pitch)[:, :C]
    v.copy_(x)
    return v


def _guarded(rows, C, pitch, offset):
    """An output for codes in a buffer of 77s, and a check that nothing else of the buffer changed"""
    buf = torch.full((offset + rows * pitch + 64,), 77, dtype=torch.int8, device="cuda")
    v = buf[offset:offset + rows * pitch].view(rows, pitch)[:, :C]

    def check():
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[offset:offset + rows * pitch].view(rows, pitch)[:, :C] = False
        assert bool((buf[keep] == 77).all())
    return v, check


def _equal(x, y):
    return torch.equal(x.nan_to_num(nan=12345.0), y.nan_to_num(nan=12345.0))


SIZES = [(1, 1), (3, 2), (21, 7), (40, 8), (25, 16), (301, 17), (64, 33), (21, 63), (1000, 64), (30, 65), (33, 127), (21, 128), (21, 250), (700, 256), (23, 257), (21, 512),
         (22, 513), (500, 1000), (499, 1001), (21, 1024), (400, 1025), (1, 4096), (321, 4096), (300, 4099), (22, 8192), (2, 12345), (21, 16384), (300, 20001), (21, 40000),
         # many rows: blocks that go on to further ones
         (200001, 4), (100003, 9), (70001, 64), (60000, 33), (20011, 100), (30000, 128), (12345, 250), (9001, 513), (5003, 1001), (3001, 2049), (4000, 4096), (1501, 8192), (700, 16383)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", SIZES)
def test_quantize_rows(rows, C, dtype):
    g = _gen("q", rows, C, dtype)
    x = _special(torch.randn((rows, C), generator=g, device="cuda").to(dtype))
    for relu in (False, True):
        want_q, want_s = _codes(torch.relu(x.double()) if relu else x.double())
        q, s = wg2x2.quantize_int8(x, relu=relu)
        assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == (rows,) and q.stride(-1) == 1 and (rows == 1 or q.stride(0) % 16 == 0)
        assert torch.equal(q, want_q) and _equal(s, want_s.float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", [(7, 5), (40, 64), (33, 257), (21, 1000), (300, 1031), (5, 5000)])
def test_quantize_any_pitch_and_alignment(rows, C, dtype):
    g = _gen("qa", rows, C, dtype)
    x = torch.randn((rows, C), generator=g, device="cuda").to(dtype)
    want_q, want_s = _codes(x.double())
    for pitch, offset, qpitch, qoffset in ((C, 1, C, 0), (C + 1, 0, C, 3), (C + 8, 2, C + 5, 16), ((C + 15) // 16 * 16, 16, C + 4, 4), (C + 16, 3, (C + 15) // 16 * 16, 0)):
        v = _placed(x, pitch, offset)
        out, check = _guarded(rows, C, qpitch, qoffset)
        q, s = wg2x2.quantize_int8(v, out=out)
        assert q.data_ptr() == out.data_ptr() and torch.equal(q, want_q) and _equal(s, want_s.float())
        check()


def _norm_oracle(x, w, res, eps):
    """(q, scale in 64 bits, h) for rows"""
    h = x if res is None else (x.double() + res.double()).to(x.dtype)
    hd = h.double()
    q, s = _codes((hd * w.double()).float().double())
    return q, s / torch.sqrt(hd.square().mean(-1) + eps), h


def _norm_tol(C):
    # squares: one rounding each and at most 64 + C / 16 additions one after the other; the root halves that; three more roundings and the scale's
    return (0.5 * (65 + C / 16) + 6) * U


def _close(s, want, rel):
    assert torch.equal(s.isnan(), want.isnan())
    ok = ~want.isnan()
    small = torch.finfo(torch.float32).tiny           # (below the normal numbers a step is 2^-149)
    assert bool(((s.double() - want)[ok].abs() <= rel * want[ok].abs() + (2.0 ** -149) * (want[ok].abs() < small)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", SIZES)
def test_norm_rows(rows, C, dtype):
    g = _gen("n", rows, C, dtype)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, res, w = _special(rnd(rows, C)), rnd(rows, C), 1 + 0.2 * rnd(C)
    res[1::4] = 0                     # (special rows as they are)
    for r in (None, res):
        for weight in (w, w.float() + 0.01):
            q0, s0, h0 = _norm_oracle(x, weight, r, 1e-5)
            got = wg2x2.rms_norm_int8(x, weight, residual=r, eps=1e-5)
            assert len(got) == (2 if r is None else 3)
            assert torch.equal(got[0], q0)
            _close(got[1], s0, _norm_tol(C))
            if r is not None:
                assert _equal(got[2], h0) and got[2].dtype == dtype


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", [(7, 5), (40, 64), (21, 1000), (300, 1031), (3, 17000)])
def test_norm_in_place_and_any_alignment(rows, C, dtype):
    g = _gen("na", rows, C, dtype)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, res, w = rnd(rows, C), rnd(rows, C), 1 + 0.2 * rnd(C)
    q0, s0, h0 = _norm_oracle(x, w, res, 1e-6)
    # x, residual, sum: pitch and offset of each (alike, or each its own)
    for px, ox, pr, orr, ph, oh in ((C, 0, C, 0, C, 0), (C, 1, C, 1, C, 1), (C + 3, 0, C, 5, C + 1, 2), (C + 8, 8, C + 16, 0, C + 24, 0), (C + 5, 3, C + 5, 3, C + 5, 3)):
        a, b, h = _placed(x, px, ox), _placed(res, pr, orr), _placed(torch.zeros_like(x), ph, oh)
        wo = _placed(w[None], C, 1)[0]
        q, s, out = wg2x2.rms_norm_int8(a, wo, residual=b, residual_out=h)
        assert out.data_ptr() == h.data_ptr() and torch.equal(q, q0) and torch.equal(h, h0) and torch.equal(a, x) and torch.equal(b, res)
        _close(s, s0, _norm_tol(C))
        for into in (0, 1):
            a, b = _placed(x, px, ox), _placed(res, pr, orr)
            q, s, out = wg2x2.rms_norm_int8(a, w, residual=b, residual_out=(a, b)[into])
            assert torch.equal(q, q0) and torch.equal((a, b)[into], h0) and torch.equal((a, b)[1 - into], (x, res)[1 - into])
    # side by side in one buffer
    buf = torch.cat([x, res, res], 1)
    q, s, h = wg2x2.rms_norm_int8(buf[:, :C], w, residual=buf[:, C:2 * C], residual_out=buf[:, 2 * C:])
    assert torch.equal(q, q0) and torch.equal(buf, torch.cat([x, res, h0], 1))


def test_norm_of_large_and_small_rows():
    """Squares beyond 32 bits, and far below them"""
    C = 700
    g = _gen("large")
    for size in (3e19, 1e30, 3e38, 1e-17, 1e-21):
        for rows, layout in ((3, "NHWC"), (200, "NHWC"), (50, "NCHW")):
            for c in (C, 60, 9000):
                x = (torch.rand((rows, c), generator=g, device="cuda") - 0.5) * (2 * min(size, 3.3e38))
                q0, s0, _ = _norm_oracle(x, torch.full((c,), 0.5, device="cuda"), None, 1e-30)
                xin = x if layout == "NHWC" else x.view(rows, c, 1, 1)
                q, s = wg2x2.rms_norm_int8(xin, torch.full((c,), 0.5, device="cuda"), eps=1e-30, layout=layout)
                assert torch.equal(q.reshape(rows, c), q0)
                _close(s.reshape(rows), s0, _norm_tol(c))


IMAGES = [(1, 1, 1, 1), (2, 3, 5, 7), (3, 4, 1, 33), (2, 63, 9, 9), (1, 64, 56, 56), (5, 65, 7, 7), (2, 128, 14, 13), (1, 200, 6, 6), (3, 256, 7, 7), (2, 300, 4, 4), (1, 512, 7, 7),
          (2, 600, 3, 5), (1, 1024, 6, 7), (2, 1025, 3, 3), (1, 2500, 2, 9), (2, 9001, 1, 3), (7, 375, 32, 30), (40, 64, 28, 28), (9, 616, 21, 20)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,C,H,W", IMAGES)
def test_images(B, C, H, W, dtype):
    """NCHW in, rows of channels out, for the quantiser and the norm"""
    g = _gen("i", B, C, H, W, dtype)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    rows = _special(rnd(B * H * W, C))
    image = lambda r: r.view(B, H, W, C).permute(0, 3, 1, 2).contiguous()  # noqa: E731
    x, res, w = image(rows), rnd(B, C, H, W), 1 + 0.2 * rnd(C)
    rres = res.permute(0, 2, 3, 1).reshape(-1, C)
    for relu in (False, True):
        want_q, want_s = _codes(torch.relu(rows.double()) if relu else rows.double())
        q, s = wg2x2.quantize_int8(x, relu=relu, layout="NCHW")
        assert q.shape == (B, H, W, C) and s.shape == (B, H, W)
        assert torch.equal(q.reshape(-1, C), want_q) and _equal(s.flatten(), want_s.float())
    for r in (None, res):
        q0, s0, h0 = _norm_oracle(rows, w, None if r is None else rres, 1e-6)
        got = wg2x2.rms_norm_int8(x, w, residual=r, layout="NCHW")
        assert torch.equal(got[0].reshape(-1, C), q0)
        _close(got[1].flatten(), s0, _norm_tol(C))
        if r is not None:
            assert _equal(got[2], image(h0))
            for into in (x.clone(), res.clone()):
                a, b = (into, res) if torch.equal(into.nan_to_num(), x.nan_to_num()) else (x, into)
                assert _equal(wg2x2.rms_norm_int8(a, w, residual=b, layout="NCHW", residual_out=into)[2], image(h0)) and _equal(into, image(h0))
    out, check = _guarded(B * H * W, C, C + 3, 1)
    q, _ = wg2x2.quantize_int8(x, layout="NCHW", out=out.unflatten(0, (B, H, W)))
    assert torch.equal(q.reshape(-1, C), _codes(rows.double())[0])
    check()


def _rand_codes(g, rows, C, low=-127):
    return torch.randint(low, 128, (rows, C), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


def _linear_oracle(q, s, w, ws, bias, relu):
    """(y, |product|) in 64 bits; the sums are whole numbers below 2^53"""
    p = (q.double() @ w.double().T) * s.double()[:, None] * ws.double()
    y = p if bias is None else p + bias.double()
    return (torch.relu(y) if relu else y), p.abs()


def _check_linear(y, want, p, dtype):
    # the sum, the scale's product and the last one: 3 roundings of the product; the result's own, and its rounding to dtype
    tol = 1.01 * (3 * U * p + (U + torch.finfo(dtype).eps / 2) * want.abs()) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -140)
    assert torch.equal(y.isnan(), want.isnan())
    big = want.abs() >= torch.finfo(dtype).max
    ok = ~want.isnan() & ~big
    assert bool(((y.double() - want).abs() <= tol)[ok].all())
    assert bool((y.double().abs() >= torch.finfo(dtype).max)[big].all())


LINEAR = [(1, 1, 1), (4, 15, 9), (4, 31, 100), (2, 500, 700), (3, 129, 33), (4, 4096, 4096), (1, 9000, 300), (1, 16, 3), (2, 17, 129), (3, 100, 64), (5, 128, 128), (7, 129, 1000), (16, 512, 1000), (17, 1000, 31), (31, 64, 257), (33, 127, 300), (64, 2048, 100),
          (100, 300, 513), (127, 4096, 128), (128, 128, 4100), (129, 1023, 255), (200, 40, 2048), (256, 512, 1000), (300, 8192, 70), (500, 384, 384), (1000, 256, 640),
          (1111, 33, 777), (2049, 1100, 300), (5000, 64, 64), (3, 4096, 4096), (20000, 96, 24), (1, 5000, 20001), (40, 2000, 19000),
          # small products, up to the limits, and those just behind them
          (16, 6144, 700), (9, 64, 5920), (9, 65, 5921), (15, 70, 9472), (16, 100, 9473), (2, 6145, 9), (6, 2000, 6001), (256, 512, 512), (40, 33, 2368), (64, 1030, 2369),
          (1, 600, 9000), (1, 64, 20000), (1, 1025, 9), (2300, 24, 65), (32, 4096, 2048), (32, 4096, 2400), (17, 4097, 31), (129, 4080, 370),
          (8, 64, 11840), (7, 70, 11841), (8, 1025, 9472), (5, 1030, 9473), (8, 8192, 100), (8, 8193, 100), (16, 4096, 300), (16, 4097, 300), (10, 130, 5921), (24, 900, 4736), (32, 2049, 4737), (288, 600, 500),
          (17, 100, 2032), (17, 100, 2033), (130, 3000, 400),
          # clusters that share a tile: few rows and long contractions
          (3, 9000, 40), (5, 8192, 128), (7, 7001, 1000), (16, 6200, 333), (31, 8000, 257), (33, 5000, 127), (64, 4500, 100), (127, 4224, 128), (6, 8200, 333), (9, 8192, 128),
          # tiles of 256 x 256 and 256 x 128 on pairs of SMs, ragged
          (4100, 700, 3001), (3000, 1024, 2048), (8192, 300, 4097), (2600, 2000, 5000), (700, 4100, 9000)]


@pytest.mark.parametrize("rows,C,K", LINEAR)
def test_linear(rows, C, K):
    g = _gen("l", rows, C, K)
    q, w = _rand_codes(g, rows, C), _rand_codes(g, K, C)
    s, ws = torch.rand(rows, generator=g, device="cuda") + 0.01, (torch.rand(K, generator=g, device="cuda") + 0.01) / C
    s[rows // 2] = 0
    if rows > 2:
        s[rows // 3] = math.nan
    bias = torch.randn(K, generator=g, device="cuda")
    for dtype, b, relu in ((torch.float32, None, False), (torch.float32, bias, True), (torch.float16, bias, False), (torch.bfloat16, None, True), (torch.bfloat16, bias, False)):
        want, p = _linear_oracle(q, s, w, ws, b, relu)
        y = wg2x2.linear_int8(q, s, w, ws, bias=b, relu=relu, dtype=dtype)
        assert y.shape == (rows, K) and y.dtype == dtype and y.is_contiguous()
        _check_linear(y, want, p, dtype)


@pytest.mark.parametrize("B,H,W,C,K", [(1, 1, 1, 5, 3), (2, 1, 2, 100, 7), (1, 1, 3, 512, 1000), (1, 7, 7, 512, 100), (2, 7, 7, 64, 64), (1, 7, 7, 5000, 100), (3, 5, 9, 4130, 33), (1, 1, 3, 7000, 1000), (1, 1, 3, 9000, 1000), (3, 4, 5, 500, 2100), (2, 2, 3, 200, 6000), (5, 1, 3, 72, 40), (3, 5, 9, 130, 33), (4, 28, 28, 64, 128), (1, 56, 56, 64, 64), (40, 14, 14, 128, 256),
                                       (64, 7, 7, 256, 512), (2, 1, 130, 2000, 17), (30, 28, 27, 33, 300), (64, 14, 14, 600, 1030), (17, 28, 28, 1024, 513)])
def test_linear_images(B, H, W, C, K):
    g = _gen("li", B, H, W, C, K)
    rows = B * H * W
    q, w = _rand_codes(g, rows, C), _rand_codes(g, K, C)
    s, ws = torch.rand(rows, generator=g, device="cuda"), torch.rand(K, generator=g, device="cuda") / C
    bias = torch.randn(K, generator=g, device="cuda")
    for dtype, b, relu in ((torch.float32, None, False), (torch.float16, bias, True), (torch.bfloat16, bias, False)):
        want, p = _linear_oracle(q, s, w, ws, b, relu)
        y = wg2x2.linear_int8(q.view(B, H, W, C), s.view(B, H, W), w, ws, bias=b, relu=relu, layout="NCHW", dtype=dtype)
        assert y.shape == (B, K, H, W) and y.is_contiguous()
        _check_linear(y.permute(0, 2, 3, 1).reshape(rows, K), want, p, dtype)


@pytest.mark.parametrize("rows,C,K", [(2, 131071, 5), (150, 70000, 130)])
def test_linear_largest_sums(rows, C, K):
    """128 * 128 * C just below 2^31, exact"""
    q, w = torch.full((rows, C), -128, dtype=torch.int8, device="cuda"), torch.full((K, C), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    one = torch.ones(rows, device="cuda"), torch.ones(K, device="cuda")
    y = wg2x2.linear_int8(q, one[0], w, one[1])
    want = torch.where(torch.arange(K, device="cuda") % 2 == 1, -128.0 * 127 * C, 128.0 * 128 * C).float()
    assert torch.equal(y, want.expand(rows, K))
    with pytest.raises(wg2x2.Wg2x2Error):
        wg2x2.linear_int8(torch.zeros((1, 131072), dtype=torch.int8, device="cuda"), one[0][:1], torch.zeros((1, 131072), dtype=torch.int8, device="cuda"), one[1][:1])


@pytest.mark.parametrize("rows,C,K", [(3, 33, 65), (200, 100, 1000), (300, 260, 140)])
def test_linear_any_pitch(rows, C, K):
    """Codes at any pitch, alignment and order; a result among other columns, which stay as they were"""
    g = _gen("lp", rows, C, K)
    q, w = _rand_codes(g, rows, C), _rand_codes(g, K, C)
    s, ws = torch.rand(rows, generator=g, device="cuda"), torch.rand(K, generator=g, device="cuda")
    plain = wg2x2.linear_int8(q, s, w, ws)
    for a, b in ((_placed(q, C + 1, 3), w), (q, _placed(w, C + 16, 5)), (_placed(q, (C + 31) // 16 * 16, 32), _placed(w, (C + 15) // 16 * 16, 16)), (q.T.contiguous().T, w.T.contiguous().T)):
        assert torch.equal(wg2x2.linear_int8(a, s, b, ws), plain)
    for dtype in TYPES:
        buf = torch.full((rows, K + 7), 3.0, dtype=dtype, device="cuda")
        out = buf[:, 2:2 + K]
        y = wg2x2.linear_int8(q, s, w, ws, dtype=dtype, out=out)
        assert y.data_ptr() == out.data_ptr() and torch.equal(out, plain.to(dtype))
        assert bool((buf[:, :2] == 3).all()) and bool((buf[:, 2 + K:] == 3).all())


def test_leading_shapes_and_nothing():
    g = _gen("shapes")
    x = torch.randn((2, 3, 4, 40), generator=g, device="cuda")
    w, ws = wg2x2.quantize_int8(torch.randn((24, 40), generator=g, device="cuda"))
    q, s = wg2x2.quantize_int8(x)
    flat_q, flat_s = wg2x2.quantize_int8(x.view(24, 40))
    assert torch.equal(q.reshape(24, 40), flat_q) and torch.equal(s.view(24), flat_s)
    y = wg2x2.linear_int8(q, s, w, ws)
    assert y.shape == (2, 3, 4, 24) and torch.equal(y.view(24, 24), wg2x2.linear_int8(flat_q, flat_s, w, ws))
    q1, s1 = wg2x2.quantize_int8(x[0, 0, 0])
    assert q1.shape == (40,) and s1.shape == () and torch.equal(wg2x2.linear_int8(q1, s1, w, ws), y[0, 0, 0])
    for lead in ((0,), (2, 0), (0, 3)):
        e = torch.empty((*lead, 40), device="cuda")
        q, s = wg2x2.quantize_int8(e)
        assert q.shape == e.shape and s.shape == lead
        assert wg2x2.linear_int8(q, s, w, ws).shape == (*lead, 24)
        q, s, h = wg2x2.rms_norm_int8(e, torch.ones(40, device="cuda"), residual=e)
        assert q.shape == e.shape and h.shape == e.shape
    for shape in ((0, 40, 3, 3), (2, 40, 0, 3)):
        e = torch.empty(shape, device="cuda")
        q, s = wg2x2.quantize_int8(e, layout="NCHW")
        assert q.shape == (shape[0], shape[2], shape[3], 40)
        assert wg2x2.linear_int8(q, s, w, ws, layout="NCHW").shape == (shape[0], 24, shape[2], shape[3])


def test_codes_and_scales_are_ordinary_tensors():
    """Each outlives the other, can be written, saved and loaded, and used as a constant of a graph"""
    import io
    g = _gen("ordinary")
    x = torch.randn((6, 5, 33), generator=g, device="cuda")
    q, s = wg2x2.quantize_int8(x)
    q0, s0 = _codes(x.double())
    keep = s
    f = io.BytesIO()
    torch.save((q, s), f)
    f.seek(0)
    q2, s2 = torch.load(f)
    assert torch.equal(q2, q0) and torch.equal(s2, s0.float())
    w = _rand_codes(g, 7, 33)
    one = torch.ones(7, device="cuda")
    assert torch.equal(wg2x2.linear_int8(q2, s2, w, one), wg2x2.linear_int8(q, s, w, one))
    q.zero_()
    assert torch.equal(s, s0.float())
    s.fill_(2.0)
    assert int(q.abs().max()) == 0 and not q.requires_grad and s.is_leaf
    del q, s
    for _ in range(5):
        wg2x2.quantize_int8(torch.randn_like(x))
    torch.cuda.synchronize()
    assert bool((keep == 2).all())
    w = torch.randn((5,), generator=g, device="cuda", requires_grad=True)
    (w * wg2x2.quantize_int8(x)[1].sum(0)).sum().backward()
    assert torch.allclose(w.grad, s0.float().sum(0))
    with torch.inference_mode():
        q, s = wg2x2.quantize_int8(x)
        assert torch.equal(q, q0)


def test_refusals():
    x = torch.randn((6, 32), device="cuda")
    w, ws = wg2x2.quantize_int8(torch.randn((8, 32), device="cuda"))
    q, s = wg2x2.quantize_int8(x)
    one = torch.ones(32, device="cuda")
    V, T, E = ValueError, TypeError, wg2x2.Wg2x2Error
    for error, call in (
            (T, lambda: wg2x2.quantize_int8(x.double())), (T, lambda: wg2x2.quantize_int8(x, out=torch.empty_like(x))), (V, lambda: wg2x2.quantize_int8(x, out=q[:5])),
            (V, lambda: wg2x2.quantize_int8(x.T)), (V, lambda: wg2x2.quantize_int8(x[:, ::2])), (V, lambda: wg2x2.quantize_int8(x[:1].expand(6, 32))), (V, lambda: wg2x2.quantize_int8(x, layout="NCHW")),
            (V, lambda: wg2x2.quantize_int8(x.view(1, 2, 3, 32).permute(0, 3, 1, 2), layout="NCHW")), (V, lambda: wg2x2.quantize_int8(torch.tensor(1.0, device="cuda"))),
            (V, lambda: wg2x2.quantize_int8(x, scale_out=torch.empty(7, device="cuda"))), (T, lambda: wg2x2.quantize_int8(x, scale_out=torch.empty(6, device="cuda", dtype=torch.float16))),
            (V, lambda: wg2x2.quantize_int8(torch.empty((3, 0), device="cuda"))),
            (V, lambda: wg2x2.rms_norm_int8(x, one[:31])), (T, lambda: wg2x2.rms_norm_int8(x, one.half())), (V, lambda: wg2x2.rms_norm_int8(x, one, residual=x[:5])),
            (T, lambda: wg2x2.rms_norm_int8(x, one, residual=x.half())), (V, lambda: wg2x2.rms_norm_int8(x, one, residual_out=x)), (E, lambda: wg2x2.rms_norm_int8(x, one, eps=0.0)),
            (E, lambda: wg2x2.rms_norm_int8(x, one, eps=1e-50)), (E, lambda: wg2x2.rms_norm_int8(x[:5], one, residual=x[:5].clone(), residual_out=x[1:])), (T, lambda: wg2x2.rms_norm_int8(x, one, eps="a")),
            (V, lambda: wg2x2.rms_norm_int8(x, one, residual=x[:1].expand(6, 32))), (T, lambda: wg2x2.rms_norm_int8(x, one.cpu())),
            (T, lambda: wg2x2.linear_int8(x, s, w, ws)), (V, lambda: wg2x2.linear_int8(q, s[:5], w, ws)), (V, lambda: wg2x2.linear_int8(q, s, w[:, :31], ws)), (V, lambda: wg2x2.linear_int8(q, s, w, ws[:7])),
            (V, lambda: wg2x2.linear_int8(q, s, w, ws, bias=ws[:7])), (T, lambda: wg2x2.linear_int8(q, s, w, ws, bias=ws.half())), (T, lambda: wg2x2.linear_int8(q, s, w, ws, dtype=torch.float64)),
            (T, lambda: wg2x2.linear_int8(q, s, w, ws, dtype="float32")), (V, lambda: wg2x2.linear_int8(q, s, w, ws, layout="NCHW")), (V, lambda: wg2x2.linear_int8(q, s, w, ws, out=torch.empty((6, 9), device="cuda"))),
            (T, lambda: wg2x2.linear_int8(q, s, w, ws, out=torch.empty((6, 8), device="cuda"), dtype=torch.float16)), (V, lambda: wg2x2.linear_int8(q, s, w[None], ws)), (T, lambda: wg2x2.linear_int8(q, s, w.cpu(), ws)),
            (V, lambda: wg2x2.linear_int8(q, s, w[:0], ws[:0])), (V, lambda: wg2x2.linear_int8(q, s, w, ws, out=torch.empty((8, 6), device="cuda").T))):
        with pytest.raises(error):
            call()


def _block(x, short, p):
    """A channels-last block end as a network has it: Winograd layer, norm with the shortcut, two per-pixel products in 8 bits"""
    y = wg2x2.layer_fwd_prepared(x, p["wino"], p["K"], layout="NHWC")
    q, s, h = wg2x2.rms_norm_int8(y, p["g"], residual=short, eps=1e-6)
    u = wg2x2.linear_int8(q, s, p["w1"][0], p["w1"][1], bias=p["b1"], relu=True)
    q, s = wg2x2.quantize_int8(u)
    return y, h, u, wg2x2.linear_int8(q, s, p["w2"][0], p["w2"][1], bias=p["b2"])


def _block_params(g, C, K, M):
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return dict(K=K, wino=wg2x2.prepare_weights(rnd(16, C, K) / (4 * C ** 0.5)), g=1 + 0.1 * rnd(K), w1=wg2x2.quantize_int8(rnd(M, K) / K ** 0.5), b1=0.1 * rnd(M),
                w2=wg2x2.quantize_int8(rnd(K, M) / M ** 0.5), b2=0.1 * rnd(K))


@pytest.mark.parametrize("B,C,K,M,H,W", [(2, 32, 48, 100, 9, 7), (8, 64, 64, 256, 28, 28)])
def test_run_of_them(B, C, K, M, H, W):
    g = _gen("block", B, C, K)
    p = _block_params(g, C, K, M)
    x, short = torch.randn((B, H, W, C), generator=g, device="cuda"), torch.randn((B, H, W, K), generator=g, device="cuda")
    y, h, u, out = _block(x, short, p)
    q0, s0, h0 = _norm_oracle(y.view(-1, K), p["g"], short.view(-1, K), 1e-6)
    assert torch.equal(h.view(-1, K), h0)
    want, prod = _linear_oracle(q0, s0, *p["w1"], p["b1"], True)
    rel = _norm_tol(K)                                            # of the norm's scale, on top of the product's own
    assert bool(((u.view(-1, M).double() - want).abs() <= 1.01 * ((3 * U + rel) * prod + 2 * U * want.abs()) + 2.0 ** -140).all())
    q0, s0 = _codes(u.view(-1, M).double())
    want, prod = _linear_oracle(q0, s0.float(), *p["w2"], p["b2"], False)
    _check_linear(out.view(-1, K), want, prod, torch.float32)


def test_streams_threads_and_graphs():
    """On other streams than the tensors' own, in two captured graphs that are replayed at once, and by several threads: the same bits"""
    g = _gen("graphs")
    p = _block_params(g, 32, 64, 128)
    sets = [(torch.randn((3, 8, 8, 32), generator=g, device="cuda"), torch.randn((3, 8, 8, 64), generator=g, device="cuda")) for _ in range(2)]
    want = [[t.clone() for t in _block(*a, p)] for a in sets]
    torch.cuda.synchronize()
    same = lambda got, k: all(torch.equal(a, b) for a, b in zip(got, want[k]))  # noqa: E731
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k, st in enumerate(streams):
        with torch.cuda.stream(st):
            got.append(_block(*sets[k], p))
    torch.cuda.synchronize()
    assert same(got[0], 0) and same(got[1], 1)
    graphs, outs = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_block(*sets[k], p))
        graphs.append(graph)
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[k].replay()
    torch.cuda.synchronize()
    assert same(outs[0], 0) and same(outs[1], 1)
    bad = []

    def work(k):
        for _ in range(10):
            with torch.cuda.stream(streams[k]):
                r = _block(*sets[k], p)
                streams[k].synchronize()
            if not same(r, k):
                bad.append(k)
    ts = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_shared_tiles_on_several_streams():
    """Products whose tiles are shared by clusters, many of them at once: no two wait for each other"""
    g = _gen("several")
    shapes = [(8, 1024, 256), (16, 4096, 128), (40, 2048, 512), (100, 8192, 1024), (9, 640, 64), (9, 8192, 256), (16, 10000, 128), (40, 8192, 512)]
    sets = []
    for rows, C, K in shapes:
        q, w = _rand_codes(g, rows, C), _rand_codes(g, K, C)
        sets.append((q, torch.rand(rows, generator=g, device="cuda"), w, torch.rand(K, generator=g, device="cuda")))
    want = [wg2x2.linear_int8(*a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(6)]
    got = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 6]):
            k = (i * 7 + i // 6) % len(sets)
            got.append((k, wg2x2.linear_int8(*sets[k])))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k]) for k, y in got) and wg2x2.last_device_status()[0] == 0


_FIRST_CALL = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import wg2x2
x, res = torch.randn((300, 1000), device="cuda"), torch.randn((300, 1000), device="cuda")
w, one = torch.randn((500, 1000), device="cuda"), torch.ones(1000, device="cuda")
im = torch.randn((2, 64, 9, 9), device="cuda")
torch.cuda.synchronize()
def f():
    q, s, h = wg2x2.rms_norm_int8(x, one, residual=res)
    t = wg2x2.quantize_int8(w)
    return wg2x2.linear_int8(q, s, *t), wg2x2.linear_int8(q[:8], s[:8], *t), wg2x2.linear_int8(q[:2], s[:2], *t), h, wg2x2.quantize_int8(im, layout="NCHW")[0]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = f()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(y, f()))
print("same")
"""


def test_first_call_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-winograd-cnn_b200")
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL, pkg], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_other_current_stream_and_reused_memory():
    """A result's memory goes back to its stream's pool while kernels that read it are queued there: in order, so nothing is disturbed"""
    g = _gen("reuse")
    w = wg2x2.quantize_int8(torch.randn((256, 512), generator=g, device="cuda"))
    x = torch.randn((64, 512), generator=g, device="cuda")
    want = wg2x2.linear_int8(*wg2x2.quantize_int8(x), *w)
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        ys = [wg2x2.linear_int8(*wg2x2.quantize_int8(x), *w) for _ in range(50)]
        torch.cuda.current_stream().synchronize()
    assert all(torch.equal(y, want) for y in ys)


@pytest.mark.parametrize("rows,C,K", [(9, 8192, 256), (3000, 256, 1024), (6000, 1024, 4096)])
def test_time_out_of_the_product(rows, C, K):
    """A load that never comes: the wait for it gives up, the status says so, and the next call is right"""
    from wg2x2._lib import lib
    g = _gen("timeout", rows)
    q, w = _rand_codes(g, rows, C), _rand_codes(g, K, C)
    s, ws = torch.ones(rows, device="cuda"), torch.ones(K, device="cuda")
    want = (q.double() @ w.double().T).float()
    assert wg2x2.last_device_status()[0] == 0
    assert lib.wg2x2_set_wait_limit(20000) == 0 and lib.wg2x2_test_drop_load(1) == 0
    try:
        wg2x2.linear_int8(q, s, w, ws)
        assert wg2x2.last_device_status()[0] == -4
    finally:
        lib.wg2x2_set_wait_limit(0)
        lib.wg2x2_test_drop_load(-1)
    assert torch.equal(wg2x2.linear_int8(q, s, w, ws), want) and wg2x2.last_device_status()[0] == 0


def test_largest_offsets():
    """More than 2^31 elements in and out"""
    rows, C = (1 << 21) + 5, 1032
    x = torch.empty((rows, C), dtype=torch.bfloat16, device="cuda").normal_(generator=_gen("offsets"))
    q, s = wg2x2.quantize_int8(x)
    at = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    q0, s0 = _codes(x[at].double())
    assert torch.equal(q[at], q0) and torch.equal(s[at], s0.float())
    del x
    w, ws = q[:1030], s[:1030]
    y = wg2x2.linear_int8(q, s, w, ws, dtype=torch.bfloat16)
    want, p = _linear_oracle(q[at], s[at], w, ws, None, False)
    _check_linear(y[at], want, p, torch.bfloat16)


@pytest.mark.parametrize("layout,fused,stage5_pool", [("NCHW", True, True), ("NHWC", True, True), ("NCHW", False, False)])
def test_network_with_pointwise_products_in_8_bits(layout, fused, stage5_pool, monkeypatch):
    """ResNet18Var(pointwise="int8"): four shortcuts and the classifier, each what its operands say"""
    import resnet18_var
    net = resnet18_var.ResNet18Var(num_classes=100, layout=layout, fused=fused, stage5_pool=stage5_pool, pointwise="int8").cuda()
    image = torch.randn((3, 3, 96, 96), generator=_gen("net"), device="cuda")
    net(image)                                       # (the weights' codes are made once)
    calls = []

    def recorded(name):
        f = getattr(wg2x2, name)

        def g(*a, **k):
            r = f(*a, **k)
            calls.append((name, a, k, r if name == "quantize_int8" else r.clone()))      # (a block's last kernel writes over its shortcut)
            return r
        monkeypatch.setattr(wg2x2, name, g)
    recorded("quantize_int8")
    recorded("linear_int8")
    logits = net(image)
    assert logits.shape == (3, 100) and bool(logits.isfinite().all())
    assert [c[0] for c in calls] == ["quantize_int8", "linear_int8"] * 5 and torch.equal(logits, calls[-1][3])
    for i, (name, a, k, r) in enumerate(calls):
        nchw = k.get("layout") == "NCHW"
        if name == "quantize_int8":
            x = a[0].permute(0, 2, 3, 1) if nchw else a[0]
            rows = x.reshape(-1, x.shape[-1]).double()
            q0, s0 = _codes(torch.relu(rows) if k.get("relu") else rows)
            assert torch.equal(r[0].reshape(q0.shape), q0) and torch.equal(r[1].flatten(), s0.float())
        else:
            assert a[0] is calls[i - 1][3][0] and a[1] is calls[i - 1][3][1]
            want, p = _linear_oracle(a[0].reshape(-1, a[0].shape[-1]), a[1].flatten(), a[2], a[3], k.get("bias"), False)
            y = r.permute(0, 2, 3, 1) if nchw else r
            _check_linear(y.reshape(want.shape), want, p, torch.float32)
    blk = net.blocks[1][0]
    q0, s0 = _codes((blk.short * blk["bn1"].scale.view(-1, 1, 1, 1)).flatten(1).double())
    assert torch.equal(blk._short_codes[0], q0) and torch.equal(blk._short_codes[1], s0.float())
    assert (calls[1][2]["bias"] is None) == fused


def test_pointwise_is_refused_by_name():
    import resnet18_var
    with pytest.raises(ValueError):
        resnet18_var.ResNet18Var(pointwise="int4")
