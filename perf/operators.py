"""Per-pixel products in 8 bits, and what feeds them: the cases by which their speed is measured.

  quantize  rows of activations (or weights) -> codes of -127 .. 127 and a scale a row: wg2x2.quantize_int8
  norm      root-mean-square norm over the channels with the shortcut's addition -> codes and scales: wg2x2.rms_norm_int8
  linear    product of codes with a scale for each row and each output channel: wg2x2.linear_int8

A row is a token, or a pixel with its channels.  Definitions, in exact arithmetic but for what is said to be held in a type:

  quantize  a = max_c |x_c|, scale = a / 127, q_c = 127 x_c / a to the nearest whole number, ties to the even one
  norm      h = x + residual, held in x's type; u_c = h_c w_c, held in 32 bits; a = max_c |u_c|, q_c = 127 u_c / a as above,
            scale = a / 127 / sqrt(mean_c h_c^2 + eps)
  linear    y_k = (sum_c q_c w_kc) scale scale_k + bias_k, optionally through a ReLU, in the type asked for

A row whose a is below 2^-119 has scale 0 and codes 0.  The codes are whole numbers, the same on both sides to the last one; they are
returned as they are, with their scales, which is what the product takes.
"""
import functools
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
TINY = 2.0 ** -119


def _quantize(name, rows, C, type, relu=False):
    return dict(name=name, op="quantize", layout="NHWC", rows=rows, C=C, type=type, relu=relu)


def _norm(name, rows, C, type, residual=True):
    return dict(name=name, op="norm", layout="NHWC", rows=rows, C=C, type=type, residual=residual)


def _linear(name, rows, C, K, type, bias=True, relu=False):
    return dict(name=name, op="linear", layout="NHWC", rows=rows, C=C, K=K, type=type, bias=bias, relu=relu)


def listed():
    return [
        # one token in front of a product: the launch counts
        _quantize("quantize_1x4096", 1, 4096, "bf16"),
        # what the first 1x1 shortcut of the benchmark's network takes, batch 256: an NCHW image through its ReLU
        dict(name="quantize_nchw_256x64x56", op="quantize", layout="NCHW", B=256, C=64, H=56, W=56, type="f32", relu=True),
        # channels off every vector size
        _quantize("quantize_7777x1001", 7777, 1001, "f16", relu=True),
        # one token behind a block
        _norm("norm_1x4096", 1, 4096, "bf16"),
        # a long batch of tokens: the bytes count
        _norm("norm_16384x4096", 16384, 4096, "bf16"),
        # channels-last pixels of a 64-channel stage in the library's own precision, batch 64 of 56 x 56
        _norm("norm_200704x64", 64 * 56 * 56, 64, "f32"),
        # odd channels, no shortcut
        _norm("norm_999x1283", 999, 1283, "f16", residual=False),
        # one token: the weights' bytes count
        _linear("linear_1x4096x4096", 1, 4096, 4096, "bf16"),
        # a few tokens, output channels off the tiles
        _linear("linear_24x2048x8191", 24, 2048, 8191, "bf16"),
        # the classifier of the benchmark's network at its batch
        _linear("linear_256x512x1000", 256, 512, 1000, "f32"),
        # the shortcut of the network's second stage at the benchmark's batch, NCHW out
        dict(name="linear_nchw_256x64x28x128", op="linear", layout="NCHW", B=256, C=64, H=28, W=28, K=128, type="f32", bias=False, relu=False),
        # a long batch of tokens through a wide layer: the tensor cores count
        _linear("linear_8192x4096x4096", 8192, 4096, 4096, "bf16", relu=True),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; every second one at a multiple of 16"""
    n = int(round(low * (high / low) ** rng.random()))
    return max(low, n // 16 * 16) if rng.random() < 0.5 and n >= 16 else n


def draw(rng):
    op = rng.choice(["quantize", "norm", "linear"])
    c = dict(op=op, type=rng.choice(["f32", "f16", "bf16"]))
    if rng.random() < 0.3:
        # an image: up to the batch of 256, sides and channels of the network's stages
        side = rng.randint(1, 56)
        c.update(layout="NCHW", H=side, W=max(1, side + rng.randint(-2, 2)), C=_size(rng, 8, 1024))
        if op == "linear":
            c["K"] = _size(rng, 8, 1024)
        values = c["H"] * c["W"] * max(c["C"], c.get("K", 0))
        c["B"] = _size(rng, 1, max(1, min(256, 2 ** 25 // values)))
    else:
        C = _size(rng, 8, 8192 if op == "linear" else 16384)
        c.update(layout="NHWC", C=C)
        if op == "linear":
            c["K"] = _size(rng, 8, 8192)
            most = min(16384, 2 ** 36 // (C * c["K"]), 2 ** 25 // max(C, c["K"]))
        else:
            most = min(65536, 2 ** 25 // C)
        c["rows"] = _size(rng, 1, max(1, most))
    if op == "norm":
        c["residual"] = rng.random() < 0.7
    else:
        c["relu"] = rng.random() < 0.5
    if op == "linear":
        c["bias"] = rng.random() < 0.5
    return c


def _rows(case):
    return case["rows"] if case["layout"] == "NHWC" else case["B"] * case["H"] * case["W"]


def _codes(gen, rows, C):
    """Codes and scales as a quantiser gives them for values from a normal distribution: rows begin on 16 bytes"""
    v = torch.randn((rows, C), generator=gen, device="cuda")
    a = v.abs().amax(1)
    q = torch.zeros((rows, (C + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :C]
    q.copy_(torch.round(v * (127 / a)[:, None]))
    return q, a / 127


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    C, t = case["C"], TYPES[case["type"]]
    s = dict(case=case)
    if case["op"] == "linear":
        q, s["scale"] = _codes(gen, _rows(case), C)
        w, t_scale = _codes(gen, case["K"], C)
        s.update(w=w, w_scale=t_scale / C ** 0.5, bias=0.1 * rnd(case["K"]) if case["bias"] else None)
        if case["layout"] == "NCHW":
            q, s["scale"] = q.unflatten(0, (case["B"], case["H"], case["W"])), s["scale"].view(case["B"], case["H"], case["W"])
        s["q"] = q
        return s
    # some channels are larger than others, as in a trained network
    spread = torch.exp(0.5 * rnd(C))
    shape, per_channel = ((case["rows"], C), spread) if case["layout"] == "NHWC" else ((case["B"], C, case["H"], case["W"]), spread[:, None, None])
    s["x"] = (rnd(*shape) * per_channel).to(t)
    if case["op"] == "norm":
        s["weight"] = (1 + 0.1 * rnd(C)).to(t)
        s["residual"] = (rnd(*shape) * per_channel).to(t) if case["residual"] else None
    return s


@functools.lru_cache(None)
def _library():
    sys.path.insert(0, os.path.abspath("sparse-winograd-cnn_b200"))
    import wg2x2
    return wg2x2


def run(s):
    case = s["case"]
    if own:
        wg = _library()
        if case["op"] == "quantize":
            return wg.quantize_int8(s["x"], relu=case["relu"], layout=case["layout"])
        if case["op"] == "norm":
            return wg.rms_norm_int8(s["x"], s["weight"], residual=s["residual"], eps=EPS, layout=case["layout"])
        return wg.linear_int8(s["q"], s["scale"], s["w"], s["w_scale"], bias=s["bias"], relu=case["relu"], layout=case["layout"],
                              dtype=TYPES[case["type"]])
    if case["op"] == "quantize":
        x = s["x"] if case["layout"] == "NHWC" else s["x"].permute(0, 2, 3, 1)
        x = x.float()
        return _plain_codes(torch.relu(x) if case["relu"] else x)
    if case["op"] == "norm":
        h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
        v = (h if case["layout"] == "NHWC" else h.permute(0, 2, 3, 1)).float()
        q, scale = _plain_codes(v * s["weight"].float())
        scale = (scale.double() / torch.sqrt(v.double().square().mean(-1) + EPS)).float()
        return (q, scale) if s["residual"] is None else (q, scale, h)
    # sums of more than 1040 products pass the whole numbers that 32 bits hold
    t = torch.float32 if case["C"] <= 1040 else torch.float64
    y = (s["q"].to(t) @ s["w"].to(t).T).float() * s["scale"][..., None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["relu"]:
        y = torch.relu(y)
    return (y if case["layout"] == "NHWC" else y.permute(0, 3, 1, 2).contiguous()).to(TYPES[case["type"]])


def _plain_codes(v):
    """Codes and scales of rows in 32 bits.  (The quotient in 64 bits: in 32 a value half way between two codes goes either way.)"""
    a = v.abs().amax(-1)
    live = a >= TINY
    q = torch.round(v.double() * 127 / torch.where(live, a, 1)[..., None].double())
    q = torch.where((live & a.isfinite())[..., None], q, 0).to(torch.int8)
    scale = torch.where(live, a / 127, torch.where(a < TINY, 0.0, float("nan")))
    return q, torch.where(scale.isinf(), float("nan"), scale)


def work(case):
    rows, C, e = _rows(case), case["C"], SIZE[case["type"]]
    if case["op"] == "quantize":
        return {"bytes": rows * C * (e + 1) + 4 * rows, "flops": 3 * rows * C}
    if case["op"] == "norm":
        return {"bytes": rows * C * ((3 if case["residual"] else 1) * e + 1) + 4 * rows + C * e, "flops": 6 * rows * C}
    K = case["K"]
    return {"bytes": rows * C + K * C + 4 * (rows + K) + (4 * K if case["bias"] else 0) + rows * K * e, "flops": 2 * rows * C * K}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "linear":
        x = s["q"].to(f64).mul_(s["scale"].to(f64).unsqueeze(-1))
        y = torch.einsum("...c,kc->...k", x, s["w"].to(f64)).mul_(s["w_scale"].to(f64))
        if case["bias"]:
            y.add_(s["bias"].to(f64))
        if case["relu"]:
            y.clamp_(min=0)
        return y if case["layout"] == "NHWC" else y.movedim(-1, 1).contiguous()
    x = s["x"]
    if case["op"] == "norm":
        h = x.to(f64)
        if case["residual"]:
            h = (h + s["residual"].to(f64)).to(x.dtype).to(f64)
        stored = h
        if case["layout"] == "NCHW":
            h = h.movedim(1, -1)
        u = (h * s["weight"].to(f64)).float().to(f64)
        norm = (torch.linalg.vector_norm(h, dim=-1).square() / case["C"] + EPS).sqrt()
    else:
        u = x.to(f64) if case["layout"] == "NHWC" else x.to(f64).movedim(1, -1)
        if case["relu"]:
            u = u.clamp(min=0)
        norm = torch.ones(u.shape[:-1], dtype=f64, device=u.device)
    a = torch.maximum(u.amax(-1), -u.amin(-1))
    none = a < TINY
    q = (u * 127 / a.masked_fill(none, 1).unsqueeze(-1)).round_()
    q = q.masked_fill(none[..., None], 0).to(torch.int8)
    scale = (a / 127 / norm).masked_fill(none, 0)
    return (q, scale, stored) if case["op"] == "norm" and case["residual"] else (q, scale)
