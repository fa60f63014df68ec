"""The operators of a block over many rows: product with epilogue, gated projections, norms with the
residual addition, against their definitions in f64.

Bounds.  A sum over K products of exact operands accumulated in f32 is off by at most
(K/16 + 32) * 2^-23 * sum_k |x_k w_k|: a tensor-core step adds sixteen products and may lose one unit in
the last place of a partial sum, which is at most the sum of the magnitudes; the joining of at most
eight parts and sixteen warps is the 32.  The activations have a slope of at most 1.13 and errors of a
few units in the last place: 4e-6 (|v| + 1).  A result is rounded by at most half a step, 2^-24 of it in
f32 and 2^-8 in bf16.
"""
import math

import numpy as np
import pytest
import torch

from cogni_ml_b200 import (ACTIVATIONS, DeviceQuantWeight, Norm, QuantWeight, gemm_glu, norm_residual,
                           synth)

pytestmark = pytest.mark.gpu
Q4_K, Q5_K, Q6_K, Q8_0, IQ4_NL = synth.Q4_K, synth.Q5_K, synth.Q6_K, synth.Q8_0, synth.IQ4_NL
TYPES = [Q4_K, Q5_K, Q6_K, Q8_0, IQ4_NL]
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Weight:
    """A synthetic weight on the device and its values: f32 (as dequantised) and rounded to bf16, in f64."""

    def __init__(self, cuda, oracle, qtype, n, k, seed):
        raw = synth.make_weight(qtype, n, k, seed=seed, tensor_id=qtype)
        self.dev = DeviceQuantWeight.upload(QuantWeight(raw, qtype, n, k), cuda)
        w = torch.from_numpy(oracle.dequantize(qtype, raw, n * k)).view(n, k).to(cuda)
        self.exact, self.rounded = w.double(), w.bfloat16().double()
        self.rms = float(w.double().square().mean().sqrt())


def rows(cuda, m, n, seed, dtype=torch.float32, scale=1.0):
    return (torch.from_numpy(synth.make_activation(m, n, seed=seed, tensor_id=77)).to(cuda) * scale).to(dtype)


def inputs(cuda, oracle, qtype, m, n, k, seed):
    w = Weight(cuda, oracle, qtype, n, k, seed)
    return w, rows(cuda, m, k, seed, torch.bfloat16, 1.5 / (w.rms * math.sqrt(k)))


def act64(v, name):
    return {"none": lambda: v, "relu": lambda: v.clamp(min=0), "silu": lambda: v * torch.sigmoid(v),
            "gelu": lambda: torch.nn.functional.gelu(v), "sigmoid": lambda: torch.sigmoid(v),
            "gelu_tanh": lambda: torch.nn.functional.gelu(v, approximate="tanh")}[name]()


def product(x, w, bias=None):
    """x W^T + bias in f64 and the bound of its f32 sum."""
    x = x.double()
    v = x @ w.T
    err = (x.shape[1] / 16 + 32) * 2.0 ** -23 * (x.abs() @ w.abs().T)
    if bias is not None:
        v = v + bias.double()
    return v, err + 2.0 ** -24 * v.abs()


def epilogue_reference(x, w, bias, act, residual, out_dtype):
    v, err = product(x, w.rounded, bias)
    y = act64(v, act)
    tol = 1.13 * err + (4e-6 * (v.abs() + 1) if act != "none" else 0)
    if residual is not None:
        y = y + residual.double()
        tol = tol + 2.0 ** -24 * y.abs()
    return y, tol + HALF_STEP[out_dtype] * (y.abs() + tol)


def glu_reference(x, wg, wu, bg, bu, act):
    (g, eg), (u, eu) = product(x, wg, bg), product(x, wu, bu)
    a = act64(g, act)
    ea = 1.13 * eg + 4e-6 * (g.abs() + 1)
    y = a * u
    tol = a.abs() * eu + u.abs() * ea + ea * eu + 2.0 ** -24 * y.abs()
    return y, tol + HALF_STEP[torch.bfloat16] * (y.abs() + tol)


def within(y, ref, tol):
    return bool(torch.isfinite(y).all()) and bool(((y.double() - ref).abs() <= tol).all())


def check(y, ref, tol):
    assert torch.isfinite(y).all()
    off = (y.double() - ref).abs() - tol
    at = int(off.argmax())
    assert off.max() <= 0, f"element {at} of {tuple(y.shape)}: {y.view(-1)[at]} for {ref.reshape(-1)[at]} +- {tol.reshape(-1)[at]}"


def healthy(engine):
    assert engine.lib.cogni_qmm_wait_timeouts() == 0


# row counts around every boundary of the kernels' tiles, and a few prompt-sized ones
SHAPES = [(5, 1, 256), (2, 3, 768), (40, 7, 512), (90, 2, 256), (1, 64, 256), (1, 2053, 1024), (2, 300, 768), (7, 129, 512), (8, 1000, 2048), (9, 16, 256), (15, 128, 1280),
          (16, 256, 4096), (17, 515, 512), (31, 33, 1024), (33, 130, 256), (63, 513, 768), (64, 384, 2048), (65, 200, 1536),
          (100, 96, 512), (127, 260, 256), (130, 1111, 512), (300, 257, 1024), (700, 300, 512), (1100, 640, 256),
          # enough rows of weights for several parts of K, waves of clusters and every kernel of the gated form
          (3, 9000, 1024), (12, 4104, 4352), (20, 4109, 4096), (29, 6002, 3328), (90, 5003, 2048)]


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_epilogue_matches_its_definition(cuda, oracle, engine, qtype, m, n, k):
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=m + n)
    bias, residual = rows(cuda, 1, n, 5).view(-1), rows(cuda, m, n, 6)
    y = w.dev.gemm_epilogue(x, bias=bias, residual=residual)
    check(y, *epilogue_reference(x, w, bias, "none", residual, torch.float32))
    y = w.dev.gemm_epilogue(x, bias=bias, activation="gelu", out_dtype=torch.bfloat16)
    check(y, *epilogue_reference(x, w, bias, "gelu", None, torch.bfloat16))
    healthy(engine)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_glu_matches_its_definition(cuda, oracle, engine, qtype, m, n, k):
    wg, x = inputs(cuda, oracle, qtype, m, n, k, seed=m + n)
    wu = Weight(cuda, oracle, qtype, n, k, seed=m + n + 1)
    bg, bu = rows(cuda, 1, n, 5).view(-1), rows(cuda, 1, n, 6).view(-1)
    for b1, b2, act in ((None, None, "silu"), (bg, bu, "gelu_tanh")):
        y = gemm_glu(wg.dev, wu.dev, x, activation=act, bias_gate=b1, bias_up=b2)
        assert y.dtype == torch.bfloat16 and y.shape == (m, n)
        # weights as bf16 or as f32, all of them the same way
        forms = [glu_reference(x, g, u, b1, b2, act) for g, u in ((wg.rounded, wu.rounded), (wg.exact, wu.exact))]
        if not any(within(y, *f) for f in forms):
            check(y, *forms[0])
    healthy(engine)


# cogni_qmm_set_kernel_choice: token-tile width 128 / 256 / 512, parts of K 1 / 2 / 4, the CTA pair off, direct loads
@pytest.mark.parametrize("choices", [(49, 53), (49, 54), (49, 59), (50, 53), (50, 54), (51, 53), (51, 54), (51, 53, 58), (49, 56), (51, 56)])
@pytest.mark.parametrize("qtype", TYPES)
def test_every_tile_and_split(cuda, oracle, engine, choices, qtype):
    m, n, k = 530, 200, 1024
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=17)
    wu = Weight(cuda, oracle, qtype, n, k, seed=18)
    bias, residual = rows(cuda, 1, n, 5).view(-1), rows(cuda, m, n, 6)
    for c in choices:
        assert engine.lib.cogni_qmm_set_kernel_choice(c) == 0
    try:
        y = w.dev.gemm_epilogue(x, bias=bias, activation="relu", residual=residual)
        g = gemm_glu(w.dev, wu.dev, x, bias_gate=bias)
    finally:
        for c in (48, 52, 55, 57):
            engine.lib.cogni_qmm_set_kernel_choice(c)
    check(y, *epilogue_reference(x, w, bias, "relu", residual, torch.float32))
    check(g, *glu_reference(x, w.rounded, wu.rounded, bias, None, "silu"))
    healthy(engine)


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("m", [3, 40, 260])
def test_every_activation_with_every_type_of_rows(cuda, oracle, engine, act, m):
    n, k = 190, 512
    w, x = inputs(cuda, oracle, Q5_K, m, n, k, seed=9)
    wu = Weight(cuda, oracle, Q5_K, n, k, seed=10)
    bias = 3.0 * rows(cuda, 1, n, 4).view(-1)
    for res_dtype in (None, torch.float32, torch.bfloat16):
        residual = None if res_dtype is None else rows(cuda, m, n, 6, res_dtype)
        for out_dtype in (torch.float32, torch.bfloat16):
            y = w.dev.gemm_epilogue(x, bias=bias, activation=act, residual=residual, out_dtype=out_dtype)
            assert y.dtype == out_dtype
            check(y, *epilogue_reference(x, w, bias, act, residual, out_dtype))
    y = gemm_glu(w.dev, wu.dev, x, activation=act, bias_gate=bias)
    forms = [glu_reference(x, g, u, bias, None, act) for g, u in ((w.rounded, wu.rounded), (w.exact, wu.exact))]
    if not any(within(y, *f) for f in forms):
        check(y, *forms[0])


@pytest.mark.parametrize("qtype", [Q4_K, Q6_K, Q8_0])
@pytest.mark.parametrize("m", [1, 5, 70, 290])
def test_strided_rows_and_untouched_gaps(cuda, oracle, engine, qtype, m):
    n, k = 134, 512
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=21)
    wu = Weight(cuda, oracle, qtype, n, k, seed=22)
    wide = torch.full((m + 1, k + 24), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:m, 8:8 + k] = x
    xs = wide[:m, 8:8 + k]
    residual = rows(cuda, m, n + 3, 6)[:, 1:1 + n]
    for out_dtype in (torch.float32, torch.bfloat16):
        buf = torch.full((m + 2, n + 5), 7.0, dtype=out_dtype, device=cuda)
        y = w.dev.gemm_epilogue(xs, residual=residual, out=buf[1:m + 1, 2:2 + n])
        assert y.data_ptr() == buf[1:, 2:].data_ptr()
        check(y, *epilogue_reference(x, w, None, "none", residual, out_dtype))
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[1:m + 1, 2:2 + n] = False
        assert (buf[keep] == 7.0).all()
    buf = torch.full((m + 2, n + 5), 7.0, dtype=torch.bfloat16, device=cuda)
    y = gemm_glu(w.dev, wu.dev, xs, out=buf[1:m + 1, 3:3 + n])
    forms = [glu_reference(x, g, u, None, None, "silu") for g, u in ((w.rounded, wu.rounded), (w.exact, wu.exact))]
    if not any(within(y, *f) for f in forms):
        check(y, *forms[0])
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[1:m + 1, 3:3 + n] = False
    assert (buf[keep] == 7.0).all()


@pytest.mark.parametrize("m,n,k", [(1, 300, 1024), (24, 512, 768), (600, 300, 512)])
def test_residual_in_place(cuda, oracle, engine, m, n, k):
    w, x = inputs(cuda, oracle, Q4_K, m, n, k, seed=31)
    for dtype in (torch.float32, torch.bfloat16):
        h = rows(cuda, m, n, 8, dtype)
        ref, tol = epilogue_reference(x, w, None, "relu", h, dtype)
        y = w.dev.gemm_epilogue(x, activation="relu", residual=h, out=h)
        assert y is h
        check(h, ref, tol)


def test_no_rows_and_leading_dimensions(cuda, oracle, engine):
    w, x = inputs(cuda, oracle, Q4_K, 6, 96, 256, seed=3)
    assert w.dev.gemm_epilogue(x[:0]).shape == (0, 96)
    assert gemm_glu(w.dev, w.dev, x[:0]).shape == (0, 96)
    y = w.dev.gemm_epilogue(x.view(2, 3, 256))
    assert y.shape == (2, 3, 96) and torch.equal(y.view(6, 96), w.dev.gemm_epilogue(x))
    assert w.dev.gemm_epilogue(x[0]).shape == (96,)
    h, z = norm_residual(rows(cuda, 4, 32, 1)[:0], norm=Norm(torch.ones(32, device=cuda)))
    assert h.shape == z.shape == (0, 32)


@pytest.mark.parametrize("m,n,k", [(3, 256, 2048), (48, 640, 1024), (90, 4096, 1024), (520, 300, 768)])
def test_same_bits_every_time(cuda, oracle, engine, m, n, k):
    w, x = inputs(cuda, oracle, Q5_K, m, n, k, seed=41)
    wu = Weight(cuda, oracle, Q5_K, n, k, seed=42)
    residual = rows(cuda, m, n, 2)
    first = w.dev.gemm_epilogue(x, residual=residual), gemm_glu(w.dev, wu.dev, x)
    for _ in range(20):
        assert torch.equal(first[0], w.dev.gemm_epilogue(x, residual=residual))
        assert torch.equal(first[1], gemm_glu(w.dev, wu.dev, x))


@pytest.mark.parametrize("m", [2, 40, 300])
def test_infinities_and_nan_stay_in_their_row(cuda, oracle, engine, m):
    w, x = inputs(cuda, oracle, Q8_0, m, 130, 512, seed=51)
    wu = Weight(cuda, oracle, Q8_0, 130, 512, seed=52)
    clean = w.dev.gemm_epilogue(x), gemm_glu(w.dev, wu.dev, x)
    x[0, 3], x[1, 5] = float("nan"), float("inf")
    y, g = w.dev.gemm_epilogue(x), gemm_glu(w.dev, wu.dev, x)
    assert y[0].isnan().all() and g[0].isnan().all() and not torch.isfinite(y[1]).any()
    assert torch.equal(y[2:], clean[0][2:]) and torch.equal(g[2:], clean[1][2:])


# ------------------------------------------------------------------------------------------- norms
def norm64(v, norm):
    if norm.kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / (v.square().mean(1, keepdim=True) + norm.eps).sqrt() * norm.weight.double()
    return v if norm.bias is None else v + norm.bias.double()


def make_norm(cuda, n, kind, seed, bias=None):
    bias = kind == "layer" if bias is None else bias
    return Norm(1 + 0.1 * rows(cuda, 1, n, seed).view(-1), eps=1e-5, kind=kind,
                bias=rows(cuda, 1, n, seed + 1).view(-1) if bias else None)


def norm_tolerance(h, norm, y, dtype, h_err):
    """Of y = norm(h) with |error of h| <= h_err.  In units of 2^-24: at most 32 values a thread one after
    the other and ten levels of the tree for the mean square and (layer) the mean, then the root,
    three products, the bias: 64 on |y - bias| and the mean's on its own; the error of h passes with a slope
    of at most |weight| / root, and shifts the root by at most its own relative size."""
    hc = h - h.mean(1, keepdim=True) if norm.kind == "layer" else h
    inv = 1 / (hc.square().mean(1, keepdim=True) + norm.eps).sqrt()
    w = norm.weight.double().abs()
    worst = h_err.amax(1, keepdim=True) + (64 * 2.0 ** -24 * h.abs().mean(1, keepdim=True) if norm.kind == "layer" else 0)
    tol = (worst * inv * w) * (2 + hc.abs() * inv) + 64 * 2.0 ** -24 * (hc.abs() * inv * w)
    tol = tol + 2.0 ** -23 * y.abs()
    return tol + HALF_STEP[dtype] * (y.abs() + tol)


WIDTHS = [1, 2, 7, 8, 31, 32, 64, 96, 255, 256, 257, 1000, 2051, 4096, 5120, 8192, 8200, 9001, 16384, 20000, 32768]


def norm_case(cuda, m, n, kind, res_dtype, block_dtype, gate, post, out_dtype, pad=0, eps=None):
    def make(dtype, seed):
        t = rows(cuda, m, n + pad, seed, dtype)
        return t[:, pad:] if pad else t

    residual, block = make(res_dtype, 1), None if block_dtype is None else make(block_dtype, 2)
    g = None if gate is None else rows(cuda, 1, n, 3).view(-1) if gate == "channels" else make(torch.float32, 3)
    p = make_norm(cuda, n, kind, 4) if post and block is not None else None
    norm = make_norm(cuda, n, kind, 6)
    scale = 0.625
    h, y = norm_residual(residual, block, post_norm=p, gate=g if block is not None else None, scale=scale, norm=norm,
                         out_dtype=out_dtype)
    ref = residual.double()
    err = torch.zeros_like(ref)
    if block is not None:
        b = block.double()
        be = torch.zeros_like(b)
        if p is not None:
            be = norm_tolerance(b, p, norm64(b, p), torch.float32, torch.zeros_like(b))
            b = norm64(b, p)
        if g is not None:
            b, be = b * g.double(), be * g.double().abs() + 2.0 ** -24 * (b * g.double()).abs()
        ref = ref + scale * b
        err = scale * be + 2.0 ** -23 * (scale * b.abs() + ref.abs())
    assert h.dtype == res_dtype and y.dtype == out_dtype and h.shape == y.shape == (m, n)
    check(h, ref, err + HALF_STEP[res_dtype] * (ref.abs() + err))
    want = norm64(ref, norm)
    check(y, want, norm_tolerance(ref, norm, want, out_dtype, err))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("n", WIDTHS)
def test_norm_residual_matches_its_definition(cuda, engine, kind, n):
    if n == 1 and kind == "layer":
        pytest.skip("the layer norm of one value is its bias: no bound to test")
    for m in (1, 5):
        norm_case(cuda, m, n, kind, torch.float32, torch.bfloat16, "channels", False, torch.bfloat16)
        norm_case(cuda, m, n, kind, torch.float32, torch.float32, "rows", True, torch.float32)
        norm_case(cuda, m, n, kind, torch.bfloat16, torch.bfloat16, None, True, torch.bfloat16)


@pytest.mark.parametrize("res", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("block", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", [None, "channels", "rows"])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_norm_residual_types_and_strides(cuda, engine, res, block, gate, pad):
    for post in (False, True):
        for out in (torch.float32, torch.bfloat16):
            norm_case(cuda, 70, 264, "rms", res, block, gate, post, out, pad=pad)


def test_norm_residual_in_place_and_alone(cuda, engine):
    m, n = 37, 520
    norm = make_norm(cuda, n, "rms", 6)
    h0, block = rows(cuda, m, n, 1), rows(cuda, m, n, 2, torch.bfloat16)
    h, y = norm_residual(h0, block, scale=0.5, norm=norm)
    hidden, out = h0.clone(), block.clone()
    h2, y2 = norm_residual(hidden, out, scale=0.5, norm=norm, hidden=hidden, out=out)
    assert h2 is hidden and y2 is out and torch.equal(h, h2) and torch.equal(y, y2)
    only, none = norm_residual(h0, block, scale=0.5)
    assert none is None and torch.equal(only, h)
    same, y3 = norm_residual(h, norm=norm)
    assert same is h and torch.equal(y3, y)  # h is f32: its norm is the same as formed from the registers


def test_norm_residual_rows_of_zeros_infinities_and_nan(cuda, engine):
    m, n = 6, 300
    norm = make_norm(cuda, n, "rms", 6, bias=True)
    h0 = rows(cuda, m, n, 1)
    clean = norm_residual(h0, norm=norm, out_dtype=torch.float32)[1]
    h0[0], h0[1, 7], h0[2, 9] = 0.0, float("nan"), float("inf")
    y = norm_residual(h0, norm=norm, out_dtype=torch.float32)[1]
    assert torch.equal(y[0], norm.bias) and y[1].isnan().all() and torch.equal(y[3:], clean[3:])
    assert y[2, 9].isnan() and y[2].isnan().sum() == 1


# ----------------------------------------------------------------------------- together, as in a layer
@pytest.mark.parametrize("m", [1, 16, 77, 513])
def test_feed_forward_half_of_a_layer(cuda, oracle, engine, m):
    """norm -> gate and up -> down onto the residual stream -> norm, eagerly, on another stream and replayed
    from a graph on new inputs: the same bits each way, and near the f64 result."""
    d, f = 512, 1280
    gate, up = Weight(cuda, oracle, Q4_K, f, d, 1), Weight(cuda, oracle, Q4_K, f, d, 2)
    down = Weight(cuda, oracle, Q6_K, d, f, 3)
    norm1 = Norm((1 + 0.1 * rows(cuda, 1, d, 4).view(-1)) * (2 / (gate.rms * math.sqrt(d))))
    norm2 = Norm(1 + 0.1 * rows(cuda, 1, d, 5).view(-1))
    h = torch.empty(m, d, device=cuda)
    attn = torch.empty(m, d, device=cuda, dtype=torch.bfloat16)

    def layer(stream=None):
        h1, x = norm_residual(h, attn, norm=norm1, stream=stream)
        g = gemm_glu(gate.dev, up.dev, x, stream=stream)
        h2 = down.dev.gemm_epilogue(g, residual=h1, stream=stream)
        return (x, g, h2) + norm_residual(h2, norm=norm2, stream=stream)[1:]

    def fill(seed):
        h.copy_(rows(cuda, m, d, seed))
        attn.copy_(rows(cuda, m, d, seed + 1, torch.bfloat16))

    fill(10)
    eager = layer()
    x, g, h2, y = eager
    want_x = norm64(h.double() + attn.double(), norm1)
    assert ((x.double() - want_x).abs() <= 2.0 ** -8 * want_x.abs() + 1e-5).all()
    forms = [glu_reference(x, a, b, None, None, "silu") for a, b in ((gate.rounded, up.rounded), (gate.exact, up.exact))]
    if not any(within(g, *t) for t in forms):
        check(g, *forms[0])
    h1 = (h.double() + attn.double()).float()
    check(h2, *epilogue_reference(g, down, None, "none", h1, torch.float32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = layer(side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer()
    for seed in (10, 20, 30):
        fill(seed)
        graph.replay()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(got, layer()))
    healthy(engine)


def test_calls_on_two_streams_at_once(cuda, oracle, engine):
    w, x = inputs(cuda, oracle, Q4_K, 12, 4096, 1024, seed=61)
    wu = Weight(cuda, oracle, Q4_K, 4096, 1024, seed=62)
    x2 = x.flip(0).contiguous()
    want = w.dev.gemm_epilogue(x), gemm_glu(w.dev, wu.dev, x2)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(30):
        got.append((w.dev.gemm_epilogue(x, stream=streams[0]), gemm_glu(w.dev, wu.dev, x2, stream=streams[1])))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


@pytest.mark.parametrize("qtype", [Q4_K, Q6_K])
@pytest.mark.parametrize("m", [1, 20, 140])
def test_columns_of_one_buffer(cuda, oracle, engine, qtype, m):
    """x, residual and results as columns of one buffer, side by side: not an overlap, and the same bits as apart."""
    n, k = 136, 512
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=71)
    residual = rows(cuda, m, n, 72, torch.bfloat16)
    want = w.dev.gemm_epilogue(x, residual=residual, out_dtype=torch.bfloat16)
    gated = gemm_glu(w.dev, w.dev, x)
    big = torch.full((m, k + 3 * n + 8), 7.0, device=cuda, dtype=torch.bfloat16)
    bx, br, by, bg = big[:, :k], big[:, k:k + n], big[:, k + n:k + 2 * n], big[:, k + 2 * n:k + 3 * n]
    bx.copy_(x)
    br.copy_(residual)
    w.dev.gemm_epilogue(bx, residual=br, out=by)
    gemm_glu(w.dev, w.dev, bx, out=bg)
    assert torch.equal(by, want) and torch.equal(bg, gated) and torch.equal(bx, x) and (big[:, k + 3 * n:] == 7).all()
    norm = make_norm(cuda, n, "rms", 73)
    h, y = norm_residual(br.contiguous(), by.contiguous(), norm=norm)
    norm_residual(br, by, norm=norm, hidden=br, out=by)
    assert torch.equal(br, h) and torch.equal(by, y)


def test_results_over_inputs_are_refused(cuda, oracle, engine):
    w = Weight(cuda, oracle, Q4_K, 512, 512, 1)
    x = rows(cuda, 4, 512, 2, torch.bfloat16)
    for call in (lambda: w.dev.gemm_epilogue(x, out=x), lambda: gemm_glu(w.dev, w.dev, x, out=x),
                 lambda: w.dev.gemm_epilogue(x[:3], residual=x[1:], out=x[:3]),
                 lambda: norm_residual(x, norm=Norm(torch.ones(512, device=cuda)), hidden=x[:], out=x)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("qtype", [Q4_K, Q8_0])
@pytest.mark.parametrize("m", [20, 40, 600])
def test_rows_past_32_bit_offsets(cuda, oracle, engine, qtype, m):
    """Rows so far apart that the last ones lie more than 2^32 elements (and bytes) behind the first."""
    n, k = 264, 512
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=81)
    stride = (1 << 32) // (m - 1) // 8 * 8 + 64
    far = torch.empty((m - 1) * stride + 1024, device=cuda, dtype=torch.bfloat16)
    fx, fr = far.as_strided((m, k), (stride, 1), 0), far.as_strided((m, n), (stride, 1), k)
    fx.copy_(x)
    residual = rows(cuda, m, n, 82, torch.bfloat16)
    want = w.dev.gemm_epilogue(x, residual=residual, out_dtype=torch.bfloat16)
    fr.copy_(residual)
    assert torch.equal(w.dev.gemm_epilogue(fx, residual=fr, out=fr), want)
    gated = gemm_glu(w.dev, w.dev, x)
    assert torch.equal(gemm_glu(w.dev, w.dev, fx, out=fr), gated)
    norm = make_norm(cuda, n, "layer", 83)
    h, y = norm_residual(residual, gated, norm=norm)
    fr.copy_(residual)
    h2, y2 = norm_residual(fr, gated, norm=norm, hidden=fr)
    assert torch.equal(h2, h) and torch.equal(y2, y)


def test_a_gate_of_one_factor_a_row_is_refused(cuda, engine):
    with pytest.raises(ValueError, match="gate"):
        norm_residual(rows(cuda, 8, 8, 1), rows(cuda, 8, 8, 2), gate=rows(cuda, 8, 1, 3))


def test_no_columns_are_refused(cuda, engine):
    with pytest.raises(ValueError, match="columns"):
        norm_residual(torch.empty(3, 0, device=cuda), norm=Norm(torch.empty(0, device=cuda)))
