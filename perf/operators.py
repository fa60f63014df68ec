"""Timing cases of the prefill and batched-serving block on quantised weights: the matrix product with
its epilogue, the gated feed-forward projections, and the norms around a block.

All three take the rows of one call together, from the single token of a decode step over the rows of
a serving batch to a chunk of a prompt.  Activations enter the products as bf16, weights as GGUF bytes,
the residual stream is f32 or bf16:

  epilogue  y = residual + act(x W^T + bias)                  W: one quantised matrix
  glu       y = act(x Wg^T + bg) * (x Wu^T + bu)              Wg, Wu: gate and up projection; y bf16, for the
                                                              down projection
  norm      h = residual + scale * gate * norm_post(block),  y = norm_pre(h)

A weight enters as its f32 dequantised value rounded to bf16, as in the framework's prefill product.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"q8_0": 8, "q4_k": 12, "q5_k": 13, "q6_k": 14, "iq4_nl": 20}
BLOCK = {8: (34, 32), 12: (144, 256), 13: (176, 256), 14: (210, 256), 20: (18, 32)}  # bytes, elements
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # down projection of one 9B-shaped layer, one token, onto the f32 residual stream
        {"name": "down_m1", "op": "epilogue", "type": "q6_k", "m": 1, "n": 4096, "k": 12288,
         "bias": False, "act": "none", "residual": "f32", "out": "f32"},
        # attention output projection for a batch of sixteen sequences
        {"name": "attn_out_m16", "op": "epilogue", "type": "q4_k", "m": 16, "n": 4096, "k": 4096,
         "bias": False, "act": "none", "residual": "f32", "out": "f32"},
        # an encoder's first feed-forward matrix: bias and gelu, odd rows, odd columns
        {"name": "ragged_gelu_m37", "op": "epilogue", "type": "q8_0", "m": 37, "n": 2053, "k": 1024,
         "bias": True, "act": "gelu", "residual": "none", "out": "bf16"},
        # the tail chunk of a prompt, bias and a bf16 residual
        {"name": "proj_m77", "op": "epilogue", "type": "q5_k", "m": 77, "n": 4096, "k": 4096,
         "bias": True, "act": "none", "residual": "bf16", "out": "bf16"},
        # down projection of a prompt chunk, onto the f32 residual stream
        {"name": "down_m2048", "op": "epilogue", "type": "q6_k", "m": 2048, "n": 4096, "k": 12288,
         "bias": False, "act": "none", "residual": "f32", "out": "f32"},
        # gate and up of a 9B-shaped layer, one token
        {"name": "glu_m1", "op": "glu", "type": "q4_k", "m": 1, "n": 12288, "k": 4096, "bias": False,
         "act": "silu"},
        # gate and up of a 27B-shaped layer, two dozen sequences
        {"name": "glu_27b_m24", "op": "glu", "type": "q4_k", "m": 24, "n": 17408, "k": 5120, "bias": False,
         "act": "silu"},
        # a short chunk, gelu gating with biases, a width that fills no tile
        {"name": "glu_gelu_m131", "op": "glu", "type": "q5_k", "m": 131, "n": 10210, "k": 2560, "bias": True,
         "act": "gelu_tanh"},
        # gate and up of a prompt chunk
        {"name": "glu_m4096", "op": "glu", "type": "q4_k", "m": 4096, "n": 12288, "k": 4096, "bias": False,
         "act": "silu"},
        # the norm in front of a block, one token
        {"name": "norm_m1", "op": "norm", "m": 1, "n": 4096, "kind": "rms", "block": "bf16", "post": False,
         "gate": "none", "h": "f32", "out": "bf16"},
        # layer norm after a block and before the next, odd sizes, everything bf16
        {"name": "layernorm_m333", "op": "norm", "m": 333, "n": 2051, "kind": "layer", "block": "bf16", "post": True,
         "gate": "rows", "h": "bf16", "out": "bf16"},
        # both norms, a channel gate and the f32 residual stream of a prompt chunk
        {"name": "norm_m4096", "op": "norm", "m": 4096, "n": 5120, "kind": "rms", "block": "f32", "post": True,
         "gate": "channels", "h": "f32", "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("epilogue", "epilogue", "glu", "glu", "norm"))
    m = _log(rng, 1, 4096)
    if op == "norm":
        n = _log(rng, 64, 16384)
        return {"op": op, "m": min(m, 20_000_000 // n), "n": n, "kind": rng.choice(("rms", "rms", "layer")),
                "block": rng.choice(("none", "bf16", "f32")), "post": rng.random() < 0.5,
                "gate": rng.choice(("none", "channels", "rows")), "h": rng.choice(("f32", "bf16")),
                "out": rng.choice(("bf16", "bf16", "f32"))}
    k = 256 * _log(rng, 1, 48)
    n = _log(rng, 64, 12288)
    case = {"op": op, "type": rng.choice(tuple(TYPES)), "m": min(m, 100_000_000_000 // (n * k)), "n": n, "k": k,
            "bias": rng.random() < 0.5, "act": rng.choice(ACTIVATIONS)}
    if op == "epilogue":
        case["residual"] = rng.choice(("none", "f32", "bf16"))
        case["out"] = rng.choice(("f32", "bf16"))
    return case


# ------------------------------------------------------------------------------------------ inputs
class _Maker:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(int(seed))

    def rows(self, *shape):
        return torch.randn(*shape, dtype=torch.float32, device="cuda", generator=self.gen)

    def raw(self, t, out_dim, in_dim):
        """GGUF bytes of an [out_dim, in_dim] weight: uniform quants and sub-block scales, fp16 block
        scales |N(0, s)| of the size trained weights have (weight rms about 0.04)."""
        bb, be = BLOCK[t]
        nb = out_dim * (in_dim // be)
        w = torch.randint(0, 256, (nb, bb), dtype=torch.uint8, device="cuda", generator=self.gen)

        def put(at, sigma):
            d = torch.randn(nb, 1, device="cuda", generator=self.gen).abs_().mul_(sigma)
            w[:, at:at + 2] = d.to(torch.float16).view(torch.uint8)

        if t in (12, 13):
            put(0, 1e-4 if t == 12 else 5e-5)
            put(2, 7.5e-4)
        elif t == 14:
            w[:, 192:208] = torch.randint(-64, 64, (nb, 16), dtype=torch.int8, device="cuda",
                                          generator=self.gen).view(torch.uint8)
            put(208, 6e-5)
        else:
            put(0, 5.5e-4)
        return w.view(-1)

    def norm(self, case):
        """Weight and, for layer norm, bias: what a trained norm holds."""
        return 1.0 + 0.1 * self.rows(case["n"]), 0.1 * self.rows(case["n"]) if case["kind"] == "layer" else None


def _inputs(case, seed):
    """All tensors of a case, the weights as raw bytes."""
    mk, m, n = _Maker(seed), case["m"], case["n"]
    s = {}
    if case["op"] == "norm":
        s["residual"] = mk.rows(m, n).to(DTYPES[case["h"]])
        s["block"] = None if case["block"] == "none" else mk.rows(m, n).to(DTYPES[case["block"]])
        s["post"] = mk.norm(case) if case["post"] and s["block"] is not None else None
        s["gate"] = None if case["gate"] == "none" or s["block"] is None else \
            mk.rows(n) if case["gate"] == "channels" else mk.rows(m, n)
        s["pre"] = mk.norm(case)
        return s
    k, t = case["k"], TYPES[case["type"]]
    s["x"] = mk.rows(m, k).to(torch.bfloat16)
    s["w"] = [mk.raw(t, n, k) for _ in range(2 if case["op"] == "glu" else 1)]
    s["bias"] = [mk.rows(n) if case["bias"] else None for _ in s["w"]]
    if case["op"] == "epilogue":
        s["residual"] = None if case["residual"] == "none" else mk.rows(m, n).to(DTYPES[case["residual"]])
    return s


EPS, SCALE = 1e-6, 0.75


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:  # the handles that a program makes when it loads its model
        import cogni_ml_b200 as engine
        s["engine"] = engine
        if case["op"] == "norm":
            for name in ("post", "pre"):
                if s[name] is not None:
                    s[name] = engine.Norm(s[name][0], eps=EPS, kind=case["kind"], bias=s[name][1])
        else:
            s["weights"] = [engine.DeviceQuantWeight(w, TYPES[case["type"]], case["n"], case["k"]) for w in s["w"]]
            for w in s["weights"]:
                w.resident = True  # complete before anything that uses it is launched
    return s


# -------------------------------------------------------------------------------------------- runs
_IQ4_NL = (-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113)


def _half(raw, at):
    return raw[:, at:at + 2].contiguous().view(torch.float16).float()


def _plain_weights(t, raw, n, k):
    """[n, k] f32 weights that hold bf16 values, by elementary operations on whole byte planes."""
    raw = raw.view(-1, BLOCK[t][0])
    if t == 8:
        w = _half(raw, 0) * raw[:, 2:].contiguous().view(torch.int8).float()
    elif t == 20:
        q = torch.cat([raw[:, 2:] & 15, raw[:, 2:] >> 4], 1)
        w = _half(raw, 0) * torch.tensor(_IQ4_NL, dtype=torch.float32, device=raw.device)[q.int()]
    elif t == 14:
        low = raw[:, :128].reshape(-1, 2, 64)
        low = torch.cat([low & 15, low >> 4], 2).view(-1, 2, 4, 32)
        high = raw[:, 128:192].reshape(-1, 2, 1, 32)
        high = torch.cat([high & 3, (high >> 2) & 3, (high >> 4) & 3, high >> 6], 2)
        q = (low + 16 * high).view(-1, 16, 16).float() - 32.0
        scale = _half(raw, 208) * raw[:, 192:208].contiguous().view(torch.int8).float()
        w = scale.unsqueeze(2) * q
    else:
        s = raw[:, 4:16]
        sc = torch.cat([s[:, 0:4] & 63, (s[:, 8:12] & 15) + ((s[:, 0:4] >> 6) << 4)], 1).float()
        mn = torch.cat([s[:, 4:8] & 63, (s[:, 8:12] >> 4) + ((s[:, 4:8] >> 6) << 4)], 1).float()
        q = raw[:, -128:].reshape(-1, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 2).view(-1, 8, 32)
        if t == 13:
            h = raw[:, 16:48].unsqueeze(1)
            q = q + 16 * torch.cat([(h >> g) & 1 for g in range(8)], 1)
        w = (_half(raw, 0) * sc).unsqueeze(2) * q.float() - (_half(raw, 2) * mn).unsqueeze(2)
    return w.reshape(n, k).to(torch.bfloat16).float()


def _plain_act(v, name):
    if name == "none":
        return v
    if name == "relu":
        return v.clamp(min=0.0)
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))


def _plain_norm(v, weight, bias):
    if bias is not None:
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * weight
    return v if bias is None else v + bias


def _plain(s):
    case = s["case"]
    out = DTYPES[case.get("out", "bf16")]
    if case["op"] == "norm":
        h = s["residual"].float()
        if s["block"] is not None:
            b = s["block"].float()
            if s["post"] is not None:
                b = _plain_norm(b, *s["post"])
            if s["gate"] is not None:
                b = b * s["gate"]
            h = h + SCALE * b
        return h.to(DTYPES[case["h"]]), _plain_norm(h, *s["pre"]).to(out)
    x = s["x"].float()

    def product(w, bias):
        y = x @ _plain_weights(TYPES[case["type"]], w, case["n"], case["k"]).T
        return y if bias is None else y + bias

    y = _plain_act(product(s["w"][0], s["bias"][0]), case["act"])
    if case["op"] == "glu":
        y = y * product(s["w"][1], s["bias"][1])
    elif s["residual"] is not None:
        y = s["residual"].float() + y
    return y.to(out)


def _own(s):
    case, engine = s["case"], s["engine"]
    if case["op"] == "glu":
        return engine.gemm_glu(*s["weights"], s["x"], activation=case["act"], bias_gate=s["bias"][0],
                               bias_up=s["bias"][1])
    out = DTYPES[case["out"]]
    if case["op"] == "norm":
        return engine.norm_residual(s["residual"], s["block"], post_norm=s["post"], gate=s["gate"], scale=SCALE,
                                    norm=s["pre"], out_dtype=out)
    return s["weights"][0].gemm_epilogue(s["x"], bias=s["bias"][0], activation=case["act"], residual=s["residual"],
                                         out_dtype=out)


def run(s):
    return _own(s) if own else _plain(s)


# -------------------------------------------------------------------------------------------- work
def work(case):
    m, n = case["m"], case["n"]
    size = {"none": 0, "f32": 4, "bf16": 2}
    if case["op"] == "norm":
        block = case["block"] != "none"
        norms = (2 if case["kind"] == "layer" else 1) * (1 + (case["post"] and block))
        gate = {"none": 0, "channels": n, "rows": m * n}[case["gate"]] if block else 0
        return {"bytes": m * n * (2 * size[case["h"]] + size[case["block"]] + size[case["out"]]) + 4 * (norms * n + gate),
                "flops": m * n * (10 if block else 5)}
    bb, be = BLOCK[TYPES[case["type"]]]
    mats = 2 if case["op"] == "glu" else 1
    return {"bytes": mats * n * (case["k"] // be * bb + (4 if case["bias"] else 0)) + 2 * m * case["k"]
            + m * n * (size[case.get("out", "bf16")] + size[case.get("residual", "none")]),
            "flops": 2 * mats * m * n * case["k"]}


# ------------------------------------------------------------------------- the same in 64 bits
def _wide_weights(t, raw, n, k):
    """[n, k] in f64: each weight from its block's definition, rounded to f32 and then to bf16."""
    b = raw.view(-1, BLOCK[t][0])
    count = BLOCK[t][1]
    dev = raw.device
    e = torch.arange(count, device=dev)
    byte = b.long()
    half = lambda at: b[:, at:at + 2].contiguous().view(torch.float16).double()  # noqa: E731
    signed = lambda v: v - 256 * (v > 127)  # noqa: E731
    if t == 8:
        v = half(0) * signed(byte[:, 2 + e]).double()
    elif t == 20:
        nib = byte[:, 2 + e % 16] >> (4 * (e // 16)) & 15
        v = half(0) * torch.tensor(_IQ4_NL, dtype=torch.float64, device=dev)[nib]
    elif t == 14:
        part, run_, at = e // 128, e % 128 // 32, e % 32
        low = byte[:, 64 * part + 32 * (run_ % 2) + at] >> (4 * (run_ // 2)) & 15
        high = byte[:, 128 + 32 * part + at] >> (2 * run_) & 3
        v = half(208) * signed(byte[:, 192 + e // 16]).double() * (low + 16 * high - 32).double()
    else:
        g = e // 32
        lo4, up4 = g % 4, (g >= 4).long()
        first, second, third = byte[:, 4 + lo4], byte[:, 8 + lo4], byte[:, 12 + lo4]
        sc = torch.where(up4 == 0, first & 63, (third & 15) | (first >> 6 << 4))
        mn = torch.where(up4 == 0, second & 63, (third >> 4) | (second >> 6 << 4))
        q = byte[:, BLOCK[t][0] - 128 + 32 * (g // 2) + e % 32] >> (4 * (g % 2)) & 15
        if t == 13:
            q = q + 16 * (byte[:, 16 + e % 32] >> g & 1)
        v = half(0) * sc.double() * q.double() - half(2) * mn.double()
    return v.float().to(torch.bfloat16).double().reshape(n, k)


def _wide_act(v, name):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name in ("silu", "sigmoid"):
        g = 0.5 + 0.5 * torch.tanh(0.5 * v)
        return g * v if name == "silu" else g
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))
    if name == "gelu_tanh":
        return v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def _wide_norm(v, weight, bias):
    if bias is None:
        return weight.double() * v / (v.square().sum(1, keepdim=True) / v.shape[1] + EPS).sqrt()
    mean = v.sum(1, keepdim=True) / v.shape[1]
    var = (v - mean).square().sum(1, keepdim=True) / v.shape[1]
    return weight.double() * (v - mean) / (var + EPS).sqrt() + bias.double()


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        h = s["residual"].double()
        if s["block"] is not None:
            b = s["block"].double()
            if s["post"] is not None:
                b = _wide_norm(b, *s["post"])
            h = h + SCALE * (b if s["gate"] is None else s["gate"].double() * b)
        return h, _wide_norm(h, *s["pre"])
    t, n, k = TYPES[case["type"]], case["n"], case["k"]
    x = s["x"].double()
    step = max(1, (1 << 24) // k)

    def product(w, bias):
        raw = w.view(n, -1)
        y = torch.cat([x @ _wide_weights(t, raw[at:at + step].reshape(-1), min(step, n - at), k).T
                       for at in range(0, n, step)], 1)
        return y if bias is None else y + bias.double()

    y = _wide_act(product(s["w"][0], s["bias"][0]), case["act"])
    if case["op"] == "glu":
        return y * product(s["w"][1], s["bias"][1])
    return y if s["residual"] is None else s["residual"].double() + y
