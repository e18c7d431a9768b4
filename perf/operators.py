"""What the 4-bit operators of this framework are timed on, and their plain forms.

The format is microscaled e2m1: 32 values along K share one e8m0 scale (2^(byte - 127)); two codes to a byte, the even element in
the low half; four scale bytes to an int32 word, words column-major with the rows padded to four.

* ``quant``    per_token_group_quant_mxfp4 (optionally of silu_and_mul), and the values that the result stands for (mxfp4_dequant):
               the round trip of a producer that checks or stores what the next linear will read.
* ``dequant``  mxfp4_dequant of a weight or of a stack of expert weights, as a path without 4-bit kernels needs them.
* ``matmul``   w4a4_mxfp4_matmul on operands that are quantised already.
* ``linear``   w4a4_mxfp4_linear: 16-bit activations in, quantisation, product, bias.
* ``moe``      fused_experts_mxfp4: a whole expert layer for a few tokens, activations in 16 bits.

Sizes are those of the projections and the expert layer that perf/cases.py runs in 8 bits, and the ranges around them.
"""
from __future__ import annotations

import math

import torch

own = False
mxfp4 = None  # the framework's module, where `own` is true

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # the activations of a decode batch on their own: a launch and a round trip to memory
        {"name": "quant_decode_32", "kind": "quant", "m": 32, "k": 7168, "dtype": "bf16", "silu": False},
        # between the two projections of a prefill chunk's feed-forward, gate_up at tensor parallel 2
        {"name": "quant_silu_4096", "kind": "quant", "m": 4096, "k": 9216, "dtype": "bf16", "silu": True},
        # the expert shard of one layer, made ready for a path that takes 16 bits
        {"name": "dequant_experts", "kind": "dequant", "e": 8, "n": 512, "k": 7168, "dtype": "fp16"},
        # the largest projection of a layer
        {"name": "dequant_weight", "kind": "dequant", "e": 1, "n": 7168, "k": 18432, "dtype": "bf16"},
        # a large decode batch behind a producer that quantises, the attention output projection
        {"name": "matmul_128", "kind": "matmul", "m": 128, "n": 7168, "k": 16384, "dtype": "bf16", "bias": False},
        # a full prefill chunk, gate_up at tensor parallel 2: the largest product
        {"name": "matmul_4096", "kind": "matmul", "m": 4096, "n": 18432, "k": 7168, "dtype": "bf16", "bias": False},
        # a decode step of one request: latency and the weight's bytes
        {"name": "linear_decode_1", "kind": "linear", "m": 1, "n": 4608, "k": 7168, "dtype": "bf16", "bias": False},
        # a decode step of a small batch of a float16 model with biases
        {"name": "linear_decode_32", "kind": "linear", "m": 32, "n": 4096, "k": 4096, "dtype": "fp16", "bias": True},
        # a ragged prefill chunk through a short-K projection
        {"name": "linear_chunk_1000", "kind": "linear", "m": 1000, "n": 24576, "k": 1536, "dtype": "bf16", "bias": True},
        # one request's decode step through the expert layer: eight experts
        {"name": "moe_decode_1", "kind": "moe", "m": 1, "experts": 256, "hidden": 7168, "inter": 2048, "topk": 8, "dtype": "bf16"},
        # a decode batch through a tensor-parallel shard of narrow experts, odd in number of tokens
        {"name": "moe_shard_13", "kind": "moe", "m": 13, "experts": 128, "hidden": 4096, "inter": 256, "topk": 6, "dtype": "fp16"},
        # a decode batch that hits most experts
        {"name": "moe_decode_64", "kind": "moe", "m": 64, "experts": 256, "hidden": 7168, "inter": 2048, "topk": 8, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    """Whole multiples of step between lo and hi, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["quant", "dequant", "matmul", "matmul", "linear", "linear", "linear", "moe", "moe", "moe"])
    dtype = "fp16" if rng.random() < 0.3 else "bf16"
    if kind == "quant":
        return {"kind": kind, "m": _log_int(rng, 1, 4096), "k": _log_int(rng, 128, 9216, 32), "dtype": rng.choice([dtype, "fp32"]),
                "silu": rng.random() < 0.4}
    if kind == "dequant":
        e = rng.choice([1, 1, 4, 8])
        return {"kind": kind, "e": e, "n": _log_int(rng, 64, 7168 // e, 8), "k": _log_int(rng, 128, 18432, 32), "dtype": rng.choice([dtype, "fp32"])}
    if kind in ("matmul", "linear"):
        n, k = _log_int(rng, 256, 28672, 8), _log_int(rng, 256, 18432, 32)
        # no more arithmetic than the full prefill chunk has
        m = _log_int(rng, 1, max(1, min(4096, 4096 * 18432 * 7168 // (n * k))))
        return {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.4}
    # whole layers, expert-parallel shares and tensor-parallel shards of the intermediate size
    return {"kind": kind, "m": _log_int(rng, 1, 64), "experts": rng.choice([16, 32, 64, 128, 256]), "hidden": rng.choice([2048, 4096, 7168]),
            "inter": rng.choice([192, 256, 512, 1024, 2048]), "topk": rng.choice([2, 4, 6, 8]), "dtype": dtype}


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------


def _activation(gen, shape, dtype):
    """N(0, 1) with one value in a thousand twenty times as large: the outliers that small blocks exist for."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 1e-3, x * 20.0, x).to(dtype)


def _quant(x):
    """float32 [n, k] -> codes 0 .. 15 (uint8 [n, k]) and scale bytes (int32 [n, k / 32])."""
    g = x.view(x.shape[0], -1, BLOCK)
    # the exponent of the largest magnitude after its rounding to one fraction bit, less the 2 of the largest code (6 = 1.5 * 2^2)
    byte = (((g.abs().amax(-1).view(torch.int32) + 0x200000) >> 23).clamp_(max=254) - 2).clamp_(min=0)
    a = g * ((254 - byte) << 23).view(torch.float32)[..., None]
    sign = (a < 0).to(torch.uint8) << 3
    a = a.abs()
    # to nearest, ties to the even code: the midpoints of 0 .5 1 1.5 2 3 4 6
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return (code | sign).view(x.shape), byte


def _pack(code, byte):
    """Codes and scale bytes in the layout that the operators take: uint8 [n, k / 2], int32 [n, ceil(k / 128)] column-major."""
    n, blocks = byte.shape
    q = code[:, 0::2] | (code[:, 1::2] << 4)
    words = torch.nn.functional.pad(byte, (0, -blocks % 4, 0, -n % 4)).view(n + -n % 4, -1, 4)
    words = words[..., 0] | (words[..., 1] << 8) | (words[..., 2] << 16) | (words[..., 3] << 24)
    return q.contiguous(), words.t().contiguous().t()[:n]


def _weights(gen, e, n, k):
    """[e, n, k] weights N(0, 0.02^2), quantised as a checkpoint holds them and with the scales laid out for the operators."""
    words, rows = -(-k // 128), n + -n % 4
    q = torch.empty((e, n, k // 2), device="cuda", dtype=torch.uint8)
    s = torch.zeros((e, words, rows), device="cuda", dtype=torch.int32)
    for i in range(e):
        q[i], part = _pack(*_quant(torch.randn((n, k), generator=gen, device="cuda").mul_(0.02)))
        s[i, :, :n] = part.t()
    return q, s.transpose(1, 2)[:, :n]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"kind": kind, "dtype": dtype}
    if kind == "quant":
        state["silu"] = case["silu"]
        state["x"] = _activation(gen, (case["m"], case["k"] * (2 if case["silu"] else 1)), dtype)
    elif kind == "dequant":
        state["q"], state["s"] = _weights(gen, case["e"], case["n"], case["k"])
    elif kind == "moe":
        m, e, hidden, inter = case["m"], case["experts"], case["hidden"], case["inter"]
        state["x"] = torch.randn((m, hidden), generator=gen, device="cuda").to(dtype)
        # what a router hands on: softmax weights of the chosen experts, renormalised
        scores, ids = torch.randn((m, e), generator=gen, device="cuda").topk(case["topk"], dim=1)
        state["weights"], state["ids"] = torch.softmax(scores, dim=1), ids.to(torch.int32)
        state["w1"], state["s1"] = _weights(gen, e, 2 * inter, hidden)
        state["w2"], state["s2"] = _weights(gen, e, hidden, inter)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        x = _activation(gen, (m, k), dtype)
        if kind == "matmul":
            state["x"], state["xs"] = _pack(*_quant(x.float()))
        else:
            state["x"] = x
        w, s = _weights(gen, 1, n, k)
        state["w"], state["s"] = w[0], s[0]
        state["bias"] = torch.randn((n,), generator=gen, device="cuda").to(dtype) if case["bias"] else None
    return state


# ---------------------------------------------------------------------------------------------------------------------------
# the pass: the framework's calls, and the plain forms
# ---------------------------------------------------------------------------------------------------------------------------

SCALING = 2.5  # routed scaling factor of the expert layer


def _scales(words, k):
    """int32 words [.., n, ceil(k / 128)] -> float32 scales [.., n, k / 32]."""
    shifts = torch.arange(0, 32, 8, device=words.device, dtype=torch.int32)
    byte = ((words[..., None] >> shifts) & 0xFF).flatten(-2)[..., : k // BLOCK]
    return torch.exp2((byte - 127).float())


def _values(q, words):
    """Packed codes and scale words -> float32 values [.., n, k]."""
    table = torch.tensor(VALUES + [-v for v in VALUES], device=q.device)
    k = q.shape[-1] * 2
    codes = torch.stack((q & 15, q >> 4), dim=-1).flatten(-2).int()
    return (table[codes].unflatten(-1, (k // BLOCK, BLOCK)) * _scales(words, k)[..., None]).flatten(-2)


def _quantised_values(x):
    code, byte = _quant(x)
    table = torch.tensor(VALUES + [-v for v in VALUES], device=x.device)
    return (table[code.int()].view(x.shape[0], -1, BLOCK) * torch.exp2((byte - 127).float())[..., None]).view(x.shape)


def _silu_and_mul(x):
    gate, up = x.float().chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _token(state, t):
    """The expert layer of token t: [hidden] float32, not scaled yet."""
    ids = state["ids"][t].long()
    x = state["x"][t].float()
    h = _silu_and_mul(_values(state["w1"][ids], state["s1"][ids]) @ x)  # [topk, inter]
    y = torch.bmm(_values(state["w2"][ids], state["s2"][ids]), h[..., None])[..., 0]  # [topk, hidden]
    return (y * state["weights"][t][:, None]).sum(0)


def _plain(state):
    kind, dtype = state["kind"], state["dtype"]
    if kind == "quant":
        return _quantised_values(_silu_and_mul(state["x"]) if state["silu"] else state["x"].float()).to(dtype)
    if kind == "dequant":
        return _values(state["q"], state["s"]).to(dtype)
    if kind == "moe":
        return (torch.stack([_token(state, t) for t in range(state["x"].shape[0])]) * SCALING).to(dtype)
    x = _values(state["x"], state["xs"]) if kind == "matmul" else _quantised_values(state["x"].float())
    y = x @ _values(state["w"], state["s"]).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(dtype)


def run(state):
    global mxfp4
    if not own:
        return _plain(state)
    if mxfp4 is None:
        from sglang_amd import mxfp4
    kind = state["kind"]
    if kind == "quant":
        q, s = mxfp4.per_token_group_quant_mxfp4(state["x"], fuse_silu_and_mul=state["silu"])
        return mxfp4.mxfp4_dequant(q, s, state["dtype"])
    if kind == "dequant":
        return mxfp4.mxfp4_dequant(state["q"], state["s"], state["dtype"])
    if kind == "matmul":
        return mxfp4.w4a4_mxfp4_matmul(state["x"], state["w"], state["xs"], state["s"], state["dtype"], bias=state["bias"])
    if kind == "linear":
        return mxfp4.w4a4_mxfp4_linear(state["x"], state["w"], state["s"], bias=state["bias"])
    return mxfp4.fused_experts_mxfp4(state["x"], state["w1"], state["w2"], state["weights"], state["ids"], state["s1"], state["s2"],
                                     routed_scaling_factor=SCALING)


# ---------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------


def _exact_values(q, words):
    """From the fields of a code: sign, two exponent bits, one fraction bit; and of the word's bytes as little-endian memory."""
    k = q.shape[-1] * 2
    c = torch.empty(q.shape[:-1] + (k,), dtype=torch.int64, device=q.device)
    c[..., 0::2], c[..., 1::2] = q.long() % 16, q.long() // 16
    exponent, fraction = (c // 2) % 4, (c % 2).double()
    size = torch.where(exponent == 0, 0.5 * fraction, (1.0 + 0.5 * fraction) * 2.0 ** (exponent - 1).double())
    value = torch.where(c >= 8, -size, size)
    byte = words.clone(memory_format=torch.contiguous_format).view(torch.uint8)[..., : k // BLOCK].double()
    return value * torch.repeat_interleave(2.0 ** (byte - 127.0), BLOCK, dim=-1)


def _exact_quantised(x):
    """Every value to the nearest multiple of its binade's step, ties to the even multiple; float64 in and out."""
    g = x.view(x.shape[0], -1, BLOCK)
    mantissa, exponent = torch.frexp(g.abs().amax(-1))  # 0.5 <= mantissa < 1
    exponent = (exponent - 1 + (mantissa >= 0.875).int() - 2).double().clamp(-127.0, 125.0)
    scale = (2.0 ** exponent)[..., None]
    a = g / scale
    step = torch.where(a.abs() < 2.0, 0.5, torch.where(a.abs() < 4.0, 1.0, 2.0)).double()
    return ((torch.round(a / step) * step).clamp(-6.0, 6.0) * scale).view(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    kind = state["kind"]
    if kind == "quant":
        x = state["x"].double()
        if state["silu"]:
            half = x.shape[1] // 2
            x = x[:, :half] * torch.sigmoid(x[:, :half]) * x[:, half:]
        return _exact_quantised(x)
    if kind == "dequant":
        return _exact_values(state["q"], state["s"])
    if kind == "moe":
        x, ids, weights = state["x"].double(), state["ids"].long(), state["weights"].double()
        out = torch.zeros_like(x)
        for e in ids.unique().tolist():
            token, place = (ids == e).nonzero(as_tuple=True)
            a = x[token] @ _exact_values(state["w1"][e], state["s1"][e]).t()
            half = a.shape[1] // 2
            h = a[:, :half] * torch.sigmoid(a[:, :half]) * a[:, half:]
            out.index_add_(0, token, (h @ _exact_values(state["w2"][e], state["s2"][e]).t()) * weights[token, place][:, None])
        return out * SCALING
    x = _exact_values(state["x"], state["xs"]) if kind == "matmul" else _exact_quantised(state["x"].double())
    y = x @ _exact_values(state["w"], state["s"]).t()
    return y if state["bias"] is None else y + state["bias"].double()


# ---------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------

BITS = 17 / 32  # bytes of an element: half a byte, and a scale byte for 32


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "quant":
        m, k = case["m"], case["k"]
        # x in, the 4-bit form out and in again, the values out
        return {"bytes": m * k * (size * (2 if case["silu"] else 1) + 2 * BITS + size), "flops": 0}
    if kind == "dequant":
        return {"bytes": case["e"] * case["n"] * case["k"] * (BITS + size), "flops": 0}
    m = case["m"]
    if kind == "moe":
        e, hidden, inter, topk = case["experts"], case["hidden"], case["inter"], case["topk"]
        hit = e * (1.0 - (1.0 - topk / e) ** m)  # experts that some token picks, on average
        return {"bytes": hit * 3 * inter * hidden * BITS + 2 * 2 * m * hidden + 8 * m * topk, "flops": 2.0 * m * topk * 3 * inter * hidden}
    n, k = case["n"], case["k"]
    return {"bytes": m * k * (BITS if kind == "matmul" else 2) + n * k * BITS + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}
