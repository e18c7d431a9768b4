"""What latent attention on this framework is timed on, and its plain forms.

A token's keys and values are one shared row of 576 numbers: a latent of 512 and a part of 64 that carries the rotary position.
The row is all that the cache holds.  Attention either works on the rows themselves (absorbed: the up-projections are folded into
the queries and into what follows, all heads share one key of 576 and one value of 512), or on per-head keys of 128 + 64 and
values of 128 that the up-projection made of the latents (expanded).

* ``write``    mla_write_cache: root-mean-square norm of the latent, rotary embedding of the position part and of the queries', and
               the row's store into its slot of the paged cache.  Into an 8-bit cache followed by mla_gather_cache, which gives the
               values that the bytes stand for.
* ``gather``   mla_gather_cache: the rows of cached prefixes, one after the other and in 16 bits, for the up-projection.
* ``decode``   mla_decode_attention: absorbed attention of one or a few new tokens of each request over the paged cache.
* ``prefill``  mla_prefill_attention: expanded causal attention over ragged sequences.
* ``merge``    merge_attention_states: two attentions over disjoint keys joined into one.

The absorbed products on either side of ``decode`` are timed by perf/cases.py; heads, types and token counts are those of its cases
and the ranges around them.
"""
from __future__ import annotations

import math

import torch

own = False
mla = None  # the framework's module, where `own` is true

LATENT, ROPE, WIDTH = 512, 64, 576
NOPE, VALUE = 128, 128
SM_SCALE = (NOPE + ROPE) ** -0.5
EPS = 1e-6
POSITIONS = 32768  # rows of the table of cosines and sines
CACHE_SCALE = 0.0125  # of the 8-bit cache: the largest of a normed latent's values, some 5, to the largest code, 448
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NEG_INF = float("-inf")


def listed():
    return [
        # a decode batch's rows and queries, all 128 heads: a launch
        {"name": "write_decode_64", "kind": "write", "tokens": 64, "heads": 128, "dtype": "bf16", "cache": "same", "page": 64, "neox": False,
         "norm": True},
        # a prefill chunk into an 8-bit cache at tensor parallel 8, and its rows read back
        {"name": "write_fp8_4096", "kind": "write", "tokens": 4096, "heads": 16, "dtype": "bf16", "cache": "fp8", "page": 64, "neox": False,
         "norm": True},
        # the cached prefixes of a few long requests, for the up-projection of a chunked prefill
        {"name": "gather_prefix_30000", "kind": "gather", "batch": 7, "len": 8192, "dtype": "bf16", "cache": "same", "page": 64},
        # short shared prefixes of a decode batch that turned into a prefill, token-sized pages of an 8-bit cache
        {"name": "gather_fp8_paged_1", "kind": "gather", "batch": 32, "len": 200, "dtype": "fp16", "cache": "fp8", "page": 1},
        # one request, all heads: latency, and the split over the cache's length
        {"name": "decode_1", "kind": "decode", "batch": 1, "queries": 1, "heads": 128, "len": 8000, "dtype": "bf16", "cache": "same", "page": 64},
        # a decode batch at tensor parallel 8 that verifies a drafted token each: bound by the cache's bytes
        {"name": "decode_shard_64", "kind": "decode", "batch": 64, "queries": 2, "heads": 16, "len": 8192, "dtype": "fp16", "cache": "same",
         "page": 16},
        # a large data-parallel batch over an 8-bit cache, all heads: the matrix cores and the bytes at once
        {"name": "decode_fp8_128", "kind": "decode", "batch": 128, "queries": 1, "heads": 128, "len": 6000, "dtype": "bf16", "cache": "fp8",
         "page": 64},
        # several short prompts in one batch, ragged, at tensor parallel 8
        {"name": "prefill_ragged_17", "kind": "prefill", "batch": 17, "queries": 300, "prefix": 0, "heads": 16, "dtype": "bf16", "causal": True},
        # a chunk of a long prompt of a float16 model against its own keys and those of the chunks before it
        {"name": "prefill_chunk_1000", "kind": "prefill", "batch": 1, "queries": 1000, "prefix": 9000, "heads": 32, "dtype": "fp16",
         "causal": True},
        # a full prompt, all heads: the largest
        {"name": "prefill_8192", "kind": "prefill", "batch": 1, "queries": 8192, "prefix": 0, "heads": 128, "dtype": "bf16", "causal": True},
        # the last chunk's own attention and its prefix's, a few tokens
        {"name": "merge_37", "kind": "merge", "tokens": 37, "heads": 16, "dtype": "fp16"},
        # a full chunk's, all heads: bound by the bytes
        {"name": "merge_4096", "kind": "merge", "tokens": 4096, "heads": 128, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    """Whole multiples of step between lo and hi, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["write", "gather", "decode", "decode", "decode", "decode", "prefill", "prefill", "prefill", "merge"])
    dtype = "fp16" if rng.random() < 0.3 else "bf16"
    page = rng.choice([1, 16, 32, 64, 64, 128])
    cache = rng.choice(["same", "same", "fp8"])
    heads = rng.choice([8, 16, 16, 32, 64, 128, 128])
    if kind == "write":
        return {"kind": kind, "tokens": _log_int(rng, 1, 8192), "heads": heads, "dtype": dtype, "cache": cache, "page": page,
                "neox": rng.random() < 0.3, "norm": rng.random() < 0.8}
    if kind == "gather":
        return {"kind": kind, "batch": _log_int(rng, 1, 32), "len": _log_int(rng, 1, 8192), "dtype": dtype, "cache": cache, "page": page}
    if kind == "decode":
        queries = rng.choice([1, 1, 1, 2, 3, 4])
        # no more scores than the large batch has
        batch = _log_int(rng, 1, 256)
        length = _log_int(rng, 1, max(1, min(32768, 128 * 6000 * 128 // (batch * queries * heads))))
        return {"kind": kind, "batch": batch, "queries": queries, "heads": heads, "len": length, "dtype": dtype, "cache": cache, "page": page}
    if kind == "prefill":
        batch = rng.choice([1, 1, 2, 5, 16])
        queries = _log_int(rng, 1, 8192 // batch)
        prefix = rng.choice([0, 0, _log_int(rng, 1, 16384 // batch)])
        # no more scores than the full prompt has
        most = 8192 * 8192 * 128 // 2
        while batch * queries * (queries // 2 + prefix) * heads > most:
            queries, prefix = queries // 2 + 1, prefix // 2
        return {"kind": kind, "batch": batch, "queries": queries, "prefix": prefix, "heads": heads, "dtype": dtype,
                "causal": prefix == 0 or rng.random() < 0.7}
    return {"kind": kind, "tokens": _log_int(rng, 1, 8192), "heads": heads, "dtype": dtype}


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------


def _lengths(batch, longest):
    """Ragged lengths of a batch, the first the longest, the others down to a third of it, in no order."""
    return [longest if i == 0 else max(1, longest - (i * 7919 % 101) * longest * 2 // 303) for i in range(batch)]


def _table(gen, lengths, page):
    """A page table int32 [batch, most pages] whose pages lie in the cache in no order, and the cache's number of pages."""
    counts = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(counts) + 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(lengths), max(counts)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(counts) + 3


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _cache(gen, state, lengths, page, dtype, kind):
    """A filled cache of normed latents: N(0, 1), the first token of a request with a position part of three times the size, as
    the tokens that everything attends to have."""
    state["table"], pages = _table(gen, lengths, page)
    rows = torch.randn((pages, page, WIDTH), generator=gen, device="cuda")
    rows[state["table"][:, 0].long(), 0, LATENT:] *= 3.0
    if kind == "fp8":
        state["scale"] = torch.full((1,), CACHE_SCALE, device="cuda")
        state["cache"] = (rows / state["scale"]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    else:
        state["scale"] = None
        state["cache"] = rows.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"kind": kind, "dtype": dtype}
    if kind == "write":
        tokens, heads, page = case["tokens"], case["heads"], case["page"]
        # the last rows of a batch that is padded to a captured size have no slot
        state["valid"] = valid = tokens - tokens // 16
        state["table"], pages = _table(gen, [valid], page)
        t = torch.arange(valid, device="cuda")
        slots = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
        slots[:valid] = state["table"][0, t // page].long() * page + t % page
        state["slots"], state["cu"] = slots, _ints([0, valid])
        state["latent"] = _rows(gen, (tokens, WIDTH), dtype)  # what the down-projection gives
        # the queries' position part is the tail of each head's 192 numbers
        state["q_pe"] = _rows(gen, (tokens, heads, NOPE + ROPE), dtype)[..., NOPE:]
        state["weight"] = (1.0 + 0.1 * torch.randn((LATENT,), generator=gen, device="cuda")).to(dtype) if case["norm"] else None
        state["positions"] = torch.randint(0, POSITIONS, (tokens,), generator=gen, device="cuda")
        inverse = 10000.0 ** (-torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float64) / ROPE)
        angles = torch.arange(POSITIONS, device="cuda", dtype=torch.float64)[:, None] * inverse
        state["cos_sin"] = torch.cat((angles.cos(), angles.sin()), dim=1).float()
        state["neox"] = case["neox"]
        if case["cache"] == "fp8":
            state["scale"] = torch.full((1,), CACHE_SCALE, device="cuda")
            state["cache"] = torch.zeros((pages, page, WIDTH), device="cuda").to(torch.float8_e4m3fn)
        else:
            state["scale"] = None
            state["cache"] = torch.zeros((pages, page, WIDTH), dtype=dtype, device="cuda")
    elif kind == "gather":
        lengths = _lengths(case["batch"], case["len"])
        _cache(gen, state, lengths, case["page"], dtype, case["cache"])
        state["cu"], state["total"] = _ints(_starts(lengths)), sum(lengths)
    elif kind == "decode":
        lengths = _lengths(case["batch"], case["len"])
        _cache(gen, state, lengths, case["page"], dtype, case["cache"])
        state["lens"] = _ints(lengths)
        # the absorbed product gives the queries head by head: [heads, tokens, 512], seen token by token
        b, n, h = case["batch"], case["queries"], case["heads"]
        state["q_nope"] = _rows(gen, (h, b * n, LATENT), dtype).transpose(0, 1).view(b, n, h, LATENT)
        state["q_pe"] = _rows(gen, (b, n, h, ROPE), dtype)
    elif kind == "prefill":
        queries = _lengths(case["batch"], case["queries"])
        keys = [n + m for n, m in zip(queries, _lengths(case["batch"], case["prefix"]) if case["prefix"] else [0] * len(queries))]
        state["cu_q"], state["cu_k"], state["most"] = _ints(_starts(queries)), _ints(_starts(keys)), max(queries)
        state["q"] = _rows(gen, (sum(queries), case["heads"], NOPE + ROPE), dtype)
        # what the up-projection gives: a head's key, then its value
        kv = _rows(gen, (sum(keys), case["heads"], NOPE + VALUE), dtype)
        state["k_nope"], state["v"] = kv[..., :NOPE], kv[..., NOPE:]
        state["k_pe"] = _rows(gen, (sum(keys), ROPE), dtype)
        state["causal"] = case["causal"]
    else:
        shape = (case["tokens"], case["heads"])
        for part in "ab":
            state["out_" + part] = _rows(gen, shape + (VALUE,), dtype)
            state["lse_" + part] = torch.randn(shape, generator=gen, device="cuda") * 2.0 + 6.0
        # tokens whose prefix holds nothing
        empty = torch.rand((case["tokens"],), generator=gen, device="cuda") < 0.1
        state["lse_b"][empty] = NEG_INF
        state["out_b"][empty] = 0.0
    return state


# ---------------------------------------------------------------------------------------------------------------------------
# the pass: the framework's calls, and the plain forms
# ---------------------------------------------------------------------------------------------------------------------------


def _rotate(x, table, neox):
    """x [.., 64] float32 by the angles whose cosines and sines are table's rows [.., 64]: pairs of neighbours, or (neox) of
    numbers that lie 32 apart."""
    cos, sin = table[..., : ROPE // 2], table[..., ROPE // 2:]
    if neox:
        a, b = x[..., : ROPE // 2], x[..., ROPE // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)


def _cached(state, rows):
    """Rows of the cache by their numbers, float32."""
    cache = state["cache"].view(-1, WIDTH)
    if state["scale"] is None:
        return cache[rows].float()
    return cache.view(torch.uint8)[rows].view(torch.float8_e4m3fn).float() * state["scale"]


def _request_rows(state, request, count):
    page = state["cache"].shape[1]
    t = torch.arange(count, device="cuda")
    return state["table"][request].long()[t // page] * page + t % page


def _attend(scores, values):
    """scores [.., q, k] float32 with -inf at what is masked, values [.., k, d] -> out, lse; rows that see nothing are 0 and -inf."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == NEG_INF, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / torch.where(total == 0.0, 1.0, total)
    return out, (torch.log(total) + torch.where(top == NEG_INF, 0.0, top))[..., 0]


def _mask(n, m, causal):
    """[n, m] of 0 and -inf: query i is the key of place i + m - n."""
    if not causal:
        return 0.0
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")
    return torch.where(j <= i + (m - n), 0.0, NEG_INF)


def _plain_write(state):
    table = state["cos_sin"][state["positions"]]
    latent = state["latent"].float()
    c, pe = latent[:, :LATENT], _rotate(latent[:, LATENT:], table, state["neox"])
    if state["weight"] is not None:
        c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * state["weight"].float()
    rows = torch.cat((c, pe), dim=1)[: state["valid"]]
    slots = state["slots"][: state["valid"]]
    cache = state["cache"].view(-1, WIDTH)
    q = _rotate(state["q_pe"].float(), table[:, None], state["neox"]).to(state["dtype"])
    if state["scale"] is None:
        cache[slots] = rows.to(state["dtype"])
        return state["cache"], q
    cache.view(torch.uint8)[slots] = (rows / state["scale"]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return _cached(state, slots).to(state["dtype"]), q


def _plain(state):
    kind, dtype = state["kind"], state["dtype"]
    if kind == "write":
        return _plain_write(state)
    if kind == "gather":
        cu = state["cu"].tolist()
        return torch.cat([_cached(state, _request_rows(state, i, cu[i + 1] - cu[i])) for i in range(len(cu) - 1)]).to(dtype)
    if kind == "decode":
        b, n, h, _ = state["q_nope"].shape
        out, lse = torch.empty((b, n, h, LATENT), dtype=dtype, device="cuda"), torch.empty((b, n, h), device="cuda")
        for i, m in enumerate(state["lens"].tolist()):
            kv = _cached(state, _request_rows(state, i, m))
            q = torch.cat((state["q_nope"][i], state["q_pe"][i]), dim=-1).float().view(n * h, WIDTH)
            scores = (q @ kv.t()).view(n, h, m) * SM_SCALE
            if n > 1:
                scores = scores + _mask(n, m, True)[:, None]
            o, s = _attend(scores.view(n * h, m), kv[:, :LATENT])
            out[i], lse[i] = o.view(n, h, LATENT).to(dtype), s.view(n, h)
        return out, lse
    if kind == "prefill":
        q, k_nope, k_pe, v = state["q"], state["k_nope"], state["k_pe"], state["v"]
        h = q.shape[1]
        out, lse = torch.empty((q.shape[0], h, VALUE), dtype=dtype, device="cuda"), torch.empty((q.shape[0], h), device="cuda")
        cu_q, cu_k = state["cu_q"].tolist(), state["cu_k"].tolist()
        for i in range(len(cu_q) - 1):
            a, b, c, d = cu_q[i], cu_q[i + 1], cu_k[i], cu_k[i + 1]
            mask = _mask(b - a, d - c, state["causal"])
            step = max(1, (1 << 28) // max(1, (b - a) * (d - c)))  # heads whose scores are held at once
            for at in range(0, h, step):
                heads = slice(at, at + step)
                key = torch.cat((k_nope[c:d, heads].float(), k_pe[c:d, None].float().expand(-1, min(step, h - at), -1)), dim=-1)
                scores = torch.matmul(q[a:b, heads].float().transpose(0, 1), key.permute(1, 2, 0).contiguous()) * SM_SCALE + mask
                o, s = _attend(scores, v[c:d, heads].float().transpose(0, 1).contiguous())
                out[a:b, heads], lse[a:b, heads] = o.transpose(0, 1).to(dtype), s.t()
        return out, lse
    a, b = state["lse_a"], state["lse_b"]
    top = torch.maximum(a, b)
    shift = torch.where(top == NEG_INF, 0.0, top)
    wa, wb = torch.exp(a - shift), torch.exp(b - shift)
    total = wa + wb
    whole = torch.where(total == 0.0, 1.0, total)
    out = state["out_a"].float() * (wa / whole)[..., None] + state["out_b"].float() * (wb / whole)[..., None]
    return out.to(dtype), torch.log(total) + shift


def run(state):
    global mla
    if not own:
        return _plain(state)
    if mla is None:
        from sglang_amd import mla
    kind = state["kind"]
    if kind == "write":
        q = mla.mla_write_cache(state["latent"], state["cache"], state["slots"], norm_weight=state["weight"], eps=EPS, cos_sin=state["cos_sin"],
                                positions=state["positions"], neox=state["neox"], q_pe=state["q_pe"], scale=state["scale"])
        if state["scale"] is None:
            return state["cache"], q
        return mla.mla_gather_cache(state["cache"], state["table"], state["cu"], state["valid"], dtype=state["dtype"], scale=state["scale"]), q
    if kind == "gather":
        return mla.mla_gather_cache(state["cache"], state["table"], state["cu"], state["total"], dtype=state["dtype"], scale=state["scale"])
    if kind == "decode":
        return mla.mla_decode_attention(state["q_nope"], state["q_pe"], state["cache"], state["table"], state["lens"], SM_SCALE,
                                        scale=state["scale"], return_lse=True)
    if kind == "prefill":
        return mla.mla_prefill_attention(state["q"], state["k_nope"], state["k_pe"], state["v"], state["cu_q"], state["cu_k"], state["most"],
                                         SM_SCALE, causal=state["causal"], return_lse=True)
    return mla.merge_attention_states(state["out_a"], state["lse_a"], state["out_b"], state["lse_b"])


# ---------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------


def _exact_rotation(x, cos_sin):
    """Complex numbers by the unit numbers of their angles; x [.., 32, 2] float64."""
    unit = torch.complex(cos_sin[..., : ROPE // 2].double(), cos_sin[..., ROPE // 2:].double())
    return torch.view_as_real(torch.view_as_complex(x.contiguous()) * unit)


def _exact_rope(x, cos_sin, neox):
    x = x.double()
    if neox:
        return _exact_rotation(x.unflatten(-1, (2, ROPE // 2)).transpose(-1, -2), cos_sin).transpose(-1, -2).flatten(-2)
    return _exact_rotation(x.unflatten(-1, (ROPE // 2, 2)), cos_sin).flatten(-2)


def _exact_e4m3(x):
    """Every value to the nearest multiple of its binade's step, ties to the even multiple, at most 448; float64 in and out."""
    exponent = (torch.frexp(x.abs())[1] - 1).clamp(min=-6)
    step = torch.ldexp(torch.ones_like(x), exponent - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_softmax(scores, seen, values):
    """Base 2 throughout; seen marks what counts."""
    s = torch.where(seen, scores * math.log2(math.e), NEG_INF)
    some = seen.any(-1, keepdim=True)
    top = torch.where(some, s.max(-1, keepdim=True).values, 0.0)
    weights = torch.exp2(s - top)
    total = weights.sum(-1, keepdim=True)
    out = torch.where(some, torch.matmul(weights, values) / total, 0.0)
    return out, ((torch.log2(total) + top) * math.log(2.0))[..., 0]


def _exact_cached(state, request, count):
    """The first tokens of a request from the cache, page by page, float64."""
    page = state["cache"].shape[1]
    pages = state["table"][request, : -(-count // page)].long()
    data = state["cache"].view(torch.uint8) if state["scale"] is not None else state["cache"]
    rows = data.index_select(0, pages).flatten(0, 1)[:count]
    if state["scale"] is None:
        return rows.double()
    code = rows.long()
    exponent, fraction = (code // 8) % 16, (code % 8).double()
    size = torch.where(exponent == 0, fraction * 2.0 ** -9, (1.0 + fraction / 8.0) * torch.exp2(exponent.double() - 7.0))
    return torch.where(code >= 128, -size, size) * state["scale"].double()


def exact(case, seed):
    state = prepare(case, seed)
    kind = state["kind"]
    if kind == "write":
        angle_rows = state["cos_sin"].index_select(0, state["positions"])
        q = _exact_rope(state["q_pe"], angle_rows.unsqueeze(1), state["neox"])
        c = state["latent"][:, :LATENT].double()
        if state["weight"] is not None:
            c = c / torch.sqrt(c.square().sum(-1, keepdim=True) / LATENT + EPS) * state["weight"].double()
        rows = torch.cat((c, _exact_rope(state["latent"][:, LATENT:], angle_rows, state["neox"])), dim=-1)
        if state["scale"] is not None:
            scale = state["scale"].double()
            return _exact_e4m3(rows[: state["valid"]] / scale) * scale, q
        cache = state["cache"].double().flatten(0, 1)
        cache.index_copy_(0, state["slots"][: state["valid"]], rows[: state["valid"]])
        return cache.view(state["cache"].shape), q
    if kind == "gather":
        lengths = (state["cu"][1:] - state["cu"][:-1]).tolist()
        return torch.cat([_exact_cached(state, i, n) for i, n in enumerate(lengths)])
    if kind == "decode":
        b, n, h, _ = state["q_nope"].shape
        outs, sums = [], []
        for i, m in enumerate(state["lens"].tolist()):
            rows = _exact_cached(state, i, m)
            scores = state["q_nope"][i].double() @ rows[:, :LATENT].t() + state["q_pe"][i].double() @ rows[:, LATENT:].t()  # [n, h, m]
            # the last query sees everything, the one before it all but the last token, and so on
            back = torch.arange(n - 1, -1, -1, device="cuda").view(n, 1, 1)
            seen = (torch.arange(m, device="cuda") < m - back).expand(n, h, m)
            o, s = _exact_softmax(scores * SM_SCALE, seen, rows[:, :LATENT])
            outs.append(o)
            sums.append(s)
        return torch.stack(outs), torch.stack(sums)
    if kind == "prefill":
        outs, sums = [], []
        cu_q, cu_k = state["cu_q"].tolist(), state["cu_k"].tolist()
        for a, b, c, d in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
            position = state["k_pe"][c:d].double()
            last = torch.arange(b - a, device="cuda")[:, None] + ((d - c) - (b - a)) if state["causal"] else d - c
            seen = (torch.arange(d - c, device="cuda")[None] <= last).expand(b - a, d - c)
            by_head = []
            for head in range(state["q"].shape[1]):
                q = state["q"][a:b, head].double()
                scores = q[:, :NOPE] @ state["k_nope"][c:d, head].double().t() + q[:, NOPE:] @ position.t()
                by_head.append(_exact_softmax(scores * SM_SCALE, seen, state["v"][c:d, head].double()))
            outs.append(torch.stack([o for o, _ in by_head], dim=1))
            sums.append(torch.stack([s for _, s in by_head], dim=1))
        return torch.cat(outs), torch.cat(sums)
    pair = torch.stack((state["lse_a"], state["lse_b"])).double()
    lse = torch.logsumexp(pair, dim=0)
    share = torch.where(lse == NEG_INF, 0.0, torch.exp(pair - lse))[..., None]
    return share[0] * state["out_a"].double() + share[1] * state["out_b"].double(), lse


# ---------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    byte = 1 if case.get("cache") == "fp8" else 2
    if kind == "write":
        tokens, heads = case["tokens"], case["heads"]
        valid = tokens - tokens // 16
        # rows in and out, the queries' part in and out, a position, its cosines and sines, a slot
        total = valid * WIDTH * (2 + byte) + tokens * (heads * ROPE * 4 + 8 + ROPE * 4 + 8)
        if byte == 1:
            total += valid * WIDTH * (1 + 2)  # the rows read back
        return {"bytes": total, "flops": 0}
    if kind == "gather":
        return {"bytes": sum(_lengths(case["batch"], case["len"])) * WIDTH * (byte + 2), "flops": 0}
    if kind == "decode":
        n, h = case["queries"], case["heads"]
        lengths = _lengths(case["batch"], case["len"])
        scores = sum(sum(max(0, m - back) for back in range(n)) for m in lengths) * h
        return {"bytes": sum(lengths) * WIDTH * byte + case["batch"] * n * h * ((WIDTH + LATENT) * 2 + 4), "flops": 2.0 * scores * (WIDTH + LATENT)}
    if kind == "prefill":
        h = case["heads"]
        queries = _lengths(case["batch"], case["queries"])
        prefixes = _lengths(case["batch"], case["prefix"]) if case["prefix"] else [0] * len(queries)
        scores = sum(n * m + (n * (n + 1) // 2 if case["causal"] else n * n) for n, m in zip(queries, prefixes)) * h
        keys = sum(queries) + sum(prefixes)
        return {"bytes": 2 * (sum(queries) * h * (NOPE + ROPE + VALUE + 2) + keys * (h * (NOPE + VALUE) + ROPE)),
                "flops": 2.0 * scores * (NOPE + ROPE + VALUE)}
    return {"bytes": case["tokens"] * case["heads"] * (3 * VALUE * 2 + 3 * 4), "flops": 0}
