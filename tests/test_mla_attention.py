"""Latent attention without a GPU: what the C entry points and the Python checks refuse, before anything is launched; shapes of the
fake implementations; the reference of the GPU tests against torch's own attention and against differences."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tests import mla_reference as R

I32, I64, BF16, F16, F32, F8 = torch.int32, torch.int64, torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _address():
    buf = ctypes.create_string_buffer(8192)
    return buf, (ctypes.addressof(buf) + 255) // 256 * 256


def _refused(rc, *words):
    from sglang_amd._lib import lib

    text = lib.fp8k_last_error().decode()
    assert rc != 0 and all(w in text for w in words), (rc, text)


def test_c_refusals_of_the_cache_operators():
    from sglang_amd import _lib

    lib = _lib.lib
    keep, p = _address()

    def write(latent=p, ld=576, cache=p, slots=p, weight=None, weight_type=0, cos=None, max_pos=0, pos=None, q=None, qt=64, qh=64, qo=None, ot=64,
              oh=64, T=4, H=0, dtype=_lib.BF16):
        return lib.fp8k_mla_write_cache(latent, ld, cache, slots, 1, weight, weight_type, 1e-6, cos, max_pos, pos, 1, 0, q, qt, qh, qo, ot, oh, None,
                                        T, H, 100, dtype, 0, None)

    assert write(T=0, latent=None) == 0
    _refused(write(dtype=_lib.F32), "Half or BFloat16")
    _refused(write(latent=None), "null")
    _refused(write(ld=575), "16-byte")
    _refused(write(ld=568), "16-byte")
    _refused(write(latent=p + 8), "16-byte")
    _refused(write(slots=p + 4), "slots")
    _refused(write(weight=p, weight_type=_lib.F16), "weight")
    _refused(write(cos=p), "positions")
    _refused(write(cos=p, pos=p, max_pos=0), "positions")
    _refused(write(q=p, qo=p, H=2), "cosines")
    _refused(write(q=p, H=2, cos=p, pos=p, max_pos=3), "place")
    _refused(write(q=p, qo=p, H=2, cos=p, pos=p, max_pos=3, qh=65), "16-byte")
    _refused(write(q=p, qo=p, H=2, cos=p, pos=p, max_pos=3, ot=-64), "negative")
    _refused(write(T=-1), "sizes")

    def gather(cache=p, width=4, stride=4, out=p, ld=576, B=2, tokens=5, pages=3, page=16, dtype=_lib.BF16):
        return lib.fp8k_mla_gather_cache(cache, p, stride, width, p, None, None, out, ld, B, tokens, pages, page, dtype, 0, None)

    assert gather(B=0) == 0 and gather(tokens=0, out=None) == 0
    _refused(gather(dtype=_lib.F32), "Half or BFloat16")
    _refused(gather(pages=0), "page table")
    _refused(gather(width=0), "page table")
    _refused(gather(stride=-4), "page table")
    _refused(gather(ld=580), "16-byte")
    _refused(gather(cache=None), "null")
    _refused(gather(tokens=1 << 31), "sizes")
    del keep


def test_c_refusals_of_the_attentions():
    from sglang_amd import _lib

    lib = _lib.lib
    keep, p = _address()

    def decode(q=p, qs=(512, 512, 512), ps=(64, 64, 64), table_stride=4, width=4, B=2, n=1, H=1, pages=3, page=16, scale=0.1, dtype=_lib.BF16, ws=p,
               ws_bytes=None):
        need = lib.fp8k_mla_decode_workspace_bytes(B, n, H, width * page)
        return lib.fp8k_mla_decode(q, *qs, p, *ps, p, p, table_stride, width, p, None, p, None, B, n, H, pages, page, scale, dtype, 0, ws,
                                   need if ws_bytes is None else ws_bytes, None)

    assert decode(B=0, q=None) == 0
    _refused(decode(dtype=_lib.F32), "Half or BFloat16")
    _refused(decode(q=None), "null")
    _refused(decode(q=p + 8), "16-byte")
    _refused(decode(qs=(512, 512, 516)), "16-byte")
    _refused(decode(ps=(64, -64, 64)), "negative")
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        _refused(decode(scale=bad), "positive")
    _refused(decode(B=65536), "sizes")
    _refused(decode(n=0), "sizes")
    _refused(decode(n=513, H=128), "sizes")
    _refused(decode(pages=0), "page table")
    _refused(decode(width=0), "page table")
    _refused(decode(width=1 << 20, page=1 << 12, ws_bytes=1 << 50), "2^30")
    _refused(decode(ws=None), "workspace")
    _refused(decode(ws_bytes=16), "workspace")
    _refused(decode(ws=p + 128), "workspace")
    assert lib.fp8k_mla_decode_workspace_bytes(0, 1, 16, 64) == 0

    def prefill(q=p, k=p, strides=(192, 192, 256, 256, 64, 256, 256), B=1, H=1, Tq=4, Tk=4, most=4, scale=0.1, dtype=_lib.BF16, ws=None):
        s = strides
        return lib.fp8k_mla_prefill(q, s[0], s[1], k, s[2], s[3], p, s[4], p, s[5], s[6], p, p, p, None, B, H, Tq, Tk, most, scale, 1, dtype, ws, 1 << 20, None)

    assert prefill(B=0) == 0 and prefill(Tq=0) == 0 and prefill(most=0) == 0
    _refused(prefill(dtype=_lib.F32), "Half or BFloat16")
    _refused(prefill(q=None), "null")
    _refused(prefill(k=None), "null")
    _refused(prefill(strides=(192, 192, 256, 256, 60, 256, 256)), "16-byte")
    _refused(prefill(strides=(192, 192, 256, -256, 64, 256, 256)), "negative")
    _refused(prefill(scale=0.0), "positive")
    _refused(prefill(most=-1), "sizes")
    _refused(prefill(strides=(192, 192, 1 << 25, 256, 64, 256, 256)), "further apart")
    _refused(prefill(Tk=1 << 16), "workspace")
    _refused(prefill(Tk=1 << 16, ws=p + 8), "workspace")
    assert lib.fp8k_mla_prefill_workspace_bytes(1, 1, 4, 64, 4) == 0 and lib.fp8k_mla_prefill_workspace_bytes(1, 1, 4, 1 << 16, 4) > 0
    _refused(prefill(B=1 << 23, H=1 << 16, Tq=1 << 30, most=1 << 30), "blocks")

    def merge(a=p, rows=4, D=128, dtype=_lib.BF16):
        return lib.fp8k_merge_attention_states(a, p, p, p, p, p, rows, D, dtype, None)

    assert merge(rows=0) == 0
    _refused(merge(D=12), "multiple of 8")
    _refused(merge(D=0), "multiple of 8")
    _refused(merge(a=None), "null")
    _refused(merge(a=p + 8), "16-byte")
    _refused(merge(dtype=9), "expected")
    del keep


def _empty(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_python_refusals():
    from sglang_amd import sgl_kernel as K

    with FakeTensorMode():
        cache, table = _empty(5, 16, 576), _empty(2, 3, dtype=I32)

        def refused(words, fn, good, **changed):
            with pytest.raises(RuntimeError, match=words):
                fn(**{**good, **changed})

        write = dict(latent=_empty(4, 576), cache=cache, slots=_empty(4, dtype=I64), norm_weight=None, eps=1e-6, cos_sin=_empty(9, 64, dtype=F32),
                     positions=_empty(4, dtype=I64), neox=False, q_pe=_empty(4, 2, 64), q_out=_empty(4, 2, 64), scale=None)
        refused("latent", K.mla_write_cache, write, latent=_empty(4, 512))
        refused("latent", K.mla_write_cache, write, latent=_empty(4, 576, dtype=F32))
        refused("latent", K.mla_write_cache, write, latent=_empty(576, 4).t())
        refused("operands' type", K.mla_write_cache, write, cache=_empty(5, 16, 576, dtype=F16))
        refused("cache must", K.mla_write_cache, write, cache=_empty(5, 16, 640)[..., :576])
        refused("cache must", K.mla_write_cache, write, cache=_empty(80, 576))
        refused("slots", K.mla_write_cache, write, slots=_empty(5, dtype=I64))
        refused("slots", K.mla_write_cache, write, slots=_empty(4, dtype=F32))
        refused("norm_weight", K.mla_write_cache, write, norm_weight=_empty(512, dtype=F16))
        refused("norm_weight", K.mla_write_cache, write, norm_weight=_empty(576))
        refused("cos_sin", K.mla_write_cache, write, cos_sin=_empty(9, 64))
        refused("cos_sin", K.mla_write_cache, write, cos_sin=_empty(0, 64, dtype=F32))
        refused("need cos_sin", K.mla_write_cache, write, cos_sin=None)
        refused("needs positions", K.mla_write_cache, write, positions=None)
        refused("q_pe", K.mla_write_cache, write, q_pe=_empty(3, 2, 64))
        refused("q_out", K.mla_write_cache, write, q_out=None)
        refused("q_out needs", K.mla_write_cache, write, q_pe=None)
        refused("scale", K.mla_write_cache, write, scale=_empty(1, dtype=F32))
        refused("scale", K.mla_write_cache, write, cache=_empty(5, 16, 576, dtype=F8), scale=_empty(2, dtype=F32))
        refused("must live on the GPU", K.mla_write_cache, write, latent=torch.empty((4, 576), dtype=BF16))

        gather = dict(cache=cache, page_table=table, cu_seqlens=_empty(3, dtype=I32), starts=None, scale=None, out=_empty(9, 576))
        refused("out must", K.mla_gather_cache, gather, out=_empty(9, 512))
        refused("operands' type", K.mla_gather_cache, gather, out=_empty(9, 576, dtype=F16))
        refused("cu_seqlens", K.mla_gather_cache, gather, cu_seqlens=_empty(3, dtype=I64))
        refused("page_table", K.mla_gather_cache, gather, cu_seqlens=_empty(4, dtype=I32))
        refused("starts", K.mla_gather_cache, gather, starts=_empty(3, dtype=I32))
        refused("without pages", K.mla_gather_cache, gather, page_table=table[:, :0])

        decode = dict(q_nope=_empty(2, 1, 8, 512), q_pe=_empty(2, 1, 8, 64), cache=cache, page_table=table, seq_lens=_empty(2, dtype=I32), sm_scale=0.1,
                      scale=None, out=_empty(2, 1, 8, 512), lse=None)
        refused("q_nope", K.mla_decode_attention, decode, q_nope=_empty(2, 8, 512))
        refused("q_nope", K.mla_decode_attention, decode, q_nope=_empty(2, 1, 8, 512, dtype=F32))
        refused("q_pe", K.mla_decode_attention, decode, q_pe=_empty(2, 1, 4, 64))
        refused("operands' type", K.mla_decode_attention, decode, cache=_empty(5, 16, 576, dtype=torch.float8_e5m2))
        refused("page_table", K.mla_decode_attention, decode, page_table=_empty(2, 3, dtype=I64))
        refused("page_table", K.mla_decode_attention, decode, page_table=_empty(3, 3, dtype=I32))
        refused("seq_lens", K.mla_decode_attention, decode, seq_lens=_empty(2, dtype=I64))
        refused("out must", K.mla_decode_attention, decode, out=_empty(2, 1, 512, 8).transpose(2, 3))
        refused("lse", K.mla_decode_attention, decode, lse=_empty(2, 1, 8))
        for bad in (0.0, -0.1, float("inf"), float("nan")):
            refused("sm_scale", K.mla_decode_attention, decode, sm_scale=bad)

        prefill = dict(q=_empty(6, 2, 192), k_nope=_empty(7, 2, 128), k_pe=_empty(7, 64), v=_empty(7, 2, 128), cu_seqlens_q=_empty(3, dtype=I32),
                       cu_seqlens_k=_empty(3, dtype=I32), max_seqlen_q=4, sm_scale=0.1, causal=True, out=_empty(6, 2, 128), lse=None)
        refused("q must", K.mla_prefill_attention, prefill, q=_empty(6, 2, 128))
        refused("one type", K.mla_prefill_attention, prefill, v=_empty(7, 2, 128, dtype=F16))
        refused("k_nope and v", K.mla_prefill_attention, prefill, v=_empty(7, 1, 128))
        refused("k_nope and v", K.mla_prefill_attention, prefill, k_pe=_empty(6, 64))
        refused("cu_seqlens_k", K.mla_prefill_attention, prefill, cu_seqlens_k=_empty(4, dtype=I32))
        refused("cu_seqlens_q", K.mla_prefill_attention, prefill, cu_seqlens_q=_empty(0, dtype=I32))
        refused("max_seqlen_q", K.mla_prefill_attention, prefill, max_seqlen_q=-1)
        refused("sm_scale", K.mla_prefill_attention, prefill, sm_scale=0.0)
        refused("out must", K.mla_prefill_attention, prefill, out=_empty(6, 2, 192))
        refused("lse", K.mla_prefill_attention, prefill, lse=_empty(6, dtype=F32))

        merge = dict(out_a=_empty(3, 2, 128), lse_a=_empty(3, 2, dtype=F32), out_b=_empty(3, 2, 128), lse_b=_empty(3, 2, dtype=F32), out=_empty(3, 2, 128),
                     lse=_empty(3, 2, dtype=F32))
        refused("one type", K.merge_attention_states, merge, out_b=_empty(3, 2, 128, dtype=F16))
        refused("lse_a", K.merge_attention_states, merge, lse_b=_empty(3, 2))
        refused("multiple of 8", K.merge_attention_states, merge, **{k: _empty(3, 2, 12) for k in ("out_a", "out_b", "out")})
        refused("float32, float16", K.merge_attention_states, merge, out_a=_empty(3, 2, 128, dtype=torch.float64))


def test_fake_shapes():
    from sglang_amd import mla

    with FakeTensorMode():
        cache, table, lens = _empty(5, 16, 576, dtype=F8), _empty(2, 3, dtype=I32), _empty(2, dtype=I32)
        scale = _empty(1, dtype=F32)
        q = mla.mla_write_cache(_empty(4, 576), cache, _empty(4, dtype=I64), cos_sin=_empty(9, 64, dtype=F32), positions=_empty(4, dtype=I64),
                                q_pe=_empty(4, 2, 192)[..., 128:], scale=scale)
        assert q.shape == (4, 2, 64) and q.is_contiguous() and q.dtype == BF16
        assert mla.mla_write_cache(_empty(4, 576), cache, _empty(4, dtype=I64)) is None
        assert mla.mla_gather_cache(cache, table, _empty(3, dtype=I32), 7, dtype=F16, scale=scale).shape == (7, 576)
        o, s = mla.mla_decode_attention(_empty(2, 8, 512), _empty(2, 8, 64), cache, table, lens, 0.1, scale=scale, return_lse=True)
        assert o.shape == (2, 8, 512) and s.shape == (2, 8) and s.dtype == F32
        o, s = mla.mla_decode_attention(_empty(2, 3, 8, 512), _empty(2, 3, 8, 64), cache, table, lens, 0.1, return_lse=True)
        assert o.shape == (2, 3, 8, 512) and s.shape == (2, 3, 8)
        o, s = mla.mla_prefill_attention(_empty(6, 2, 192), _empty(7, 2, 128), _empty(7, 1, 64), _empty(7, 2, 128), lens, lens, 6, 0.1, return_lse=True)
        assert o.shape == (6, 2, 128) and s.shape == (6, 2)
        o, s = mla.merge_attention_states(o, s, o, s)
        assert o.shape == (6, 2, 128) and s.shape == (6, 2)


def test_reference_is_attention():
    """The float64 definition against torch's softmax, log-sum-exp and their derivative: d lse / d q = scale * softmax . k, by differences."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 32), (9, 32), (9, 8)))
    limit = torch.tensor([0, 1, 4, 9, 12])
    out, lse, tol, _ = R.softmax_rows(q, k, v, 0.3, limit, BF16)
    for i, n in enumerate(limit.tolist()):
        n = min(n, 9)
        if n == 0:
            assert not out[i].any() and lse[i] == float("-inf")
            continue
        s = q[i] @ k[:n].t() * 0.3
        assert torch.allclose(out[i], torch.softmax(s, 0) @ v[:n]) and torch.allclose(lse[i], torch.logsumexp(s, 0))
        step = 1e-6
        up = R.softmax_rows(q + step * torch.eye(5, 32, dtype=torch.float64), k, v, 0.3, limit, BF16)[1]
        assert abs((up[i] - lse[i]) / step - 0.3 * (torch.softmax(s, 0) @ k[:n])[i]) < 1e-5
    assert bool((tol >= R.half_step(BF16) * out.abs()).all())
    x, cs = torch.randn((3, 64), generator=g, dtype=torch.float64), torch.randn((3, 32), generator=g, dtype=torch.float64)
    table = torch.cat((cs.cos(), cs.sin()), 1)
    pairs = torch.view_as_complex(x.view(3, 32, 2)) * torch.polar(torch.ones_like(cs), cs)
    assert torch.allclose(R.rotate(x, table, False)[0], torch.view_as_real(pairs).reshape(3, 64))
    halves = torch.complex(x[:, :32], x[:, 32:]) * torch.polar(torch.ones_like(cs), cs)
    assert torch.allclose(R.rotate(x, table, True)[0], torch.cat((halves.real, halves.imag), 1))


def test_the_joined_logarithm_is_memory_of_its_own():
    """A row's numbers may be several workgroups', which all read both logarithms: none may be overwritten."""
    from sglang_amd import _lib

    keep, p = _address()
    merge = _lib.lib.fp8k_merge_attention_states
    _refused(merge(p, p + 1024, p, p + 2048, p, p + 1024, 2, 192, _lib.BF16, None), "memory of its own")
    _refused(merge(p, p + 1024, p, p + 2048, p, p + 2048, 2, 192, _lib.BF16, None), "memory of its own")
    del keep


def test_places_of_rotated_queries_do_not_overlap():
    """An expanded or otherwise overlapping output of the writer is refused."""
    from sglang_amd import _lib

    keep, p = _address()

    def write(ot, oh, T=4, H=3):
        return _lib.lib.fp8k_mla_write_cache(p, 576, p, p, 1, None, 0, 1e-6, p, 10, p, 1, 0, p, 192, 64, p, ot, oh, None, T, H, 100, _lib.BF16, 0, None)

    for ot, oh in ((0, 64), (64, 64), (192, 0), (128, 64), (64, 192), (184, 64), (32, 256)):
        _refused(write(ot, oh), "overlap")
    _refused(write(0, 64, H=1), "overlap")
    _refused(write(192, 0, T=1), "overlap")
    del keep
