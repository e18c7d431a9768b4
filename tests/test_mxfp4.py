"""MXFP4 without a GPU: the oracle against the format's definition, scale layouts, refusals, and the shapes that tracing sees."""
import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import mxfp4_oracle as O
from sglang_amd import _host, _lib, custom_ops, mxfp4, sgl_kernel


def test_oracle_rounds_to_nearest_even():
    v = np.array([0.0, 0.25, 0.2500001, 0.75, 0.7499999, 1.25, 1.26, 1.75, 1.74, 2.5, 2.51, 3.5, 3.49, 5.0, 5.01, 6.9, 100.0])
    want = [0, 0, 0.5, 1, 0.5, 1, 1.5, 2, 1.5, 2, 3, 4, 3, 4, 6, 6, 6]
    assert O.decode(O.encode(v)).tolist() == want
    assert O.decode(O.encode(-v)).tolist() == [-w for w in want]


def test_oracle_scale_is_that_of_the_rounded_maximum():
    # 1 .. 1.74 round to binade 1, 1.75 and above to the next one; 2 less for the codes' own exponent
    for a, e in ((1.0, 0), (1.7499, 0), (1.75, 1), (2.0, 1), (0.0, -1000), (2.0**-126, -126), (2.0**-140, -140), (3.0e38, 127), (np.inf, None)):
        assert O.scale_byte(np.array([a]))[0] == (255 if e is None else max(e - 2 + 127, 0))


def test_oracle_packs_and_unpacks():
    code = np.random.default_rng(0).integers(0, 16, (3, 64)).astype(np.uint8)
    assert np.array_equal(O.unpack(O.pack(code)), code) and O.pack(code)[0, 0] == code[0, 0] + 16 * code[0, 1]


@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (4, 4), (7, 9), (2, 5, 3)])
def test_scale_words(shape):
    gen = torch.Generator().manual_seed(1)
    byte = torch.randint(0, 256, shape, generator=gen).to(torch.uint8)
    words = mxfp4.pack_mxfp4_scales(byte)
    rows, blocks = shape[-2:]
    assert words.shape == shape[:-1] + ((blocks + 3) // 4,) and words.stride()[-2:] == (1, (rows + 3) // 4 * 4)
    for j in range(blocks):  # byte j % 4 of word j / 4
        assert torch.equal((words[..., j // 4] >> (8 * (j % 4))) & 255, byte[..., j].int())
    if blocks % 4:
        assert not ((words[..., -1].long() & 0xFFFFFFFF) >> (8 * (blocks % 4))).any()
    assert torch.equal(mxfp4.unpack_mxfp4_scales(words, blocks * 32), byte)
    made = mxfp4.create_mxfp4_scales(shape[:-1] + (blocks * 32,), "cpu")
    assert made.shape == words.shape and made.stride() == words.stride()
    with pytest.raises(RuntimeError):
        mxfp4.pack_mxfp4_scales(byte.int())
    with pytest.raises(RuntimeError):
        mxfp4.unpack_mxfp4_scales(words, blocks * 32 + 16)


def test_native_calls_decline_host_memory():
    x, q, s = torch.zeros((4, 128), dtype=torch.bfloat16), torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 1), dtype=torch.int32)
    assert _host.mx_quant(x, False) is None
    assert _host.mx_dequant(q, s, torch.bfloat16) is None
    assert _host.mx_matmul(q, q, s, s, torch.bfloat16, None) is None
    assert _host.mx_linear(x, q, s, None) is None
    assert _host.mx_experts(x, q[None], q[None], torch.zeros(4, 2), torch.zeros((4, 2), dtype=torch.int32), s[None], s[None], False, False,
                            1.0, False) is None


def test_host_tensors_are_refused():
    x, q, s = torch.zeros((4, 128), dtype=torch.bfloat16), torch.zeros((8, 64), dtype=torch.uint8), torch.zeros((8, 1), dtype=torch.int32)
    for fn in (lambda: sgl_kernel.mxfp4_quant(x, q[:4], s[:4]), lambda: sgl_kernel.mxfp4_dequant(q, s, torch.empty((8, 128))),
               lambda: sgl_kernel.mxfp4_scaled_mm(q, q, s, s, torch.bfloat16)):
        with pytest.raises(RuntimeError, match="GPU"):
            fn()


@pytest.fixture
def mem():
    buf = ctypes.create_string_buffer(8192)
    yield (ctypes.addressof(buf) + 255) // 256 * 256
    del buf


def _refused(rc, text):
    assert rc != 0 and text in _lib.lib.fp8k_last_error(), (rc, _lib.lib.fp8k_last_error())


def test_quant_arguments(mem):
    f, p, B = _lib.lib.fp8k_mxfp4_quant, mem, _lib.BF16
    _refused(f(p, p, p, 4, 100, 104, 1, 4, B, 0, None), b"multiple of 32")
    _refused(f(p, p, p, 4, 0, 8, 1, 4, B, 0, None), b"multiple of 32")
    _refused(f(p, p, p, 4, 128, 128, 1, 4, 9, 0, None), b"bfloat16")
    _refused(f(None, p, p, 4, 128, 128, 1, 4, B, 0, None), b"null")
    _refused(f(p, p, None, 4, 128, 128, 1, 4, B, 0, None), b"scales")
    _refused(f(p + 2, p, p, 4, 128, 128, 1, 4, B, 0, None), b"aligned")
    _refused(f(p, p, p, 4, 128, 132, 1, 4, B, 0, None), b"row stride")
    _refused(f(p, p, p, 4, 128, 64, 1, 4, B, 0, None), b"row stride")
    _refused(f(p, p, p, 4, 128, 128, 1, 4, B, 1, None), b"row stride")  # the fused form reads rows of 2 K
    _refused(f(p, p, p, 4, 128, 128, 0, 4, B, 0, None), b"strides")
    _refused(f(p, p, p, 4, 128, 128, -1, 4, B, 0, None), b"strides")
    _refused(f(p, p, p, 1 << 20, 128, 128, 1, 4, B, 0, None), b"too many")
    assert f(None, None, None, 0, 128, 128, 1, 4, B, 0, None) == 0


def test_dequant_arguments(mem):
    f, p = _lib.lib.fp8k_mxfp4_dequant, mem
    _refused(f(p, p, p, 1, 4, 100, 0, 1, 4, _lib.BF16, None), b"multiple of 32")
    _refused(f(p, p, p, 1, 4, 128, 0, 1, 4, 7, None), b"bfloat16")
    _refused(f(p + 4, p, p, 1, 4, 128, 0, 1, 4, _lib.BF16, None), b"aligned")
    _refused(f(p, p, None, 1, 4, 128, 0, 1, 4, _lib.BF16, None), b"aligned")
    _refused(f(p, p, p, 1, 4, 128, 0, -1, 4, _lib.BF16, None), b"strides")
    _refused(f(p, p, p, 1, 4, 128, -1, 1, 4, _lib.BF16, None), b"strides")
    _refused(f(p, p, p, 70000, 4, 128, 0, 1, 4, _lib.BF16, None), b"too large")
    _refused(f(p, p, p, 1, 1 << 20, 128, 0, 1, 1 << 20, _lib.BF16, None), b"too large")
    assert f(None, None, None, 0, 4, 128, 0, 1, 4, _lib.BF16, None) == 0


def test_gemm_arguments(mem):
    p, B, F = mem, _lib.BF16, _lib.F32

    def f(A=p, Bq=p, As=p, Bs=p, bias=None, C=p, M=4, N=16, K=128, lda=64, ldb=64, am=1, aw=4, bn=1, bw=16, ldc=16, dt=B, bdt=F):
        return _lib.lib.fp8k_mxfp4_gemm(A, Bq, As, Bs, bias, C, M, N, K, lda, ldb, am, aw, bn, bw, ldc, dt, bdt, None)

    for kw, text in (({"K": 80, "lda": 48, "ldb": 48}, b"multiple of 32"), ({"N": 12}, b"16 bytes"), ({"dt": F}, b"Half or BFloat16"),
                     ({"lda": 56}, b"16-byte"), ({"ldb": 72}, b"16-byte"), ({"lda": 48}, b"16-byte"), ({"A": p + 8}, b"16-byte"),
                     ({"Bq": p + 8}, b"16-byte"), ({"A": None}, b"16-byte"), ({"C": None}, b"null"), ({"As": None}, b"scales"), ({"Bs": p + 2}, b"scales"),
                     ({"am": -1}, b"strides"), ({"bw": 1 << 60}, b"strides"), ({"bias": p, "bdt": _lib.F16}, b"bias"), ({"ldc": 8}, b"8-byte"),
                     ({"ldc": 18}, b"8-byte"), ({"M": -1}, b"sizes")):
        _refused(f(**kw), text)
    assert f(M=0, A=None, C=None) == 0
    lin = _lib.lib.fp8k_mxfp4_linear
    need = _lib.lib.fp8k_mxfp4_linear_workspace_bytes(300, 16, 128)
    assert need >= 300 * 64 + 300 * 4
    _refused(lin(p, p, p, None, p, 300, 16, 128, 128, 64, 1, 16, 16, B, F, None, 0, None), b"workspace")
    _refused(lin(p, p, p, None, p, 300, 16, 128, 128, 64, 1, 16, 16, B, F, p, need - 1, None), b"workspace")
    _refused(lin(p, p, p, None, p, 300, 16, 128, 128, 64, 1, 16, 16, B, F, p + 16, need, None), b"workspace")
    _refused(lin(p, p, p, None, p, 300, 16, 128, 100, 64, 1, 16, 16, B, F, p, need, None), b"row stride")
    # the scale words of the activations are addressed in 32 bits
    _refused(lin(p, p, p, None, p, 1 << 17, 16, 1 << 20, 1 << 20, 1 << 19, 1, 16, 16, B, F, p, 1 << 60, None), b"too many activations")


def test_experts_arguments(mem):
    p, B = mem, _lib.BF16

    def f(x=p, w1=p, w2=p, s1=p, s2=p, tw=p, ids=p, out=p, T=2, topk=2, E=2, H=64, I=32, ldx=64, act=0, dt=B, ws=p, n=1 << 20, w1e=64 * 32, s1n=1):
        return _lib.lib.fp8k_mxfp4_experts(x, w1, w2, s1, s2, tw, ids, 0, out, T, topk, E, H, I, ldx, w1e, 64 * 16, 64, s1n, 64, 64, 1, 64, act,
                                           0, 1.0, dt, ws, n, None)

    for kw, text in (({"H": 40, "ldx": 40}, b"multiples of 32"), ({"I": 48}, b"multiples of 32"), ({"T": 129}, b"at most 128"),
                     ({"T": 128, "topk": 9}, b"1024"), ({"dt": _lib.F32}, b"Half or BFloat16"), ({"act": 2}, b"silu or gelu"), ({"x": None}, b"null"),
                     ({"ids": None}, b"null"), ({"x": p + 2}, b"16-byte"), ({"ldx": 60}, b"16-byte"), ({"w1e": 8}, b"16-byte"), ({"s1n": -1}, b"strides"),
                     ({"ws": None}, b"workspace"), ({"n": 100}, b"workspace"), ({"ws": p + 64}, b"workspace"), ({"E": 0}, b"sizes"), ({"topk": 0}, b"sizes")):
        _refused(f(**kw), text)
    assert f(T=0, x=None) == 0


def test_fake_tensors_have_the_shapes():
    with FakeTensorMode():
        x = torch.empty((6, 256), dtype=torch.bfloat16, device="cuda")
        w, s = torch.empty((64, 128), dtype=torch.uint8, device="cuda"), mxfp4.create_mxfp4_scales((64, 256), "cuda")
        assert custom_ops.mxfp4_scaled_mm(torch.empty((6, 128), dtype=torch.uint8, device="cuda"), w, s[:6], s, torch.float16).shape == (6, 64)
        q, qs = mxfp4.per_token_group_quant_mxfp4(x)
        assert q.shape == (6, 128) and qs.shape == (6, 2) and qs.stride() == (1, 8)
        q, qs = mxfp4.per_token_group_quant_mxfp4(x, fuse_silu_and_mul=True)
        assert q.shape == (6, 64) and qs.shape == (6, 1)
        assert mxfp4.w4a4_mxfp4_linear(x.view(2, 3, 256), w, s).shape == (2, 3, 64)
        assert mxfp4.mxfp4_dequant(w, s, torch.float32).shape == (64, 256)
        e1, e2 = torch.empty((4, 64, 128), dtype=torch.uint8, device="cuda"), torch.empty((4, 256, 16), dtype=torch.uint8, device="cuda")
        out = mxfp4.fused_experts_mxfp4(x, e1, e2, torch.empty((6, 2), device="cuda"), torch.empty((6, 2), dtype=torch.int32, device="cuda"),
                                        mxfp4.create_mxfp4_scales((4, 64, 256), "cuda"), mxfp4.create_mxfp4_scales((4, 256, 32), "cuda"))
        assert out.shape == (6, 256) and out.dtype == torch.bfloat16
