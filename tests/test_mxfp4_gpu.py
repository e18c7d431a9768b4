"""MXFP4 quantisation, products and linears on the GPU against the float64 oracle.

Products are compared bit for bit: the operands' values are multiples of a power of two and the sum of the magnitudes of a result's terms
stays under 2^24 of the product's step, so that float32 sums are exact in any order and only the last rounding is left."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as O
from sglang_amd import mxfp4, sgl_kernel

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = [torch.bfloat16, torch.float16]


def _np(t):
    return t.detach().double().cpu().numpy()


def _unpacked(q, s):
    """codes and scale bytes of a device pair, as the oracle has them"""
    k = q.shape[-1] * 2
    return O.unpack(q.cpu().numpy()), mxfp4.unpack_mxfp4_scales(s.cpu(), k).numpy()


def _check_quant(x, q, s, fused=False):
    ref_code, ref_byte = O.quant(_np(x))
    code, byte = _unpacked(q, s)
    np.testing.assert_array_equal(byte, ref_byte)
    np.testing.assert_array_equal(code, ref_code)


def _activations(shape, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    return torch.where(torch.rand(shape, generator=gen) < 0.02, x * 30, x).to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 32), (3, 64), (4, 128), (5, 160), (17, 512), (33, 544), (130, 1056), (2, 7168)])
def test_quant_is_the_definition(dev, m, k, dtype):
    x = _activations((m, k), dtype, m + k)
    x[m // 2, :32] = 0
    q, s = mxfp4.per_token_group_quant_mxfp4(x)
    assert q.shape == (m, k // 2) and s.shape == (m, (k + 127) // 128) and s.stride() == (1, (m + 3) // 4 * 4)
    _check_quant(x, q, s)
    # bytes that no block has are zero
    if k % 128:
        assert not ((s[:, -1].long() & 0xFFFFFFFF) >> (8 * (k % 128 // 32))).any()


@pytest.mark.parametrize("dtype", HALF)
def test_quant_of_every_16_bit_value(dev, dtype):
    """Every bit pattern, in blocks of neighbours (subnormals, infinities, NaN) and in blocks of mixed magnitudes."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(torch.int16)
    for order in (torch.arange(65536), (torch.arange(65536) * 40503) % 65536):
        x = bits[order].view(64, 1024).view(dtype).cuda()
        _check_quant(x, *mxfp4.per_token_group_quant_mxfp4(x))


def test_quant_of_float32_bit_patterns(dev):
    gen = torch.Generator().manual_seed(3)
    exponent = torch.randint(0, 256, (64, 32, 1), generator=gen)
    near = (exponent + torch.randint(-3, 1, (64, 32, 32), generator=gen)).clamp(0, 255)
    # fractions that end in ties as often as not
    fraction = torch.randint(0, 8, near.shape, generator=gen) << 20
    fraction += torch.where(torch.rand(near.shape, generator=gen) < 0.5, torch.randint(0, 1 << 20, near.shape, generator=gen), 0)
    sign = torch.randint(0, 2, near.shape, generator=gen)
    x = ((sign << 31) | (near << 23) | fraction).to(torch.int64).numpy().astype(np.uint32).view(np.float32).reshape(64, 1024)
    t = torch.from_numpy(x).cuda()
    _check_quant(t, *mxfp4.per_token_group_quant_mxfp4(t))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 32), (6, 96), (19, 640), (64, 1056)])
def test_fused_silu_and_mul(dev, dtype, m, k):
    """silu(gate) * up in float32: the device's exponential and reciprocal are within 2^-20, so a code may differ from the oracle's only
    where the value is that near to the middle between two codes, and a scale only where the maximum is that near to 1.75 of a binade."""
    x = _activations((m, 2 * k), dtype, m)
    q, s = mxfp4.per_token_group_quant_mxfp4(x, fuse_silu_and_mul=True)
    v = _np(x)
    v = O.act(v[:, :k], "silu") * v[:, k:]
    code, byte = _unpacked(q, s)
    lo, hi = O.quant(v * (1 - 2.0**-20)), O.quant(v * (1 + 2.0**-20))
    assert ((byte == lo[1]) | (byte == hi[1])).all()
    settled = np.repeat((lo[1] == hi[1]), 32, axis=1)
    assert settled.mean() > 0.9
    small = np.minimum(O.decode(lo[0]), O.decode(hi[0])), np.maximum(O.decode(lo[0]), O.decode(hi[0]))
    got = O.decode(code)
    assert ((got >= small[0]) & (got <= small[1]) | ~settled).all()


def test_quant_of_strided_rows_leaves_the_rest(dev):
    wide = _activations((9, 512), torch.bfloat16)
    x = wide[:, 64:64 + 160]  # rows 1024 bytes apart, 128 bytes in
    words = torch.full((2, 12), -7, dtype=torch.int32, device=dev)
    q = torch.empty((9, 80), dtype=torch.uint8, device=dev)
    sgl_kernel.mxfp4_quant(x, q, words.t()[:9])
    _check_quant(x, q, words.t()[:9])
    assert (words[:, 9:] == -7).all()
    row_major = torch.empty((9, 2), dtype=torch.int32, device=dev)
    sgl_kernel.mxfp4_quant(x, q, row_major)
    assert torch.equal(row_major, words.t()[:9])
    odd = wide[:, 3:3 + 160]  # not 16-byte aligned: the layer-level call makes it so, the op refuses it
    _check_quant(odd, *mxfp4.per_token_group_quant_mxfp4(odd))
    with pytest.raises(RuntimeError, match="aligned"):
        sgl_kernel.mxfp4_quant(odd, q, row_major)
    _check_quant(x.t().contiguous().t(), *mxfp4.per_token_group_quant_mxfp4(x.t().contiguous().t()))


@pytest.mark.parametrize("dtype", TYPES)
def test_dequant_is_exact(dev, dtype):
    """Every code with every scale byte; one rounding to the output type (bfloat16 and float32 need none above the subnormals)."""
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 4))
    byte = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 2, axis=1)
    q, s = torch.from_numpy(O.pack(code)).cuda(), mxfp4.pack_mxfp4_scales(torch.from_numpy(byte)).cuda()
    got = mxfp4.mxfp4_dequant(q, s, dtype)
    want = torch.from_numpy(O.values(code, byte)).to(torch.float32).to(dtype)
    assert torch.equal(got.cpu().nan_to_num(nan=77.0), want.nan_to_num(nan=77.0)) and torch.equal(got.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("e,n,k", [(1, 1, 32), (3, 7, 160), (2, 18, 1024), (5, 4, 544)])
def test_dequant_of_stacks_and_weights(dev, e, n, k):
    w = _activations((e, n, k), torch.bfloat16)
    q, s = mxfp4.quant_weight_mxfp4(w)
    one = [mxfp4.quant_weight_mxfp4(w[i]) for i in range(e)]
    assert all(torch.equal(q[i], a) and torch.equal(s[i], b) for i, (a, b) in enumerate(one))
    got = mxfp4.mxfp4_dequant(q, s, torch.float32)
    np.testing.assert_array_equal(_np(got), O.values(*_unpacked(q, s)))
    assert torch.equal(mxfp4.mxfp4_dequant(q[0], s[0], torch.float32), got[0])
    assert torch.equal(mxfp4.mxfp4_dequant(q, s.contiguous(), torch.float32), got)  # row-major words


# ------------------------------------------------------------------------------------------------------------------ products


def _operand(rng, rows, k, device, row_major=False, spread=1):
    code = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    byte = rng.integers(127 - spread, 128 + spread, (rows, k // 32)).astype(np.uint8)
    q = torch.from_numpy(O.pack(code)).to(device)
    s = mxfp4.pack_mxfp4_scales(torch.from_numpy(byte)).to(device)
    return O.values(code, byte), q, s.contiguous() if row_major else s


def _rounded(v, dtype):
    return torch.from_numpy(v).to(torch.float32).to(dtype)


SHAPES = [(1, 8, 32), (1, 16, 128), (3, 24, 96), (16, 64, 256), (17, 40, 288), (31, 136, 512), (33, 264, 544), (48, 72, 1024), (64, 256, 800),
          (65, 128, 256), (100, 520, 1536), (128, 384, 2048), (129, 200, 640), (200, 1032, 1056), (256, 256, 4096), (300, 512, 288),
          (513, 776, 1312), (1, 4096, 4096), (8, 1000, 7168), (5, 8, 18432), (1000, 1096, 768), (2050, 2056, 512)]


@pytest.fixture
def plan():
    """Pins the kernel that products take."""
    from sglang_amd._lib import lib

    yield lib.fp8k_tune_force_mxfp4_plan
    lib.fp8k_tune_force_mxfp4_plan(-1)


def _exact(dev, m, n, k):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    for dtype, row_major in ((torch.bfloat16, False), (torch.float16, True)):
        spread = 1 if k <= 8192 else 0
        av, a, sa = _operand(rng, m, k, dev, row_major, spread)
        bv, b, sb = _operand(rng, n, k, dev, row_major, spread)
        sums = np.abs(av) @ np.abs(bv).T
        assert sums.max() < 2**24 * 0.25 * 4.0**-spread  # the premise: terms are multiples of 0.25 * 4^-spread
        ref = av @ bv.T
        got = mxfp4.w4a4_mxfp4_matmul(a, b, sa, sb, dtype)
        assert torch.equal(got.cpu(), _rounded(ref, dtype)), (m, n, k)
        for bias_type in (dtype, torch.float32):
            bias = torch.from_numpy(rng.integers(-64, 65, n) / 8.0).to(bias_type).to(dev)
            got = mxfp4.w4a4_mxfp4_matmul(a, b, sa, sb, dtype, bias=bias)
            assert torch.equal(got.cpu(), _rounded(ref + _np(bias), dtype)), (m, n, k, bias_type)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_is_exact(dev, m, n, k):
    _exact(dev, m, n, k)


@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (15, 72, 256), (64, 64, 288), (65, 72, 512), (127, 136, 736), (129, 264, 1024), (130, 256, 1280), (200, 520, 1568),
                                   (257, 248, 2048), (300, 1032, 2304), (520, 776, 4640)])
def test_every_kernel_is_exact(dev, plan, kind, m, n, k):
    """One, two, three .. K blocks, remainders of every unrolling, rows and columns around the edges of every tile."""
    plan(kind)
    _exact(dev, m, n, k)


@pytest.mark.parametrize("kind", range(1, 5))
@pytest.mark.parametrize("blocks", range(1, 12))
def test_operands_from_memory_arrive_in_time(dev, plan, kind, blocks):
    """Every count of K blocks with operands that no cache holds: a wait that lets a block's loads pass shows as rows of stale operands."""
    k, gen = blocks * 256, torch.Generator(device=dev).manual_seed(blocks)

    def operand(rows):
        q = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device=dev, generator=gen)
        byte = torch.randint(126, 128, (rows, k // 32), dtype=torch.uint8, device=dev, generator=gen)
        return q, mxfp4.pack_mxfp4_scales(byte)

    def values(q, s):
        return mxfp4.mxfp4_dequant(q, s, torch.float32)

    flush = torch.empty(1 << 27, dtype=torch.float32, device=dev)
    plan(kind)
    for _ in range(6):
        (a, sa), (b, sb) = operand(130), operand(1032)
        ref = (values(a, sa).double() @ values(b, sb).double().t()).bfloat16()  # terms are multiples of 1/16 and at most 36: float32 sums are exact
        for _ in range(3):
            flush.zero_()
            assert torch.equal(mxfp4.w4a4_mxfp4_matmul(a, b, sa, sb), ref)


@pytest.mark.parametrize("kind", range(5))
def test_every_kernel_stores_unaligned_rows(dev, plan, kind):
    """Rows of the result that start at multiples of 8 bytes only, through the C interface; what lies between them stays."""
    from sglang_amd import _lib

    rng = np.random.default_rng(kind)
    plan(kind)
    m, n, k = 150, 328, 544
    av, a, sa = _operand(rng, m, k, dev)
    bv, b, sb = _operand(rng, n, k, dev)
    wide = torch.full((m, n + 20), 7.0, dtype=torch.bfloat16, device=dev)
    out = wide[:, 4:4 + n]
    _lib.check(_lib.lib.fp8k_mxfp4_gemm(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), None, out.data_ptr(), m, n, k, k // 2, k // 2,
                                        sa.stride(0), sa.stride(1), sb.stride(0), sb.stride(1), n + 20, _lib.BF16, _lib.F32, _lib.stream_ptr(dev)))
    assert torch.equal(out.cpu(), _rounded(av @ bv.T, torch.bfloat16))
    assert (wide[:, :4] == 7).all() and (wide[:, 4 + n:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(4, 64, 512), (40, 128, 288), (300, 264, 1056), (520, 512, 800)])
def test_matmul_of_strided_operands(dev, m, n, k):
    rng = np.random.default_rng(5)
    av, a, sa = _operand(rng, m, k, dev)
    bv, b, sb = _operand(rng, n, k, dev)
    wide_a, wide_b = (torch.full((t.shape[0], k // 2 + 48), 0x77, dtype=torch.uint8, device=dev) for t in (a, b))
    wide_a[:, 16:16 + k // 2], wide_b[:, 32:32 + k // 2] = a, b
    words = torch.full((3 * sb.shape[1], 2 * n), -1, dtype=torch.int32, device=dev)  # what is not ours are NaN scales
    words[::3, ::2] = sb.t()
    got = mxfp4.w4a4_mxfp4_matmul(wide_a[:, 16:16 + k // 2], wide_b[:, 32:32 + k // 2], sa, words[::3, ::2].t(), torch.bfloat16)
    assert torch.equal(got.cpu(), _rounded(av @ bv.T, torch.bfloat16))
    # every second row of the activations
    got = mxfp4.w4a4_mxfp4_matmul(wide_a[::2, 16:16 + k // 2], b, sa[::2], sb, torch.bfloat16)
    assert torch.equal(got.cpu(), _rounded(av[::2] @ bv.T, torch.bfloat16))


@pytest.mark.parametrize("m", [2, 20, 70, 300, 600])
def test_nan_and_extreme_scales_stay_in_their_rows(dev, m):
    rng = np.random.default_rng(m)
    n, k = 72, 544
    av, a, sa = _operand(rng, m, k, dev)
    bv, b, sb = _operand(rng, n, k, dev)
    byte_a, byte_b = mxfp4.unpack_mxfp4_scales(sa, k), mxfp4.unpack_mxfp4_scales(sb, k)
    byte_a[1, 3], byte_b[5, 16] = 255, 255  # the last block of a row among them
    byte_a[0], byte_b[7] = 0, 254           # 2^-127 and 2^127 meet
    got = _np(mxfp4.w4a4_mxfp4_matmul(a, b, mxfp4.pack_mxfp4_scales(byte_a), mxfp4.pack_mxfp4_scales(byte_b), torch.bfloat16))
    nan = np.zeros((m, n), bool)
    nan[1], nan[:, 5] = True, True
    # column 7 has terms of up to 36 * 2^127 wherever the other scale is not 2^-127: beyond float32, infinities of both signs
    known = np.ones((m, n), bool)
    known[2:, 7] = False
    np.testing.assert_array_equal(np.isnan(got)[known], nan[known])
    rest = np.ones((m, n), bool)
    rest[:2], rest[:, 5], rest[:, 7] = False, False, False
    ref = _np(_rounded(av @ bv.T, torch.bfloat16))
    np.testing.assert_array_equal(got[rest], ref[rest])
    code_a, code_b = O.unpack(a[0].cpu().numpy()), O.unpack(b[7].cpu().numpy())
    want = float(O.decode(code_a) @ O.decode(code_b))  # exact: the scales' product is 1
    assert got[0, 7] == float(torch.tensor(want).to(torch.bfloat16))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k", [(1, 64, 96), (1, 512, 7168), (4, 264, 1056), (13, 1000, 2048), (16, 128, 288), (33, 512, 4096), (130, 136, 544),
                                   (700, 520, 1024)])
def test_linear_is_quant_and_matmul(dev, m, n, k, dtype):
    rng = np.random.default_rng(k)
    x = _activations((m, k), dtype, n)
    _, w, s = _operand(rng, n, k, dev)
    q, qs = mxfp4.per_token_group_quant_mxfp4(x)
    for bias in (None, _activations((n,), dtype), _activations((n,), torch.float32)):
        got = mxfp4.w4a4_mxfp4_linear(x, w, s, bias=bias)
        want = mxfp4.w4a4_mxfp4_matmul(q, w, qs, s, dtype, bias=bias)
        # sums of a few rows are added up in another order; terms below 2^-24 of the largest differ
        size = np.abs(O.values(*_unpacked(q, qs))) @ np.abs(O.values(*_unpacked(w, s))).T
        step = torch.finfo(dtype).eps * np.abs(_np(want)) + k * 2.0**-24 * size
        assert (np.abs(_np(got) - _np(want)) <= step).all()
        ref = O.values(*O.quant(_np(x))) @ O.values(*_unpacked(w, s)).T + (0 if bias is None else _np(bias))
        # half a step of the result's type, and float32 sums of k terms
        assert (np.abs(_np(got) - ref) <= torch.finfo(dtype).eps / 2 * np.abs(ref) * 1.01 + k * 2.0**-24 * size + 1e-7).all()


def test_linear_shapes_and_forms(dev):
    rng = np.random.default_rng(0)
    n, k = 136, 288
    _, w, s = _operand(rng, n, k, dev)
    x = _activations((2, 3, 5, k), torch.bfloat16)
    flat = mxfp4.w4a4_mxfp4_linear(x.view(-1, k), w, s)
    assert torch.equal(mxfp4.w4a4_mxfp4_linear(x, w, s), flat.view(2, 3, 5, n))
    assert torch.equal(mxfp4.w4a4_mxfp4_linear(x[0, 0, 0], w, s), flat[0]) or torch.allclose(mxfp4.w4a4_mxfp4_linear(x[0, 0, 0], w, s), flat[0], rtol=2**-6)
    assert mxfp4.w4a4_mxfp4_linear(x[:0], w, s).shape == (0, 3, 5, n)
    wide = _activations((7, 2 * k), torch.bfloat16)
    assert torch.equal(mxfp4.w4a4_mxfp4_linear(wide[:, :k], w, s), mxfp4.w4a4_mxfp4_linear(wide[:, :k].contiguous(), w, s))
    assert torch.equal(mxfp4.w4a4_mxfp4_linear(x.transpose(0, 2), w, s), mxfp4.w4a4_mxfp4_linear(x.transpose(0, 2).contiguous(), w, s))
    q, qs = mxfp4.per_token_group_quant_mxfp4(wide[:, :k])
    assert torch.equal(mxfp4.w4a4_mxfp4_linear(q, w, s, input_scale=qs), mxfp4.w4a4_mxfp4_matmul(q, w, qs, s, torch.bfloat16))
    for bad in (lambda: mxfp4.w4a4_mxfp4_linear(x.float(), w, s), lambda: mxfp4.w4a4_mxfp4_linear(x, w[:, :128], s),
                lambda: mxfp4.w4a4_mxfp4_linear(x, w, s[:64]), lambda: mxfp4.w4a4_mxfp4_linear(x, w[:12], s[:12]),
                lambda: mxfp4.w4a4_mxfp4_linear(x, w, s, bias=torch.zeros(n - 1, device=dev)), lambda: mxfp4.w4a4_mxfp4_linear(x, w, s.float()),
                lambda: mxfp4.w4a4_mxfp4_linear(x, w, s, input_scale=qs), lambda: mxfp4.w4a4_mxfp4_linear(x, w.cpu(), s)):
        with pytest.raises(RuntimeError):
            bad()


def test_native_calls_are_the_dispatcher_path(dev, monkeypatch):
    from sglang_amd import _host

    rng = np.random.default_rng(0)
    n, k = 264, 544
    _, w, s = _operand(rng, n, k, dev)
    x, bias = _activations((21, k), torch.float16), _activations((n,), torch.float16)
    q, qs = mxfp4.per_token_group_quant_mxfp4(x)
    calls = [lambda: mxfp4.per_token_group_quant_mxfp4(x), lambda: (mxfp4.mxfp4_dequant(w, s, torch.float16),),
             lambda: (mxfp4.w4a4_mxfp4_matmul(q, w, qs, s, torch.float16, bias=bias),)]
    native = [c() for c in calls]
    for name in ("mx_quant", "mx_dequant", "mx_matmul", "mx_linear"):
        assert hasattr(_host, name)
        monkeypatch.setattr(_host, name, lambda *a: None)
    for a, c in zip(native, calls):
        for t, u in zip(a, c()):
            assert t.stride() == u.stride() and torch.equal(t, u)
    assert torch.equal(mxfp4.w4a4_mxfp4_linear(x, w, s, bias=bias), native[2][0])


def _feed_forward(x, w):
    """up projections, silu_and_mul into the next quantisation, down projection"""
    a = mxfp4.w4a4_mxfp4_linear(x, *w["up"])
    q, s = mxfp4.per_token_group_quant_mxfp4(a, fuse_silu_and_mul=True)
    return mxfp4.w4a4_mxfp4_linear(q, *w["down"], input_scale=s)


@pytest.mark.parametrize("m", [1, 24, 200])
def test_feed_forward_captured_and_on_another_stream(dev, m):
    k, inter = 544, 288
    w = {"up": mxfp4.quant_weight_mxfp4(_activations((2 * inter, k), torch.bfloat16) * 0.05),
         "down": mxfp4.quant_weight_mxfp4(_activations((k, inter), torch.bfloat16) * 0.05)}
    xs = [_activations((m, k), torch.bfloat16, i) for i in range(4)]
    eager = [_feed_forward(x, w) for x in xs]
    # against float64 on what the 4-bit tensors stand for, quantising the same intermediate values
    a = mxfp4.w4a4_mxfp4_linear(xs[0], *w["up"])
    q, s = mxfp4.per_token_group_quant_mxfp4(a, fuse_silu_and_mul=True)
    ref = O.values(*_unpacked(q, s)) @ O.values(*_unpacked(*w["down"])).T
    size = np.abs(O.values(*_unpacked(q, s))) @ np.abs(O.values(*_unpacked(*w["down"]))).T
    assert (np.abs(_np(eager[0]) - ref) <= 1.01 * 2.0**-8 * np.abs(ref) + inter * 2.0**-24 * size).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [_feed_forward(x, w) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _feed_forward(static, w)
    for x, e in zip(xs, eager):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, e)
        assert torch.equal(_feed_forward(x, w), e)
