"""The expert layer on MXFP4 weights: as near to float64 as the rounding of its result in every form, and scales at the ends of their range.

The intermediate is held as a pair of bfloat16 numbers: the first is off by 2^-8 of it at most, the second by 2^-8 of that, so the pair by
2^-16.  Float32 sums of h (+ i) terms add (h + i) * 2^-24, the activation 2^-18.  The roundings of different terms are independent: in the
norm they add up like the terms themselves, whose sizes add up to under 32 times the result (checked), their squares' root to a few times it.
That is under a tenth of what the result's one rounding makes of the norm, some 0.4 of half a step (2^-8 or 2^-11), and with it within 1.1
of that rounding alone.  An intermediate of one 16-bit number would make it 1.4 times."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as O
from sglang_amd import mxfp4

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]


def _np(t):
    return t.double().cpu().numpy()


def _values(q, s):
    return O.values(O.unpack(q.cpu().numpy()), mxfp4.unpack_mxfp4_scales(s.cpu(), q.shape[-1] * 2).numpy())


def _layer(e, h, i, seed):
    gen = torch.Generator().manual_seed(seed)
    return [mxfp4.quant_weight_mxfp4((torch.randn(shape, generator=gen) * 0.1).cuda()) for shape in ((e, 2 * i, h), (e, h, i))]


def _inputs(t, h, e, topk, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((t, h), generator=gen).to(dtype).cuda()
    scores, ids = torch.rand((t, e), generator=gen).topk(topk, dim=1)
    return x, torch.softmax(scores, 1).cuda(), ids.to(torch.int32).cuda()


def _as_near_as_its_rounding(out, x, layer, weights, ids, kind="silu", on_input=False, scaling=1.0):
    (w1, s1), (w2, s2) = layer
    ref, size = O.experts(_np(x), _values(w1, s1), _values(w2, s2), _np(weights), ids.cpu().numpy(), kind, on_input, scaling)
    assert out.isfinite().all() and np.linalg.norm(size) < 32 * np.linalg.norm(ref)
    rounded = torch.from_numpy(ref).to(out.dtype).double().numpy()
    assert np.linalg.norm(_np(out) - ref) <= 1.1 * np.linalg.norm(rounded - ref)


# one slot to an expert, a few, five to eight (two tiles of 8 or one), many; over 16, 32 and 64 tokens, and K blocks that end early
SHAPES = [(1, 8, 4, 512, 288), (9, 6, 2, 160, 96), (20, 20, 5, 288, 160), (40, 32, 5, 256, 96), (60, 32, 3, 544, 64), (64, 64, 8, 256, 96),
          (70, 6, 2, 256, 288), (100, 16, 1, 128, 288), (128, 64, 4, 160, 96)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind,on_input", [("silu", False), ("gelu", False), ("silu", True), ("gelu", True)])
@pytest.mark.parametrize("t,e,topk,h,i", SHAPES)
def test_every_form_costs_one_rounding(dev, t, e, topk, h, i, kind, on_input, dtype):
    layer = _layer(e, h, i, t)
    (w1, s1), (w2, s2) = layer
    x, weights, ids = _inputs(t, h, e, topk, dtype, e)
    if on_input:
        weights = weights + 0.5  # or the activation sees next to nothing
    ids[:, topk // 2] = torch.where(torch.arange(t, device=dev) % 3 == 1, torch.tensor(-1, dtype=torch.int32, device=dev), ids[:, topk // 2])
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2, activation=kind, apply_router_weight_on_input=on_input, routed_scaling_factor=1.5)
    _as_near_as_its_rounding(out, x, layer, weights, ids, kind, on_input, 1.5)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("t,e,topk", [(1, 4, 2), (6, 4, 2), (40, 4, 2)])
@pytest.mark.parametrize("h,i", [(32, 32), (128, 96), (160, 128), (224, 160), (256, 256), (288, 224), (416, 288)])
def test_scales_at_the_ends_of_their_range(dev, t, e, topk, h, i, dtype):
    """Up rows with the largest scales (2^126, 2^127; their codes keep the values in float32's range, the rows next to them have every
    code), W2 with the smallest (2^-127 .. 2^-122; the values are subnormal floats), and a product of the two that is neither."""
    layer = _layer(e, h, i, t)
    (w1, s1), (w2, s2) = layer
    rng = np.random.default_rng(h)
    code, byte = O.unpack(w1.cpu().numpy()), mxfp4.unpack_mxfp4_scales(s1.cpu(), h).numpy().copy()
    high = np.zeros(2 * i, bool)
    high[i::2] = True  # every second up row
    byte[:, high] = rng.integers(253, 255, byte[:, high].shape)
    small = rng.integers(0, 4, code[:, high].shape) | (rng.integers(0, 2, code[:, high].shape) << 3)  # 0 .. 1.5
    code[:, high] = small
    byte[:, i + 1::2] = np.minimum(byte[:, i + 1::2] + 125, 252)
    w1 = torch.from_numpy(O.pack(code)).to(dev)
    s1 = mxfp4.pack_mxfp4_scales(torch.from_numpy(byte)).to(dev)
    low = rng.integers(0, 6, (e, h, i // 32)).astype(np.uint8)
    s2 = mxfp4.pack_mxfp4_scales(torch.from_numpy(low)).to(dev)
    layer = [(w1, s1), (w2, s2)]
    x, weights, ids = _inputs(t, h, e, topk, dtype, e)
    x = x * 2.0**-9
    v1 = _values(w1, s1)
    gate, up = np.einsum("tk,enk->ten", _np(x), v1[:, :i]), np.einsum("tk,enk->ten", np.abs(_np(x)), np.abs(v1[:, i:]))
    assert (np.abs(v1) < 2.0**128).all() and up.max() < 2.0**127 and np.abs(gate).max() < 1  # the premise: nothing overflows float32
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)
    _as_near_as_its_rounding(out, x, layer, weights, ids)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("t,e,topk", [(1, 4, 2), (6, 4, 2), (40, 4, 2)])
@pytest.mark.parametrize("h,i", [(32, 64), (160, 96), (288, 352), (448, 32)])
def test_scale_bytes_that_no_block_has(dev, t, e, topk, h, i, dtype):
    """What the last word of a row holds behind its blocks is not looked at."""
    (w1, s1), (w2, s2) = _layer(e, h, i, t)
    x, weights, ids = _inputs(t, h, e, topk, dtype, e)
    want = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)

    def spoiled(s, blocks, byte):
        words = s.clone(memory_format=torch.contiguous_format)
        as_bytes = words.view(torch.uint8)
        assert not as_bytes[..., blocks:].any() and blocks % 4
        as_bytes[..., blocks:] = byte
        return words.transpose(-1, -2).contiguous().transpose(-1, -2)

    for byte in (1, 127, 252, 253, 254, 255):
        got = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, spoiled(s1, h // 32, byte), spoiled(s2, i // 32, byte))
        assert torch.equal(got, want), byte
