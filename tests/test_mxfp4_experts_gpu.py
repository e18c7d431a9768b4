"""The expert layer on MXFP4 weights against the float64 oracle.

Tolerance: the result is rounded once and the intermediate once, each off by at most half a step of the type (finfo.eps / 2 relative), and
the intermediate's error reaches the result through the magnitudes of the second stage's terms; the activation function and float32 sums
of K terms add K * 2^-24 and 2^-18 (the device's exponential, reciprocal and error function, relative) of the same sizes."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as O
from sglang_amd import mxfp4

pytestmark = pytest.mark.gpu


def _layer(e, h, i, seed=0, scale=0.1):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for shape in ((e, 2 * i, h), (e, h, i)):
        out.append(mxfp4.quant_weight_mxfp4((torch.randn(shape, generator=gen) * scale).cuda()))
    return out


def _np(t):
    return t.double().cpu().numpy()


def _values(q, s):
    return O.values(O.unpack(q.cpu().numpy()), mxfp4.unpack_mxfp4_scales(s.cpu(), q.shape[-1] * 2).numpy())


def _inputs(t, h, e, topk, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((t, h), generator=gen).to(dtype).cuda()
    scores, ids = torch.rand((t, e), generator=gen).topk(min(topk, e), dim=1)
    return x, torch.softmax(scores, 1).cuda(), ids.to(torch.int32).cuda()


def _check(out, x, layer, weights, ids, kind="silu", on_input=False, scaling=1.0):
    (w1, s1), (w2, s2) = layer
    v1, v2 = _values(w1, s1), _values(w2, s2)
    xs, tw = x.double().cpu().numpy(), weights.double().cpu().numpy()
    ref, size = O.experts(xs, v1, v2, tw, ids.cpu().numpy(), kind, on_input, scaling)
    half = torch.finfo(x.dtype).eps / 2
    h, i = v1.shape[2], v2.shape[2]
    # the first stage's float32 sums: relative to the magnitudes of their terms, at most (h + i) * 2^-24 of a size that the intermediate
    # has at least a thousandth of in these tests
    got = out.double().cpu().numpy()
    tol = half * np.abs(ref) + size * (half + 2.0**-12) * 1.01 + torch.finfo(x.dtype).tiny
    assert np.isfinite(got).all() and (np.abs(got - ref) <= tol).all(), np.max(np.abs(got - ref) / tol)
    # and together: independent roundings, so far less than their bounds added up
    norm = np.linalg.norm(ref)
    if norm:
        assert np.linalg.norm(got - ref) <= 2 * half * norm


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,topk,h,i", [(1, 4, 1, 32, 32), (1, 8, 2, 256, 64), (2, 256, 8, 128, 32), (3, 5, 3, 288, 96), (7, 16, 4, 544, 160),
                                          (13, 8, 2, 1024, 256), (16, 1, 1, 256, 288), (33, 1, 1, 128, 64), (17, 3, 2, 512, 512), (64, 32, 8, 256, 96),
                                          (100, 4, 2, 160, 128), (128, 16, 8, 128, 64), (5, 4, 2, 2048, 544), (1, 2, 2, 4096, 1312)])
def test_experts_against_float64(dev, t, e, topk, h, i, dtype):
    layer = _layer(e, h, i, t)
    x, weights, ids = _inputs(t, h, e, topk, dtype, e)
    (w1, s1), (w2, s2) = layer
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2, routed_scaling_factor=2.5)
    assert out.shape == x.shape and out.dtype == dtype
    _check(out, x, layer, weights, ids, scaling=2.5)
    assert torch.equal(out, mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2, routed_scaling_factor=2.5))  # whatever the timing


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("on_input", [False, True])
def test_options(dev, kind, on_input):
    layer = _layer(6, 160, 96)
    (w1, s1), (w2, s2) = layer
    x, weights, ids = _inputs(9, 160, 6, 2, torch.bfloat16)
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2, activation=kind, apply_router_weight_on_input=on_input)
    _check(out, x, layer, weights, ids, kind, on_input)
    # int64 ids, row-major scales, float64 weights, a padded batch
    assert torch.equal(out, mxfp4.fused_experts_mxfp4(x, w1, w2, weights.double(), ids.long(), s1.contiguous(), s2.contiguous(), activation=kind,
                                                      apply_router_weight_on_input=on_input))
    wide = torch.randn((9, 320), device=dev).to(torch.bfloat16)
    wide[:, 64:224] = x
    assert torch.equal(out, mxfp4.fused_experts_mxfp4(wide[:, 64:224], w1, w2, weights, ids, s1, s2, activation=kind,
                                                      apply_router_weight_on_input=on_input))
    assert torch.equal(out, mxfp4.fused_experts_mxfp4(x, w1, w2, weights.t().contiguous().t(), ids.t().contiguous().t(), s1, s2, activation=kind,
                                                      apply_router_weight_on_input=on_input))
    same = x.clone()
    got = mxfp4.fused_experts_mxfp4(same, w1, w2, weights, ids, s1, s2, activation=kind, apply_router_weight_on_input=on_input, inplace=True)
    assert got.data_ptr() == same.data_ptr() and torch.equal(same, out)


@pytest.mark.parametrize("t,topk", [(1, 3), (6, 4), (40, 8)])
def test_experts_of_other_ranks_and_repeated_ones(dev, t, topk):
    e = 7
    layer = _layer(e, 128, 64, 3)
    (w1, s1), (w2, s2) = layer
    gen = torch.Generator().manual_seed(t)
    x = torch.randn((t, 128), generator=gen).to(torch.bfloat16).cuda()
    weights = torch.rand((t, topk), generator=gen).cuda()
    # ids below and above the range contribute nothing, the same expert twice counts twice, some tokens have none at all
    ids = torch.randint(-2, e + 3, (t, topk), generator=gen).to(torch.int32)
    ids[0] = ids[0, 0].clamp(0, e - 1)
    ids[-1] = torch.where(torch.tensor(t > 1), torch.full((topk,), -1, dtype=torch.int32), ids[-1])
    ids = ids.cuda()
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)
    _check(out, x, layer, weights, ids)
    if t > 1:
        assert not out[-1].any()
    far = ids.long() + torch.where(ids < 0, -(1 << 40), 0)
    assert torch.equal(out, mxfp4.fused_experts_mxfp4(x, w1, w2, weights, far, s1, s2))
    none = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, torch.full_like(ids, -1), s1, s2)
    assert not none.any() and none.isfinite().all()


@pytest.mark.parametrize("t,e,topk,h,i", [(5, 4, 4, 288, 544), (16, 10, 4, 544, 288), (20, 20, 5, 160, 96), (64, 64, 8, 256, 96), (60, 32, 3, 4128, 64),
                                          (100, 16, 1, 128, 288), (128, 64, 4, 160, 512)])
def test_five_to_eight_slots_to_an_expert(dev, t, e, topk, h, i):
    """Between the few-slot tiles and the large ones, with experts that have more than one tile and experts that have none."""
    layer = _layer(e, h, i, t)
    x, weights, ids = _inputs(t, h, e, topk, torch.bfloat16, e)
    ids[: t // 2] = ids[: t // 2].clamp(max=e // 2)
    (w1, s1), (w2, s2) = layer
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)
    _check(out, x, layer, weights, ids)
    assert torch.equal(out, mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,topk,h,i", [(1, 8, 4, 512, 288), (9, 16, 4, 1024, 256), (40, 6, 2, 256, 544), (70, 64, 4, 256, 96)])
def test_the_intermediate_costs_no_precision(dev, t, e, topk, h, i, dtype):
    """The whole error is that of the result's rounding, 2^-8 or 2^-11 at most and some 0.4 of it in the norm.  The pairs of the intermediate
    are off by 2^-16 of a term at most, float32 sums by (h + i) * 2^-24 and the activation by 2^-18; the roundings of different terms are
    independent, so that in the norm they add up like the terms themselves do, whose sizes add up to under 32 times the result (checked)
    and their squares' root to a few times it: a tenth of float16's 0.4 * 2^-11, whose square is within the 1.1."""
    layer = _layer(e, h, i, t)
    (w1, s1), (w2, s2) = layer
    x, weights, ids = _inputs(t, h, e, topk, dtype, e)
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)
    ref, size = O.experts(x.double().cpu().numpy(), _values(w1, s1), _values(w2, s2), weights.double().cpu().numpy(), ids.cpu().numpy(), "silu", False, 1.0)
    assert np.linalg.norm(size) < 32 * np.linalg.norm(ref)
    rounded = torch.from_numpy(ref).to(dtype).double().numpy()
    assert np.linalg.norm(_np(out) - ref) <= 1.1 * np.linalg.norm(rounded - ref)


def test_intermediate_beyond_float16(dev):
    """gate * up above 65504 with results that float16 holds."""
    layer = [mxfp4.quant_weight_mxfp4((torch.randn((3, n, k), generator=torch.Generator().manual_seed(n)) * c).cuda()) for n, k, c in
             ((192, 128, 3.0), (128, 96, 2.0**-12))]
    (w1, s1), (w2, s2) = layer
    x, weights, ids = _inputs(5, 128, 3, 2, torch.float16)
    x = x * 20
    v1 = _values(w1, s1)
    products = np.einsum("tk,enk->ten", x.double().cpu().numpy(), v1)
    assert (products[..., :96] * products[..., 96:]).max() > 2 * 65504
    _check(mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2), x, layer, weights, ids)


def test_what_no_expert_takes_is_never_multiplied(dev):
    """NaN and infinity in the weights of masked choices, and in tokens all of whose choices are masked."""
    layer = _layer(5, 160, 96)
    (w1, s1), (w2, s2) = layer
    for t in (1, 6, 50):
        x, weights, ids = _inputs(t, 160, 5, 3, torch.float16, t)
        ids[:, 1] = -1
        if t > 1:
            ids[t // 2] = 5
        zero = weights.clone()
        zero[(ids < 0) | (ids > 4)] = 0
        clean = mxfp4.fused_experts_mxfp4(x, w1, w2, zero, ids, s1, s2)
        bad, dirty = weights.clone(), x.clone()
        bad[(ids < 0) | (ids > 4)] = float("nan")
        if t > 1:
            bad[t // 2] = float("inf")
            dirty[t // 2] = float("nan")
            assert not clean[t // 2].any()
        for on_input in (False, True):
            want = clean if not on_input else mxfp4.fused_experts_mxfp4(x, w1, w2, zero, ids, s1, s2, apply_router_weight_on_input=True)
            assert torch.equal(mxfp4.fused_experts_mxfp4(dirty, w1, w2, bad, ids, s1, s2, apply_router_weight_on_input=on_input), want)


def test_a_token_that_is_not_finite_stays_alone(dev):
    layer = _layer(4, 160, 64)
    (w1, s1), (w2, s2) = layer
    x, weights, ids = _inputs(20, 160, 4, 2, torch.bfloat16)
    clean = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)
    bad = x.clone()
    bad[3, 7], bad[11, 150] = float("nan"), float("inf")
    out = mxfp4.fused_experts_mxfp4(bad, w1, w2, weights, ids, s1, s2)
    rest = torch.tensor([r not in (3, 11) for r in range(20)], device=dev)
    assert torch.equal(out[rest], clean[rest]) and out[3].isnan().all() and not out[11].isfinite().all()
    # a NaN scale of one expert reaches the tokens that use it, and no other
    broken = mxfp4.unpack_mxfp4_scales(s1, 160)
    broken[2, 5, 4] = 255
    out = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, mxfp4.pack_mxfp4_scales(broken), s2)
    uses = (ids == 2).any(1)
    assert out[uses].isnan().all() and torch.equal(out[~uses], clean[~uses])


def test_refusals(dev):
    layer = _layer(4, 128, 64)
    (w1, s1), (w2, s2) = layer
    x, weights, ids = _inputs(4, 128, 4, 2, torch.bfloat16)
    call = mxfp4.fused_experts_mxfp4
    big = torch.zeros((129, 128), dtype=torch.bfloat16, device=dev)
    for bad in (lambda: call(x.float(), w1, w2, weights, ids, s1, s2), lambda: call(x[:, :96], w1, w2, weights, ids, s1, s2),
                lambda: call(x, w2, w1, weights, ids, s2, s1), lambda: call(x, w1, w2, weights, ids[:3], s1, s2),
                lambda: call(x, w1, w2, weights, ids.float(), s1, s2), lambda: call(x, w1[:3], w2, weights, ids, s1, s2),
                lambda: call(x, w1, w2, weights, ids, s1, s2[:, :64]), lambda: call(x, w1.float(), w2, weights, ids, s1, s2),
                lambda: call(big, w1, w2, weights.new_zeros((129, 1)), ids.new_zeros((129, 1)), s1, s2),
                lambda: call(big[:128], w1, w2, weights.new_zeros((128, 9)), ids.new_zeros((128, 9)), s1, s2),
                lambda: call(x.cpu(), w1, w2, weights, ids, s1, s2)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        call(x, w1, w2, weights, ids, s1, s2, activation="relu2")
    assert call(x[:0], w1, w2, weights[:0], ids[:0], s1, s2).shape == (0, 128)


def test_router_and_experts_captured(dev, monkeypatch):
    """The grouped router and the layer, as a decode step makes them: eager, on another stream, captured and replayed with new tokens, and
    two graphs at once that know nothing of each other."""
    from sglang_amd import _host, fused_moe

    e, h, i, t = 32, 288, 96, 6
    layer = _layer(e, h, i)
    (w1, s1), (w2, s2) = layer
    bias = torch.zeros((e,), device=dev)

    def step(x, logits):
        weights, ids = fused_moe.biased_grouped_topk(x, logits, bias, 4, True, 4, 2)
        return mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2, routed_scaling_factor=2.0)

    xs = [_inputs(t, h, e, 4, torch.bfloat16, k)[0] for k in range(4)]
    logits = [torch.randn((t, e), generator=torch.Generator().manual_seed(k)).cuda() for k in range(4)]
    eager = [step(x, g) for x, g in zip(xs, logits)]
    weights, ids = fused_moe.biased_grouped_topk(xs[0], logits[0], bias, 4, True, 4, 2)
    _check(eager[0], xs[0], layer, weights, ids, scaling=2.0)
    graphs = []
    for _ in range(2):
        sx, sl = xs[0].clone(), logits[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(sx, sl)
        graphs.append((g, sx, sl, out, torch.cuda.Stream()))
    for k in range(4):
        for j, (g, sx, sl, out, st) in enumerate(graphs):
            sx.copy_(xs[(k + j) % 4])
            sl.copy_(logits[(k + j) % 4])
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for j, (g, sx, sl, out, st) in enumerate(graphs):
            assert torch.equal(out, eager[(k + j) % 4])
        assert torch.equal(step(xs[k], logits[k]), eager[k])
    monkeypatch.setattr(_host, "mx_experts", lambda *a: None)
    assert torch.equal(step(xs[1], logits[1]), eager[1])
    again = xs[1].clone()
    weights, ids = fused_moe.biased_grouped_topk(again, logits[1], bias, 4, True, 4, 2)
    mxfp4.fused_experts_mxfp4(again, w1, w2, weights, ids, s1, s2, routed_scaling_factor=2.0, inplace=True)
    assert torch.equal(again, eager[1])
