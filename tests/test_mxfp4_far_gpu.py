"""MXFP4 on tensors of more than 2^32 bytes or values: what lies far behind their start is what it is in a small tensor."""
import pytest
import torch

from sglang_amd import mxfp4

pytestmark = pytest.mark.gpu


def _codes(shape, seed):
    return torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _scales(shape, seed):
    return torch.randint(120, 125, shape, dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def test_quantised_and_back(dev):
    m, k = 280001, 16384  # 4.6e9 values: 9.2 GB of bfloat16
    x = torch.empty((m, k), dtype=torch.bfloat16, device=dev)
    tail = torch.randn((9, k), generator=torch.Generator(device=dev).manual_seed(0), device=dev).bfloat16()
    x[:-9], x[-9:] = 1.5, tail
    q, s = mxfp4.per_token_group_quant_mxfp4(x)
    tq, ts = mxfp4.per_token_group_quant_mxfp4(tail)
    assert torch.equal(q[-9:], tq) and torch.equal(s[-9:], ts)
    del x
    got = mxfp4.mxfp4_dequant(q, s, torch.bfloat16)
    assert torch.equal(got[-9:], mxfp4.mxfp4_dequant(tq, ts, torch.bfloat16)) and (got[:-9:1000, 5] == 1.5).all()


@pytest.mark.parametrize("kind", range(5))
def test_product_with_a_far_result(dev, kind):
    from sglang_amd._lib import lib

    m, n, k = 131073, 34816, 288  # 4.6e9 results
    a, sa = _codes((m, k // 2), 1), mxfp4.pack_mxfp4_scales(_scales((m, k // 32), 2))
    b, sb = _codes((n, k // 2), 3), mxfp4.pack_mxfp4_scales(_scales((n, k // 32), 4))
    lib.fp8k_tune_force_mxfp4_plan(kind)
    try:
        got = mxfp4.w4a4_mxfp4_matmul(a, b, sa, sb)
    finally:
        lib.fp8k_tune_force_mxfp4_plan(-1)
    # terms are multiples of 2^-16 and at most 36 * 2^-6: float32 sums of 288 are exact
    av, bv = mxfp4.mxfp4_dequant(a[-5:].contiguous(), sa[-5:], torch.float32).double(), mxfp4.mxfp4_dequant(b, sb, torch.float32).double()
    assert torch.equal(got[-5:], (av @ bv.t()).bfloat16())


@pytest.mark.parametrize("t,e", [(2, 640), (40, 640)])
def test_experts_far_behind_the_first(dev, t, e):
    h, i = 4096, 2048  # 5.4 GB of gate and up codes, 2.7 GB of the others
    w1, s1 = _codes((e, 2 * i, h // 2), 1), mxfp4.pack_mxfp4_scales(_scales((e, 2 * i, h // 32), 2) - 6)
    w2, s2 = _codes((e, h, i // 2), 3), mxfp4.pack_mxfp4_scales(_scales((e, h, i // 32), 4) - 6)
    gen = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn((t, h), generator=gen, device=dev).bfloat16()
    weights = torch.rand((t, 3), generator=gen, device=dev)
    ids = torch.randint(e - 4, e, (t, 3), generator=gen, device=dev)
    got = mxfp4.fused_experts_mxfp4(x, w1, w2, weights, ids, s1, s2)
    # a stack of the last 32 experts, enough for tiles of as many slots (which decide the order of the sums)
    last = [p[-32:].clone() for p in (w1, w2)] + [p[-32:].clone(memory_format=torch.contiguous_format) for p in (s1, s2)]
    want = mxfp4.fused_experts_mxfp4(x, last[0], last[1], weights, ids - (e - 32), last[2], last[3])
    assert got.isfinite().all() and got.any(1).all()
    assert torch.equal(got, want)
