"""MXFP4 entry points on operands whose rows the kernels cannot read as they lie: the calls copy them, and give what the copy gives."""
import pytest
import torch

from sglang_amd import mxfp4

pytestmark = pytest.mark.gpu


def _random(shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def test_expanded_operands(dev):
    """One row of codes for all rows: a row stride of zero."""
    q, s = mxfp4.per_token_group_quant_mxfp4(_random((1, 288)))
    w, ws = mxfp4.quant_weight_mxfp4(_random((72, 288), seed=1))
    one = mxfp4.w4a4_mxfp4_matmul(q, w, s, ws)
    for m in (2, 8, 70):
        got = mxfp4.w4a4_mxfp4_matmul(q.expand(m, -1), w, s.expand(m, -1), ws)
        assert torch.equal(got, mxfp4.w4a4_mxfp4_matmul(q.repeat(m, 1), w, s.repeat(m, 1), ws))
        assert torch.equal(got, got[:1].expand(m, -1)) and (m > 16 or torch.equal(got[:1], one))
    x = _random((5, 288), seed=2)
    for rows in (x, x[:1], x.expand(3, 5, 288), x[:1].expand(4, 288)):
        got = mxfp4.w4a4_mxfp4_linear(rows, w[:1].expand(16, -1), ws[:1].expand(16, -1))
        assert torch.equal(got, mxfp4.w4a4_mxfp4_linear(rows.contiguous(), w[:1].repeat(16, 1), ws[:1].repeat(16, 1)))
