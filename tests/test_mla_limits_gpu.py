"""Latent attention at the limits of what its calls allow, against the definition in float64 (mla_reference.py)."""
import pytest
import torch

from tests import mla_reference as R
from tests.test_mla_attention_gpu import BF16, F16, _filled, _gen, _prefill_inputs, _queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("H,width", [(128, 4), (32, 800), (128, 300), (128, 600)])
def test_decode_of_scores_scaled_to_nothing(dev, H, width, dtype):
    """A scale of the scores and one of the cache whose product is no float32 any more, in every block of rows: all tokens that a query sees
    weigh the same, those that it does not see nothing."""
    from sglang_amd import mla

    g = _gen(H + width)
    lens = [70, 1, 0, 200]
    cache, table, pt, _ = _filled(g, lens, 64, dtype, True, width=width)
    scale = torch.full((1,), 1e-25, device="cuda")
    q, qp = _queries(g, len(lens), 1, H, dtype)
    out, lse = mla.mla_decode_attention(q, qp, cache, pt, torch.tensor(lens, dtype=torch.int32, device="cuda"), 1e-25, scale=scale, return_lse=True)
    want, want_lse, tol, lse_tol = R.decode(q, qp, cache, table, lens, 1e-25, scale)
    R.close(out, want, tol, "out")
    R.close(lse, want_lse, lse_tol, "lse")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_of_scores_scaled_to_nothing(dev, causal, dtype):
    from sglang_amd import mla

    q, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(_gen(3), [70, 5], [70, 130], 2, dtype, slack=0)
    out, lse = mla.mla_prefill_attention(q, kn, kp, v, tq, tk, 70, 1e-45, causal=causal, return_lse=True)
    want, want_lse, tol, lse_tol = R.prefill(q, kn, kp, v, cu_q, cu_k, 1e-45, causal)
    R.close(out, want, tol, "out")
    R.close(lse, want_lse, lse_tol, "lse")
