"""Latent attention at the limits of what its calls allow, against the definition in float64 (mla_reference.py)."""
import pytest
import torch

from tests import mla_reference as R
from tests.test_mla_attention_gpu import BF16, F16, SCALE, _filled, _gen, _prefill_inputs, _queries

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


def _decode_by_abi(q, qp, cache, pt, sl, guard=4096):
    """fp8k_mla_decode with just the workspace that it asks for, full of ones, and bytes behind it that must stay as they are."""
    from sglang_amd._lib import BF16 as CODE, check, lib, stream_ptr

    B, n, H, _ = q.shape
    out = torch.full((B, n, H, 512), 9.0, dtype=q.dtype, device="cuda")
    lse = torch.full((B, n, H), 9.0, device="cuda")
    need = lib.fp8k_mla_decode_workspace_bytes(B, n, H, pt.shape[1] * cache.shape[1])
    ws = torch.full((need + guard,), 255, dtype=torch.uint8, device="cuda")
    check(lib.fp8k_mla_decode(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), qp.data_ptr(), qp.stride(0), qp.stride(1), qp.stride(2), cache.data_ptr(),
                              pt.data_ptr(), pt.stride(0), pt.shape[1], sl.data_ptr(), None, out.data_ptr(), lse.data_ptr(), B, n, H, cache.shape[0],
                              cache.shape[1], SCALE, CODE, 0, ws.data_ptr(), need, stream_ptr(q.device)))
    assert bool((ws[need:] == 255).all())
    return out, lse


@pytest.mark.parametrize("n,H,lens,width", [(1, 128, [64 * 40, 100, 0, 64 * 33], 40), (1, 16, [(i * 53) % 900 for i in range(300)], 16),
                                            (2, 32, [(i * 37) % 250 if i % 5 else 0 for i in range(700)], 4), (1, 128, [0, 0, 0], 2),
                                            (1, 8, [0] * 600, 2), (1, 128, [130] * 256, 3), (1, 16, [700] * 257, 11)], ids=lambda x: None if isinstance(x, list) else str(x))
def test_decode_stays_in_its_workspace(dev, n, H, lens, width):
    """Batches with fewer requests than runs and with more, with and without empty ones, in a workspace that held something else."""
    g = _gen(len(lens) + H)
    cache, table, pt, _ = _filled(g, lens, 64, BF16, False, width=width)
    q, qp = _queries(g, len(lens), n, H, BF16)
    out, lse = _decode_by_abi(q, qp, cache, pt, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    want, want_lse, tol, lse_tol = R.decode(q, qp, cache, table, lens, SCALE, None)
    R.close(out, want, tol, "out")
    R.close(lse, want_lse, lse_tol, "lse")


@pytest.mark.parametrize("n,H,B,width", [(1, 16, 5, 4), (1, 128, 300, 3), (2, 40, 1100, 2)])
def test_decode_cuts_by_one_reading_of_the_lengths(dev, n, H, B, width):
    """Calls one behind the other in one workspace, each with other lengths: what one has left there - which runs hold a request, partials - never
    reaches the next, requests that have lost all their tokens among them."""
    from sglang_amd._lib import BF16 as CODE, check, lib, stream_ptr

    g = _gen(B)
    most = [64 * width] * B
    cache, table, pt, _ = _filled(g, most, 64, BF16, False, width=width)
    q, qp = _queries(g, B, n, H, BF16)
    need = lib.fp8k_mla_decode_workspace_bytes(B, n, H, 64 * width)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty((B, n, H, 512), dtype=BF16, device="cuda"), torch.empty((B, n, H), device="cuda")
    for turn, lens in enumerate((most, [0] * B, [(29 * i) % (64 * width + 1) if i % 3 else 0 for i in range(B)], [0] * (B - 1) + [64 * width], [1] + [0] * (B - 1))):
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        check(lib.fp8k_mla_decode(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), qp.data_ptr(), qp.stride(0), qp.stride(1), qp.stride(2), cache.data_ptr(),
                                  pt.data_ptr(), pt.stride(0), width, sl.data_ptr(), None, out.data_ptr(), lse.data_ptr(), B, n, H, cache.shape[0], 64, SCALE,
                                  CODE, 0, ws.data_ptr(), need, stream_ptr(q.device)))
        want, want_lse, tol, lse_tol = R.decode(q, qp, cache, table, lens, SCALE, None)
        R.close(out, want, tol, "out %d" % turn)
        R.close(lse, want_lse, lse_tol, "lse %d" % turn)


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
@pytest.mark.parametrize("rows,D", [(5, 8), (37, 192), (3, 8192)])
def test_merge_in_place(dev, rows, D, dtype):
    """The result may take the place of either operand, rows of several workgroups among them."""
    from sglang_amd import mla, sgl_kernel

    g = _gen(D)
    a, b = (torch.randn((rows, D), generator=g, device="cuda").to(dtype) for _ in range(2))
    la, lb = (torch.randn((rows,), generator=g, device="cuda") * 3 for _ in range(2))
    la[0] = lb[1] = float("-inf")
    want, want_lse = mla.merge_attention_states(a, la, b, lb)
    for which in (0, 1):
        x, y, lse = a.clone(), b.clone(), torch.empty_like(la)
        sgl_kernel.merge_attention_states(x, la, y, lb, (x, y)[which], lse)
        assert torch.equal((x, y)[which], want) and torch.equal((y, x)[which], (b, a)[which]) and torch.equal(lse, want_lse)
    both = torch.cat((a, a))
    with pytest.raises(RuntimeError, match="out must be"):
        sgl_kernel.merge_attention_states(both[:rows], la, b, lb, both[1:rows + 1], torch.empty_like(la))


@pytest.mark.parametrize("T,H", [(1, 1), (5, 16), (30, 8), (1, 128)])
def test_rotated_queries_in_slices_of_one_buffer(dev, T, H):
    """Queries and their place as slices of one buffer: the part of a head in front of its queries, a block behind a token's heads, another order of rows."""
    from sglang_amd import mla
    from tests.test_mla_attention_gpu import _table_of_angles

    g = _gen(T * H)
    latent = torch.randn((T, 576), generator=g, device="cuda").to(BF16)
    cache, slots = torch.zeros((2, 64, 576), dtype=BF16, device="cuda"), torch.arange(T, device="cuda")
    rest = dict(cos_sin=_table_of_angles(64), positions=torch.arange(T, device="cuda"))
    width = H * 192 + H * 64 + 576
    for place in (lambda b: b[:, :H * 192].view(T, H, 192)[..., :64], lambda b: b[:, H * 192:H * 256].view(T, H, 64)):
        buffer = torch.randn((T, width), generator=g, device="cuda").to(BF16)
        q, out = buffer[:, :H * 192].view(T, H, 192)[..., 128:], place(buffer)
        before, kept = buffer.clone(), q.clone()
        want = mla.mla_write_cache(latent, cache, slots, q_pe=kept, **rest)
        assert mla.mla_write_cache(latent, cache, slots, q_pe=q, q_out=out, **rest) is out
        assert torch.equal(out, want) and torch.equal(q, kept)
        place(before).copy_(want)
        assert torch.equal(buffer, before)
    if T > 1:
        buffer = torch.randn((T * H + H, 64), generator=g, device="cuda").to(BF16)
        with pytest.raises(RuntimeError, match="overlap"):
            mla.mla_write_cache(latent, cache, slots, q_pe=buffer[:T * H].view(T, H, 64), q_out=buffer[H:].view(T, H, 64), **rest)
        with pytest.raises(RuntimeError, match="overlap"):
            torch.ops.fp8k.mla_write_cache(latent, cache, slots, None, 1e-6, rest["cos_sin"], rest["positions"], False, buffer[:T * H].view(T, H, 64),
                                           buffer[H:].view(T, H, 64), None)


@pytest.mark.parametrize("n,H,lens,width", [(1, 16, [70, 0, 300], 5), (2, 32, [5000, 1, 64], 800), (1, 128, [(97 * i) % 700 for i in range(90)], 11),
                                            (1, 128, [4000], 63), (3, 50, [200] * 300, 4)], ids=lambda x: None if isinstance(x, list) else str(x))
def test_decode_in_the_queries_place(dev, n, H, lens, width):
    """The result may take the queries' place, in requests that one run holds and in those that several share, in every block of rows."""
    from sglang_amd import mla

    g = _gen(H)
    cache, table, pt, _ = _filled(g, lens, 64, BF16, False, width=width)
    q, qp = _queries(g, len(lens), n, H, BF16)
    q = q.contiguous()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = mla.mla_decode_attention(q, qp, cache, pt, sl, SCALE)
    for _ in range(3):
        place = q.clone()
        assert mla.mla_decode_attention(place, qp, cache, pt, sl, SCALE, out=place) is place
        assert torch.equal(place, want)
    whole = torch.cat((q.view(-1), q.view(-1)))
    with pytest.raises(RuntimeError, match="overlaps"):
        mla.mla_decode_attention(whole[:q.numel()].view(q.shape), qp, cache, pt, sl, SCALE, out=whole[512:512 + q.numel()].view(q.shape))
    assert torch.equal(whole, torch.cat((q.view(-1), q.view(-1))))


def test_results_beside_their_operands(dev):
    """Results and operands as pieces of one buffer, each beginning where another ends."""
    from sglang_amd import mla

    g = _gen(8)
    q, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(g, [70, 5], [70, 130], 2, BF16, slack=0)
    want = mla.mla_prefill_attention(q, kn, kp, v, tq, tk, 70, SCALE)
    buffer = torch.empty((q.numel() + want.numel() + kp.numel(),), dtype=BF16, device="cuda")
    q2, out, kp2 = (x.view(s) for x, s in zip(buffer.split((q.numel(), want.numel(), kp.numel())), (q.shape, want.shape, kp.shape)))
    q2.copy_(q), kp2.copy_(kp)
    assert mla.mla_prefill_attention(q2, kn, kp2, v, tq, tk, 70, SCALE, out=out) is out and torch.equal(out, want)
    cache, table, pt, _ = _filled(g, [70, 33], 64, BF16, False)
    buffer = torch.empty((cache.numel() + 103 * 576,), dtype=BF16, device="cuda")
    cache2, rows = buffer[:cache.numel()].view(cache.shape), buffer[cache.numel():].view(103, 576)
    cache2.copy_(cache)
    cu = torch.tensor([0, 70, 103], dtype=torch.int32, device="cuda")
    assert torch.equal(mla.mla_gather_cache(cache2, pt, cu, 103, out=rows), mla.mla_gather_cache(cache, pt, cu, 103))
    with pytest.raises(RuntimeError, match="overlaps"):
        mla.mla_gather_cache(cache2, pt, cu, 103, out=buffer[cache.numel() - 576:-576].view(103, 576))


@pytest.mark.parametrize("lq,lk,H,most", [([300], [300], 3, 100), ([300, 600], [300, 900], 2, 128), ([700], [9000], 2, 250), ([1024, 1000], [5000, 8000], 1, 512),
                                          ([700, 20], [700, 700], 64, 1)], ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_of_more_queries_than_stated(dev, lq, lk, H, most, causal):
    """A bound below the longest sequence: its queries up to the bound are as they are, those behind the bound's block are not written; keys split and not, blocks
    of 128 and of 256."""
    from sglang_amd import mla

    q, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(_gen(most), lq, lk, H, BF16)
    out = torch.full((q.shape[0], H, 128), 7.0, dtype=BF16, device="cuda")
    _, lse = mla.mla_prefill_attention(q, kn, kp, v, tq, tk, most, SCALE, causal=causal, return_lse=True, out=out)
    want, want_lse, tol, lse_tol = R.prefill(q, kn, kp, v, cu_q, cu_k, SCALE, causal)
    for at, n in zip(cu_q, lq):
        first = slice(at, at + min(n, most))
        R.close(out[first], want[first], tol[first], "out")
        R.close(lse[first], want_lse[first], lse_tol[first], "lse")
        assert bool((out[at + min(n, -(-most // 256) * 256):at + n] == 7.0).all())
    assert bool((out[cu_q[-1]:] == 7.0).all())


def test_decode_of_the_most_requests(dev):
    """65535 requests of one token or none: a single token's weight is 1, its result the row itself."""
    from sglang_amd import mla

    g = _gen(65535)
    B = 65535
    cache = torch.randn((700, 2, 576), generator=g, device="cuda").to(BF16)
    table = torch.randint(0, 700, (B, 1), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, 2, (B,), generator=g, device="cuda", dtype=torch.int32)
    q, qp = _queries(g, B, 1, 1, BF16)
    out, lse = mla.mla_decode_attention(q[:, 0], qp[:, 0], cache, table, lens, SCALE, return_lse=True)
    rows = cache[table[:, 0].long(), 0, :512]
    assert torch.equal(out[:, 0], torch.where((lens > 0)[:, None], rows, torch.zeros_like(rows)))
    assert torch.equal(torch.isinf(lse[:, 0]), lens == 0)


@pytest.mark.parametrize("n,H", [(512, 128), (1, 65536), (65536, 1)])
def test_decode_of_the_most_rows(dev, n, H):
    """65536 rows to a request, new tokens by heads; more new tokens than the request has among them."""
    g = _gen(n)
    lens = [300, 0]
    cache, table, pt, _ = _filled(g, lens, 64, BF16, False)
    q, qp = _queries(g, 2, n, H, BF16)
    from sglang_amd import mla

    out, lse = mla.mla_decode_attention(q, qp, cache, pt, torch.tensor(lens, dtype=torch.int32, device="cuda"), SCALE, return_lse=True)
    want, want_lse, tol, lse_tol = R.decode(q, qp, cache, table, lens, SCALE, None)
    R.close(out, want, tol, "out")
    R.close(lse, want_lse, lse_tol, "lse")


@pytest.mark.parametrize("lq,lk,H,slack", [([16], [9000], 4, 4000), ([16], [9000], 8, 0), ([130, 0, 5], [5000, 3000, 0], 2, 700), ([256], [4000], 3, 9), ([512, 512], [4000, 97], 8, 0),
                                           ([40] * 12, [700 + 100 * i for i in range(12)], 1, 2000)], ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_stays_in_its_workspace(dev, lq, lk, H, slack, causal):
    """Split keys with just the workspace asked for, full of ones, and bytes behind it that must stay as they are; queries with many more rows than the sequences have."""
    from sglang_amd._lib import BF16 as CODE, check, lib, stream_ptr

    q, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(_gen(H), lq, lk, H, BF16, slack=slack)
    Tq, Tk, B = q.shape[0], kn.shape[0], len(lq)
    out, lse = torch.full((Tq, H, 128), 7.0, dtype=BF16, device="cuda"), torch.full((Tq, H), 7.0, device="cuda")
    need = lib.fp8k_mla_prefill_workspace_bytes(B, H, Tq, Tk, max(lq))
    assert need > 0
    ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device="cuda")
    check(lib.fp8k_mla_prefill(q.data_ptr(), q.stride(0), q.stride(1), kn.data_ptr(), kn.stride(0), kn.stride(1), kp.data_ptr(), kp.stride(0), v.data_ptr(), v.stride(0),
                               v.stride(1), tq.data_ptr(), tk.data_ptr(), out.data_ptr(), lse.data_ptr(), B, H, Tq, Tk, max(lq), SCALE, 1 if causal else 0, CODE, ws.data_ptr(),
                               need, stream_ptr(q.device)))
    n = cu_q[-1]
    assert bool((ws[need:] == 255).all()) and bool((out[n:] == 7.0).all()) and bool((lse[n:] == 7.0).all())
    want, want_lse, tol, lse_tol = R.prefill(q, kn, kp, v, cu_q, cu_k, SCALE, causal)
    R.close(out[:n], want, tol, "out")
    R.close(lse[:n], want_lse, lse_tol, "lse")
