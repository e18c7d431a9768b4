"""Latent attention (sglang_amd/mla.py) against its definition in float64 (mla_reference.py, which derives the tolerances): every way that a
call is cut, lengths from nothing to several runs, pages that end inside a tile, rows that see nothing, infinities and NaN where nothing
looks, strides, far caches, captured graphs, other streams; and the operators as a layer runs them together."""
import pytest
import torch

from tests import mla_reference as R

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5
BF16, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
NAN = float("nan")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _filled(g, lens, page, dtype, fp8, spare=2, width=None, sharp=1.0):
    """A cache whose pages lie in no order, NaN wherever no request has a token; table (list and tensor), scale."""
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = width or max(max(counts), 1)
    table, at = [], 0
    for n in counts:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    rows = torch.randn((pages, page, 576), generator=g, device="cuda") * sharp
    used = torch.zeros((pages * page,), dtype=torch.bool, device="cuda")
    for pages_of, n in zip(table, lens):
        t = torch.arange(n, device="cuda")
        used[torch.tensor(pages_of, device="cuda")[t // page] * page + t % page] = True
    rows[~used.view(pages, page)] = NAN
    scale = torch.full((1,), 0.0125, device="cuda") if fp8 else None
    cache = (rows / 0.0125).clamp(-448, 448).to(F8) if fp8 else rows.to(dtype)
    return cache, table, torch.tensor(table, dtype=torch.int32, device="cuda"), scale


def _queries(g, B, n, H, dtype):
    q = torch.randn((H, B * n, 512), generator=g, device="cuda").to(dtype).transpose(0, 1).view(B, n, H, 512)
    return q, torch.randn((B, n, H, 64), generator=g, device="cuda").to(dtype)


def _check_decode(lens, n, H, page, dtype, fp8, seed=0, sharp=1.0, width=None):
    from sglang_amd import mla

    g = _gen(seed)
    cache, table, pt, scale = _filled(g, lens, page, dtype, fp8, sharp=sharp, width=width)
    q, qp = _queries(g, len(lens), n, H, dtype)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = mla.mla_decode_attention(q, qp, cache, pt, sl, SCALE, scale=scale, return_lse=True)
    want, want_lse, tol, lse_tol = R.decode(q, qp, cache, table, lens, SCALE, scale)
    R.close(out, want, tol, "out")
    R.close(lse, want_lse, lse_tol, "lse")
    again, lse2 = mla.mla_decode_attention(q, qp, cache, pt, sl, SCALE, scale=scale, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    return out


LENS = [[1], [64], [65, 0, 1, 63], [0], [0, 0, 130], [200, 64, 128, 127, 129, 5, 1, 17]]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("n,H,page", [(1, 16, 64), (1, 1, 1), (2, 7, 3), (1, 128, 64), (3, 17, 16), (1, 40, 128)])
def test_decode(dev, lens, n, H, page, dtype, fp8):
    _check_decode(lens, n, H, page, dtype, fp8, seed=sum(lens) + n * H)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,H", [(1, 8), (1, 32), (2, 32), (1, 128), (4, 128), (3, 50)])
@pytest.mark.parametrize("lens", [[5000], [1700, 900, 0, 2600], [300] * 40], ids=["one", "four", "forty"])
def test_decode_over_several_runs(dev, lens, n, H, fp8):
    _check_decode(lens, n, H, 64, BF16, fp8, seed=H)


@pytest.mark.parametrize("rows,H", [(16, 16), (32, 32), (64, 64), (128, 128)])
def test_decode_of_every_block_of_rows(dev, rows, H):
    """A batch with tiles enough for every CU takes the largest block of rows that its heads fill; its runs hold parts of several requests."""
    _check_decode([333 + 7 * i for i in range(130)], 1, H, 64, BF16 if H != 64 else F16, H == 32, seed=H)


@pytest.mark.parametrize("dtype,fp8", [(BF16, False), (F16, True), (BF16, True), (F16, False)])
@pytest.mark.parametrize("H,width", [(128, 1), (128, 16), (128, 64), (128, 300), (64, 300), (32, 300), (70, 300), (257, 64)])
def test_decode_of_every_cut(dev, H, width, dtype, fp8):
    """The width of the page table bounds the lengths, and that decides how many rows a workgroup takes: from 16 to 128 of 128 heads, blocks that
    the heads do not fill, more blocks than one.  Lengths are few, or none, or end a step before, at and behind the steps that run ahead."""
    lens = [1, 31, 32, 33, 63, 64] if width == 1 else [0, 1, 64, 95, 96, 97, 128, 129, 160, 161, 192, 193, 257, 321, 400, 33]
    _check_decode(lens, 1, H, 64, dtype, fp8, seed=H + width, width=width)


@pytest.mark.parametrize("n,H,B,width", [(2, 8, 700, 4), (1, 16, 1500, 4), (3, 24, 600, 40), (1, 128, 520, 8)])
def test_decode_of_more_requests_than_threads(dev, n, H, B, width):
    """A thread of the prefix sum counts several requests, empty ones among them."""
    _check_decode([(i * 37) % 250 if i % 5 else 0 for i in range(B)], n, H, 64, BF16, n == 2, seed=B, width=width)


@pytest.mark.parametrize("B,H,width", [(200, 16, 5), (40, 128, 6), (90, 64, 8), (257, 128, 4), (16, 128, 36), (1, 128, 129)])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_of_short_requests(dev, B, H, width, fp8):
    """A run counts a new request as some tiles more: its borders may lie in front of a request's tiles, in them or behind them, and a run may hold
    no tile at all; 16 to 128 rows to a workgroup."""
    _check_decode([(64 * width - 79 * i) % (64 * width + 1) for i in range(B)], 1, H, 64, BF16, fp8, seed=B, width=width)


def test_decode_lengths_below_zero(dev):
    from sglang_amd import mla

    g = _gen(1)
    cache, table, pt, _ = _filled(g, [70, 70], 64, BF16, False)
    q, qp = _queries(g, 2, 1, 16, BF16)
    out, lse = mla.mla_decode_attention(q, qp, cache, pt, torch.tensor([-3, -(1 << 31)], dtype=torch.int32, device="cuda"), SCALE, return_lse=True)
    assert not out.any() and bool((lse == float("-inf")).all())


@pytest.mark.parametrize("order", ["rising", "falling", "spike"])
@pytest.mark.parametrize("H,fp8", [(16, False), (128, False), (128, True)])
def test_decode_scores_that_raise_the_maximum(dev, order, H, fp8):
    """The running maximum rises in every tile, in the first alone, or jumps once far from either end: scores up to 60 apart."""
    from sglang_amd import mla

    n = 700
    g = _gen(7)
    cache, table, pt, scale = _filled(g, [n], 64, BF16, fp8)
    q, qp = _queries(g, 1, 1, H, BF16)
    direction = torch.sign(torch.randn((576,), generator=g, device="cuda"))
    size = torch.linspace(0, 1, n, device="cuda")
    size = {"rising": size, "falling": size.flip(0), "spike": (torch.arange(n, device="cuda") == 400).float()}[order]
    rows = torch.randn((n, 576), generator=g, device="cuda") * 0.1 + 1.2 * size[:, None] * direction
    t = torch.arange(n, device="cuda")
    index = torch.tensor(table[0], device="cuda")[t // 64] * 64 + t % 64
    if fp8:
        cache.view(-1, 576).view(torch.uint8)[index] = (rows / 0.0125).clamp(-448, 448).to(F8).view(torch.uint8)
    else:
        cache.view(-1, 576)[index] = rows.to(BF16)
    q, qp = (direction[:512].to(BF16) + 0.1 * q).to(BF16), (direction[512:].to(BF16) + 0.1 * qp).to(BF16)
    sl = torch.tensor([n], dtype=torch.int32, device="cuda")
    out, lse = mla.mla_decode_attention(q, qp, cache, pt, sl, SCALE, scale=scale, return_lse=True)
    want, want_lse, tol, lse_tol = R.decode(q, qp, cache, table, [n], SCALE, scale)
    R.close(out, want, tol, "out")
    R.close(lse, want_lse, lse_tol, "lse")


def test_decode_layouts(dev):
    """3-D queries; queries, tables and caches that lie otherwise; a caller's output; no lse: one result."""
    from sglang_amd import mla

    g = _gen(3)
    lens = [90, 200, 33]
    cache, table, pt, _ = _filled(g, lens, 16, BF16, False)
    q, qp = _queries(g, 3, 1, 24, BF16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = mla.mla_decode_attention(q, qp, cache, pt, sl, SCALE)
    q3, qp3 = q[:, 0], qp[:, 0]
    assert torch.equal(mla.mla_decode_attention(q3, qp3, cache, pt, sl, SCALE), want[:, 0])
    wide = torch.zeros((3, 24, 516), dtype=BF16, device="cuda")  # rows at multiples of 8 bytes: copied
    wide[..., 4:] = q3
    assert torch.equal(mla.mla_decode_attention(wide[..., 4:], qp3, cache, pt, sl, SCALE), want[:, 0])
    strange = torch.zeros((3, 24, 64, 2), dtype=BF16, device="cuda")
    strange[..., 0] = qp3
    assert torch.equal(mla.mla_decode_attention(q3, strange[..., 0], cache, pt, sl, SCALE), want[:, 0])
    tables = torch.full((3, 40), 1 << 30, dtype=torch.int32, device="cuda")
    tables[:, 5:5 + pt.shape[1]] = pt
    assert torch.equal(mla.mla_decode_attention(q, qp, cache, tables[:, 5:5 + pt.shape[1]], sl, SCALE), want)
    assert torch.equal(mla.mla_decode_attention(q, qp, cache, pt.t().contiguous().t(), sl, SCALE), want)
    assert torch.equal(mla.mla_decode_attention(q, qp, cache.unsqueeze(2), pt, sl, SCALE), want)
    out = torch.empty_like(want, memory_format=torch.contiguous_format)
    assert mla.mla_decode_attention(q, qp, cache, pt, sl, SCALE, out=out) is out and torch.equal(out, want)
    # lengths beyond the table are held to it, entries that are no pages to the nearest page
    pt2 = pt.clone()
    pt2[1, 3], pt2[2, 0] = 1 << 30, -5
    long = torch.tensor([90, 1 << 30, 33], dtype=torch.int32, device="cuda")
    clean = torch.nan_to_num(cache)
    got = mla.mla_decode_attention(q, qp, clean, pt2, long, SCALE)
    table2 = [list(r) for r in table]
    table2[1][3], table2[2][0] = cache.shape[0] - 1, 0
    w, _, tol, _ = R.decode(q, qp, clean, table2, [90, pt.shape[1] * 16, 33], SCALE, None)
    R.close(got, w, tol)
    # no requests, no pages
    assert mla.mla_decode_attention(q[:0], qp[:0], cache, pt[:0], sl[:0], SCALE).shape == (0, 1, 24, 512)
    o, s = mla.mla_decode_attention(q, qp, cache[:0], pt, sl, SCALE, return_lse=True)
    assert not o.any() and bool((s == float("-inf")).all())
    assert not mla.mla_decode_attention(q, qp, cache, pt[:, :0], sl, SCALE).any()


def test_decode_of_far_pages(dev):
    """Pages beyond 2^32 bytes, and beyond 2^32 numbers, of a cache."""
    from sglang_amd import mla

    g = _gen(11)
    pages = (1 << 33) // (64 * 576 * 2) + 40
    cache = torch.empty((pages, 64, 576), dtype=BF16, device="cuda")
    places = [3, pages // 2 + 5, pages - 1, pages - 7]
    cache[places] = torch.randn((4, 64, 576), generator=g, device="cuda").to(BF16)
    q, qp = _queries(g, 1, 1, 16, BF16)
    pt, sl = torch.tensor([places], dtype=torch.int32, device="cuda"), torch.tensor([250], dtype=torch.int32, device="cuda")
    out = mla.mla_decode_attention(q, qp, cache, pt, sl, SCALE)
    want, _, tol, _ = R.decode(q, qp, cache[places], [[0, 1, 2, 3]], [250], SCALE, None)
    R.close(out, want, tol)
    rows = mla.mla_gather_cache(cache, pt, torch.tensor([0, 250], dtype=torch.int32, device="cuda"), 250)
    assert torch.equal(rows, cache[places].view(-1, 576)[:250])
    slots = torch.tensor([(pages - 1) * 64 + 63, 5], device="cuda")
    latent = torch.randn((2, 576), generator=g, device="cuda").to(BF16)
    mla.mla_write_cache(latent, cache, slots)
    assert torch.equal(cache.view(-1, 576)[slots], latent)


# ---------------------------------------------------------------------------------------------------------------- prefill


def _prefill_inputs(g, lq, lk, H, dtype, slack=3):
    """Queries and keys of all sequences, with NaN behind the last; keys and values as halves of one tensor."""
    cu_q, cu_k = [0], [0]
    for a, b in zip(lq, lk):
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
    q = torch.randn((cu_q[-1] + slack, H, 192), generator=g, device="cuda").to(dtype)
    kv = torch.randn((cu_k[-1] + slack, H, 256), generator=g, device="cuda").to(dtype)
    pe = torch.randn((cu_k[-1] + slack, 64), generator=g, device="cuda").to(dtype)
    q[cu_q[-1]:], kv[cu_k[-1]:], pe[cu_k[-1]:] = NAN, NAN, NAN
    to = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, kv[..., :128], pe, kv[..., 128:], cu_q, cu_k, to(cu_q), to(cu_k)


def _check_prefill(lq, lk, H, dtype, causal, seed=0):
    from sglang_amd import mla

    q, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(_gen(seed), lq, lk, H, dtype)
    out = torch.full((q.shape[0], H, 128), 7.0, dtype=dtype, device="cuda")
    got, lse = mla.mla_prefill_attention(q, kn, kp, v, tq, tk, max(lq), SCALE, causal=causal, return_lse=True, out=out)
    assert got is out and bool((out[cu_q[-1]:] == 7.0).all())
    want, want_lse, tol, lse_tol = R.prefill(q, kn, kp, v, cu_q, cu_k, SCALE, causal)
    R.close(out[:cu_q[-1]], want, tol, "out")
    R.close(lse[:cu_q[-1]], want_lse, lse_tol, "lse")
    # a larger bound may cut the keys otherwise; the same call gives the same bits
    again = mla.mla_prefill_attention(q, kn, kp, v, tq, tk, max(lq) + 500, SCALE, causal=causal)
    R.close(again[:cu_q[-1]], want, tol, "out")
    assert torch.equal(mla.mla_prefill_attention(q, kn, kp, v, tq, tk, max(lq), SCALE, causal=causal)[:cu_q[-1]], out[:cu_q[-1]])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1], [200]), ([130], [130]), ([64, 0, 3, 129], [64, 5, 70, 129]), ([5, 100], [0, 40]), ([300], [1000]),
                                   ([128, 127, 1, 33, 32, 31], [128, 191, 64, 33, 96, 500]), ([200], [17])], ids=str)
@pytest.mark.parametrize("H", [1, 5, 16])
def test_prefill(dev, lq, lk, H, causal, dtype):
    _check_prefill(lq, lk, H, dtype, causal, seed=sum(lq) + H)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,lk,H", [([2000, 777], [2000, 3333], 3), ([16], [9000], 4), ([1], [4097], 1), ([130, 0, 5], [5000, 3000, 0], 2), ([40], [20], 3)], ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_over_split_keys(dev, lq, lk, H, causal, dtype):
    """Few queries over long keys: the keys of a block are split, down to splits without a tile, and joined."""
    _check_prefill(lq, lk, H, dtype, causal, seed=H)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,lk,H,causal", [([256], [256], 3, False), ([256], [1100], 3, True), ([251, 256], [1600, 650], 2, True), ([480], [480], 150, False),
                                            ([1000], [4100], 40, True), ([230, 256, 250], [0, 900, 7], 2, False), ([512, 512], [4000, 97], 1, True)], ids=str)
def test_prefill_in_large_blocks(dev, lq, lk, H, causal, dtype):
    """Queries that fill blocks of 256 and have many keys: eight waves to a workgroup, the keys split and not; sequences without keys, and with few, among them."""
    _check_prefill(lq, lk, H, dtype, causal, seed=H)


def test_prefill_of_many_blocks(dev):
    """More workgroups than run at once: no splits, long and short blocks by turns."""
    _check_prefill([700, 130, 1500], [700, 400, 1500], 64, BF16, True)


def test_prefill_of_far_keys(dev):
    """Keys and values whose rows lie beyond 2^32 bytes, split and not."""
    from sglang_amd import mla

    g = _gen(13)
    tk = (1 << 33) // (128 * 256 * 2) + 700
    kv = torch.empty((tk, 128, 256), dtype=BF16, device="cuda")
    pe = torch.randn((tk, 64), generator=g, device="cuda").to(BF16)
    ends = [tk - 1500, tk - 700, tk]
    for h in (0, 1):
        kv[ends[0]:, h] = torch.randn((1500, 256), generator=g, device="cuda").to(BF16)
    q = torch.randn((150, 2, 192), generator=g, device="cuda").to(BF16)
    tq = torch.tensor([0, 30, 150], dtype=torch.int32, device="cuda")
    tk_ = torch.tensor(ends, dtype=torch.int32, device="cuda")
    for most in (120, 1 << 15):
        out = mla.mla_prefill_attention(q, kv[:, :2, :128], pe, kv[:, :2, 128:], tq, tk_, most, SCALE)
        want, _, tol, _ = R.prefill(q, kv[:, :2, :128], pe, kv[:, :2, 128:], [0, 30, 150], ends, SCALE, True)
        R.close(out, want, tol)


def test_prefill_layouts(dev):
    from sglang_amd import mla

    q, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(_gen(5), [70, 90], [70, 200], 4, BF16, slack=0)
    want, lse = mla.mla_prefill_attention(q, kn, kp, v, tq, tk, 90, SCALE, return_lse=True)
    for args in ((q, kn, kp.unsqueeze(1), v), (q, kn.contiguous(), kp, v.contiguous()), (q.transpose(0, 1).contiguous().transpose(0, 1), kn, kp, v)):
        got, s = mla.mla_prefill_attention(*args, tq, tk, 90, SCALE, return_lse=True)
        assert torch.equal(got, want) and torch.equal(s, lse)
    odd = torch.zeros((160, 4, 196), dtype=BF16, device="cuda")
    odd[..., 4:] = q
    wide = torch.zeros((270, 2, 64), dtype=BF16, device="cuda")
    wide[:, 1] = kp
    assert torch.equal(mla.mla_prefill_attention(odd[..., 4:], kn, wide[:, 1], v, tq, tk, 90, SCALE), want)
    # queries beyond the stated maximum, 128 to a block, are left out: those of the first block are not
    assert torch.equal(mla.mla_prefill_attention(q, kn, kp, v, tq, tk, 90, SCALE, out=torch.zeros_like(want)), want)
    assert mla.mla_prefill_attention(q[:0], kn, kp, v, tq * 0, tk, 0, SCALE).shape == (0, 4, 128)
    o, s = mla.mla_prefill_attention(q, kn[:0], kp[:0], v[:0], tq, tk * 0, 90, SCALE, return_lse=True)
    assert not o.any() and bool((s == float("-inf")).all())
    # bounds outside the tensors are held to them: no read leaves them
    far = torch.tensor([0, 70, 1 << 30], dtype=torch.int32, device="cuda")
    got = mla.mla_prefill_attention(q, kn, kp, v, far, torch.tensor([0, 70, 1 << 30], dtype=torch.int32, device="cuda"), 90, SCALE)
    assert torch.equal(got, want)


@pytest.mark.parametrize("order", [1, -1])
def test_prefill_scores_that_raise_the_maximum(dev, order):
    from sglang_amd import mla

    q, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(_gen(9), [150], [700], 2, BF16, slack=0)
    direction = torch.sign(torch.randn((128,), generator=_gen(1), device="cuda"))
    size = torch.linspace(0, 1, 700, device="cuda")
    size = size if order > 0 else size.flip(0)
    kn.copy_((kn.float() * 0.1 + 5.0 * size[:, None, None] * direction).to(BF16))
    q[..., :128] = (q[..., :128].float() * 0.1 + direction).to(BF16)
    for causal in (True, False):
        out, lse = mla.mla_prefill_attention(q, kn, kp, v, tq, tk, 150, SCALE, causal=causal, return_lse=True)
        want, want_lse, tol, lse_tol = R.prefill(q, kn, kp, v, cu_q, cu_k, SCALE, causal)
        R.close(out, want, tol, "out")
        R.close(lse, want_lse, lse_tol, "lse")


# ---------------------------------------------------------------------------------------------------------------- cache


def _table_of_angles(positions):
    inverse = 10000.0 ** (-torch.arange(0, 64, 2, device="cuda", dtype=torch.float64) / 64)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inverse
    return torch.cat((a.cos(), a.sin()), 1).float()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H,norm,neox,ints", [(1, 1, "own", False, torch.int64), (5, 16, "f32", True, torch.int32), (67, 3, None, False, torch.int32),
                                                (300, 128, "own", True, torch.int64), (4, 0, "own", None, torch.int64)])
def test_write_cache(dev, T, H, norm, neox, ints, dtype, fp8):
    from sglang_amd import mla

    g = _gen(T + H)
    pages, page = T // 16 + 3, 16
    latent = (torch.randn((T, 640), generator=g, device="cuda") * 3).to(dtype)[:, :576]
    weight = 1 + 0.3 * torch.randn((512,), generator=g, device="cuda")
    weight = {None: None, "own": weight.to(dtype), "f32": weight}[norm]
    order = torch.randperm(pages * page, generator=g, device="cuda")[:T].to(ints)
    slots = order.clone()
    if T > 4:
        slots[1], slots[3] = -1, pages * page
    table = _table_of_angles(5000) if neox is not None else None
    pos = torch.randint(0, 5000, (T,), generator=g, device="cuda").to(ints) if neox is not None else None
    if T > 4:
        pos[2] = 0
    q = torch.randn((T, H, 192), generator=g, device="cuda").to(dtype)[..., 128:] if H else None
    scale = torch.full((1,), 0.02, device="cuda") if fp8 else None
    cache = torch.full((pages, page, 576), 5.0, device="cuda").to(F8 if fp8 else dtype)
    before = cache.clone()
    kept = q.clone() if H else None
    got_q = mla.mla_write_cache(latent, cache, slots, norm_weight=weight, eps=1e-5, cos_sin=table, positions=pos, neox=bool(neox), q_pe=q, scale=scale)

    x = latent.double()
    c, pe = x[:, :512], x[:, 512:]
    if weight is not None:
        c = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * weight.double()
    size = pe.abs()
    if table is not None:
        pe, size = R.rotate(pe, table.double()[pos.long()], neox)
    want = torch.cat((c, pe), 1)
    slack = torch.cat((c.abs() * 2.0 ** -19, size * 2.0 ** -22), 1)
    stored = [i for i in range(T) if not (T > 4 and i in (1, 3))]
    where = slots[stored].long()
    if fp8:
        code = cache.view(-1, 576).view(torch.uint8)[where].view(F8).double()
        exact = (want[stored] / 0.02).clamp(-448, 448)
        slack = slack[stored] / 0.02 + exact.abs() * 2.0 ** -22
        # half a step of e4m3 around the value: 2^-4 relative, 2^-10 below the normal range
        R.close(code, exact, torch.maximum(exact.abs() * 2.0 ** -4, torch.full_like(exact, 2.0 ** -10)) + slack, "codes")
    else:
        R.close(cache.view(-1, 576)[where], want[stored], want[stored].abs() * R.half_step(dtype) + slack[stored] + 2.0 ** -25, "rows")
    untouched = torch.ones((pages * page,), dtype=torch.bool, device="cuda")
    untouched[where] = False
    assert torch.equal(cache.view(-1, 576).view(torch.uint8)[untouched], before.view(-1, 576).view(torch.uint8)[untouched])
    if not H:
        assert got_q is None
        return
    w, size = R.rotate(q.double(), table.double()[pos.long()][:, None], neox)
    tol = w.abs() * R.half_step(dtype) + size * 2.0 ** -22 + 2.0 ** -25
    R.close(got_q, w, tol, "queries")
    assert torch.equal(q, kept) and got_q.is_contiguous()
    # in place, and into a place that is copied to
    whole = torch.randn((T, H, 192), generator=g, device="cuda").to(dtype)
    whole[..., 128:] = q
    place = whole[..., 128:]
    head = whole[..., :128].clone()
    assert mla.mla_write_cache(latent, cache, slots, norm_weight=weight, eps=1e-5, cos_sin=table, positions=pos, neox=bool(neox), q_pe=place, q_out=place,
                               scale=scale) is place
    assert torch.equal(place, got_q) and torch.equal(whole[..., :128], head)
    odd = torch.zeros((T, H, 66), dtype=dtype, device="cuda")
    mla.mla_write_cache(latent, cache, slots, norm_weight=weight, eps=1e-5, cos_sin=table, positions=pos, neox=bool(neox), q_pe=q, q_out=odd[..., 1:65], scale=scale)
    assert torch.equal(odd[..., 1:65], got_q)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_write_cache_of_unusual_values(dev, dtype):
    """Zeros, the smallest and the largest numbers, infinities, NaN; an 8-bit cache takes what is too large as 448 and keeps NaN."""
    from sglang_amd import mla

    latent = torch.zeros((4, 576), dtype=dtype, device="cuda")
    top = torch.finfo(dtype).max
    latent[1, :8] = torch.tensor([top, -top, float("inf"), -float("inf"), NAN, 1e-30, 449.0, -465.0], device="cuda").to(dtype)
    latent[2] = 2.0 ** -10
    latent[3, 512:520] = latent[1, :8]
    slots = torch.arange(4, device="cuda")
    cache = torch.empty((1, 4, 576), dtype=dtype, device="cuda")
    mla.mla_write_cache(latent, cache, slots)
    assert torch.equal(cache[0].view(torch.int16), latent.view(torch.int16))
    cache8 = torch.empty((1, 4, 576), dtype=F8, device="cuda")
    mla.mla_write_cache(latent, cache8, slots)
    want = latent.float().clamp(-448, 448).to(F8)
    assert torch.equal(torch.nan_to_num(cache8[0].float(), nan=1e9), torch.nan_to_num(want.float(), nan=1e9))
    # a row of zeros stays one under the norm
    mla.mla_write_cache(latent[:1].contiguous(), cache, slots[:1], norm_weight=torch.ones((512,), device="cuda"))
    assert not cache[0, 0].any()


@pytest.mark.parametrize("dtype,fp8", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("lens,starts", [([5], None), ([100, 0, 1, 64, 33], None), ([0], None), ([7, 20, 0, 64], [60, 0, 3, 1])])
@pytest.mark.parametrize("page", [1, 16, 5])
def test_gather_cache(dev, lens, starts, page, dtype, fp8):
    from sglang_amd import mla

    whole = [a + b for a, b in zip(lens, starts or [0] * len(lens))]
    cache, table, pt, scale = _filled(_gen(page), whole, page, dtype, fp8)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    to = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    total = cu[-1] + 4
    out = torch.full((total, 584), 3.0, dtype=dtype, device="cuda")[:, :576]
    got = mla.mla_gather_cache(cache, pt, to(cu), total, starts=None if starts is None else to(starts), dtype=dtype, scale=scale, out=out)
    assert got is out and bool((out[cu[-1]:] == 3.0).all())
    flat = cache.view(-1, 576)
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda") + (starts[b] if starts else 0)
        rows = torch.tensor(table[b], device="cuda")[t // page] * page + t % page
        if fp8:
            want = (flat.view(torch.uint8)[rows].view(F8).float() * scale).to(dtype)
        else:
            want = flat[rows]
        assert torch.equal(out[cu[b]:cu[b + 1]], want)
    fresh = mla.mla_gather_cache(cache, pt, to(cu), total, starts=None if starts is None else to(starts), dtype=dtype, scale=scale)
    assert fresh.shape == (total, 576) and fresh.dtype == dtype and torch.equal(fresh[:cu[-1]], out[:cu[-1]])
    odd = torch.full((total, 577), 3.0, dtype=dtype, device="cuda")
    mla.mla_gather_cache(cache, pt, to(cu), total, starts=None if starts is None else to(starts), dtype=dtype, scale=scale, out=odd[:, 1:])
    assert torch.equal(odd[:, 1:], out) and bool((odd[:, 0] == 3.0).all())


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
@pytest.mark.parametrize("shape,D", [((1,), 8), ((37, 16), 128), ((5, 3, 7), 512), ((0, 4), 128), ((2000,), 64)])
def test_merge(dev, shape, D, dtype):
    from sglang_amd import mla

    g = _gen(D)
    a, b = (torch.randn(shape + (D,), generator=g, device="cuda").to(dtype) for _ in range(2))
    la, lb = (torch.randn(shape, generator=g, device="cuda") * 5 for _ in range(2))
    if la.numel() > 30:
        la.view(-1)[3], lb.view(-1)[4] = float("-inf"), float("-inf")
        la.view(-1)[5] = lb.view(-1)[5] = float("-inf")
        la.view(-1)[6], la.view(-1)[7] = 100.0, -300.0
        a.view(-1, D)[3], b.view(-1, D)[4], a.view(-1, D)[5] = NAN, float("inf"), NAN
    out, lse = mla.merge_attention_states(a, la, b, lb)
    assert out.shape == a.shape and out.dtype == dtype and lse.shape == la.shape and lse.dtype == torch.float32
    both = torch.stack((la, lb)).double()
    want_lse = torch.logsumexp(both, 0)
    share = torch.where(both == float("-inf"), 0.0, torch.exp(both - want_lse))[..., None]
    za, zb = (torch.where((s == 0), 0.0, t.double()) for s, t in zip(share, (a, b)))
    want = share[0] * za + share[1] * zb
    # an exponential's relative error: the rounding of its argument, up to |la - lb| * 1.44 * 2^-23, and its own; a float32 sum and quotient
    gap = torch.where(torch.isfinite(both).all(0), (both[0] - both[1]).abs(), 0.0)
    slack = (gap * 2.0 ** -22 + 2.0 ** -20)[..., None] * (share[0] * za.abs() + share[1] * zb.abs())
    R.close(out, want, want.abs() * R.half_step(dtype) + slack + (2.0 ** -25 if dtype == F16 else 1e-30), "out")
    R.close(lse, want_lse, torch.where(torch.isfinite(want_lse), want_lse, 0.0).abs() * 2.0 ** -22 + 2.0 ** -20, "lse")
    if len(shape) == 2 and shape[0]:
        wide = torch.zeros(shape + (D + 4,), dtype=dtype, device="cuda")
        wide[..., 4:] = a
        o2, l2 = mla.merge_attention_states(wide[..., 4:], la.t().contiguous().t(), b, lb)
        assert torch.equal(torch.nan_to_num(o2), torch.nan_to_num(out)) and torch.equal(l2, lse)


# ---------------------------------------------------------------------------------------------------------------- streams, graphs, compile


def test_decode_in_graphs(dev):
    """Two captured calls on buffers of their own; lengths and queries change between replays, eager calls run between them."""
    from sglang_amd import mla

    g = _gen(21)
    cases = []
    for lens, H in (([700, 90], 128), ([64] * 6, 16)):
        cache, table, pt, _ = _filled(g, [800] * len(lens), 64, BF16, False)
        q, qp = (t.contiguous() for t in _queries(g, len(lens), 1, H, BF16))
        cases.append((q, qp, cache, pt, torch.tensor(lens, dtype=torch.int32, device="cuda")))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for c in cases:
        with torch.cuda.stream(side):
            mla.mla_decode_attention(*c, SCALE, return_lse=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = mla.mla_decode_attention(*c, SCALE, return_lse=True)
        graphs.append((graph, res))
    for turn in range(4):
        for i, c in enumerate(cases):
            c[0].normal_(generator=g)
            c[4].copy_(torch.randint(0, 801, c[4].shape, generator=g, device="cuda"))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in cases]
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for c, (_, (out, lse)) in zip(cases, graphs):
            want, want_lse = mla.mla_decode_attention(*c, SCALE, return_lse=True)
            assert torch.equal(out, want) and torch.equal(lse, want_lse), turn


def test_whole_step_in_a_graph_and_on_another_stream(dev):
    from sglang_amd import mla

    g = _gen(31)
    B, H = 6, 16
    lens = [100, 64, 1, 65, 300, 2]
    cache, table, pt, scale = _filled(g, [400] * B, 64, BF16, True)
    table_cs = _table_of_angles(500)
    latent, w = torch.randn((B, 576), generator=g, device="cuda").to(BF16), torch.ones((512,), dtype=BF16, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, qp = (t.contiguous()[:, 0] for t in _queries(g, B, 1, H, BF16))

    def step():
        pos = (sl - 1).long()
        slots = pt.gather(1, (pos // 64)[:, None])[:, 0].long() * 64 + pos % 64
        rot = mla.mla_write_cache(latent, cache, slots, norm_weight=w, cos_sin=table_cs, positions=pos, q_pe=qp, scale=scale)
        return mla.mla_decode_attention(q, rot, cache, pt, sl, SCALE, scale=scale)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        latent.normal_(generator=g)
        sl.copy_(torch.randint(1, 401, (B,), generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, step()), turn
    assert first.shape == (B, H, 512)


def test_prefill_in_graphs(dev):
    """Two captured chains, each a prompt's chunk over split keys and its cached prefix's rows, joined; lengths change between replays on two streams."""
    from sglang_amd import mla

    g = _gen(33)
    to = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cases = []
    for H, dtype in ((3, BF16), (2, F16)):
        cache, table, pt, _ = _filled(g, [1900], 64, dtype, False)
        rand = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)  # noqa: E731, B023
        cases.append([rand(256, H, 192), rand(3000, H, 128), rand(3000, 64), rand(3000, H, 128), to(0, 256), to(0, 3000), cache, pt, to(0, 1900)])

    def chain(q, kn, kp, v, cu_q, cu_k, cache, pt, cu_p):
        own, s = mla.mla_prefill_attention(q, kn, kp, v, cu_q, cu_k, 256, SCALE, return_lse=True)
        rows = mla.mla_gather_cache(cache, pt, cu_p, 1900, dtype=q.dtype)
        keys = rows[:, None, :128].expand(-1, q.shape[1], -1).contiguous()
        pre, ps = mla.mla_prefill_attention(q, keys, rows[:, 512:], keys, cu_q, cu_p, 256, SCALE, causal=False, return_lse=True)
        return mla.merge_attention_states(own, s, pre, ps)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for c in cases:
        with torch.cuda.stream(side):
            chain(*c)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = chain(*c)
        graphs.append((graph, res))
    for turn in range(4):
        for i, c in enumerate(cases):
            c[0].normal_(generator=g)
            c[4].copy_(to(0, 256 - 50 * turn))
            c[5].copy_(to(0, 3000 - 700 * turn * i))
            c[8].copy_(to(0, (1900, 64, 0, 1000)[turn]))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in cases]
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for c, (_, got) in zip(cases, graphs):
            n = 256 - 50 * turn
            for a, b in zip(got, chain(*c)):
                assert torch.equal(a[:n], b[:n]) and bool(torch.isfinite(a[:n]).all()), turn


def test_calls_of_two_threads(dev):
    """Two threads, a stream each, make calls at once; every result is that of a call alone."""
    import threading

    from sglang_amd import mla

    g = _gen(35)
    work = []
    for lens, H in (([1200, 30, 500], 128), ([90] * 20, 16)):
        cache, table, pt, _ = _filled(g, lens, 64, BF16, False)
        q, qp = _queries(g, len(lens), 1, H, BF16)
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        pq, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(g, [40], [2000 + H], 2, BF16, slack=0)
        work.append(lambda a=(q, qp, cache, pt, sl, SCALE), b=(pq, kn, kp, v, tq, tk, 40, SCALE): (mla.mla_decode_attention(*a), mla.mla_prefill_attention(*b)))
    want = [fn() for fn in work]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] += [work[i]() for _ in range(10)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for w, results in zip(want, got):
        assert len(results) == 10 and all(torch.equal(x, y) for r in results for x, y in zip(w, r))


def test_decode_of_a_shared_row_of_pages(dev):
    """Requests that share one row of the page table, which is expanded rather than copied; one request twice."""
    from sglang_amd import mla

    g = _gen(37)
    cache, table, pt, _ = _filled(g, [700], 16, BF16, False)
    q, qp = _queries(g, 4, 2, 16, BF16)
    q[3], qp[3] = q[1], qp[1]
    sl = torch.tensor([700, 65, 1, 65], dtype=torch.int32, device="cuda")
    out = mla.mla_decode_attention(q, qp, cache, pt.expand(4, -1), sl, SCALE)
    assert torch.equal(out, mla.mla_decode_attention(q, qp, cache, pt.repeat(4, 1), sl, SCALE))
    want, _, tol, _ = R.decode(q, qp, cache, table * 4, sl.tolist(), SCALE, None)
    R.close(out, want, tol, "out")


def test_compiled(dev):
    from sglang_amd import mla

    g = _gen(41)
    lens = [100, 30]
    cache, table, pt, _ = _filled(g, lens, 16, BF16, False)
    q, qp = _queries(g, 2, 1, 16, BF16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pq, kn, kp, v, cu_q, cu_k, tq, tk = _prefill_inputs(g, [20, 30], [20, 60], 2, BF16, slack=0)
    latent, slots = torch.randn((2, 576), generator=g, device="cuda").to(BF16), torch.tensor([0, 1], device="cuda")
    table_cs, pos = _table_of_angles(64), torch.tensor([5, 9], device="cuda")

    def step(cache):
        rot = mla.mla_write_cache(latent, cache, slots, cos_sin=table_cs, positions=pos, q_pe=qp[:, 0])
        o, s = mla.mla_decode_attention(q[:, 0], rot, cache, pt, sl, SCALE, return_lse=True)
        rows = mla.mla_gather_cache(cache, pt, torch.tensor([0, 100, 130], dtype=torch.int32, device="cuda"), 130)
        po, ps = mla.mla_prefill_attention(pq, kn, kp, v, tq, tk, 30, SCALE, return_lse=True)
        return o, s, rows, mla.merge_attention_states(po, ps, po, ps)[0]

    ours, theirs = cache.clone(), cache.clone()
    eager = step(ours)
    traced = torch.compile(step, backend="aot_eager")(theirs)
    for a, b in zip(eager, traced):
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))
    assert torch.equal(torch.nan_to_num(ours), torch.nan_to_num(theirs))


# ---------------------------------------------------------------------------------------------------------------- together


def test_prefill_behind_a_prefix_then_decode(dev):
    """A layer's attention as it runs: a prompt's first chunk, a second one behind the cached first (gathered rows, up-projection, attention without
    mask, join), then a decoded token on the absorbed path, all against one attention over the whole in float64.

    Both forms round the up-projected keys and values (or the absorbed queries and results) to bf16: every score is off by up to
    2 u * scale * sum |q k|, which is taken twice; results by u * a on top."""
    from sglang_amd import mla

    g = _gen(51)
    H, first, second = 4, 150, 90
    T = first + second + 1
    hidden = torch.randn((T, 576), generator=g, device="cuda").to(BF16)
    weight = torch.ones((512,), dtype=BF16, device="cuda")
    up = torch.randn((H, 256, 512), generator=g, device="cuda").mul_(512 ** -0.5).to(BF16)  # keys' rows, then values'
    q = torch.randn((T, H, 192), generator=g, device="cuda").to(BF16)
    cs, pos = _table_of_angles(T), torch.arange(T, device="cuda")
    cache = torch.full((6, 64, 576), NAN, dtype=BF16, device="cuda")
    pages = torch.tensor([[4, 1, 3, 0]], dtype=torch.int32, device="cuda")
    slots = pages[0].long()[pos // 64] * 64 + pos % 64
    to = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def expand(rows):
        kv = (rows[:, :512].float() @ up.float().view(H * 256, 512).t()).to(BF16).view(-1, H, 256)
        return kv[..., :128], rows[:, 512:], kv[..., 128:]

    outs = []
    rotated = torch.empty((T, H, 64), dtype=BF16, device="cuda")
    for a, b in ((0, first), (first, first + second), (T - 1, T)):
        rotated[a:b] = mla.mla_write_cache(hidden[a:b], cache, slots[a:b], norm_weight=weight, cos_sin=cs, positions=pos[a:b], q_pe=q[a:b, :, 128:])
        qr = torch.cat((q[a:b, :, :128], rotated[a:b]), -1)
        if b == T:
            absorbed = torch.matmul(q[a:b, :, :128].float().transpose(0, 1), up[:, :128].float()).to(BF16).transpose(0, 1)
            o = mla.mla_decode_attention(absorbed, rotated[a:b], cache, pages, to(T), SCALE)
            outs.append(torch.matmul(o.float().transpose(0, 1), up[:, 128:].float().transpose(1, 2).contiguous()).to(BF16).transpose(0, 1))
            continue
        kn, kp, v = expand(cache.view(-1, 576)[slots[a:b]])
        o, s = mla.mla_prefill_attention(qr, kn, kp, v, to(0, b - a), to(0, b - a), b - a, SCALE, return_lse=True)
        if a:
            kn, kp, v = expand(mla.mla_gather_cache(cache, pages, to(0, a), a))
            po, ps = mla.mla_prefill_attention(qr, kn, kp, v, to(0, b - a), to(0, a), b - a, SCALE, causal=False, return_lse=True)
            o, s = mla.merge_attention_states(o, s, po, ps)
        outs.append(o)
    got = torch.cat(outs)

    rows = cache.view(-1, 576)[slots].double()
    u = R.half_step(BF16)
    for h in range(H):
        k = torch.cat((rows[:, :512] @ up[h, :128].double().t(), rows[:, 512:]), -1)
        v = rows[:, :512] @ up[h, 128:].double().t()
        qh = torch.cat((q[:, h, :128], rotated[:, h]), -1).double()
        s = (qh @ k.t()) * SCALE
        seen = torch.arange(T, device="cuda")[None] <= torch.arange(T, device="cuda")[:, None]
        p = torch.softmax(torch.where(seen, s, float("-inf")), -1)
        # the absorbed query is a rounded sum over 128, what multiplies it rows of 512: |row| . (|up| |q|) bounds the size of its error
        size = rows[:, :512].abs() @ up[h, :128].double().abs().t()
        ds = 2 * u * SCALE * torch.where(seen, qh[:, :128].abs() @ size.t(), 0.0).max(-1, keepdim=True).values
        mean = p @ (rows[:, :512].abs() @ up[h, 128:].double().abs().t())
        R.close(got[:, h], p @ v, u * (p @ v).abs() + (4 * u + 2 * ds) * mean, "head %d" % h)


def test_decode_between_the_absorbed_products(dev):
    """per_tensor_quant_mla_fp8 and bmm_fp8 on either side of the attention, as the layer calls them; against the same products of the
    values that the 8-bit operands stand for, to the tolerance of the products' own tests (1e-2 of the largest)."""
    from sglang_amd import mla
    from sglang_amd.fp8_kernel import per_tensor_quant_mla_fp8
    from sglang_amd.sgl_kernel import bmm_fp8

    g = _gen(61)
    H, B = 16, 5
    lens = [70, 1, 200, 64, 33]
    cache, table, pt, scale = _filled(g, lens, 64, BF16, True)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((B, H, 192), generator=g, device="cuda").to(BF16)
    w_kc, w_vc = ((torch.randn(s, generator=g, device="cuda") * 0.05 / 0.001).clamp(-448, 448).to(F8) for s in ((H, 512, 128), (H, 128, 512)))
    ws = torch.full((1,), 0.001, device="cuda")

    def product(x, w):  # x [B, H, k] -> [B, H, n]
        zero = torch.zeros((1,), device="cuda")
        xq, xs = per_tensor_quant_mla_fp8(x.transpose(0, 1), zero)
        return bmm_fp8(xq, w.transpose(1, 2), xs, ws, BF16).transpose(0, 1), torch.matmul(xq.float() * xs, (w.float() * ws).transpose(1, 2).contiguous()).transpose(0, 1)

    absorbed, plain = product(q[..., :128], w_kc)
    assert float((absorbed.float() - plain).abs().max() / plain.abs().max()) <= 1e-2
    out = mla.mla_decode_attention(absorbed, q[..., 128:], cache, pt, sl, SCALE, scale=scale)
    want, _, tol, _ = R.decode(absorbed[:, None], q[:, None, :, 128:], cache, table, lens, SCALE, scale)
    R.close(out[:, None], want, tol)
    result, plain = product(out, w_vc)
    assert float((result.float() - plain).abs().max() / plain.abs().max()) <= 1e-2
