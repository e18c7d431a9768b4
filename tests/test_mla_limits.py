"""Latent attention at the limits of what its calls allow, without a GPU: sizes of workspaces, and what the C entry points refuse."""
import pytest


@pytest.mark.parametrize("n,H,max_len", [(1, 128, 256), (1, 16, 4096), (2, 128, 64), (4, 64, 131072), (1, 1, 1)])
def test_decode_workspace_goes_by_runs(n, H, max_len):
    """A run leaves at most two partials, and there are at most 256 runs, whatever the batch; beside them 8 bytes to a request."""
    from sglang_amd._lib import lib

    size = lambda B: lib.fp8k_mla_decode_workspace_bytes(B, n, H, max_len)  # noqa: E731
    for B in (1, 2, 100, 255, 256, 257, 600, 2048, 4096, 65535):
        if B * (max_len // 64 + 1) >= 1 << 30:
            continue
        assert size(B) <= min(512, 256 + B) * n * H * (512 + 1) * 4 + 8 * B + 3 * 256
    if 65535 * (max_len // 64 + 1) < 1 << 30:
        assert size(65535) - size(4096) <= 8 * (65535 - 4096) + 256


def test_assembly_names_the_registers_that_it_sets():
    """An asm statement that sets m0 says so, or the compiler may keep something of its own there across it."""
    import pathlib
    import re

    import sglang_amd

    found = 0
    for path in (pathlib.Path(sglang_amd.__file__).parent / "csrc").glob("*.h*"):
        for text in re.findall(r"\basm\b[^;]*;", path.read_text()):
            if re.search(r"s_mov_b32 m0", text):
                found += 1
                assert '"m0"' in text, (path.name, text)
    assert found == 3


def _address(size):
    import ctypes

    buf = ctypes.create_string_buffer(size + 256)
    return buf, (ctypes.addressof(buf) + 255) // 256 * 256


def _refused(rc, *words):
    from sglang_amd._lib import lib

    text = lib.fp8k_last_error().decode()
    assert rc != 0 and all(w in text for w in words), (rc, text)


def test_joined_rows_and_logarithms_are_memory_of_their_own():
    """3 rows of 192 numbers, 1152 bytes in 16 bits: a result that begins or ends inside an operand, or holds its own logarithms, is refused."""
    from sglang_amd import _lib

    keep, p = _address(1 << 14)
    a, b, out, la, lb, lse = (p + 2048 * i for i in range(6))

    def merge(out=out, lse=lse, a=a, b=b, la=la, lb=lb, dtype=_lib.BF16):
        return _lib.lib.fp8k_merge_attention_states(a, la, b, lb, out, lse, 3, 192, dtype, None)

    for x in (a, b):
        for off in (16, -16, 1136, -1136):
            _refused(merge(out=x + off), "out must be")
    _refused(merge(out=a + 1152, b=a, dtype=_lib.F32), "out must be")
    for x in (la, lb):
        for off in (4, 8, -4, -8):
            _refused(merge(lse=x + off), "lse must be")
    _refused(merge(lse=a + 1148), "lse must be")
    _refused(merge(lse=b - 8), "lse must be")
    _refused(merge(lse=out + 1148), "lse must be")
    _refused(merge(la=out + 1144), "out must be")
    _refused(merge(lb=out - 8), "out must be")
    del keep


def _write_with_bad_weight(q, qt, qh, out, ot, oh, T, H):
    """What the writer says of these queries and their places.  Nothing is ever launched: the norm's weight is of a wrong type, and looked at last."""
    from sglang_amd import _lib

    p = 1 << 20
    rc = _lib.lib.fp8k_mla_write_cache(p, 576, p, p, 1, p, _lib.F16, 1e-6, p, 10, p, 1, 0, q, qt, qh, out, ot, oh, None, T, H, 100, _lib.BF16, 0, None)
    text = _lib.lib.fp8k_last_error().decode()
    assert rc != 0 and ("weight" in text or "overlap" in text), text
    return "overlap" in text


def test_rotated_queries_share_no_memory_with_others():
    """Every place among some thousand random ones against the numbers that it holds: what overlaps is refused, the queries' own place and places with their
    strides are taken whenever they may be."""
    import random

    rng = random.Random(3)
    base = 1 << 30
    seen = {"overlap": 0, "apart": 0, "in place": 0, "other strides": 0}
    for _ in range(4000):
        T, H = rng.choice([(1, 1), (1, 5), (4, 1), (3, 4), (2, 7), (6, 3)])
        nest = lambda: rng.choice([(64 * H, 64), (192 * H, 192), (192 * H + 64, 192), (64, 64 * T), (72, 72 * T), (192 * H + 576, 192), (64 * H + 8, 64)])  # noqa: E731
        (qt, qh), (ot, oh) = nest(), nest()
        if rng.random() < 0.6:
            ot, oh = qt, qh
        if rng.random() < 0.1:
            qh = 0
        delta = rng.choice([0, 0, 64, -64, 128, 8 * rng.randint(-300, 300), rng.choice([1, -1]) * (ot * rng.randint(0, 3) + oh * rng.randint(0, 3)), qt * rng.randint(-2, 2) + 64])
        rows = lambda st, sh, at: {at + t * st + h * sh + i for t in range(T) for h in range(H) for i in range(64)}  # noqa: E731
        own = delta == 0 and (T == 1 or qt == ot) and (H == 1 or qh == oh)
        if len(rows(ot, oh, 0)) < T * H * 64:
            continue  # places that overlap each other are another refusal
        refused = _write_with_bad_weight(base, qt, qh, base + 2 * delta, ot, oh, T, H)
        collide = bool(rows(qt, qh, 0) & rows(ot, oh, delta)) and not own
        what = (T, H, qt, qh, ot, oh, delta)
        if collide:
            assert refused, what
        elif (T == 1 or qt == ot) and (H == 1 or qh == oh):
            assert not refused, what
        seen["overlap" if collide else "in place" if own else "apart" if (qt, qh) == (ot, oh) else "other strides"] += 1
    assert min(seen.values()) > 50, seen
    # slices of one buffer: heads' 64 of 192, tokens of 8 heads and 576 more; the result behind the heads, or between them
    assert not _write_with_bad_weight(base + 256, 8 * 192 + 576, 192, base + 2 * 8 * 192, 8 * 192 + 576, 64, 30, 8)
    assert not _write_with_bad_weight(base + 256, 8 * 192, 192, base, 8 * 192, 192, 30, 8)
    assert not _write_with_bad_weight(base, 8 * 192, 192, base + 2 * 64, 64 * 192, 192, 30, 8)  # other strides, a common divisor
    assert _write_with_bad_weight(base, 8 * 192, 192, base + 2 * 192, 8 * 192, 192, 30, 8)  # one head on
    assert _write_with_bad_weight(base, 8 * 192, 192, base + 2 * 8 * 192, 8 * 192, 192, 30, 8)  # one token on
    assert _write_with_bad_weight(base, 8 * 64, 64, base + 16, 8 * 64, 64, 1, 1)


def test_results_of_attentions_are_no_part_of_their_operands():
    """Addresses of an imagined layout, each refused before anything is launched: results that begin or end inside an operand or each other."""
    from sglang_amd import _lib

    lib, M = _lib.lib, 1 << 20
    B, n, H, pages, page = 3, 2, 16, 4, 64
    at = {k: (i + 1) * (M << 4) for i, k in enumerate(("q", "qp", "cache", "table", "lens", "out", "lse", "ws", "k", "kp", "v", "cu"))}
    size = dict(q=B * n * H * 1024, qp=B * n * H * 128, cache=pages * page * 1152, out=B * n * H * 1024, lse=B * n * H * 4)

    def decode(out=at["out"], lse=at["lse"], heads_first=False):
        strides = (n * 512, 512, B * n * 512) if heads_first else (n * H * 512, H * 512, 512)
        return lib.fp8k_mla_decode(at["q"], *strides, at["qp"], n * H * 64, H * 64, 64, at["cache"], at["table"], 4, 4, at["lens"], None, out, lse, B, n, H, pages, page,
                                   0.1, _lib.BF16, 0, at["ws"], 1 << 40, None)

    for k in ("q", "qp", "cache"):
        _refused(decode(out=at[k] + size[k] - 16), "overlaps")
        _refused(decode(out=at[k] - size["out"] + 16), "overlaps")
        _refused(decode(lse=at[k] + size[k] - 4), "overlaps")
        _refused(decode(lse=at[k] - size["lse"] + 4), "overlaps")
    _refused(decode(lse=at["out"] + size["out"] - 4), "overlaps")
    _refused(decode(out=at["q"], heads_first=True), "overlaps")
    _refused(decode(out=at["q"] + 16), "overlaps")
    _refused(decode(out=at["q"], lse=at["q"]), "overlaps")

    Tq, Tk = 5, 7
    size = dict(q=Tq * H * 384, k=(Tk - 1) * H * 512 + (H - 1) * 512 + 256, v=(Tk - 1) * H * 512 + (H - 1) * 512 + 256, kp=Tk * 128, out=Tq * H * 256, lse=Tq * H * 4)

    def prefill(out=at["out"], lse=at["lse"]):
        return lib.fp8k_mla_prefill(at["q"], H * 192, 192, at["k"], H * 256, 256, at["kp"], 64, at["v"], H * 256, 256, at["cu"], at["cu"], out, lse, 1, H, Tq, Tk, Tq, 0.1,
                                    1, _lib.BF16, None, 0, None)

    for k in ("q", "k", "kp", "v"):
        _refused(prefill(out=at[k] + size[k] - 16), "overlaps")
        _refused(prefill(out=at[k] - size["out"] + 16), "overlaps")
        _refused(prefill(lse=at[k] + size[k] - 4), "overlaps")
        _refused(prefill(lse=at[k] - size["lse"] + 4), "overlaps")
    _refused(prefill(out=at["q"]), "overlaps")
    _refused(prefill(lse=at["out"] + size["out"] - 4), "overlaps")

    def gather(out):
        return lib.fp8k_mla_gather_cache(at["cache"], at["table"], 4, 4, at["cu"], None, None, out, 640, 2, 9, pages, page, _lib.BF16, 0, None)

    _refused(gather(at["cache"] + pages * page * 1152 - 16), "overlaps")
    _refused(gather(at["cache"] - (8 * 640 + 576) * 2 + 16), "overlaps")


def test_prefill_workspace_goes_by_blocks():
    """Keys are split where there are fewer blocks of queries than CUs: at most two workgroups of 128 rows to each of 256 CUs (and an eighth more, where heads go by XCDs), 516 bytes to
    a row.  Rows of q that no sequence has, as a padded call's, take no memory."""
    import random

    from sglang_amd._lib import lib

    size = lib.fp8k_mla_prefill_workspace_bytes
    most = 2 * 256 * 128 * 516 * 9 // 8 + 512
    rng = random.Random(5)
    some = 0
    for _ in range(3000):
        B, H = rng.choice([1, 2, 5, 16, 64]), rng.choice([1, 4, 16, 17, 33, 128])
        longest = int(2 ** rng.uniform(0, 13))
        Tq, Tk = rng.choice([B * longest, rng.randint(longest, B * longest), 8192 + B * longest]), int(2 ** rng.uniform(0, 21))
        need = size(B, H, Tq, Tk, longest)
        assert 0 <= need <= most, (B, H, Tq, Tk, longest, need)
        some += need > 0
        assert size(B, H, (1 << 30) + Tq, Tk, longest) <= most
    assert some > 300
    assert size(1, 16, 8192, 1 << 17, 16) == size(1, 16, 16384, 1 << 17, 16) > 0
