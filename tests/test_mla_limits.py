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
