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
