"""The weight-streaming kernel of MXFP4 products (and the linear that quantises inside it): every width of its strips and every count of
K blocks that its eight waves can have, with operands that no cache holds.  Its waits are counted by hand: one that lets a block's loads
pass shows as rows of stale operands.

Results are compared bit for bit.  Values are multiples of 1/4 and at most 6, terms multiples of 1/16 and at most 36: up to 40 * 256 of them
stay under 2^24 sixteenths, so float32 sums are exact in any order."""
import pytest
import torch

from sglang_amd import mxfp4

pytestmark = pytest.mark.gpu


@pytest.fixture
def strips():
    """Pins the kernel that products take."""
    from sglang_amd._lib import lib

    lib.fp8k_tune_force_mxfp4_plan(0)
    yield
    lib.fp8k_tune_force_mxfp4_plan(-1)


def _operand(rows, k, gen):
    q = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    byte = torch.randint(126, 128, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=gen)
    s = mxfp4.pack_mxfp4_scales(byte)
    return q, s, mxfp4.mxfp4_dequant(q, s, torch.float32).double()


def _cold(call, ref):
    flush = torch.empty(1 << 27, dtype=torch.float32, device="cuda")
    for _ in range(3):
        flush.zero_()
        assert torch.equal(call(), ref)


# a wave has every eighth block: none, one, two (all the slots of the wider forms), three, four (all of the others), five
BLOCKS = [3, 8, 11, 17, 25, 33, 40]


@pytest.mark.parametrize("blocks", BLOCKS)
@pytest.mark.parametrize("m,n", [(1, 1032), (16, 1032), (13, 16368), (17, 1032), (32, 520), (27, 16368), (33, 520), (64, 1032), (130, 264)])
def test_products_from_memory(dev, strips, m, n, blocks):
    gen = torch.Generator(device=dev).manual_seed(blocks)
    for rest in (0, 32, 160):  # K blocks that end early
        k = blocks * 256 - rest
        a, sa, av = _operand(m, k, gen)
        b, sb, bv = _operand(n, k, gen)
        _cold(lambda: mxfp4.w4a4_mxfp4_matmul(a, b, sa, sb), (av @ bv.t()).bfloat16())


@pytest.mark.parametrize("m,n,blocks", [(1, 1032, 3), (1, 1032, 17), (1, 1032, 40), (2, 520, 33), (2, 520, 40), (4, 1032, 25), (9, 520, 11), (16, 264, 6),
                                        (1, 16368, 8), (3, 16368, 25), (1, 32720, 11), (4, 32720, 17)])
def test_quantising_linears_from_memory(dev, m, n, blocks):
    """The activations are values that 4 bits hold, so that quantising them loses nothing."""
    gen = torch.Generator(device=dev).manual_seed(blocks)
    for rest in (0, 32, 160):
        k = blocks * 256 - rest
        assert m * k <= 28672  # one launch
        _, _, av = _operand(m, k, gen)
        b, sb, bv = _operand(n, k, gen)
        _cold(lambda: mxfp4.w4a4_mxfp4_linear(av.bfloat16(), b, sb), (av @ bv.t()).bfloat16())


@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("k", [32, 96, 288, 480, 1184])
def test_scale_bytes_that_no_block_has(dev, kind, k):
    """Every kernel of the products: what the last word of a row holds behind its blocks is multiplied by nothing but zeros."""
    from sglang_amd._lib import lib

    gen = torch.Generator(device=dev).manual_seed(k)
    (a, sa, av), (b, sb, bv) = _operand(70, k, gen), _operand(136, k, gen)
    ref = (av @ bv.t()).bfloat16()

    def spoiled(s, byte):
        words = s.clone(memory_format=torch.contiguous_format)
        as_bytes = words.view(torch.uint8)
        assert not as_bytes[:, k // 32:].any()
        as_bytes[:, k // 32:] = byte
        return words

    lib.fp8k_tune_force_mxfp4_plan(kind)
    try:
        for x, w in ((0, 0), (1, 254), (254, 1), (254, 254), (253, 127)):
            assert torch.equal(mxfp4.w4a4_mxfp4_matmul(a, b, spoiled(sa, x), spoiled(sb, w)), ref), (x, w)
    finally:
        lib.fp8k_tune_force_mxfp4_plan(-1)
