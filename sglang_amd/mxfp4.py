"""MXFP4 on this path: 4-bit weights and activations with one power-of-two scale per 32 values.

The format is the OCP microscaling one: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) in blocks of 32 along K, each
block with an e8m0 scale 2^(byte - 127), byte 255 being NaN.  A tensor of it is a pair:

  codes    uint8 [.., rows, K/2]: element 2i in the low half of byte i, 2i + 1 in the high half - what checkpoints hold
  scales   int32 [.., rows, ceil(K/128)]: the four scale bytes of 128 values in a word, blocks 4j .. 4j+3 of a row in word j from byte 0
           on; column-major, rows padded to 4, bytes that no block has zero.  ``pack_mxfp4_scales`` makes them, once after loading, of
           the uint8 [.., rows, K/32] of a checkpoint.  Other strides are taken as well; the kernels read these fastest.

K is a multiple of 32, the number of weight rows of a product a multiple of 8.

Entry points: ``per_token_group_quant_mxfp4`` and ``mxfp4_dequant``; ``w4a4_mxfp4_matmul`` and ``w4a4_mxfp4_linear`` on 4-bit
activations; ``fused_experts_mxfp4``, a whole expert layer for a few tokens, whose activations stay in 16 bits.  All launch on the
current stream of their operands' device, never synchronise, and may be captured into a graph.  They compute no gradients.  Activations and
codes whose rows the kernels cannot read as they lie (not contiguous, overlapping, not at multiples of 16 bytes) are copied first; the weights
of the expert layer are not.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _host
from . import custom_ops as _ops

BLOCK = 32


def create_mxfp4_scales(shape: Tuple[int, ...], device) -> torch.Tensor:
    """Uninitialised scale words for codes of `shape` [.., rows, K] (K in values): int32 [.., rows, ceil(K/128)], column-major with the
    rows padded to a multiple of 4."""
    *batch, rows, k = shape
    words, padded = (k + 127) // 128, (rows + 3) // 4 * 4
    return torch.empty((*batch, words, padded), dtype=torch.int32, device=device).transpose(-1, -2)[..., :rows, :]


def pack_mxfp4_scales(scales: torch.Tensor) -> torch.Tensor:
    """e8m0 bytes uint8 [.., rows, K/32], one per block as checkpoints hold them -> the int32 words that the operators take.  Plain tensor
    ops, meant for weight loading."""
    if scales.dtype != torch.uint8 or scales.dim() < 2:
        raise RuntimeError("pack_mxfp4_scales: uint8 [.., rows, K/32] expected")
    rows, blocks = scales.shape[-2:]
    padded = scales.new_zeros(scales.shape[:-1] + ((blocks + 3) // 4 * 4,))
    padded[..., :blocks] = scales
    words = padded.view(torch.int32)
    out = scales.new_zeros(scales.shape[:-2] + (words.shape[-1], (rows + 3) // 4 * 4), dtype=torch.int32)
    out[..., :rows] = words.transpose(-1, -2)
    return out.transpose(-1, -2)[..., :rows, :]


def unpack_mxfp4_scales(words: torch.Tensor, k: int) -> torch.Tensor:
    """The inverse of pack_mxfp4_scales: int32 words [.., rows, ceil(k/128)] -> e8m0 bytes uint8 [.., rows, k/32], contiguous."""
    if words.dtype != torch.int32 or k % BLOCK != 0 or words.shape[-1] != (k + 127) // 128:
        raise RuntimeError("unpack_mxfp4_scales: int32 [.., rows, ceil(k/128)] and k a multiple of 32 expected")
    return words.clone(memory_format=torch.contiguous_format).view(torch.uint8)[..., : k // BLOCK].contiguous()


def per_token_group_quant_mxfp4(x: torch.Tensor, fuse_silu_and_mul: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] float32 / float16 / bfloat16 -> (codes, scales), blocks of 32 along K.

    The scale's exponent is that of the block's largest magnitude rounded to one fraction bit, minus 2 (at least -127); values are
    rounded to nearest, ties to the even code, and end at 6.  A block with an infinity or a NaN becomes NaN.
    fuse_silu_and_mul: x is [M, 2K], gate columns then up columns; silu(gate) * up is formed in float32 and quantised unrounded."""
    if not torch.compiler.is_compiling():
        out = _host.mx_quant(x, fuse_silu_and_mul)
        if out is not None:
            return out
    if x.dim() != 2:
        raise RuntimeError("per_token_group_quant_mxfp4: x must be 2-D")
    if fuse_silu_and_mul and x.shape[1] % 2 != 0:
        raise RuntimeError("fuse_silu_and_mul needs an even last dimension")
    m, k = x.shape[0], x.shape[1] // 2 if fuse_silu_and_mul else x.shape[1]
    q = torch.empty((m, k // 2), dtype=torch.uint8, device=x.device)
    s = create_mxfp4_scales((m, k), x.device)
    _ops.mxfp4_quant(x, q, s, fuse_silu_and_mul)
    return q, s


def quant_weight_mxfp4(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """A weight [.., N, K] of any float type -> (codes, scales), once after loading; expert stacks [E, N, K] matrix by matrix.  Types other
    than float32, float16 and bfloat16 are taken as their float32 values."""
    if weight.dim() not in (2, 3):
        raise RuntimeError("quant_weight_mxfp4: [N, K] or [E, N, K] expected")

    def readable(w: torch.Tensor) -> torch.Tensor:
        return w.float() if w.is_floating_point() and w.dtype not in (torch.float32, torch.float16, torch.bfloat16) else w

    if weight.dim() == 2:
        return per_token_group_quant_mxfp4(readable(weight))
    e, n, k = weight.shape
    q = torch.empty((e, n, k // 2), dtype=torch.uint8, device=weight.device)
    s = create_mxfp4_scales((e, n, k), weight.device)
    for i in range(e):
        _ops.mxfp4_quant(readable(weight[i]), q[i], s[i])
    return q, s


def mxfp4_dequant(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Values [N, K] of codes [N, K/2] and their scales, or [E, N, K] of a stack: exact in float32, rounded once to `dtype` (float32,
    float16, bfloat16)."""
    if not torch.compiler.is_compiling():
        out = _host.mx_dequant(q, s, dtype)
        if out is not None:
            return out
    out = torch.empty(q.shape[:-1] + (q.shape[-1] * 2,), dtype=dtype, device=q.device)
    _ops.mxfp4_dequant(q, s, out)
    return out


def w4a4_mxfp4_matmul(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, output_dtype: torch.dtype = torch.bfloat16,
                      bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """C [M, N] = A . B^T (+ bias) of two quantised operands: codes A [M, K/2], B [N, K/2], scales As, Bs.  Float32 sums, the bias (of the
    output's type or float32) added in float32, one rounding to output_dtype (float16 or bfloat16)."""
    if not torch.compiler.is_compiling():
        out = _host.mx_matmul(A, B, As, Bs, output_dtype, bias)
        if out is not None:
            return out
    return _ops.mxfp4_scaled_mm(A, B, As, Bs, output_dtype, bias)


def w4a4_mxfp4_linear(input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, input_scale: Optional[torch.Tensor] = None,
                      bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """input [.., K] float16 / bfloat16, weight codes [N, K/2] -> [.., N] of the input's type: the activations are quantised as
    per_token_group_quant_mxfp4 does, then multiplied: for a few rows in one launch, traced by torch.compile in two (float32 sums may
    differ in order).  With input_scale the input holds codes [.., K/2] already (quantised upstream,
    scales [tokens, ceil(K/128)]) and the result is bfloat16."""
    if input_scale is None and not torch.compiler.is_compiling():
        output = _host.mx_linear(input, weight, weight_scale, bias)
        if output is not None:
            return output
    input_2d = input.reshape(-1, input.shape[-1])
    shape = [*input.shape[:-1], weight.shape[0]]
    if input_scale is not None:
        if input_2d.dtype != torch.uint8:
            raise RuntimeError("w4a4_mxfp4_linear: input_scale given, so input must hold uint8 codes already")
        return w4a4_mxfp4_matmul(input_2d, weight, input_scale, weight_scale, torch.bfloat16, bias).view(shape)
    if input_2d.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("w4a4_mxfp4_linear: float16 or bfloat16 input expected")
    q, s = per_token_group_quant_mxfp4(input_2d)
    return w4a4_mxfp4_matmul(q, weight, s, weight_scale, input_2d.dtype, bias).view(shape)


def fused_experts_mxfp4(
    hidden_states: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    topk_weights: torch.Tensor,
    topk_ids: torch.Tensor,
    w1_scale: torch.Tensor,
    w2_scale: torch.Tensor,
    activation: str = "silu",
    inplace: bool = False,
    apply_router_weight_on_input: bool = False,
    routed_scaling_factor: Optional[float] = None,
) -> torch.Tensor:
    """The gated experts of a few tokens - at most 128, and at most 1024 (token, choice) pairs - in two launches.

    hidden_states [T, H] float16 / bfloat16; w1 codes [E, 2I, H/2] (gate rows, then up rows), w2 codes [E, H, I/2], contiguous; topk_weights [T, k]
    and topk_ids [T, k] as the routers of fused_moe return them; an id that is not 0 .. E-1 (-1: an expert of another rank)
    contributes nothing.  Activations stay in 16 bits: with few tokens the layer is bound by the weights' bytes.

      h = act(x . gate^T) * (x . up^T), out = round(routed_scaling_factor * sum of weight * h . w2^T), sums in float32

    h is held as the sum of two bfloat16 numbers, so that the rounding of the result is the only one that counts.  Weights beyond
    float32's range (4 and 6 times 2^126, 2 to 6 times 2^127) may count as infinite, as mxfp4_dequant gives them.
    More tokens are refused: dequantise the experts (mxfp4_dequant) for a grouped product in 16 bits, or call in pieces of 128.

    apply_router_weight_on_input: the weight multiplies both products of the first stage instead.  activation: "silu" or "gelu"."""
    scaling = 1.0 if routed_scaling_factor is None else float(routed_scaling_factor)
    if topk_weights.dtype != torch.float32:
        topk_weights = topk_weights.float()
    if activation in ("silu", "gelu") and not torch.compiler.is_compiling():
        out = _host.mx_experts(hidden_states, w1, w2, topk_weights, topk_ids, w1_scale, w2_scale, activation == "gelu",
                               apply_router_weight_on_input, scaling, inplace)
        if out is not None:
            return out
    out = torch.empty(hidden_states.shape, dtype=hidden_states.dtype, device=hidden_states.device)
    _ops.mxfp4_experts(hidden_states, w1, w2, topk_weights.contiguous(), topk_ids.contiguous(), w1_scale, w2_scale, out,
                       activation, apply_router_weight_on_input, scaling)
    return hidden_states.copy_(out) if inplace else out
