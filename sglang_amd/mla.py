"""Latent attention on this path: the paged cache of latents, and attention over it in its absorbed and its expanded form.

A token's keys and values are one row of 576 numbers that all heads share: a latent of 512 and a part of 64 that carries the rotary
position.  The cache holds those rows and nothing else, [pages, page_size, 576] in the operands' 16-bit type or in float8_e4m3fn with one
scale (value = code * scale, a float32 tensor of one positive element; None: 1).  A request's pages are a row of an int32 page table.

  a layer's new tokens      mla_write_cache: norm of the latent, rotation of the position part and of the queries', store
  decode (absorbed)         per_tensor_quant_mla_fp8 and bmm_fp8 fold the keys' up-projection into the queries, mla_decode_attention, then the
                            same pair with the values' up-projection
  prefill (expanded)        the up-projection of the new latents, mla_prefill_attention
  prefill behind a prefix   mla_gather_cache, its up-projection, mla_prefill_attention without causal, merge_attention_states

All launch on the current stream of their operands' device, never synchronise, and may be captured into a graph: lengths and pages are read on
the device.  They compute no gradients.  Queries, keys and values whose rows the kernels cannot read as they lie (a last dimension that is
not contiguous, rows that do not start at multiples of 16 bytes) are copied first; a cache must be contiguous.  Sums, maxima and norms are
float32; results are rounded once.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _host
from . import custom_ops as _ops

LATENT, ROPE, ROW = 512, 64, 576
NOPE, VALUE = 128, 128


def mla_write_cache(latent: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                    cos_sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, neox: bool = False,
                    q_pe: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                    q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Stores the rows of new tokens, latent [T, 576] float16 / bfloat16 (what the down-projection gives), at slots [T] (int32 or int64; slot
    page * page_size + place) of the cache.  Slots are distinct (of rows that share one, each number may be any row's); one that the cache does not
    have (-1: the padding of a batch) is skipped.

    norm_weight [512] (of the rows' type or float32): the latent becomes x / sqrt(mean(x^2) + eps) * norm_weight.
    cos_sin float32 [P, 64] (32 cosines, 32 sines of a position) and positions [T] (int32 or int64; held within 0 .. P - 1): the position
    part is rotated, by pairs of neighbours, or with neox of numbers that lie 32 apart.
    q_pe [T, heads, 64]: rotated likewise; returned as a fresh tensor, or in q_out, which may be q_pe itself; one that overlaps it otherwise is refused.

    A float8_e4m3fn cache takes x / scale, to nearest, ties to even, values beyond 448 as 448; NaN stays NaN."""
    if not torch.compiler.is_compiling():
        done, q = _host.mla_write(latent, cache, slots, norm_weight, eps, cos_sin, positions, neox, q_pe, scale, q_out)
        if done:
            return q
    if q_pe is not None and q_out is None:
        q_out = torch.empty(q_pe.shape, dtype=q_pe.dtype, device=q_pe.device)
    _ops.mla_write_cache(latent, cache, slots, norm_weight, eps, cos_sin, positions, neox, q_pe, q_out, scale)
    return q_out


def mla_gather_cache(cache: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor, num_tokens: int, starts: Optional[torch.Tensor] = None,
                     dtype: torch.dtype = torch.bfloat16, scale: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Cached rows one after the other, [num_tokens, 576] of dtype (a 16-bit cache's own): row cu_seqlens[b] + i is token starts[b] + i (None: i) of
    request b.  cu_seqlens int32 [B + 1] does not decrease; starts int32 [B].  Rows of no request - behind cu_seqlens[B] - are not written:
    those of `out`, which is no part of the cache, stay as they were.  Tokens beyond a request's row of the table are read as its last one."""
    if not torch.compiler.is_compiling():
        got = _host.mla_gather(cache, page_table, cu_seqlens, num_tokens, starts, dtype, scale, out)
        if got is not None:
            return got
    if out is None:
        out = torch.empty((num_tokens, ROW), dtype=dtype, device=cache.device)
    elif out.shape[0] != num_tokens or out.dtype != dtype:
        raise RuntimeError("out must be [num_tokens, 576] of dtype")
    _ops.mla_gather_cache(cache, page_table, cu_seqlens, starts, scale, out)
    return out


def mla_decode_attention(q_nope: torch.Tensor, q_pe: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                         sm_scale: float, scale: Optional[torch.Tensor] = None, return_lse: bool = False,
                         out: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Absorbed attention of the newest token of each request, q_nope [B, heads, 512] and q_pe [B, heads, 64], or of its n newest,
    [B, n, heads, ..], over the seq_lens [B] (int32) tokens that it has in the cache, the newest among them:

      s[r] = sm_scale * (q_nope . row[r][:512] + q_pe . row[r][512:]),   result = softmax(s) . rows[:, :512]

    of q_nope's type and shape; with return_lse also log(sum exp(s)), float32.  out may be q_nope itself, else no part of an operand.  The last
    query of a request sees all its tokens, the one before it all but the last, and so on.  A query that sees nothing gets 0 and -inf.  The absorbed queries may be a transposed view.

    The exponentials are rounded to 16 bits for their product with the rows (their sum is not).  Lengths are held within the page table's width, and that
    bound decides how a batch is cut: pass the columns that the longest request needs, page_table[:, :n] (one request of 4000 tokens, 128 heads, takes
    30 us rather than 20 with a table for 131072).  Of a page what lies behind the last token may hold anything, the request's own rows are finite.  The whole batch's tokens are cut into equal runs, whose float32 partials
    are joined in the order of the tokens: results do not depend on timing, but on how the batch is cut."""
    if not torch.compiler.is_compiling():
        got = _host.mla_decode(q_nope, q_pe, cache, page_table, seq_lens, sm_scale, scale, return_lse, out)
        if got is not None:
            return got
    if out is None:
        out = torch.empty(q_nope.shape, dtype=q_nope.dtype, device=q_nope.device)
    lse = torch.empty(q_nope.shape[:-1], dtype=torch.float32, device=q_nope.device) if return_lse else None
    if q_nope.dim() == 3 and q_pe.dim() == 3 and out.dim() == 3:
        _ops.mla_decode_attention(q_nope.unsqueeze(1), q_pe.unsqueeze(1), cache, page_table, seq_lens, sm_scale, scale, out.unsqueeze(1),
                                  lse.unsqueeze(1) if lse is not None else None)
    else:
        _ops.mla_decode_attention(q_nope, q_pe, cache, page_table, seq_lens, sm_scale, scale, out, lse)
    return (out, lse) if return_lse else out


def mla_prefill_attention(q: torch.Tensor, k_nope: torch.Tensor, k_pe: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                          cu_seqlens_k: torch.Tensor, max_seqlen_q: int, sm_scale: float, causal: bool = True, return_lse: bool = False,
                          out: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Expanded attention over ragged sequences.  q [Tq, heads, 192], a head's 128 numbers and its 64 rotated ones; k_nope and v
    [Tk, heads, 128], as a rule the two halves of what the up-projection gives; k_pe [Tk, 64] (or [Tk, 1, 64]), read by all heads.  Sequence b has the queries
    cu_seqlens_q[b] .. cu_seqlens_q[b + 1] and the keys cu_seqlens_k[b] .. cu_seqlens_k[b + 1] (int32 [B + 1], not decreasing); max_seqlen_q is at least the
    most queries that one has: of a longer one, queries behind the bound's block (128 or 256 queries, by the call's cut) are not computed, their rows not written.

    causal: of lq queries and lk keys, query i sees the keys j <= i + lk - lq (the queries are the last of the keys); else all.  Returns [Tq, heads, 128]
    of q's type, with return_lse also log(sum exp(s)), float32 [Tq, heads]; out is no part of an operand.  A query that sees nothing gets 0 and -inf; those of no sequence are not
    written.  What lies between and behind the sequences' keys may hold anything; a sequence's own keys and values are finite.

    The exponentials are rounded to 16 bits for their product with the values (their sum is not)."""
    if not torch.compiler.is_compiling():
        got = _host.mla_prefill(q, k_nope, k_pe, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, sm_scale, causal, return_lse, out)
        if got is not None:
            return got
    if out is None:
        out = torch.empty(q.shape[:-1] + (VALUE,), dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    if k_pe.dim() == 3 and k_pe.shape[1] == 1:
        k_pe = k_pe.squeeze(1)
    _ops.mla_prefill_attention(q, k_nope, k_pe, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, sm_scale, causal, out, lse)
    return (out, lse) if return_lse else out


def merge_attention_states(out_a: torch.Tensor, lse_a: torch.Tensor, out_b: torch.Tensor, lse_b: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Two attentions of the same queries over disjoint keys as one: out_a, out_b [.., D] float32, float16 or bfloat16 (D a multiple of 8),
    lse_a, lse_b float32 [..], as the attentions here return them.

      out = (exp(lse_a) out_a + exp(lse_b) out_b) / (exp(lse_a) + exp(lse_b)),   lse = log(exp(lse_a) + exp(lse_b))

    A part with an lse of -inf counts nothing, whatever its rows hold; two of them give 0 and -inf."""
    if not torch.compiler.is_compiling():
        got = _host.merge_states(out_a, lse_a, out_b, lse_b)
        if got is not None:
            return got
    out = torch.empty(out_a.shape, dtype=out_a.dtype, device=out_a.device)
    lse = torch.empty(lse_a.shape, dtype=torch.float32, device=lse_a.device)
    _ops.merge_attention_states(out_a, lse_a, out_b, lse_b, out, lse)
    return out, lse
