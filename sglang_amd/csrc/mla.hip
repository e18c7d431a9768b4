// Latent attention: C entry points, the cache's writer and reader, and the join of two attentions.  The attention kernels are in
// mla_decode.h and mla_prefill.h.
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "mla_decode.h"
#include "mla_prefill.h"

namespace fp8k {
namespace {

bool is_half_type(int dtype) { return dtype == FP8K_BF16 || dtype == FP8K_F16; }

// whether two pieces of memory share a byte
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a_bytes > 0 && b_bytes > 0 && x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}
// Memory from its first byte to its last.
struct Piece {
  const void* at;
  int64_t bytes;
};
// rows of `last` 16-bit numbers, their sizes and strides from the outer dimension in
Piece rows_of(const void* at, std::initializer_list<std::pair<int64_t, int64_t>> dims, int64_t last) {
  int64_t n = last;
  for (const auto& d : dims) {
    if (d.first <= 0) return {at, 0};
    n += (d.first - 1) * d.second;
  }
  return {at, 2 * n};
}
// An attention's results are written while other workgroups still read its operands, and its two results by different threads.
bool results_apart(Piece out, Piece lse, std::initializer_list<Piece> operands) {
  for (const Piece& x : operands)
    if (x.at && (overlap(out.at, out.bytes, x.at, x.bytes) || (lse.at && overlap(lse.at, lse.bytes, x.at, x.bytes)))) return false;
  return !lse.at || !overlap(out.at, out.bytes, lse.at, lse.bytes);
}

// ---------------------------------------------------------------------------------------------- cache
struct MlaWriteArgs {
  const u16 *latent, *q_pe;
  void* cache;
  u16* q_out;
  const void *slots, *norm_weight, *positions;
  const float *cos_sin, *scale;
  int64_t ld_latent, q_t, q_h, o_t, o_h, num_slots, max_pos;
  int T, H, row_blocks;
  bool slots64, positions64, weight_f32, neox;
  float eps;
};

// The cosines and sines of eight pairs: those from 8 part on of a row's 32 and 32.
struct Angles {
  v4f co[2], si[2];
};
__device__ __forceinline__ Angles angles_of(const float* row, int part) {
  const v4f* const at = (const v4f*)row + 2 * part;
  return Angles{{at[0], at[1]}, {at[8], at[9]}};
}
// 16 numbers of a position part, eight pairs, rotated: pairs of neighbours (x the 16 numbers from 16 part on), or (neox) of numbers that lie
// 32 apart (x the eight from 8 part on, then the eight from 32 + 8 part on).
__device__ __forceinline__ void rotate16(float* x, const Angles& a, bool neox) {
  if (neox) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float cs = a.co[i >> 2][i & 3], sn = a.si[i >> 2][i & 3], u = x[i], v = x[8 + i];
      x[i] = u * cs - v * sn;
      x[8 + i] = v * cs + u * sn;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float cs = a.co[i >> 2][i & 3], sn = a.si[i >> 2][i & 3], u = x[2 * i], v = x[2 * i + 1];
      x[2 * i] = u * cs - v * sn;
      x[2 * i + 1] = v * cs + u * sn;
    }
  }
}

template <int DT>
__device__ __forceinline__ void load8(const u16* p, float* x) {
  const v4i v = *(const v4i*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const v2f f = unpack2<DT>((uint32_t)v[i]);
    x[2 * i] = f[0];
    x[2 * i + 1] = f[1];
  }
}
template <int DT>
__device__ __forceinline__ void store8(u16* p, const float* x) {
  *(v4i*)p = v4i{(int)pack2<DT>(x[0], x[1]), (int)pack2<DT>(x[2], x[3]), (int)pack2<DT>(x[4], x[5]), (int)pack2<DT>(x[6], x[7])};
}
// x / scale to e4m3: nearest, ties to even, at most 448; NaN stays NaN.  The quotient of a scale whose reciprocal is an ordinary number is the product
// with that and one correction by its remainder, the division's own result but for the last place at times: a division is ten instructions, and
// there are 576 to a row.
struct Fp8Scale {
  float scale, inverse;
  bool ordinary;
};
__device__ __forceinline__ Fp8Scale fp8_scale(const float* p) {
  Fp8Scale s{p ? *p : 1.0f, 0.0f, false};
  s.inverse = 1.0f / s.scale;
  s.ordinary = fabsf(s.inverse) >= 0x1p-100f && fabsf(s.inverse) <= 0x1p100f;
  return s;
}
__device__ __forceinline__ float to_fp8_range(float x, const Fp8Scale& s) {
  float v = x * s.inverse;
  if (s.ordinary) v = fabsf(v) <= kFp8Max ? fmaf(fmaf(-v, s.scale, x), s.inverse, v) : v;
  else v = x / s.scale;
  return v != v ? v : fminf(fmaxf(v, -kFp8Max), kFp8Max);
}
__device__ __forceinline__ void store8_fp8(uint8_t* p, const float* x, const Fp8Scale& s) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_fp8_range(x[i], s);
  *(v2i*)p = v2i{(int)cvt4_fp8(v[0], v[1], v[2], v[3]), (int)cvt4_fp8(v[4], v[5], v[6], v[7])};
}

// One wave to a token's row, then four threads to the position part of a token's head: lanes hold 16 bytes of what they read and write, and nothing is
// read twice.  Bound by the launch up to some hundred tokens (64 of 16 heads 3.1 us, of 128 3.2), then by the bytes: 4096 tokens into an 8-bit cache, 16 heads' queries 6.8 us,
// 24 MB at 3.5 TB/s.
template <int DT, bool FP8>
__global__ __launch_bounds__(256) void mla_write_kernel(const MlaWriteArgs p) {
  const int tid = threadIdx.x, lane = tid & 63;
  auto table_of = [&](int t) {
    const int64_t pos = p.positions64 ? ((const int64_t*)p.positions)[t] : ((const int32_t*)p.positions)[t];
    return p.cos_sin + min(max(pos, (int64_t)0), p.max_pos - 1) * kRope;
  };
  if ((int)blockIdx.x >= p.row_blocks) {
    const int64_t i = (int64_t)(blockIdx.x - p.row_blocks) * 256 + tid;
    const int part = (int)(i & 3);
    const int64_t th = i >> 2;
    if (th >= (int64_t)p.T * p.H) return;
    const int t = (int)(th / p.H), h = (int)(th - (int64_t)t * p.H);
    const int first = p.neox ? 8 * part : 16 * part, second = p.neox ? 32 + 8 * part : 16 * part + 8;
    const u16* const from = p.q_pe + t * p.q_t + h * p.q_h;
    u16* const to = p.q_out + t * p.o_t + h * p.o_h;
    float x[16];
    load8<DT>(from + first, x);
    load8<DT>(from + second, x + 8);
    rotate16(x, angles_of(table_of(t), part), p.neox);
    store8<DT>(to + first, x);
    store8<DT>(to + second, x + 8);
    return;
  }
  const int t = (int)blockIdx.x * 4 + (tid >> 6);
  if (t >= p.T) return;
  // Everything is asked for before anything is looked at: a row is short, and what it costs is the loads that wait for others.
  const u16* const from = p.latent + t * p.ld_latent;
  const int64_t slot = p.slots64 ? ((const int64_t*)p.slots)[t] : ((const int32_t*)p.slots)[t];
  const Fp8Scale scale = fp8_scale(FP8 ? p.scale : nullptr);
  float x[8], weight[8];
  load8<DT>(from + 8 * lane, x);
  // lanes 0 .. 31: a pair of the position part each, neighbours or numbers 32 apart
  const int pair = lane & 31, first = p.neox ? pair : 2 * pair, second = p.neox ? 32 + pair : 2 * pair + 1;
  float u = 0.0f, v = 0.0f, cs = 1.0f, sn = 0.0f;
  if (lane < 32) {
    u = unpack2<DT>(from[kLatent + first])[0];
    v = unpack2<DT>(from[kLatent + second])[0];
    if (p.cos_sin) {
      const float* const row = table_of(t);
      cs = row[pair];
      sn = row[32 + pair];
    }
  }
  if (p.norm_weight) {
    if (p.weight_f32) {
      *(v4f*)weight = *(const v4f*)((const float*)p.norm_weight + 8 * lane);
      *(v4f*)(weight + 4) = *(const v4f*)((const float*)p.norm_weight + 8 * lane + 4);
    } else load8<DT>((const u16*)p.norm_weight + 8 * lane, weight);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    const float f = 1.0f / sqrtf(sum * (1.0f / kLatent) + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * f * weight[i];
  }
  if (slot < 0 || slot >= p.num_slots) return;
  if (p.cos_sin) {
    const float a = u * cs - v * sn;
    v = v * cs + u * sn;
    u = a;
  }
  if (FP8) {
    uint8_t* const to = (uint8_t*)p.cache + slot * kLatentRow;
    store8_fp8(to + 8 * lane, x, scale);
    const uint32_t w = cvt_pk_fp8_lo(to_fp8_range(u, scale), to_fp8_range(v, scale), 0);
    if (lane < 32) {
      to[kLatent + first] = (uint8_t)w;
      to[kLatent + second] = (uint8_t)(w >> 8);
    }
  } else {
    u16* const to = (u16*)p.cache + slot * kLatentRow;
    store8<DT>(to + 8 * lane, x);
    const uint32_t w = pack2<DT>(u, v);
    if (lane < 32) {
      to[kLatent + first] = (u16)w;
      to[kLatent + second] = (u16)(w >> 16);
    }
  }
}

struct MlaGatherArgs {
  const uint8_t* cache;
  const int32_t *table, *cu, *starts;
  const float* scale;
  u16* out;
  int64_t table_stride, ld_out;
  int B, tokens, pages, page_size, table_width;
};

// One wave to a row: 72 (8-bit: 36) chunks of 16 bytes.  A row's request is found by bisection, for all of its lanes at once.  Bound by the
// bytes: 43600 rows of 16 bits 20 us, 5.0 TB/s, a large copy's rate.  Few rows by the loads that wait for each other: 4400 of 32 requests, 8 bits, 4.7 us.
template <int DT, bool FP8>
__global__ __launch_bounds__(256) void mla_gather_kernel(const MlaGatherArgs p) {
  const int lane = threadIdx.x & 63;
  const int i = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (i >= p.tokens || i >= p.cu[p.B] || i < p.cu[0]) return;
  // the last request that begins at or before row i and is not empty
  int lo = 0, hi = p.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid] <= i) lo = mid;
    else hi = mid;
  }
  const int64_t tok = min(max((int64_t)i - p.cu[lo] + (p.starts ? p.starts[lo] : 0), (int64_t)0), (int64_t)p.table_width * p.page_size - 1);
  const int page = (int)(tok / p.page_size);
  const int64_t e = min(max(p.table[lo * p.table_stride + page], 0), p.pages - 1);
  const int64_t row = e * p.page_size + (tok - (int64_t)page * p.page_size);
  u16* const to = p.out + (int64_t)i * p.ld_out;
  if (FP8) {
    const float scale = p.scale ? *p.scale : 1.0f;
    if (lane < 36) {
      const v4i raw = *(const v4i*)(p.cache + row * kLatentRow + lane * 16);
      float x[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(raw[k], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(raw[k], true);
        x[4 * k] = a[0] * scale;
        x[4 * k + 1] = a[1] * scale;
        x[4 * k + 2] = b[0] * scale;
        x[4 * k + 3] = b[1] * scale;
      }
      store8<DT>(to + lane * 16, x);
      store8<DT>(to + lane * 16 + 8, x + 8);
    }
  } else {
    const v4i* const from = (const v4i*)(p.cache + row * (2 * kLatentRow));
    const v4i a = from[lane];
    ((v4i*)to)[lane] = a;
    if (lane < 8) ((v4i*)to)[64 + lane] = from[64 + lane];
  }
}

// ---------------------------------------------------------------------------------------------- merge
// out = (e^la a + e^lb b) / (e^la + e^lb), a row of D numbers, eight to a thread.  Bound by the bytes: 4096 tokens of
// 128 heads of 128, bf16, 70 us, 5.8 TB/s; 37 tokens of 16 heads 2.4 us, the launch.
template <int DT>
__global__ __launch_bounds__(256) void mla_merge_kernel(const void* a, const float* la, const void* b, const float* lb, void* out, float* lse,
                                                        int64_t rows, int D8) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / D8;
  if (row >= rows) return;
  const float x = la[row], y = lb[row], top = fmaxf(x, y), shift = shift_of(top);
  const float ex = __builtin_amdgcn_exp2f((x - shift) * kLog2e), ey = __builtin_amdgcn_exp2f((y - shift) * kLog2e), sum = ex + ey;
  const float f = sum == 0.0f ? 0.0f : 1.0f / sum, fx = ex * f, fy = ey * f;
  if (i - row * D8 == 0) lse[row] = sum == 0.0f ? -INFINITY : __builtin_amdgcn_logf(sum) * kLn2 + shift;
  float u[8], v[8];
  if constexpr (DT == FP8K_F32) {
    *(v4f*)u = ((const v4f*)a)[2 * i];
    *(v4f*)(u + 4) = ((const v4f*)a)[2 * i + 1];
    *(v4f*)v = ((const v4f*)b)[2 * i];
    *(v4f*)(v + 4) = ((const v4f*)b)[2 * i + 1];
  } else {
    load8<DT>((const u16*)a + 8 * i, u);
    load8<DT>((const u16*)b + 8 * i, v);
  }
  // a part that holds nothing counts nothing, whatever stands in its rows
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = (x == -INFINITY ? 0.0f : u[k] * fx) + (y == -INFINITY ? 0.0f : v[k] * fy);
  if constexpr (DT == FP8K_F32) {
    ((v4f*)out)[2 * i] = *(v4f*)u;
    ((v4f*)out)[2 * i + 1] = *(v4f*)(u + 4);
  } else store8<DT>((u16*)out + 8 * i, u);
}

// T x H rows of kRope numbers, `t` and `h` apart (0 where there is one alone).
struct QueryRows {
  int64_t t, h;
};
// Whether rows o, at `delta` numbers from rows q, share no number with them; o's lie apart from each other.  Exact where the strides are q's; else what the ends,
// the strides' common divisor, or a period that the outer rows of both have tell: that finds slices of one buffer apart, and takes for a collision what it cannot tell.
bool queries_apart(int64_t delta, QueryRows q, QueryRows o, int64_t T, int64_t H) {
  const auto extent = [&](QueryRows r) { return (T - 1) * r.t + (H - 1) * r.h + kRope; };
  if (delta >= extent(q) || -delta >= extent(o)) return true;
  const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b != 0 && (a < 0) != (b < 0)); };
  const auto mod = [&](int64_t a, int64_t b) { return a - floor_div(a, b) * b; };
  if (q.t == o.t && q.h == o.h) {
    // Rows of differences a inner + b outer, |a| < n, |b| < m.  The outer stride is more than the inner rows' extent, so that only its two
    // multiples around delta come near, and then the inner one's two around the rest.
    const bool h_inner = H > 1 && (T == 1 || q.h < q.t);
    const int64_t inner = h_inner ? q.h : q.t, n = h_inner ? H : T, outer = h_inner ? q.t : q.h, m = h_inner ? T : H;
    for (int64_t i = 0; i < 2; ++i) {
      const int64_t b = m == 1 ? 0 : std::min(std::max(floor_div(delta, outer) + i, 1 - m), m - 1), rest = delta - b * outer;
      for (int64_t j = 0; j < 2; ++j) {
        const int64_t a = n == 1 ? 0 : std::min(std::max(floor_div(rest, inner) + j, 1 - n), n - 1), gap = rest - a * inner;
        if (gap > -kRope && gap < kRope) return false;
      }
    }
    return true;
  }
  int64_t common = 0;
  for (int64_t x : {q.t, q.h, o.t, o.h})
    while (x) {
      const int64_t y = common % x;
      common = x;
      x = y;
    }
  if (common && mod(delta, common) >= kRope && mod(delta, common) <= common - kRope) return true;
  const auto in_period = [&](int64_t period, int64_t q_inner, int64_t o_inner, int64_t n) {
    const int64_t q_size = (n - 1) * q_inner + kRope, o_size = (n - 1) * o_inner + kRope;
    return mod(delta, period) >= q_size && mod(delta, period) + o_size <= period;
  };
  return (q.t == o.t && q.t > 0 && in_period(q.t, q.h, o.h, H)) || (q.h == o.h && q.h > 0 && in_period(q.h, q.t, o.t, T));
}

int64_t up_to(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// How a decode call is cut: rows of a workgroup (16, 32, 64 or 128), and runs of tiles.  `walkers` workgroups to a block of rows, one
// workgroup to a CU.  Few rows to a workgroup read the cache more often, but put more CUs on a row's tokens for the same number of partials, and begin
// and end sooner: the fewest rows with which a CU meets at most 12 tiles, by the most that the page table allows and with what beginning a request costs.
// 128 heads, bf16, us with 16 / 32 / 64 / 128 rows: one request of 32000 tokens 41 / 43 / 43 / 49, 16 of up to 4000 54 / 50 / 48 / 47, 32 of 4000 91 / 74 / 71 / 66,
// 64 of 4000 155 / 118 / 101 / 91, 256 of 200 100 / 79 / 64 / 61.  (At most 6 tiles: 31 for 27 us with 8 of 2000; at most 24: 49 for 43 with 30 of 3000, 64 heads.)
struct DecodePlan {
  int rows, mblocks, walkers;
};
DecodePlan decode_plan(int64_t B, int64_t M, int64_t max_len) {
  DecodePlan d;
  const int64_t tiles = B * ((max_len + kMlaTile - 1) / kMlaTile), units = tiles + B * kMlaNew;
  d.rows = 16;
  while (d.rows < 128 && d.rows < M && units * ((M + d.rows - 1) / d.rows) > 12 * num_cu()) d.rows *= 2;
  d.mblocks = (int)((M + d.rows - 1) / d.rows);
  d.walkers = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(num_cu(), 256) / d.mblocks, tiles));
  return d;
}

// How a prefill call is cut.  Workgroups of four waves (128 queries), two to a CU, or of eight (256), one to a CU.  Eight fetch the keys half as often, four
// waste less on sequences' last blocks and on the diagonal, and two workgroups do not wait at each other's barriers.  Eight where the queries fill
// their blocks by seven eighths and there are many keys to a query: all are seen and as many as there are queries, or (causal) four times as many.  us with four /
// eight: 2000 queries of 32 heads with 18000 keys causal 641 / 608, all 656 / 621; 1000 with 4000 keys 106 / 105, 115 / 107; 8192 of 16 heads with 16384 keys 875 / 852,
// 1160 / 1116; but 2048 of 128 heads with their own keys, causal, 200 / 210, 4 x 512 66 / 77, and 384 of 64 heads with 8384 keys 155 / 168.
//
// Splits of the keys, where the blocks of queries leave CUs idle: as many as a model of the call's time has fewest us for, at least two tiles of keys to
// each.  A tile of a workgroup of four waves takes 1.25 us alone on a CU, 2.5 beside another, of eight 2.2; a join 5 and its partials, written and read at 4.5 TB/s.  us,
// causal: 1024 queries of 32 heads 30 whole, 41 in two; 2048 of 16 48, 56 in two; of 8 44, 35 in two, 40 in four; 16 with 2016 keys of 16 heads 42 whole, 21 in three, 15 so.
struct PrefillPlan {
  int waves, splits;
  int64_t blocks;
};
PrefillPlan prefill_cut(int waves, int64_t B, int64_t H, int64_t Tq, int64_t Tk, int64_t max_seqlen_q) {
  const int64_t rows = 32 * waves, blocks = (std::min(max_seqlen_q, Tq) + rows - 1) / rows, groups = B * H * blocks;
  PrefillPlan d{waves, 1, blocks};
  if (groups <= 0 || groups > num_cu()) return d;
  const int64_t tiles = (Tk / B + kPreKeys - 1) / kPreKeys, most = std::min<int64_t>(std::min<int64_t>(num_cu() * 8 / waves / groups, 32), tiles / 2);
  const double partials = (double)std::min(Tq * H, groups * rows) * (2 * 4 * kPreValue) / 4.5e6;
  double least = 0;
  for (int64_t n = 1; n <= most; ++n) {
    const double us = (waves == 8 ? 2.2 : groups * n > num_cu() ? 2.5 : 1.25) * (double)((tiles + n - 1) / n) + (n > 1 ? 5 + n * (partials + 0.25) : 0);
    if (n > 1 && us >= least) continue;
    least = us;
    d.splits = (int)n;
  }
  return d;
}
// Heads by XCDs, unless that leaves more than an eighth of them idle (1000 queries of 4 heads with 10000 keys 79 us by XCDs, 49 over all)
int prefill_xcd_bits(int64_t B, int64_t H) { return up_to(B * H, 8) * 8 > B * H * 9 ? 0 : 3; }
int64_t prefill_workgroups(const PrefillPlan& d, int64_t B, int64_t H) { return (prefill_xcd_bits(B, H) ? up_to(B * H, 8) : B * H) * d.blocks; }
// Of the splits' partials and their logarithms.  Splits are made of few blocks alone: at most two workgroups to a CU, 38 MB in all, however many rows q has.
int64_t prefill_rows(const PrefillPlan& d, int64_t B, int64_t H) { return d.splits == 1 ? 0 : d.splits * prefill_workgroups(d, B, H) * 32 * d.waves; }
int64_t prefill_workspace(int64_t rows) { return up_to(rows * kPreValue * 4, 256) + up_to(rows * 4, 256); }
PrefillPlan prefill_plan(int64_t B, int64_t H, int64_t Tq, int64_t Tk, int64_t max_seqlen_q, bool causal) {
  const PrefillPlan d = prefill_cut(8, B, H, Tq, Tk, max_seqlen_q);
  return Tk >= (causal ? 4 : 1) * Tq && Tq * 8 >= B * d.blocks * 256 * 7 ? d : prefill_cut(4, B, H, Tq, Tk, max_seqlen_q);
}

}  // namespace
}  // namespace fp8k

using namespace fp8k;

extern "C" int fp8k_mla_write_cache(const void* latent, int64_t ld_latent, void* cache, const void* slots, int slots_are_64bit,
                                    const void* norm_weight, int norm_weight_dtype, float eps, const float* cos_sin, int64_t max_pos,
                                    const void* positions, int positions_are_64bit, int neox, const void* q_pe, int64_t q_stride_t,
                                    int64_t q_stride_h, void* q_out, int64_t o_stride_t, int64_t o_stride_h, const float* scale, int64_t T,
                                    int64_t H, int64_t num_slots, int dtype, int cache_is_fp8, void* stream) {
  clear_error();
  FP8K_REQUIRE(is_half_type(dtype), "mla write: Half or BFloat16 rows expected");
  FP8K_REQUIRE(T >= 0 && T < (1ll << 30) && num_slots >= 0 && H >= 0 && H <= (1 << 16), "mla write: bad sizes");
  if (T == 0) return FP8K_OK;
  FP8K_REQUIRE(latent && (cache || num_slots == 0) && slots, "mla write: null pointer");
  FP8K_REQUIRE(aligned(latent, 16) && aligned(cache, 16) && ld_latent % 8 == 0 && ld_latent >= kLatentRow, "mla write: rows must be 16-byte aligned");
  FP8K_REQUIRE(aligned(slots, slots_are_64bit ? 8 : 4), "mla write: misaligned slots");
  FP8K_REQUIRE(!cos_sin || (positions && max_pos > 0 && aligned(cos_sin, 16) && aligned(positions, positions_are_64bit ? 8 : 4)),
               "mla write: the rotation needs positions and a 16-byte aligned table");
  FP8K_REQUIRE(!q_pe || (cos_sin && q_out && H > 0), "mla write: queries need a table of cosines and sines, and a place");
  if (q_pe) {
    FP8K_REQUIRE(aligned(q_pe, 16) && aligned(q_out, 16) && q_stride_t % 8 == 0 && q_stride_h % 8 == 0 && o_stride_t % 8 == 0 && o_stride_h % 8 == 0,
                 "mla write: queries must be 16-byte aligned");
    FP8K_REQUIRE(q_stride_t >= 0 && q_stride_h >= 0 && o_stride_t >= 0 && o_stride_h >= 0, "mla write: negative stride");
    const auto apart = [](int64_t inner, int64_t n, int64_t outer, int64_t m) {
      return (n == 1 || inner >= kRope) && (m == 1 || outer >= (n - 1) * inner + kRope);
    };
    FP8K_REQUIRE(apart(o_stride_h, H, o_stride_t, T) || apart(o_stride_t, T, o_stride_h, H), "mla write: the rotated queries' places overlap each other");
    const QueryRows q{T > 1 ? q_stride_t : 0, H > 1 ? q_stride_h : 0}, o{T > 1 ? o_stride_t : 0, H > 1 ? o_stride_h : 0};
    const int64_t delta = ((intptr_t)q_out - (intptr_t)q_pe) / 2;
    FP8K_REQUIRE((delta == 0 && q.t == o.t && q.h == o.h) || queries_apart(delta, q, o, T, H),
                 "mla write: the rotated queries' places overlap queries other than their own");
  }
  FP8K_REQUIRE(!norm_weight || ((norm_weight_dtype == dtype || norm_weight_dtype == FP8K_F32) && aligned(norm_weight, 16)),
               "mla write: the norm's weight must be of the rows' type or float32, 16-byte aligned");
  MlaWriteArgs p{};
  p.latent = (const u16*)latent; p.q_pe = (const u16*)q_pe; p.cache = cache; p.q_out = (u16*)q_out;
  p.slots = slots; p.norm_weight = norm_weight; p.positions = positions; p.cos_sin = cos_sin; p.scale = scale;
  p.ld_latent = ld_latent; p.q_t = q_stride_t; p.q_h = q_stride_h; p.o_t = o_stride_t; p.o_h = o_stride_h;
  p.num_slots = num_slots; p.max_pos = max_pos; p.T = (int)T; p.H = (int)H;
  p.row_blocks = (int)((T + 3) / 4);
  p.slots64 = slots_are_64bit != 0; p.positions64 = positions_are_64bit != 0; p.weight_f32 = norm_weight_dtype == FP8K_F32; p.neox = neox != 0;
  p.eps = eps;
  const int64_t q_blocks = q_pe ? (T * H * 4 + 255) / 256 : 0;
  FP8K_REQUIRE(p.row_blocks + q_blocks < (1ll << 31), "mla write: too large");
  const dim3 grid((unsigned)(p.row_blocks + q_blocks));
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == FP8K_BF16) {
    if (cache_is_fp8) mla_write_kernel<FP8K_BF16, true><<<grid, 256, 0, st>>>(p);
    else mla_write_kernel<FP8K_BF16, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (cache_is_fp8) mla_write_kernel<FP8K_F16, true><<<grid, 256, 0, st>>>(p);
    else mla_write_kernel<FP8K_F16, false><<<grid, 256, 0, st>>>(p);
  }
  return check_launch("mla write");
}

extern "C" int fp8k_mla_gather_cache(const void* cache, const int32_t* page_table, int64_t table_stride, int64_t table_width,
                                     const int32_t* cu_seqlens, const int32_t* starts, const float* scale, void* out, int64_t ld_out, int64_t B,
                                     int64_t num_tokens, int64_t pages, int64_t page_size, int dtype, int cache_is_fp8, void* stream) {
  clear_error();
  FP8K_REQUIRE(is_half_type(dtype), "mla gather: Half or BFloat16 rows expected");
  FP8K_REQUIRE(B >= 0 && B < (1 << 24) && num_tokens >= 0 && num_tokens < (1ll << 31), "mla gather: bad sizes");
  if (B == 0 || num_tokens == 0) return FP8K_OK;
  FP8K_REQUIRE(pages > 0 && pages < (1ll << 31) && page_size > 0 && page_size < (1ll << 31) && table_width > 0 && table_width < (1ll << 31) && table_stride >= 0,
               "mla gather: bad sizes of the cache or the page table");
  FP8K_REQUIRE(cache && page_table && cu_seqlens && out, "mla gather: null pointer");
  FP8K_REQUIRE(aligned(cache, 16) && aligned(out, 16) && ld_out % 8 == 0 && ld_out >= kLatentRow, "mla gather: rows must be 16-byte aligned");
  const Piece rows = rows_of(out, {{num_tokens, ld_out}}, kLatentRow);
  FP8K_REQUIRE(!overlap(rows.at, rows.bytes, cache, pages * page_size * kLatentRow * (cache_is_fp8 ? 1 : 2)), "mla gather: out overlaps the cache");
  MlaGatherArgs p{};
  p.cache = (const uint8_t*)cache; p.table = page_table; p.cu = cu_seqlens; p.starts = starts; p.scale = scale; p.out = (u16*)out;
  p.table_stride = table_stride; p.ld_out = ld_out;
  p.B = (int)B; p.tokens = (int)num_tokens; p.pages = (int)pages; p.page_size = (int)page_size; p.table_width = (int)table_width;
  const dim3 grid((unsigned)((num_tokens + 3) / 4));
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == FP8K_BF16) {
    if (cache_is_fp8) mla_gather_kernel<FP8K_BF16, true><<<grid, 256, 0, st>>>(p);
    else mla_gather_kernel<FP8K_BF16, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (cache_is_fp8) mla_gather_kernel<FP8K_F16, true><<<grid, 256, 0, st>>>(p);
    else mla_gather_kernel<FP8K_F16, false><<<grid, 256, 0, st>>>(p);
  }
  return check_launch("mla gather");
}

extern "C" int64_t fp8k_mla_decode_workspace_bytes(int64_t B, int64_t n, int64_t H, int64_t max_len) {
  if (B <= 0 || n <= 0 || H <= 0 || max_len <= 0) return 0;
  const int64_t M = n * H, slots = mla_slots(B, decode_plan(B, M, max_len).walkers);
  return up_to(slots * M * kLatent * 4, 256) + up_to(slots * M * 4, 256) + up_to(B * 8, 256);
}

extern "C" int fp8k_mla_decode(const void* q_nope, int64_t qn_stride_b, int64_t qn_stride_n, int64_t qn_stride_h, const void* q_pe,
                               int64_t qp_stride_b, int64_t qp_stride_n, int64_t qp_stride_h, const void* cache, const int32_t* page_table,
                               int64_t table_stride, int64_t table_width, const int32_t* seq_lens, const float* scale, void* out, float* lse,
                               int64_t B, int64_t n, int64_t H, int64_t pages, int64_t page_size, float sm_scale, int dtype, int cache_is_fp8,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  FP8K_REQUIRE(is_half_type(dtype), "mla decode: Half or BFloat16 queries expected");
  FP8K_REQUIRE(B >= 0 && B <= 65535 && n > 0 && H > 0 && n * H <= (1 << 16), "mla decode: bad sizes");
  FP8K_REQUIRE(sm_scale > 0.0f && sm_scale < INFINITY, "mla decode: the scale of the scores must be positive and finite");
  if (B == 0) return FP8K_OK;
  FP8K_REQUIRE(pages > 0 && pages < (1ll << 31) && page_size > 0 && page_size <= (1 << 20) && table_width > 0 && table_stride >= 0,
               "mla decode: bad sizes of the cache or the page table");
  FP8K_REQUIRE(q_nope && q_pe && cache && page_table && seq_lens && out, "mla decode: null pointer");
  FP8K_REQUIRE(aligned(q_nope, 16) && aligned(q_pe, 16) && aligned(cache, 16) && aligned(out, 16), "mla decode: operands must be 16-byte aligned");
  FP8K_REQUIRE((qn_stride_b | qn_stride_n | qn_stride_h | qp_stride_b | qp_stride_n | qp_stride_h) % 8 == 0, "mla decode: queries must be 16-byte aligned");
  FP8K_REQUIRE(qn_stride_b >= 0 && qn_stride_n >= 0 && qn_stride_h >= 0 && qp_stride_b >= 0 && qp_stride_n >= 0 && qp_stride_h >= 0,
               "mla decode: negative stride");
  const int64_t max_len = table_width * page_size;
  FP8K_REQUIRE(table_width < (1ll << 31) && max_len <= (1ll << 30) && B * (max_len / kMlaTile + 1) < (1ll << 30),
               "mla decode: the page table holds more than 2^30 tokens to a request, or 2^36 in all");
  const int64_t need = fp8k_mla_decode_workspace_bytes(B, n, H, max_len);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
    return fail(FP8K_ERR_WORKSPACE, "mla decode: workspace of %lld bytes needed, 256-byte aligned", (long long)need);
  const int64_t M = n * H;
  const Piece out_rows = rows_of(out, {}, B * M * kLatent), lse_rows{lse, B * M * 4};
  // In the queries' own place: a workgroup has read the rows of a request that it writes, and nobody else reads them.
  const bool in_place = out == q_nope && (H == 1 || qn_stride_h == kLatent) && (n == 1 || qn_stride_n == H * kLatent) && (B == 1 || qn_stride_b == M * kLatent);
  const Piece queries = rows_of(q_nope, {{B, qn_stride_b}, {n, qn_stride_n}, {H, qn_stride_h}}, kLatent);
  FP8K_REQUIRE(results_apart(out_rows, lse_rows, {rows_of(q_pe, {{B, qp_stride_b}, {n, qp_stride_n}, {H, qp_stride_h}}, kRope),
                                                  Piece{cache, pages * page_size * kLatentRow * (cache_is_fp8 ? 1 : 2)}, in_place ? Piece{} : queries}),
               "mla decode: out or lse overlaps an operand");
  const DecodePlan d = decode_plan(B, M, max_len);
  const int64_t slots = mla_slots(B, d.walkers);
  MlaDecodeArgs p{};
  p.q_nope = q_nope; p.q_pe = q_pe;
  p.qn_b = qn_stride_b; p.qn_n = qn_stride_n; p.qn_h = qn_stride_h;
  p.qp_b = qp_stride_b; p.qp_n = qp_stride_n; p.qp_h = qp_stride_h;
  p.cache = (const uint8_t*)cache; p.table = page_table; p.table_stride = table_stride; p.lens = seq_lens; p.scale = scale;
  p.out = out; p.lse = lse;
  p.part = (float*)workspace;
  p.part_lse = (float*)((uint8_t*)workspace + up_to(slots * M * kLatent * 4, 256));
  p.spans = (v2i*)((uint8_t*)p.part_lse + up_to(slots * M * 4, 256));
  p.B = (int)B; p.n = (int)n; p.H = (int)H; p.M = (int)M;
  p.page_size = (int)page_size; p.page_shift = (page_size & (page_size - 1)) ? -1 : __builtin_ctzll(page_size); p.pages = (int)pages; p.max_len = (int)max_len;
  p.walkers = d.walkers; p.mblocks = d.mblocks; p.sm_scale = sm_scale;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((d.walkers + 7) / 8 * 8 * d.mblocks));
  const bool few = B * M <= 2 * num_cu();  // rows to join: few of them have many partials each
#define MLA_DECODE(DT, FP8)                                                          \
  do {                                                                               \
    if (d.rows == 16) mla_decode_kernel<DT, FP8, 1><<<grid, 256, 0, st>>>(p);        \
    else if (d.rows == 32) mla_decode_kernel<DT, FP8, 2><<<grid, 512, 0, st>>>(p);   \
    else if (d.rows == 64) mla_decode_kernel<DT, FP8, 4><<<grid, 512, 0, st>>>(p);   \
    else mla_decode_kernel<DT, FP8, 8><<<grid, 512, 0, st>>>(p);                     \
    if (const int rc = check_launch("mla decode")) return rc;                        \
    if (few) mla_join_kernel<DT, 4><<<dim3((unsigned)M, (unsigned)B), 256, 0, st>>>(p);             \
    else mla_join_kernel<DT, 1><<<dim3((unsigned)((M + 3) / 4), (unsigned)B), 256, 0, st>>>(p);     \
  } while (0)
  if (dtype == FP8K_BF16) {
    if (cache_is_fp8) MLA_DECODE(FP8K_BF16, true);
    else MLA_DECODE(FP8K_BF16, false);
  } else {
    if (cache_is_fp8) MLA_DECODE(FP8K_F16, true);
    else MLA_DECODE(FP8K_F16, false);
  }
#undef MLA_DECODE
  return check_launch("mla decode");
}

extern "C" int64_t fp8k_mla_prefill_workspace_bytes(int64_t B, int64_t H, int64_t Tq, int64_t Tk, int64_t max_seqlen_q) {
  if (B <= 0 || H <= 0 || Tq <= 0 || Tk <= 0 || max_seqlen_q <= 0) return 0;
  return prefill_workspace(std::max(prefill_rows(prefill_cut(4, B, H, Tq, Tk, max_seqlen_q), B, H), prefill_rows(prefill_cut(8, B, H, Tq, Tk, max_seqlen_q), B, H)));
}

extern "C" int fp8k_mla_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_nope, int64_t kn_stride_t,
                                int64_t kn_stride_h, const void* k_pe, int64_t kp_stride_t, const void* v, int64_t v_stride_t,
                                int64_t v_stride_h, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, void* out, float* lse, int64_t B,
                                int64_t H, int64_t Tq, int64_t Tk, int64_t max_seqlen_q, float sm_scale, int causal, int dtype, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  clear_error();
  FP8K_REQUIRE(is_half_type(dtype), "mla prefill: Half or BFloat16 operands expected");
  FP8K_REQUIRE(B >= 0 && H > 0 && B < (1 << 24) && H <= (1 << 16) && Tq >= 0 && Tk >= 0 && Tq < (1ll << 31) - 1024 && Tk < (1ll << 31) - 1024 && max_seqlen_q >= 0,
               "mla prefill: bad sizes");
  FP8K_REQUIRE(sm_scale > 0.0f && sm_scale < INFINITY, "mla prefill: the scale of the scores must be positive and finite");
  if (B == 0 || Tq == 0 || max_seqlen_q == 0) return FP8K_OK;
  FP8K_REQUIRE(q && cu_seqlens_q && cu_seqlens_k && out && (Tk == 0 || (k_nope && k_pe && v)), "mla prefill: null pointer");
  FP8K_REQUIRE(aligned(q, 16) && aligned(k_nope, 16) && aligned(k_pe, 16) && aligned(v, 16) && aligned(out, 16) &&
                   (q_stride_t | q_stride_h | kn_stride_t | kn_stride_h | kp_stride_t | v_stride_t | v_stride_h) % 8 == 0,
               "mla prefill: operands must be 16-byte aligned");
  FP8K_REQUIRE(q_stride_t >= 0 && q_stride_h >= 0 && kn_stride_t >= 0 && kn_stride_h >= 0 && kp_stride_t >= 0 && v_stride_t >= 0 && v_stride_h >= 0,
               "mla prefill: negative stride");
  FP8K_REQUIRE(kn_stride_t < (1 << 24) && kp_stride_t < (1 << 24) && v_stride_t < (1 << 24), "mla prefill: rows of keys further apart than 2^24");
  const PrefillPlan d = prefill_plan(B, H, Tq, Tk, max_seqlen_q, causal != 0);
  const int64_t units = up_to(B * H, 8);
  FP8K_REQUIRE(units * d.blocks < (1ll << 31), "mla prefill: too many blocks of queries");
  MlaPrefillArgs p{};
  p.q = q; p.k_nope = k_nope; p.k_pe = k_pe; p.v = v;
  p.q_t = q_stride_t; p.q_h = q_stride_h; p.kn_t = kn_stride_t; p.kn_h = kn_stride_h; p.kp_t = kp_stride_t; p.v_t = v_stride_t; p.v_h = v_stride_h;
  p.cu_q = cu_seqlens_q; p.cu_k = cu_seqlens_k; p.out = out; p.lse = lse;
  p.B = (int)B; p.H = (int)H; p.Tq = (int)Tq; p.Tk = (int)Tk; p.blocks = (int)d.blocks; p.causal = causal != 0; p.sm_scale = sm_scale;
  p.splits = d.splits;
  p.xcd_bits = prefill_xcd_bits(B, H);
  const int64_t workgroups = prefill_workgroups(d, B, H);
  p.groups = (int)((workgroups / d.blocks) >> p.xcd_bits);
  const int64_t need = fp8k_mla_prefill_workspace_bytes(B, H, Tq, Tk, max_seqlen_q);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
    return fail(FP8K_ERR_WORKSPACE, "mla prefill: workspace of %lld bytes needed, 256-byte aligned", (long long)need);
  FP8K_REQUIRE(results_apart(rows_of(out, {}, Tq * H * kPreValue), Piece{lse, Tq * H * 4},
                             {rows_of(q, {{Tq, q_stride_t}, {H, q_stride_h}}, kPreNope + kRope), rows_of(k_nope, {{Tk, kn_stride_t}, {H, kn_stride_h}}, kPreNope),
                              rows_of(k_pe, {{Tk, kp_stride_t}}, kRope), rows_of(v, {{Tk, v_stride_t}, {H, v_stride_h}}, kPreValue)}),
               "mla prefill: out or lse overlaps an operand");
  p.part = (float*)workspace;
  p.part_lse = (float*)((uint8_t*)workspace + up_to(prefill_rows(d, B, H) * kPreValue * 4, 256));
  const dim3 grid((unsigned)workgroups, (unsigned)p.splits), join_grid((unsigned)workgroups, 16);
  const hipStream_t st = (hipStream_t)stream;
#define MLA_PREFILL(DT, NW)                                                       \
  do {                                                                            \
    mla_prefill_kernel<DT, NW><<<grid, 64 * NW, 0, st>>>(p);                      \
    if (p.splits > 1) {                                                           \
      if (const int rc = check_launch("mla prefill")) return rc;                  \
      mla_prefill_join_kernel<DT, NW><<<join_grid, 256, 0, st>>>(p);              \
    }                                                                             \
  } while (0)
  if (dtype == FP8K_BF16) {
    if (d.waves == 4) MLA_PREFILL(FP8K_BF16, 4);
    else MLA_PREFILL(FP8K_BF16, 8);
  } else {
    if (d.waves == 4) MLA_PREFILL(FP8K_F16, 4);
    else MLA_PREFILL(FP8K_F16, 8);
  }
#undef MLA_PREFILL
  return check_launch("mla prefill");
}

extern "C" int fp8k_merge_attention_states(const void* out_a, const float* lse_a, const void* out_b, const float* lse_b, void* out, float* lse,
                                           int64_t rows, int64_t D, int dtype, void* stream) {
  clear_error();
  FP8K_REQUIRE(is_half_type(dtype) || dtype == FP8K_F32, "merge states: float32, Half or BFloat16 expected");
  FP8K_REQUIRE(rows >= 0 && D > 0 && D % 8 == 0 && D <= (1 << 16), "merge states: the last dimension must be a multiple of 8, at most 65536");
  if (rows == 0) return FP8K_OK;
  FP8K_REQUIRE(out_a && lse_a && out_b && lse_b && out && lse, "merge states: null pointer");
  FP8K_REQUIRE(aligned(out_a, 16) && aligned(out_b, 16) && aligned(out, 16), "merge states: operands must be 16-byte aligned");
  const int64_t blocks = (rows * (D / 8) + 255) / 256;
  FP8K_REQUIRE(rows < (1ll << 40) && blocks < (1ll << 31), "merge states: too large");
  // a row's numbers may be several workgroups', and each reads both logarithms; of the rows a thread reads what it overwrites, and nothing else
  const int64_t bytes = rows * D * (dtype == FP8K_F32 ? 4 : 2), lse_bytes = rows * 4;
  const void* const parts[2] = {out_a, out_b};
  const void* const logs[2] = {lse_a, lse_b};
  for (int i = 0; i < 2; ++i) {
    FP8K_REQUIRE(!overlap(lse, lse_bytes, logs[i], lse_bytes) && !overlap(lse, lse_bytes, parts[i], bytes), "merge states: lse must be memory of its own");
    FP8K_REQUIRE((out == parts[i] || !overlap(out, bytes, parts[i], bytes)) && !overlap(out, bytes, logs[i], lse_bytes),
                 "merge states: out must be out_a, out_b or memory of its own");
  }
  FP8K_REQUIRE(!overlap(out, bytes, lse, lse_bytes), "merge states: lse must be memory of its own");
  const dim3 grid((unsigned)blocks);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == FP8K_BF16) mla_merge_kernel<FP8K_BF16><<<grid, 256, 0, st>>>(out_a, lse_a, out_b, lse_b, out, lse, rows, (int)(D / 8));
  else if (dtype == FP8K_F16) mla_merge_kernel<FP8K_F16><<<grid, 256, 0, st>>>(out_a, lse_a, out_b, lse_b, out, lse, rows, (int)(D / 8));
  else mla_merge_kernel<FP8K_F32><<<grid, 256, 0, st>>>(out_a, lse_a, out_b, lse_b, out, lse, rows, (int)(D / 8));
  return check_launch("merge states");
}
