// Expanded latent attention over ragged sequences, gfx950: per-head keys of 128 numbers and a position part of 64 that all heads share,
// values of 128.
//
//   s[i, j] = scale * (q[i, :128] . k_nope[j] + q[i, 128:] . k_pe[j]),   o[i] = sum over j <= i + Lk - Lq of softmax(s[i])[j] v[j]
//
// A workgroup is four waves with 32 query rows each, on tiles of 64 keys, and two workgroups share a CU; or eight waves, one workgroup to a CU.  Scores are formed transposed, S^T = K . Q^T, in
// 32x32x16 products: a lane holds 32 scores of one query row, a row's maximum is a lane's own and that of the lane 32 away, and what a lane
// holds is the operand of O^T = V^T . P^T as it lies, the order of the keys inside a product being free as long as V^T, read from LDS by
// transposed reads, has the same.
//
// The products of tile t + 1 with the queries run beside the exponentials of tile t, those of tile t with the values beside the exponentials' sum and the
// maximum of tile t + 1, one instruction behind the other: a product keeps the matrix core busy for 32 clocks, in which the wave issues the exponentials
// of two scores.
//
// LDS: two stages of k_nope [64, 128] and k_pe [64, 64], and two of v [64, 128], one tile behind, filled by global_load_lds; the position part is
// read where it lies, once for each head, and never copied beside the keys.  16-byte chunks of a row are permuted by the row so that the
// operand reads (16 rows, one chunk) and the transposed ones (8 rows, two chunks) spread over all banks.
//
// The loop is 20 KB of instructions, which a short sequence runs through once: one tile of keys takes 6.4 us, where a loop without that overlap, 7 KB, takes 5.2.
//
// Measured, bf16: 8192 queries of 128 heads with their own keys, causal, 2.5 - 2.65 ms by the card or 1.04 - 1.1 PFLOP/s, where a library's matrix product of 8192^3 reaches 1.55; the
// matrix cores are busy 65 % of the clocks, at the 1.6 GHz that the power limit leaves; a tile of four waves costs LDS some 1160 clocks (at the rates that its
// reads and fills reach alone) and the vector instructions 1020, beside the products' 1280.  1000 queries of 32 heads with 10000 keys, float16, 207 us or 0.94 PFLOP/s, the join 9 us of it.  17
// prompts of 100 to 300 tokens, 16 heads, 24 - 25 us: 2.8 TB/s, latency (a workgroup alone takes 6 to 9 us).
#pragma once

#include "mla_common.h"

namespace fp8k {

struct MlaPrefillArgs {
  const void *q, *k_nope, *k_pe, *v;
  int64_t q_t, q_h, kn_t, kn_h, kp_t, v_t, v_h;  // strides in elements
  const int32_t *cu_q, *cu_k;
  void* out;   // [Tq, H, 128]
  float* lse;  // [Tq, H] or null
  float *part, *part_lse;  // of split keys: [splits, gridDim.x, rows of a workgroup, 128], [splits, gridDim.x, rows]
  int B, H, Tq, Tk, blocks;  // blocks: of a workgroup's queries, that a sequence has at most
  int splits;              // of a block's keys, each a workgroup's
  int xcd_bits;            // of the number of heads side by side: 8, one to an XCD, or 1
  int groups;              // of them
  int causal;
  float sm_scale;
};

constexpr int kPreKeys = 64, kPreNope = 128, kPreValue = 128;

// position of the 16-byte chunks of a value's row of 256 bytes: c ^ swizzle(r), as the transposed reads of 16 rows x 32 bytes spread best
__device__ __forceinline__ int mla_value_swizzle(int r) { return ((r & 1) ? 12 : 0) ^ ((r & 2) ? 10 : 0) ^ ((r & 4) ? 6 : 0); }

// A workgroup's 128 (256) queries.  The blocks of a sequence's head follow each other on one XCD (workgroup i runs on XCD i % 8): they read the same
// keys.  (Few heads, or some more than a multiple of 8, would leave XCDs idle: their blocks go to all of them.)  Of a causal head the last queries, which have most keys, come first, in every other head the first ones: the workgroups that start
// together, two to a CU, are long and short ones.
struct MlaBlock {
  int b, h, q_begin, lq, q0, rows;
};
template <int ROWS>
__device__ __forceinline__ MlaBlock mla_block(const MlaPrefillArgs& p) {
  MlaBlock x;
  const int line = (int)blockIdx.x >> p.xcd_bits, group = p.blocks == 1 ? line : line / p.blocks, place = line - group * p.blocks;
  const int unit = (group << p.xcd_bits) + ((int)blockIdx.x & ((1 << p.xcd_bits) - 1));
  x.rows = 0;
  if (unit >= p.B * p.H) return x;
  x.b = unit / p.H;
  x.h = unit - x.b * p.H;
  x.q_begin = min(max(p.cu_q[x.b], 0), p.Tq);
  x.lq = min(max(p.cu_q[x.b + 1], x.q_begin), p.Tq) - x.q_begin;
  x.q0 = ((p.groups - group) & 1 ? p.blocks - 1 - place : place) * ROWS;
  x.rows = min(ROWS, x.lq - x.q0);
  return x;
}

// Where a split's rows of this workgroup's block begin, among those of all.
template <int ROWS>
__device__ __forceinline__ int64_t mla_split_row(int split) {
  return ((int64_t)split * gridDim.x + blockIdx.x) * ROWS;
}

template <int DT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void mla_prefill_kernel(const MlaPrefillArgs p) {
  constexpr int kWaveRows = kPreKeys / NW;  // of a tile of keys, fetched by a wave
  constexpr int kKey = kPreKeys * 384, kVal = kPreKeys * 256, kPe = kPreKeys * 256;  // bytes of a stage, and where k_pe begins in it
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kKey + 2 * kVal];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, half = lane >> 5;
  const MlaBlock at = mla_block<32 * NW>(p);
  if (at.rows <= 0) return;
  const int h = at.h, q_begin = at.q_begin, q0 = at.q0, lq = at.lq;
  const int k_begin = min(max(p.cu_k[at.b], 0), p.Tk), k_end = min(max(p.cu_k[at.b + 1], k_begin), p.Tk), lk = k_end - k_begin;
  const int shift_k = lk - lq;  // query i is the key of place i + shift_k
  const int last_row = q0 + at.rows - 1;
  const int keys = p.causal ? min(max(last_row + shift_k + 1, 0), lk) : lk;  // that any row of the block sees
  // this workgroup's share of their tiles
  const int all_tiles = (keys + kPreKeys - 1) / kPreKeys, split = blockIdx.y;
  int first = 0, tiles = all_tiles;
  if (p.splits > 1) {  // at most 2^25 tiles and 32 splits
    first = (uint32_t)all_tiles * split / p.splits;
    tiles = (uint32_t)all_tiles * (split + 1) / p.splits;
  }

  const int row0 = q0 + w * 32, qi = min(row0 + l31, lq - 1);
  const int lim = p.causal ? min(qi + shift_k + 1, lk) : lk;  // keys that this lane's row sees
  const int wave_keys = p.causal ? min(min(row0 + 31, lq - 1) + shift_k + 1, lk) : lk, wave_free = p.causal ? min(row0 + shift_k + 1, lk) : lk;
  const float c = p.sm_scale * kLog2e;

  v4i q[12];
  {
    const u16* const from = (const u16*)p.q + (int64_t)(q_begin + qi) * p.q_t + h * p.q_h + 8 * half;
#pragma unroll
    for (int ks = 0; ks < 12; ++ks) q[ks] = *(const v4i*)(from + 16 * ks);
  }

  // A wave fetches 16 rows (of eight waves: 8) of each part of a stage: four wave-loads of k_nope and of v, of four rows each, two of k_pe, of eight.  Load j is of row
  // 4 j (8 j) + lane / 16 (lane / 8) of the wave's: the lane's offset is that row's, which j moves by a number that all lanes share, and a chunk, which j
  // moves by an exclusive or.  Rows past the sequence's last are that row again (masked).
  const uint32_t lds0 = lds_address(smem);
  const int r16 = w * kWaveRows + (lane >> 4), r8 = w * kWaveRows + (lane >> 3);
  const int n_chunk = (lane & 15) ^ (r16 & 15), p_chunk = (lane & 7) ^ ((r8 >> 1) & 7), v_part = (lane & 15) ^ mla_value_swizzle(r16);
  const uint32_t n_stride = (uint32_t)p.kn_t * 2, p_stride = (uint32_t)p.kp_t * 2, v_stride = (uint32_t)p.v_t * 2;  // bytes
  const uint8_t* const n_from = (const uint8_t*)p.k_nope + ((int64_t)k_begin * p.kn_t + h * p.kn_h) * 2;
  const uint8_t* const p_from = (const uint8_t*)p.k_pe + (int64_t)k_begin * p.kp_t * 2;
  const uint8_t* const v_from = (const uint8_t*)p.v + ((int64_t)k_begin * p.v_t + h * p.v_h) * 2;
  auto fetch_keys = [&](int t) {
    const uint32_t to = lds0 + (t & 1) * kKey + w * kWaveRows * 256, to_pe = lds0 + (t & 1) * kKey + kPe + w * kWaveRows * 128;
    const uint8_t* const n_tile = n_from + (uint64_t)(uint32_t)(t * kPreKeys) * n_stride;
    const uint8_t* const p_tile = p_from + (uint64_t)(uint32_t)(t * kPreKeys) * p_stride;
    if ((t + 1) * kPreKeys <= lk) {
#pragma unroll
      for (int j = 0; j < kWaveRows / 4; ++j) load16_to_lds(n_tile + 4 * j * n_stride, r16 * n_stride + ((n_chunk ^ (4 * j)) << 4), to + j * 1024);
#pragma unroll
      for (int j = 0; j < kWaveRows / 8; ++j) load16_to_lds(p_tile + 8 * j * p_stride, r8 * p_stride + ((p_chunk ^ (4 * j)) << 4), to_pe + j * 1024);
    } else {
      const int last = lk - 1 - t * kPreKeys;
#pragma unroll
      for (int j = 0; j < kWaveRows / 4; ++j) load16_to_lds(n_tile, min(r16 + 4 * j, last) * n_stride + ((n_chunk ^ (4 * j)) << 4), to + j * 1024);
#pragma unroll
      for (int j = 0; j < kWaveRows / 8; ++j) load16_to_lds(p_tile, min(r8 + 8 * j, last) * p_stride + ((p_chunk ^ (4 * j)) << 4), to_pe + j * 1024);
    }
  };
  auto fetch_values = [&](int t) {
    const uint32_t to = lds0 + 2 * kKey + (t & 1) * kVal + w * kWaveRows * 256;
    const uint8_t* const tile = v_from + (uint64_t)(uint32_t)(t * kPreKeys) * v_stride;
    if ((t + 1) * kPreKeys <= lk) {
#pragma unroll
      for (int j = 0; j < kWaveRows / 4; ++j) load16_to_lds(tile + 4 * j * v_stride, r16 * v_stride + ((v_part ^ (j & 1 ? 6 : 0)) << 4), to + j * 1024);
    } else {
      const int last = lk - 1 - t * kPreKeys;
#pragma unroll
      for (int j = 0; j < kWaveRows / 4; ++j) load16_to_lds(tile, min(r16 + 4 * j, last) * v_stride + ((v_part ^ (j & 1 ? 6 : 0)) << 4), to + j * 1024);
    }
  };

  // LDS offsets of a lane in a stage: row l31 of a 32-key tile, chunk `half` of k_nope and of k_pe; a transposed read of v.  Other chunks differ in
  // bits 4 .. 7 alone: an exclusive or.
  const int n_off = l31 * 256 + ((half ^ (l31 & 15)) << 4), p_off = kPe + l31 * 128 + ((half ^ ((l31 >> 1) & 7)) << 4);
  const int v_row = 4 * half + ((lane & 15) >> 2), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int v_off = 2 * kKey + v_row * 256 + ((v_chunk ^ mla_value_swizzle(v_row)) << 4) + ((lane & 1) << 3);
  auto anew = [](int x) {  // computed where it is used, rather than a dozen addresses kept
    asm volatile("" : "+v"(x));
    return x;
  };

  v16f o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
  float m = -INFINITY, l = 0.0f, l_odd = 0.0f;  // of the odd scores: two sums that do not wait for each other

  // operand i of a tile's scores: 24 products, the two 32-key tiles by turns
  auto key_operand = [&](int n_at, int p_at, int i) {
    const int ks = i >> 1, nt = i & 1;
    return *(const v4i*)(smem + (ks < 8 ? (n_at ^ (ks << 5)) + nt * 32 * 256 : (p_at ^ ((ks - 8) << 5)) + nt * 32 * 128));
  };
  auto first_scores = [&](v16f* s) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[nt][i] = 0.0f;
  };

  auto score = [](v16f* s, int i) -> float { return s[i >> 4][i & 15]; };
  auto top_of = [&](v16f* s) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, score(s, i));
    return top;
  };

  // One tile: the weights of the scores s of tile t, whose largest is top, and their product with v; and, if there are any, the scores `next` of tile
  // t + 1, whose largest is returned.
  auto step = [&](int t, v16f* s, float top, v16f* next) -> float {
    wait_loads<0>();
    lds_only_barrier();  // keys of t + 1 and values of t have arrived, and nobody reads those of t and t - 1 any more
    if (t + 2 < tiles) fetch_keys(t + 2);
    if (t + 1 < tiles) fetch_values(t + 1);
    if (t * kPreKeys >= wave_keys) return top;  // nothing that this wave's rows see

    // a lane's scores are those of query row l31, keys 32 nt + 8 (i / 4) + 4 half + i % 4
    if (__builtin_expect((t + 1) * kPreKeys > wave_free, 0)) {
      const int key0 = t * kPreKeys + 4 * half;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + nt * 32 + 8 * (i >> 2) + (i & 3) >= lim) s[nt][i] = -INFINITY;
      top = top_of(s);
    }
    // c > 0.  The row's maximum, over two lanes, is asked for only when one of them has passed the old one by far.
    if (__builtin_expect(__any(top * c > m + kMaxSlack), 0)) {
      top = max_across32(top) * c;
      const float raised = top > m + kMaxSlack ? top : m;
      const float alpha = raised != m ? __builtin_amdgcn_exp2f(m - raised) : 1.0f;
      m = raised;
      l *= alpha;
      l_odd *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
    }
    const float shift = shift_of(m);
    uint32_t pk[16];
    // scores 2 j and 2 j + 1: arguments, exponentials, and their rounding to the 16-bit type, as the matrix core takes them; the sum is of the unrounded ones
    auto argument = [&](int j) {
      s[j >> 3][(2 * j) & 15] = fmaf(s[j >> 3][(2 * j) & 15], c, -shift);
      s[j >> 3][(2 * j + 1) & 15] = fmaf(s[j >> 3][(2 * j + 1) & 15], c, -shift);
    };
    auto exponential = [&](int j) {
      s[j >> 3][(2 * j) & 15] = __builtin_amdgcn_exp2f(s[j >> 3][(2 * j) & 15]);
      s[j >> 3][(2 * j + 1) & 15] = __builtin_amdgcn_exp2f(s[j >> 3][(2 * j + 1) & 15]);
    };
    auto round = [&](int j) { pk[j] = pack2<DT>(score(s, 2 * j), score(s, 2 * j + 1)); };
    argument(0);
    argument(1);
    exponential(0);
    const bool more = t + 1 < tiles && (t + 1) * kPreKeys < wave_keys;
    if (more) {
      constexpr int kAhead = 5;
      v4i ring[kAhead];
      const int n_at = anew(n_off + ((t + 1) & 1) * kKey), p_at = anew(p_off + ((t + 1) & 1) * kKey);
      first_scores(next);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ring[i] = key_operand(n_at, p_at, i);
#pragma unroll
      for (int i = 0; i < 24; ++i) {
        next[i & 1] = mfma32<DT>(ring[i % kAhead], q[i >> 1], next[i & 1]);
        if (i + kAhead < 24) ring[i % kAhead] = key_operand(n_at, p_at, i + kAhead);
        if (i % 3 != 2) {  // two pairs to three products
          const int j = i / 3 * 2 + i % 3;
          if (j + 2 < 16) argument(j + 2);
          if (j + 1 < 16) exponential(j + 1);
          round(j);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j + 2 < 16) argument(j + 2);
        if (j + 1 < 16) exponential(j + 1);
        round(j);
      }
    }

    top = -INFINITY;
    {
      constexpr int kAhead = 5;
      v2i ring[kAhead][2];
      const int v_at = anew(v_off + (t & 1) * kVal);
      auto read = [&](int i, v2i* to) {
        const uint8_t* const at = smem + (v_at ^ ((i & 3) << 6)) + (i >> 2) * 16 * 256;
        to[0] = lds_read_transposed(at);
        to[1] = lds_read_transposed(at + 8 * 256);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) read(i, ring[i]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const v2i* const a = ring[i % kAhead];
        const int k = i >> 2;
        o[i & 3] = mfma32<DT>(v4i{a[0][0], a[0][1], a[1][0], a[1][1]}, v4i{(int)pk[4 * k], (int)pk[4 * k + 1], (int)pk[4 * k + 2], (int)pk[4 * k + 3]}, o[i & 3]);
        if (i + kAhead < 16) read(i + kAhead, ring[i % kAhead]);
        l += score(s, 2 * i);
        l_odd += score(s, 2 * i + 1);
        // (stale, and not used, after the last tile)
        top = fmaxf(fmaxf(top, score(next, 2 * i)), score(next, 2 * i + 1));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    return top;
  };

  v16f s0[2], s1[2];
  first_scores(s0);
  first_scores(s1);
  if (first < tiles) {
    // all that the first tile takes, and the next keys, asked for at once: a short sequence waits for memory once
    fetch_keys(first);
    fetch_values(first);
    if (first + 1 < tiles) fetch_keys(first + 1);
    wait_loads<0>();
    lds_only_barrier();
    if (first * kPreKeys < wave_keys) {
      const int n_at = n_off + (first & 1) * kKey, p_at = p_off + (first & 1) * kKey;
#pragma unroll
      for (int i = 0; i < 24; ++i) s0[i & 1] = mfma32<DT>(key_operand(n_at, p_at, i), q[i >> 1], s0[i & 1]);
    }
  }
  float top = top_of(s0);
  for (int t = first; t < tiles; t += 2) {
    top = step(t, s0, top, s1);
    if (t + 1 < tiles) top = step(t + 1, s1, top, s0);
  }

  l = sum_across32(l + l_odd);
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (row0 + l31 < lq) {
    const int64_t row = (int64_t)(q_begin + row0 + l31) * p.H + h;
    const float lse2 = l == 0.0f ? -INFINITY : __builtin_amdgcn_logf(l) + shift_of(m);
    if (p.splits == 1) {
      u16* const to = (u16*)p.out + row * kPreValue + 4 * half;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *(v2i*)(to + dt * 32 + k * 8) = v2i{(int)pack2<DT>(o[dt][4 * k] * f, o[dt][4 * k + 1] * f), (int)pack2<DT>(o[dt][4 * k + 2] * f, o[dt][4 * k + 3] * f)};
      if (half == 0 && p.lse) p.lse[row] = lse2 * kLn2;
    } else {
      const int64_t place = mla_split_row<32 * NW>(split) + w * 32 + l31;
      float* const to = p.part + place * kPreValue + 4 * half;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int k = 0; k < 4; ++k) *(v4f*)(to + dt * 32 + k * 8) = v4f{o[dt][4 * k] * f, o[dt][4 * k + 1] * f, o[dt][4 * k + 2] * f, o[dt][4 * k + 3] * f};
      if (half == 0) p.part_lse[place] = lse2;
    }
  }
}

// Adds up the splits of a block's rows, in the order of their keys: 32 lanes of four columns to a row.
template <int DT, int NW>
__global__ __launch_bounds__(256) void mla_prefill_join_kernel(const MlaPrefillArgs p) {
  const MlaBlock at = mla_block<32 * NW>(p);
  const int col = 4 * (int)(threadIdx.x & 31);
  for (int r = (int)blockIdx.y * 8 + (int)(threadIdx.x >> 5); r < at.rows; r += (int)gridDim.y * 8) {
    const int64_t row = (int64_t)(at.q_begin + at.q0 + r) * p.H + at.h, from = mla_split_row<32 * NW>(0) + r, step = mla_split_row<32 * NW>(1) - mla_split_row<32 * NW>(0);
    float top = -INFINITY;
    for (int i = 0; i < p.splits; ++i) top = fmaxf(top, p.part_lse[from + i * step]);
    const float shift = shift_of(top);
    float sum = 0.0f;
    v4f x = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < p.splits; ++i) {
      const float weight = __builtin_amdgcn_exp2f(p.part_lse[from + i * step] - shift);
      sum += weight;
      x += weight * *(const v4f*)(p.part + (from + i * step) * kPreValue + col);
    }
    x *= sum == 0.0f ? 0.0f : 1.0f / sum;
    *(v2i*)((u16*)p.out + row * kPreValue + col) = v2i{(int)pack2<DT>(x[0], x[1]), (int)pack2<DT>(x[2], x[3])};
    if (col == 0 && p.lse) p.lse[row] = sum == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(sum) + shift) * kLn2;
  }
}

}  // namespace fp8k
