// Absorbed latent attention of a few new tokens over the paged cache, gfx950.
//
// A request has M = queries x heads rows that all read the same cached rows: keys of 576, values their first 512.  With r over its tokens
//   s[m, r] = scale * q[m] . row[r],   p = exp(s - max s),   o[m] = sum p[r] row[r, :512] / sum p[r]
//
// The scores are formed transposed, S^T = K . Q^T, so that a lane holds scores of one query row, and what it holds is the operand of
// O^T = V^T . P^T as it lies: the order of the tokens inside a product is free, as long as V^T, read from LDS by transposed reads,
// has the same.  P never goes through LDS, and the rescaling factors of O are a lane's own.
//
// A workgroup is eight waves (four with WM = 1) on tiles of 64 tokens.  WM of them split the R = 16 WM query rows, the other factor splits the
// tokens of a tile; each has its own running maximum and sum, and waves that share rows are joined through LDS at the end.  A wave holds
// its 16 rows' queries and all 512 columns of O, 200 registers.  With WM = 1 a wave reads nothing but the 16 rows that it fetched itself, and the
// loop has no barrier.
//
// LDS: two tiles of 9 blocks of [64 rows][64 numbers], filled by global_load_lds with per-lane addresses (pages lie anywhere, beyond 4 GB
// too).  A wave-load is 8 rows of a block, so a lane fetches from one row of a tile (WM = 1: two), at multiples of 128 bytes.  The
// 16-byte chunk c of row r of a block sits at c ^ swizzle(r), which keeps both the operand reads (16 rows, one chunk) and the transposed
// ones (8 rows, two chunks) off each other's banks.  8-bit rows are fetched to a stage of their own, 16 rows x 64 bytes to a wave-load, and
// widened into one 16-bit tile.
//
// Work: the tiles of all requests in a row are cut into equal runs, one to a workgroup, from the lengths on the device: a captured graph
// needs no plan.  A run that holds all of a request writes its result; others write normalised float32 partials and the base-2
// logarithm of their sums, which mla_join_kernel adds up.
#pragma once

#include "mla_common.h"

namespace fp8k {

struct MlaDecodeArgs {
  const void *q_nope, *q_pe;
  int64_t qn_b, qn_n, qn_h, qp_b, qp_n, qp_h;  // strides in elements
  const uint8_t* cache;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const float* scale;  // of the 8-bit cache, or null
  void* out;           // [B, n, H, 512]
  float* lse;          // [B, n, H] or null
  float *part, *part_lse;  // [walkers + B, M, 512], [walkers + B, M]
  int B, n, H, M;
  int page_size, pages, max_len;
  int walkers, mblocks;
  float sm_scale;
};

constexpr int kMlaTile = 64;         // tokens of a tile
constexpr int kMlaBlock = kMlaTile * 128;  // bytes of a block of 64 numbers of a tile in LDS
constexpr int kMlaMinRun = 2;        // tiles that a run has at least

__device__ __forceinline__ int mla_len(const MlaDecodeArgs& p, int b) { return min(max(p.lens[b], 0), p.max_len); }
__device__ __forceinline__ int mla_tiles(int len) { return (len + kMlaTile - 1) / kMlaTile; }
// tiles of a run, from all requests' tiles
__device__ __forceinline__ int mla_run(int total, int walkers) { return max((total + walkers - 1) / walkers, kMlaMinRun); }

// Tiles of all requests, by a workgroup of NW waves; every thread returns the total.  Thread t counts requests [t * per, + per): `before`
// is what lies in front of them.
template <int NW>
__device__ __forceinline__ int mla_scan(const MlaDecodeArgs& p, int per, int& before, int* lds) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int sum = 0;
  for (int b = tid * per; b < min((tid + 1) * per, p.B); ++b) sum += mla_tiles(mla_len(p, b));
  int run = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(run, d);
    if (lane >= d) run += v;
  }
  if (lane == 63) lds[w] = run;
  __syncthreads();
  int total = 0, base = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    if (i < w) base += lds[i];
    total += lds[i];
  }
  before = base + run - sum;
  return total;
}

// position of a row's 16-byte chunks in a block: c ^ swizzle(r).  Rows are 128 bytes: neighbours use different halves of the banks already.  Of the
// linear maps of bits 1 .. 3 of r, those with full rate for either kind of read (operand reads 225 bytes a clock and CU, transposed ones 161; (r >> 1) & 7
// does as well for the first alone, its rotation has half the rate there).
__device__ __forceinline__ int mla_swizzle(int r) { return ((r & 2) ? 6 : 0) ^ ((r & 4) ? 5 : 0) ^ ((r & 8) ? 4 : 0); }

template <int DT, bool FP8, int WM>
__global__ __launch_bounds__(WM == 1 ? 256 : 512) void mla_decode_kernel(const MlaDecodeArgs p) {
  constexpr int NW = WM == 1 ? 4 : 8, WT = NW / WM, R = 16 * WM, NT = 4 / WT;  // NT: 16-token tiles of a wave
  constexpr int kTileBytes = 9 * kMlaBlock, kStageBytes = FP8 ? kTileBytes / 2 : kTileBytes;
  constexpr int kRow = FP8 ? kLatentRow : 2 * kLatentRow;  // bytes of a cached row
  constexpr int kRowsOfLane = FP8 || NW == 8 ? 1 : 2;       // that a lane fetches from
  // 16-bit: two tiles.  8-bit: a tile, then two stages of raw rows.
  __shared__ __attribute__((aligned(1024))) uint8_t smem[FP8 ? kTileBytes + 2 * kStageBytes : 2 * kTileBytes];
  __shared__ int found[2], scan[NW];
  __shared__ float join_m[NW][16], join_l[NW][16];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w % WM, wt = w / WM, l15 = lane & 15, g = lane >> 4;
  // the workgroups of a run's row blocks read the same rows: on one XCD (workgroup i runs on XCD i % 8), side by side
  const int per8 = p.mblocks * 8;
  const int walker = (int)(blockIdx.x / per8) * 8 + (int)(blockIdx.x % 8), mblk = (int)(blockIdx.x % per8) / 8;
  if (walker >= p.walkers) return;

  const int per = (p.B + NW * 64 - 1) / (NW * 64);
  int before;
  const int total = mla_scan<NW>(p, per, before, scan);
  const int run = mla_run(total, p.walkers);
  if ((int64_t)walker * run >= total) return;
  const int first = walker * run, last = min(first + run, total);
  {
    int at = before;
    for (int b = tid * per; b < min((tid + 1) * per, p.B); ++b) {
      const int t = mla_tiles(mla_len(p, b));
      if (first >= at && first < at + t) {
        found[0] = b;
        found[1] = at;
      }
      at += t;
    }
  }
  __syncthreads();
  int b = __builtin_amdgcn_readfirstlane(found[0]), at = __builtin_amdgcn_readfirstlane(found[1]);

  const float kscale = FP8 && p.scale ? *p.scale : 1.0f;
  const float c = p.sm_scale * kLog2e * kscale;

  const int row = mblk * R + wm * 16 + l15;  // this lane's, of the M of a request

  // LDS offsets: operand reads of K (row l15 of a 16-token tile, chunk 4 ks + g), transposed reads of V
  const int k_off = (wt * NT * 16 + l15) * 128 + ((g ^ mla_swizzle(l15)) << 4);
  const int v_row = 4 * g + (l15 >> 2);
  const int v_off = (wt * NT * 16 + v_row) * 128 + ((((l15 & 3) >> 1) ^ mla_swizzle(v_row)) << 4) + ((l15 & 1) << 3);

  for (int pos = first; pos < last; ++b) {
    const int len = mla_len(p, b), tiles = mla_tiles(len);
    const int t_begin = pos - at, t_end = min(last - at, tiles);
    at += tiles;
    if (t_begin >= t_end) continue;
    pos += t_end - t_begin;

    // ---- the rows' queries, and how many tokens each sees
    const int r_in = min(row, p.M - 1), qi = r_in / p.H, qh = r_in - qi * p.H;
    const int lim = len - (p.n - 1 - qi);
    v4i q[18];
    {
      const u16* qn = (const u16*)p.q_nope + b * p.qn_b + qi * p.qn_n + qh * p.qn_h + 8 * g;
      const u16* qp = (const u16*)p.q_pe + b * p.qp_b + qi * p.qp_n + qh * p.qp_h + 8 * g;
#pragma unroll
      for (int ks = 0; ks < 16; ++ks) q[ks] = *(const v4i*)(qn + 32 * ks);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) q[16 + ks] = *(const v4i*)(qp + 32 * ks);
    }

    v4f o[32];
#pragma unroll
    for (int dt = 0; dt < 32; ++dt) o[dt] = v4f{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;

    // ---- fetching.  Tokens past the end are the last one's row again (masked).  16 bits: a wave has 8 rows of a tile (four waves: 16).  8 bits:
    // wave w has 16 rows, from row 16 (w % 4) on; of eight waves, two share them, by blocks.
    struct Rows {
      const uint8_t* at[kRowsOfLane];
    };
    auto rows_of = [&](int t) {
      Rows rows;
#pragma unroll
      for (int k = 0; k < kRowsOfLane; ++k) {
        const int r = FP8 ? 16 * (w & 3) + (lane >> 2) : 8 * (w * kRowsOfLane + k) + (lane >> 3);
        const int tok = min(t * kMlaTile + r, len - 1), page = tok / p.page_size;
        const int e = min(max(p.table[b * p.table_stride + page], 0), p.pages - 1);
        rows.at[k] = p.cache + ((int64_t)e * p.page_size + (tok - page * p.page_size)) * kRow + (FP8 ? (lane & 3) : (lane & 7) ^ mla_swizzle(r)) * 16;
      }
      return rows;
    };
    auto fetch = [&](const Rows& rows, uint8_t* stage) {
      if constexpr (FP8) {
        uint8_t* const to = stage + (w & 3) * 9 * 1024;
        if (NW == 4) load_blocks_to_lds<64, 1024, 0, 9>(rows.at[0], to);
        else if (w < 4) load_blocks_to_lds<64, 1024, 0, 5>(rows.at[0], to);
        else load_blocks_to_lds<64, 1024, 5, 9>(rows.at[0], to);
      } else {
#pragma unroll
        for (int k = 0; k < kRowsOfLane; ++k) load_blocks_to_lds<128, kMlaBlock, 0, 9>(rows.at[k], stage + 8 * (w * kRowsOfLane + k) * 128);
      }
    };

    Rows rows = rows_of(t_begin);
    uint8_t* const stages = smem + (FP8 ? kTileBytes : 0);
    fetch(rows, stages);
    rows = rows_of(min(t_begin + 1, t_end - 1));
    for (int t = t_begin; t < t_end; ++t) {
      uint8_t* const stage = stages + ((t - t_begin) & 1) * kStageBytes;
      uint8_t* const other = stages + ((t - t_begin + 1) & 1) * kStageBytes;
      // this tile's rows have arrived, and nobody reads the tile before any more
      if (WM > 1) wait_all_barrier();
      else wait_all();
      if (t + 1 < t_end) {
        const Rows next = rows;
        rows = rows_of(min(t + 2, t_end - 1));
        fetch(next, other);
      }
      const uint8_t* tile = stage;
      if (FP8) {
        uint8_t* const to = smem + (16 * (w & 3) + (lane >> 2)) * 128;
        const int at0 = ((2 * (lane & 3)) ^ mla_swizzle(lane >> 2)) << 4;
        const uint8_t* const from = stage + (w & 3) * 9 * 1024 + lane * 16;
        auto widen = [&](int j) {
          const v4i raw = *(const v4i*)(from + j * 1024);
          *(v4i*)(to + j * kMlaBlock + at0) = v4i{(int)fp8_to_16bit<DT, false>(raw[0]), (int)fp8_to_16bit<DT, true>(raw[0]),
                                                  (int)fp8_to_16bit<DT, false>(raw[1]), (int)fp8_to_16bit<DT, true>(raw[1])};
          *(v4i*)(to + j * kMlaBlock + (at0 ^ 16)) = v4i{(int)fp8_to_16bit<DT, false>(raw[2]), (int)fp8_to_16bit<DT, true>(raw[2]),
                                                         (int)fp8_to_16bit<DT, false>(raw[3]), (int)fp8_to_16bit<DT, true>(raw[3])};
        };
        if (NW == 4 || w < 4) {
#pragma unroll
          for (int j = 0; j < (NW == 4 ? 9 : 5); ++j) widen(j);
        } else {
#pragma unroll
          for (int j = 5; j < 9; ++j) widen(j);
        }
        if (WM > 1) {
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
        tile = smem;
      }

      // ---- S^T = K . Q^T
      v4f s[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < 18; ++ks)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          s[nt] = mfma16<DT>(*(const v4i*)(tile + ((k_off ^ ((ks & 1) << 6)) + (ks >> 1) * kMlaBlock + nt * 16 * 128)), q[ks], s[nt]);

      // ---- softmax: a lane's scores are those of query row l15, tokens 16 nt + 4 g + i
      const int tok0 = t * kMlaTile + wt * NT * 16 + 4 * g;
      const bool masked = (t + 1) * kMlaTile > len - (p.n - 1);
      float top = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = s[nt][i] * c;
          if (masked && tok0 + nt * 16 + i >= lim) v = -INFINITY;
          s[nt][i] = v;
          top = fmaxf(top, v);
        }
      top = max_across32(max_across16(top));
      const float raised = top > m + kMaxSlack ? top : m;
      if (__any(raised != m)) {
        const float alpha = raised != m ? __builtin_amdgcn_exp2f(m - raised) : 1.0f;
        m = raised;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < 32; ++dt) o[dt] *= alpha;
      }
      const float shift = shift_of(m);
      uint32_t pk[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(s[nt][i] - shift);
          l += e[i];
        }
        // weights rounded to the 16-bit type, as the matrix core takes them; their sum is of the unrounded ones
        pk[nt][0] = pack2<DT>(e[0], e[1]);
        pk[nt][1] = pack2<DT>(e[2], e[3]);
      }

      // ---- O^T += V^T . P^T
#pragma unroll
      for (int dt = 0; dt < 32; ++dt) {
        const uint8_t* const v = tile + ((v_off ^ ((dt & 3) << 5)) + (dt >> 2) * kMlaBlock);
        if constexpr (NT == 1) {
          o[dt] = mfma16_half<DT>(lds_read_transposed(v), v2i{(int)pk[0][0], (int)pk[0][1]}, o[dt]);
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; nt += 2) {
            const v2i a0 = lds_read_transposed(v + nt * 16 * 128), a1 = lds_read_transposed(v + (nt + 1) * 16 * 128);
            o[dt] = mfma16<DT>(v4i{a0[0], a0[1], a1[0], a1[1]}, v4i{(int)pk[nt][0], (int)pk[nt][1], (int)pk[nt + 1][0], (int)pk[nt + 1][1]}, o[dt]);
          }
        }
      }
    }

    // ---- join the waves that share rows, normalise, write
    const bool whole = t_end - t_begin == tiles;
    const int64_t slot = walker + b;
    l = sum_across32(sum_across16(l));
    if (g == 0) {
      join_m[w][l15] = m;
      join_l[w][l15] = l;
    }
    __syncthreads();  // and nobody reads a tile any more
    {
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < WT; ++i) top = fmaxf(top, join_m[i * WM + wm][l15]);
      const float shift = shift_of(top);
#pragma unroll
      for (int i = 0; i < WT; ++i) sum += join_l[i * WM + wm][l15] * __builtin_amdgcn_exp2f(join_m[i * WM + wm][l15] - shift);
      // a NaN sum is not 0 and stays one
      const float f = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - shift) / sum * kscale;
#pragma unroll
      for (int dt = 0; dt < 32; ++dt) o[dt] *= f;
      if (wt == 0 && g == 0 && row < p.M) {
        const float lse2 = sum == 0.0f ? -INFINITY : __builtin_amdgcn_logf(sum) + shift;
        if (!whole) p.part_lse[slot * p.M + row] = lse2;
        else if (p.lse) p.lse[(int64_t)b * p.M + row] = lse2 * kLn2;
      }
    }
    // a quarter of the 512 columns at a time through LDS: [WT][R] rows of 128 floats (and 4 of padding)
    constexpr int kLd = 132;
    float* const buf = (float*)smem;
#pragma unroll
    for (int quarter = 0; quarter < 4; ++quarter) {
#pragma unroll
      for (int d = 0; d < 8; ++d) *(v4f*)(buf + (wt * R + wm * 16 + l15) * kLd + d * 16 + 4 * g) = o[quarter * 8 + d];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < R * 16 / (NW * 64); ++k) {
        const int row_in = (k * NW * 64 + tid) >> 4, col = (tid & 15) * 8, r = mblk * R + row_in;
        v4f x = *(const v4f*)(buf + row_in * kLd + col), y = *(const v4f*)(buf + row_in * kLd + col + 4);
#pragma unroll
        for (int i = 1; i < WT; ++i) {
          x += *(const v4f*)(buf + (i * R + row_in) * kLd + col);
          y += *(const v4f*)(buf + (i * R + row_in) * kLd + col + 4);
        }
        if (r < p.M) {
          if (whole) {
            const v4i v = {(int)pack2<DT>(x[0], x[1]), (int)pack2<DT>(x[2], x[3]), (int)pack2<DT>(y[0], y[1]), (int)pack2<DT>(y[2], y[3])};
            *(v4i*)((u16*)p.out + ((int64_t)b * p.M + r) * kLatent + quarter * 128 + col) = v;
          } else {
            float* const to = p.part + (slot * p.M + r) * kLatent + quarter * 128 + col;
            *(v4f*)to = x;
            *(v4f*)(to + 4) = y;
          }
        }
      }
      __syncthreads();
    }
  }
}

// Adds up the partials of requests that several runs share, in the order of their tokens, and gives requests without tokens their zeros.
// One workgroup to a row and request; 128 threads of four columns.
template <int DT>
__global__ __launch_bounds__(256) void mla_join_kernel(const MlaDecodeArgs p) {
  __shared__ int mine[2], scan4[4];
  __shared__ float weights[256];
  const int r = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int per = (p.B + 255) / 256;
  int before;
  const int total = mla_scan<4>(p, per, before, scan4);
  if (tid == b / per) {
    for (int i = tid * per; i < b; ++i) before += mla_tiles(mla_len(p, i));
    mine[0] = before;
  }
  __syncthreads();
  const int tiles = mla_tiles(mla_len(p, b));
  const int64_t row = (int64_t)b * p.M + r;
  u16* const out = (u16*)p.out + row * kLatent;
  if (tiles == 0) {
    if (tid < 128) *(v2i*)(out + 4 * tid) = v2i{0, 0};
    if (tid == 0 && p.lse) p.lse[row] = -INFINITY;
    return;
  }
  const int run = mla_run(total, p.walkers), w0 = mine[0] / run, w1 = (mine[0] + tiles - 1) / run, n = w1 - w0 + 1;
  if (n == 1) return;
  // n <= walkers <= 256
  const int64_t slot = (int64_t)(w0 + b);
  float top = -INFINITY;
  for (int i = 0; i < n; ++i) top = fmaxf(top, p.part_lse[(slot + i) * p.M + r]);
  const float shift = shift_of(top);
  if (tid < n) weights[tid] = __builtin_amdgcn_exp2f(p.part_lse[(slot + tid) * p.M + r] - shift);
  __syncthreads();
  float sum = 0.0f;
  for (int i = 0; i < n; ++i) sum += weights[i];
  if (tid < 128) {
    v4f acc = {0, 0, 0, 0};
    const float* from = p.part + (slot * p.M + r) * kLatent + 4 * tid;
#pragma unroll 8
    for (int i = 0; i < n; ++i) acc += weights[i] * *(const v4f*)(from + (int64_t)i * p.M * kLatent);
    acc *= sum == 0.0f ? 0.0f : 1.0f / sum;
    *(v2i*)(out + 4 * tid) = v2i{(int)pack2<DT>(acc[0], acc[1]), (int)pack2<DT>(acc[2], acc[3])};
  }
  if (tid == 0 && p.lse) p.lse[row] = sum == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(sum) + shift) * kLn2;
}

}  // namespace fp8k
