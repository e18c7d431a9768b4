// A whole mixture-of-experts layer on MXFP4 weights for a few tokens, in two launches (gfx950).
//
//   h[slot]  = round16(act(g) * u),  (g, u) = x[token] . W1[expert]^T        mx_experts_up_kernel
//   y[token] = round16(f * sum over its slots of weight * h[slot] . W2[expert]^T)   mx_experts_down_kernel
//
// A slot is one (token, choice) pair.  With few tokens the layer is a stream of the chosen experts' weights, so activations stay in 16
// bits: quantising them would move no byte less.  The codes become exact 16-bit floats in registers (v_cvt_scalef32_pk_*_fp4, two a
// instruction), a product of 32 along K is one block of the scales, and its float32 result is added to the sum times the block's scale.
//
// The weights are operand B of v_mfma_f32_16x16x32 and the slots of an expert are operand A: a lane holds one weight row
// (lane & 15) and 8 values of K, so the scale that it multiplies its four results with is that of its own row.
#pragma once

#include "mx_common.h"

namespace fp8k {

constexpr int kMxMaxSlots = 1024;  // (token, choice) pairs of a call
constexpr int kMxMaxTokens = 128;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
  if (DT == FP8K_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// eight codes -> eight 16-bit floats, unscaled (all of them exact)
template <int DT>
__device__ __forceinline__ v4i fp4_to_16(uint32_t c) {
  v4i r;
  if (DT == FP8K_BF16) {
    r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 0));
    r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 1));
    r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 2));
    r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.0f, 3));
  } else {
    r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 0));
    r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 1));
    r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 2));
    r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 3));
  }
  return r;
}

struct MxExpertArgs {
  const void* x;        // [T, H] 16-bit
  const uint8_t* w1;    // [E, 2I, H/2]
  const uint8_t* w2;    // [E, H, I/2]
  const uint8_t* s1;    // words of scales, int32 strides below
  const uint8_t* s2;
  const float* topk_w;  // [T, topk]
  const void* ids;      // [T, topk] int32 or int64
  void* out;            // [T, H]
  void* h;              // [slots, I] 16-bit: the workspace, as is the table
  int32_t* tiles;       // [slots * 4]: of tile t its expert, its first place in `order`, its number of slots (1 .. 16)
  int32_t* order;       // [slots] slots sorted by expert
  int32_t* ntiles;
  int T, topk, E, H, I, slots;
  int ids64, on_input;
  int64_t ldx;          // elements
  int64_t w1_e, w2_e;   // bytes
  int64_t s1_e, s1_n, s1_w, s2_e, s2_n, s2_w;  // int32 words
  float scaling;
};

__device__ __forceinline__ int mx_expert_of(const MxExpertArgs& p, int slot) {
  const int64_t id = p.ids64 ? ((const int64_t*)p.ids)[slot] : (int64_t)((const int32_t*)p.ids)[slot];
  return id >= 0 && id < p.E ? (int)id : -1;  // -1 and anything out of range: an expert of another rank, contributes nothing
}

// the weights of one K block (256 values) of 16 rows in flight, and their way into operand form
struct MxRows {
  v4i reg[2];
  uint2 scale;  // eight scale bytes of row lane & 15
};

// 16 weight rows from `row0` of a matrix with `row_bytes` bytes to a row
struct MxStrip {
  rsrc_t w, s;
  uint32_t vo0, vo1, vs, word;
  int row_bytes, words, wc;
  __device__ __forceinline__ MxStrip(const uint8_t* W, const uint8_t* S, int64_t row0, int rows, int K, int64_t s_n, int64_t s_w, int lane) {
    row_bytes = K >> 1;
    words = (K + 127) >> 7;
    wc = lane & 7;
    w = make_rsrc(W + row0 * row_bytes, rows > 0 ? (uint32_t)(rows * row_bytes) : 0u);
    s = mx_scale_rsrc(S, row0, rows, words, s_n, s_w);
    vo0 = (uint32_t)((lane >> 3) * row_bytes) + wc * 16;
    vo1 = vo0 + (uint32_t)(8 * row_bytes);
    vs = (uint32_t)((lane & 15) * s_n * 4);
    word = (uint32_t)(s_w * 4);
  }
  __device__ __forceinline__ void load(MxRows& r, int kb, bool in) const {
    const uint32_t ko = (uint32_t)kb * kMxStepBytes;
    const bool ok = in && (int)ko + wc * 16 < row_bytes;
    r.reg[0] = buf_load16_stream(w, ok ? vo0 + ko : kOutOfRange);
    r.reg[1] = buf_load16_stream(w, ok ? vo1 + ko : kOutOfRange);
    r.scale.x = __builtin_amdgcn_raw_buffer_load_b32(s, in ? vs + 2 * kb * word : kOutOfRange, 0, 0);
    r.scale.y = __builtin_amdgcn_raw_buffer_load_b32(s, in && 2 * kb + 1 < words ? vs + (2 * kb + 1) * word : kOutOfRange, 0, 0);
  }
};

// through the wave's 2 KB LDS slot: codes of (row lane & 15, block j, values 8 kq ..) as 16-bit floats
struct MxRelay {
  uint8_t* slot;
  uint32_t st0, st1, rd;
  int key;
  __device__ __forceinline__ MxRelay(uint8_t* base, int lane) : slot(base) {
    const int wrow = lane >> 3, wc = lane & 7, r = lane & 15;
    st0 = (uint32_t)(wrow * kMxStepBytes + ((wc ^ ((wrow >> 1) & 7)) << 4));
    st1 = (uint32_t)((wrow + 8) * kMxStepBytes + ((wc ^ (((wrow + 8) >> 1) & 7)) << 4));
    rd = (uint32_t)(r * kMxStepBytes + (lane >> 4) * 4);
    key = (r >> 1) & 7;
  }
  __device__ __forceinline__ void put(const MxRows& r) const {
    *reinterpret_cast<v4i*>(slot + st0) = r.reg[0];
    *reinterpret_cast<v4i*>(slot + st1) = r.reg[1];
  }
  __device__ __forceinline__ uint32_t get(int j) const { return *reinterpret_cast<const uint32_t*>(slot + rd + ((j ^ key) << 4)); }
};
__device__ __forceinline__ float mx_block_scale(const uint2& s, int j) { return e8m0_f32(((j < 4 ? s.x : s.y) >> ((j & 3) * 8)) & 255u); }

// ------------------------------------------------------------------------------------------------
// grid (I / 16 strips + 1, units).  Units are slots (the first slot of an expert does the work, the others end at once) or experts,
// whichever are fewer.  The last strip's workgroup of unit 0 sorts the slots by expert for the second launch.
// ------------------------------------------------------------------------------------------------
template <int DT, bool GELU>
__global__ __launch_bounds__(512, 1) void mx_experts_up_kernel(const MxExpertArgs p) {
  __shared__ __attribute__((aligned(16))) uint8_t wl[8][2][16 * kMxStepBytes];
  __shared__ __attribute__((aligned(16))) float red[8][2][64][4];
  __shared__ int list[kMxMaxSlots];
  __shared__ int counts[16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int strips = (p.I + 15) >> 4;

  if ((int)blockIdx.x == strips) {
    if (blockIdx.y != 0) return;
    // place of a slot: the valid slots of a smaller expert, or of the same expert in front of it
    int* const rank = reinterpret_cast<int*>(red);
    static_assert(sizeof(red) >= kMxMaxSlots * sizeof(int), "the ranks lie where the sums of the products do");
    for (int s = tid; s < p.slots; s += 512) list[s] = mx_expert_of(p, s);
    if (tid == 0) counts[0] = 0;
    __syncthreads();
    int place[2], total[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int s = j * 512 + tid;
      if (s >= p.slots || list[s] < 0) continue;
      const int e = list[s];
      int before = 0, same = 0, of_expert = 0;
      for (int o = 0; o < p.slots; ++o) {
        const int f = list[o];
        before += f >= 0 && f < e;
        of_expert += f == e;
        same += f == e && o < s;
      }
      rank[s] = same;
      place[j] = before + same;
      total[j] = of_expert;
      p.order[before + same] = s;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int s = j * 512 + tid;
      if (s >= p.slots || list[s] < 0 || rank[s] % 16 != 0) continue;
      // the first slot of a tile: in front of it are the tiles of smaller experts and those of its own
      int tile = rank[s] / 16;
      for (int o = 0; o < p.slots; ++o) tile += list[o] >= 0 && list[o] < list[s] && rank[o] % 16 == 0;
      p.tiles[tile * 4] = list[s];
      p.tiles[tile * 4 + 1] = place[j];
      p.tiles[tile * 4 + 2] = min(16, total[j] - rank[s]);
      atomicMax(&counts[0], tile + 1);
    }
    __syncthreads();
    if (tid == 0) p.ntiles[0] = counts[0];
    return;
  }

  // ---- the unit's expert and the list of its slots, ascending
  const bool by_slot = (int)gridDim.y == p.slots;
  const int expert = by_slot ? mx_expert_of(p, blockIdx.y) : (int)blockIdx.y;
  if (expert < 0) return;
  int mine[2];
  uint64_t masks[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = j * 512 + tid;
    mine[j] = s < p.slots && mx_expert_of(p, s) == expert;
    masks[j] = __ballot(mine[j]);
    if (lane == 0) counts[j * 8 + w] = __popcll(masks[j]);
  }
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int at = 0;
    for (int k = 0; k < j * 8 + w; ++k) at += counts[k];
    if (mine[j]) list[at + __popcll(masks[j] & ((1ull << lane) - 1))] = j * 512 + tid;
  }
  for (int k = 0; k < 16; ++k) total += counts[k];
  __syncthreads();
  if (total == 0 || (by_slot && list[0] != (int)blockIdx.y)) return;

  const int c0 = blockIdx.x * 16;  // columns of h
  const uint8_t* const W = p.w1 + (int64_t)expert * p.w1_e;
  const uint8_t* const S = p.s1 + (int64_t)expert * p.s1_e * 4;
  const MxStrip gate(W, S, c0, min(16, p.I - c0), p.H, p.s1_n, p.s1_w, lane);
  const MxStrip up(W, S, (int64_t)p.I + c0, min(16, p.I - c0), p.H, p.s1_n, p.s1_w, lane);
  const MxRelay relay_g(wl[w][0], lane), relay_u(wl[w][1], lane);
  const int kbs = (p.H + kMxStep - 1) / kMxStep, per = (kbs + 7) >> 3;
  const int kb0 = w * per, kb1 = min(kbs, kb0 + per);
  const rsrc_t rX = make_rsrc(p.x, (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2));

  for (int t0 = 0; t0 < total; t0 += 16) {
    const int slot = t0 + r < total ? list[t0 + r] : -1;
    const uint32_t xrow = slot >= 0 ? (uint32_t)((slot / p.topk) * p.ldx * 2) + kq * 16 : kOutOfRange;
    v4f ag = {0.f, 0.f, 0.f, 0.f}, au = {0.f, 0.f, 0.f, 0.f};
    for (int kb = kb0; kb < kb1; ++kb) {
      MxRows g, u;
      gate.load(g, kb, true);
      up.load(u, kb, true);
      v4i x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = kb * kMxStep + j * 32 + kq * 8;
        x[j] = buf_load16(rX, slot >= 0 && k < p.H ? xrow + (uint32_t)(kb * kMxStep + j * 32) * 2 : kOutOfRange);
      }
      relay_g.put(g);
      relay_u.put(u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const v4f z = {0.f, 0.f, 0.f, 0.f};
        const v4f pg = mfma16<DT>(x[j], fp4_to_16<DT>(relay_g.get(j)), z);
        const v4f pu = mfma16<DT>(x[j], fp4_to_16<DT>(relay_u.get(j)), z);
        const float sg = mx_block_scale(g.scale, j), su = mx_block_scale(u.scale, j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ag[i] = __builtin_fmaf(pg[i], sg, ag[i]);
          au[i] = __builtin_fmaf(pu[i], su, au[i]);
        }
      }
    }
    *reinterpret_cast<v4f*>(red[w][0][lane]) = ag;
    *reinterpret_cast<v4f*>(red[w][1][lane]) = au;
    __syncthreads();
    if (tid < 256) {
      // value (slot row, column) of the tile: lane (row / 4) * 16 + column, element row % 4
      const int row = tid >> 4, col = tid & 15, l = (row >> 2) * 16 + col, i = row & 3;
      float g = 0.f, u = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        g += red[k][0][l][i];
        u += red[k][1][l][i];
      }
      if (t0 + row < total && c0 + col < p.I) {
        const int s = list[t0 + row];
        if (p.on_input) {
          g *= p.topk_w[s];
          u *= p.topk_w[s];
        }
        const float v = (GELU ? gelu_f32(g) : silu_f32(g)) * u;
        ((u16*)p.h)[(int64_t)s * p.I + c0 + col] = (u16)(DT == FP8K_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------
// grid H / 16: a workgroup owns 16 output columns and goes through all tiles of the table.  The K blocks of all tiles are one list,
// which the waves share out in runs; a wave adds a tile's results, times the routed weights, to sums of its own in LDS ([T][16] floats),
// and the eight sets are added in order at the end: no atomics between waves, so results do not depend on timing.
// ------------------------------------------------------------------------------------------------
template <int DT, int TC>  // TC: tokens that the sums have room for
__global__ __launch_bounds__(512, 1) void mx_experts_down_kernel(const MxExpertArgs p) {
  __shared__ __attribute__((aligned(16))) float sums[8 * TC * 16];  // [8][T][16]
  __shared__ __attribute__((aligned(16))) uint8_t wl[8][16 * kMxStepBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  float* const mine = sums + w * p.T * 16;
  for (int i = lane; i < p.T * 16; i += 64) mine[i] = 0.f;

  const int ntiles = p.ntiles[0];
  const int kbs = (p.I + kMxStep - 1) / kMxStep;
  const int all = ntiles * kbs, per = (all + 7) >> 3;
  const int b0 = w * per, b1 = min(all, b0 + per);
  const MxRelay relay(wl[w], lane);
  const rsrc_t rH = make_rsrc(p.h, (uint32_t)((int64_t)p.slots * p.I * 2));
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  for (int b = b0; b < b1; ++b) {
    const int t = b / kbs, kb = b - t * kbs;
    const int expert = p.tiles[t * 4], first = p.tiles[t * 4 + 1], count = p.tiles[t * 4 + 2];
    const MxStrip strip(p.w2 + (int64_t)expert * p.w2_e, p.s2 + (int64_t)expert * p.s2_e * 4, n0, min(16, p.H - n0), p.I, p.s2_n, p.s2_w, lane);
    MxRows rows;
    strip.load(rows, kb, true);
    const uint32_t hrow = r < count ? (uint32_t)p.order[first + r] * (uint32_t)(p.I * 2) + kq * 16 : kOutOfRange;
    v4i x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = kb * kMxStep + j * 32 + kq * 8;
      x[j] = buf_load16(rH, r < count && k < p.I ? hrow + (uint32_t)(kb * kMxStep + j * 32) * 2 : kOutOfRange);
    }
    relay.put(rows);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const v4f part = mfma16<DT>(x[j], fp4_to_16<DT>(relay.get(j)), v4f{0.f, 0.f, 0.f, 0.f});
      const float s = mx_block_scale(rows.scale, j);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(part[i], s, acc[i]);
    }
    if (kb == kbs - 1 || b == b1 - 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = kq * 4 + i;
        if (row < count) {
          const int slot = p.order[first + row];
          // two slots of a tile may be of one token: an LDS atomic, whose order within the wave is fixed
          atomicAdd(&mine[(slot / p.topk) * 16 + r], p.on_input ? acc[i] : acc[i] * p.topk_w[slot]);
        }
        acc[i] = 0.f;
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < p.T * 16; i += 512) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += sums[k * p.T * 16 + i];
    v *= p.scaling;
    const int n = n0 + (i & 15);
    if (n < p.H) ((u16*)p.out)[(int64_t)(i >> 4) * p.H + n] = (u16)(DT == FP8K_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
  }
}

}  // namespace fp8k
