// A whole mixture-of-experts layer on MXFP4 weights for a few tokens, in two launches (gfx950).
//
//   h[slot]  = act(g) * u,  (g, u) = x[token] . W1[expert]^T                 mx_experts_up_kernel
//   y[token] = round16(f * sum over its slots of weight * h[slot] . W2[expert]^T)   mx_experts_down_kernel
//
// A slot is one (token, choice) pair.  With few tokens the layer is a stream of the chosen experts' weights, so activations stay in 16
// bits: quantising them would move no byte less.  All sums, the routed weights and the last sum are float32.  The second product takes
// 16-bit operands, so h travels as a pair of bfloat16, rounded and what the rounding left, whose products are added: one 16-bit h would be
// an error as large as the result's own rounding (1.4 times the whole error), the pair is off by 2^-16 and has float32's range.  The
// codes become exact 16-bit floats in registers (v_cvt_scalef32_pk_*_fp4, two a instruction), and a product of 32 along K is one block
// of the scales.
//
// The weights are operand B of v_mfma_f32_16x16x32 and the slots of an expert are operand A: a lane holds 8 values of one weight row
// (lane & 15) and results of that row's column, so the one scale it needs for either is that of its own row.
#pragma once

#include "gemm_tile64.h"
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
// Eight codes become eight 16-bit floats, for bfloat16 times their scale: it has float32's exponents (subnormal ones too), so that code *
// scale is exact wherever float32 holds it - with every scale up to 2^125, the largest that quantisation makes.  4 and 6 times 2^126 and
// 2 to 6 times 2^127 are infinite, as mxfp4_dequant gives them.
template <int DT>
__device__ __forceinline__ v4i mx_floats(uint32_t c, float scale) {
  v4i b;
  if (DT == FP8K_BF16) {
    b[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
    b[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
    b[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
    b[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
  } else {
    b[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 0));
    b[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 1));
    b[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 2));
    b[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 3));
  }
  return b;
}
// acc += a . (codes of a weight row * scale), 32 values along K that share the scale.  bfloat16 adds up in place.  float16's codes are
// unscaled, and the result of the 32 is multiplied (four more multiplications per product).
template <int DT>
__device__ __forceinline__ v4f mx_mac(v4f acc, v4i a, uint32_t c, float scale) {
  const v4i b = mx_floats<DT>(c, scale);
  if (DT == FP8K_BF16) return mfma16<DT>(a, b, acc);
  const v4f part = mfma16<DT>(a, b, v4f{0.f, 0.f, 0.f, 0.f});
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(part[i], scale, acc[i]);
  return acc;
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
  void* h;              // [slots, 2, I] bfloat16, the pairs' first and second parts: the workspace, as are the four arrays of the table
  int32_t* tiles;       // [slots] tile t: some slots of one expert (mx_tile below)
  int32_t* order;       // [slots] slots sorted by expert
  float* weights;       // [slots] their routed weights, in that order
  int32_t* ntiles;
  int T, topk, E, H, I, slots;
  int ids64, on_input;
  int run;              // mx_experts_up_kernel: strips of a workgroup
  int tile;             // slots of a tile of the second launch (4 or 8)
  int64_t ldx;          // elements
  int64_t w1_e, w2_e;   // bytes
  int64_t s1_e, s1_n, s1_w, s2_e, s2_n, s2_w;  // int32 words
  float scaling;
};

__device__ __forceinline__ int mx_expert_of(const MxExpertArgs& p, int slot) {
  const int64_t id = p.ids64 ? ((const int64_t*)p.ids)[slot] : (int64_t)((const int32_t*)p.ids)[slot];
  return id >= 0 && id < p.E ? (int)id : -1;  // -1 and anything out of range: an expert of another rank, contributes nothing
}
// a tile of the table in one word: expert (below 2^16), first place in `order` (below 2^10), number of slots less one
__device__ __forceinline__ int mx_tile(int expert, int first, int count) { return (expert << 14) | (first << 4) | (count - 1); }

// The weights of a K block (256 values) of 16 rows, from lines in the wave's LDS slot to 16-bit floats: the lane's eight codes of
// block j, values 8 kq .. 8 kq + 7 of row lane & 15.  Chunk c of row r lies at position c ^ ((r >> 1) & 7).
struct MxCodes {
  uint32_t rd;
  int key;
  __device__ __forceinline__ explicit MxCodes(int lane) : rd((uint32_t)((lane & 15) * kMxStepBytes + (lane >> 4) * 4)), key(((lane & 15) >> 1) & 7) {}
  __device__ __forceinline__ uint32_t get(const uint8_t* slot, int j) const { return *reinterpret_cast<const uint32_t*>(slot + rd + ((j ^ key) << 4)); }
};
// the scale of block j, byte j & 3 of one of two words.  The conversion to bfloat16 takes a scale's exponent field as the e8m0 byte it is
// (255, infinity's, makes NaN), which saves telling 0 and 255 apart.
template <int DT>
__device__ __forceinline__ float mx_block_scale(uint32_t lo, uint32_t hi, int j) {
  const uint32_t word = j < 4 ? lo : hi;
  if (DT != FP8K_BF16) return e8m0_f32((word >> ((j & 3) * 8)) & 255u);
  const int up = 23 - (j & 3) * 8;
  return __uint_as_float((up < 0 ? word >> 1 : word << (up < 0 ? 0 : up)) & 0x7f800000u);
}

// Takes the bytes of blocks at or past the end of the rows out of the two scale words of K block kb, the last one of rows of k values.  A
// row's last word stands in place of one behind it, and the codes there are those of the next row: their product must not meet the zeros
// of the activations as an infinity.  A branch, kept one by the empty statement: masking every block took 1 % of the layer.
__device__ __forceinline__ void mx_scales_there(uint32_t& lo, uint32_t& hi, int k, int kb) {
  const uint64_t there = (1ull << (8 * ((k >> 5) - kb * (kMxStep / kMxBlock)))) - 1;
  lo &= (uint32_t)there;
  hi &= (uint32_t)(there >> 32);
  asm volatile("" : "+v"(lo), "+v"(hi));
}

// The table of the second launch: slots sorted by expert (and by their number within one), cut into tiles of up to p.tile slots of one
// expert.  One workgroup of 256 threads; keys, sorted: LDS for kMxMaxSlots words, aux: for 33.
__device__ __forceinline__ void mx_sort_slots(const MxExpertArgs& p, int* keys, int* sorted, int* aux) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  constexpr int kNone = 0x7fffffff;
  constexpr int NT = 256, J = kMxMaxSlots / NT;
  const int padded = (p.slots + 3) & ~3;
  for (int s = tid; s < padded; s += NT) {
    const int e = s < p.slots ? mx_expert_of(p, s) : -1;
    keys[s] = e < 0 ? kNone : (e << 10) | s;
  }
  if (tid < 16) aux[tid] = -1;
  if (tid == 32) aux[tid] = 0;
  __syncthreads();
  // a key's place is the number of smaller ones
  int own = 0;
  for (int s = tid; s < padded; s += NT) {
    const int key = keys[s];
    int at = 0;
#pragma unroll 4
    for (int o = 0; o < padded; o += 4) {
      const int4 k = *reinterpret_cast<const int4*>(keys + o);
      at += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
    }
    if (key != kNone) {
      ++own;
      sorted[at] = key;
      p.order[at] = s;
      p.weights[at] = p.topk_w[s];
    }
  }
  atomicAdd(&aux[32], own);
  __syncthreads();
  const int valid = aux[32];
  // places 64 (4 j + w) + lane: the first of an expert; a place's rank is its distance to the last of those at or before it
  const uint64_t upto = (2ull << lane) - 1;
  uint64_t heads[J], starts[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int at = j * NT + tid, chunk = j * 4 + w;
    heads[j] = __ballot(at < valid && (at == 0 || (sorted[at - 1] >> 10) != (sorted[at] >> 10)));
    if (lane == 0 && heads[j]) aux[chunk] = chunk * 64 + 63 - __clzll((long long)heads[j]);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int at = j * NT + tid, chunk = j * 4 + w;
    int head = -1;
    for (int c = 0; c < chunk; ++c) head = max(head, aux[c]);
    if (heads[j] & upto) head = chunk * 64 + 63 - __clzll((long long)(heads[j] & upto));
    starts[j] = __ballot(at < valid && (at - head) % p.tile == 0);
    if (lane == 0) aux[16 + chunk] = __popcll(starts[j]);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int at = j * NT + tid, chunk = j * 4 + w;
    if (!((starts[j] >> lane) & 1)) continue;
    int t = __popcll(starts[j] & (upto >> 1));
    for (int c = 0; c < chunk; ++c) t += aux[16 + c];
    int n = 1;
    while (n < p.tile && at + n < valid && (sorted[at + n] >> 10) == (sorted[at] >> 10)) ++n;
    p.tiles[t] = mx_tile(sorted[at] >> 10, at, n);
  }
  if (tid == 0) {
    int total = 0;
    for (int c = 0; c < 16; ++c) total += aux[16 + c];
    p.ntiles[0] = total;
  }
}

// ------------------------------------------------------------------------------------------------
// First launch.  Grid (runs of strips + 1, units).  Units are slots (the first slot of an expert does the work, the others end at once)
// or experts, whichever are fewer; the workgroup behind the last run of unit 0 makes the table of the second launch.
//
// A workgroup takes a run of strips of 16 columns of h: 16 gate and 16 up rows, all of K, for the expert's slots, RX at a time.  Its four
// waves take every fourth K block each.  What a block needs - the lines of 32 rows, their scale words, the slots' activations - goes
// straight to an LDS slot of the wave, requested as soon as the operands of the block before are out of it and on across the strips of
// the run, and no other load stands in the loop.  The four sums meet in LDS; the last wave, which has the fewest blocks, adds them up,
// applies the activation and writes h; the others wait for it at a barrier, with their next requests on the way.
// Bound: the weights' bytes.  One slot to a wave and four workgroups to a CU (RX = 4) beat two slots and two workgroups: 626 against
// 645 us (64 tokens, 256 experts of 7168 x 2048), 21.0 against 28 (13 tokens, 128 of 4096 x 256): the conversions of one wave run
// while another waits.  Weights that several tiles read stay in the caches, those that one reads go past them: 166 -> 151 us with 32
// slots to an expert (64 tokens, 16 experts of 7168 x 2048), 85 -> 80 with 4 (128 of 4096 x 512); for all, 4 % slower with one tile.
// ------------------------------------------------------------------------------------------------
template <int DT, bool GELU, int RX>
__global__ __launch_bounds__(256, RX == 4 ? 4 : 2) void mx_experts_up_kernel(const MxExpertArgs p) {
  constexpr int NW = 4, kSlot = 4096 + RX * 512 + 256, kX = 4096, kS = 4096 + RX * 512;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NW * kSlot];
  __shared__ __attribute__((aligned(16))) v4f red[NW - 1][2][64];
  __shared__ u16 list[kMxMaxSlots];
  static_assert(sizeof(smem) >= (2 * kMxMaxSlots + 33) * 4, "the sort works where the slots are");

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int strips = p.I >> 4, runs = (strips + p.run - 1) / p.run;
  int* const scratch = reinterpret_cast<int*>(smem);

  if ((int)blockIdx.x == runs) {
    if (blockIdx.y == 0) mx_sort_slots(p, scratch, scratch + kMxMaxSlots, scratch + 2 * kMxMaxSlots);
    return;
  }

  // ---- the unit's expert and the list of its slots, ascending
  const bool by_slot = (int)gridDim.y == p.slots;
  const int expert = __builtin_amdgcn_readfirstlane(by_slot ? mx_expert_of(p, blockIdx.y) : (int)blockIdx.y);
  if (expert < 0) return;
  constexpr int J = kMxMaxSlots / 256;
  uint64_t masks[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int s = j * 256 + tid;
    masks[j] = __ballot(s < p.slots && mx_expert_of(p, s) == expert);
    if (lane == 0) scratch[j * 4 + w] = __popcll(masks[j]);
  }
  __syncthreads();
  int total = 0;
  for (int k = 0; k < 16; ++k) total += scratch[k];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    int at = __popcll(masks[j] & ((1ull << lane) - 1));
    for (int k = 0; k < j * 4 + w; ++k) at += scratch[k];
    if ((masks[j] >> lane) & 1) list[at] = (u16)(j * 256 + tid);
  }
  total = __builtin_amdgcn_readfirstlane(total);
  __syncthreads();
  if (total == 0 || (by_slot && list[0] != (int)blockIdx.y)) return;

  const int row_bytes = p.H >> 1, words = (p.H + 127) >> 7, kbs = (p.H + kMxStep - 1) / kMxStep;
  const int strip0 = blockIdx.x * p.run, nstrips = min(p.run, strips - strip0), ntiles = (total + RX - 1) / RX;
  const int nb = kbs > w ? (kbs - w + NW - 1) / NW : 0;  // blocks of the wave: w, w + 4, ..
  const rsrc_t rW = make_rsrc(p.w1 + (int64_t)expert * p.w1_e, (uint32_t)(2 * p.I * row_bytes));
  const rsrc_t rS = mx_scale_rsrc(p.s1 + (int64_t)expert * p.s1_e * 4, 0, 2 * p.I, words, p.s1_n, p.s1_w);
  const rsrc_t rX = make_rsrc(p.x, (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2));
  const int rl = lane >> 3, cp = lane & 7;
  const uint32_t vo0 = (uint32_t)(rl * row_bytes + (cp ^ (rl >> 1)) * 16), vo1 = (uint32_t)((rl + 8) * row_bytes + (cp ^ (4 + (rl >> 1))) * 16);
  const uint32_t up_rows = (uint32_t)(p.I * row_bytes);
  // scale words of a block: lanes 0 .. 15 word 0 of the gate rows, then word 1, then those of the up rows
  const uint32_t voS = (uint32_t)((r + (kq >> 1) * p.I) * p.s1_n * 4);
  uint8_t* const own = smem + w * kSlot;
  const MxCodes codes(lane);

  // ---- requests: the wave's blocks of a tile, the tiles of a strip, the strips of the run
  int ri = 0, rtile = 0, rstrip = 0;
  uint32_t xoff[RX / 2];  // of the activations that the lane fetches: two slots a load, 16-byte piece c of slot i at position c ^ (4 (i & 3))
  auto rows_of = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RX / 2; ++i) {
      const int row = 2 * i + (lane >> 5), k = tile * RX + row;
      xoff[i] = k < total ? (uint32_t)((list[k] / p.topk) * p.ldx * 2) + (((lane & 31) ^ ((row & 3) << 2)) << 4) : kOutOfRange;
    }
  };
  rows_of(0);
  auto request = [&] __attribute__((always_inline)) {
    const int kb = w + NW * ri, c0 = (strip0 + rstrip) * 16;
    const uint32_t ko = (uint32_t)kb * kMxStepBytes + (uint32_t)(c0 * row_bytes);
    const auto lines = [&](auto once) __attribute__((always_inline)) {
      buf_load16_to_lds<once.value>(rW, vo0 + ko, 0, own);
      buf_load16_to_lds<once.value>(rW, vo1 + ko, 0, own + 1024);
      buf_load16_to_lds<once.value>(rW, vo0 + (ko + up_rows), 0, own + 2048);
      buf_load16_to_lds<once.value>(rW, vo1 + (ko + up_rows), 0, own + 3 * 1024);
    };
    if (ntiles == 1) lines(std::true_type{});
    else lines(std::false_type{});  // the next tile reads them again
#pragma unroll
    for (int i = 0; i < RX / 2; ++i) {
      const int row = 2 * i + (lane >> 5), k = kb * kMxStep + ((lane & 31) ^ ((row & 3) << 2)) * 8;
      buf_load16_to_lds(rX, xoff[i] != kOutOfRange && k < p.H ? xoff[i] + (uint32_t)(kb * kMxStep * 2) : kOutOfRange, 0, own + kX + i * 1024);
    }
    buf_load4_to_lds(rS, voS + (uint32_t)(c0 * p.s1_n * 4) + (uint32_t)min(2 * kb + (kq & 1), words - 1) * (uint32_t)(p.s1_w * 4), 0, own + kS);
    SB();
    if (++ri == nb) {
      ri = 0;
      if (++rtile == ntiles) { rtile = 0; ++rstrip; }
      if (ntiles > 1) rows_of(rtile);
    }
  };

  v4f ag = {0.f, 0.f, 0.f, 0.f}, au = {0.f, 0.f, 0.f, 0.f};
  const uint32_t xrd = (uint32_t)(kX + (r & (RX - 1)) * 512);
  const int xkey = (r & 3) << 2;
  auto block = [&](int kb, bool more) __attribute__((always_inline)) {
    wait_vm<0>();
    uint32_t s[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = *reinterpret_cast<const uint32_t*>(own + kS + k * 64 + r * 4);
    uint32_t cg[8], cu[8];
    v4i x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = *reinterpret_cast<const v4i*>(own + xrd + (((j * 4 + kq) ^ xkey) << 4));
      cg[j] = codes.get(own, j);
      cu[j] = codes.get(own + 2048, j);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // everything is out of its slot
    SB();
    if (more) request();
    if (kb * kMxStep + kMxStep > p.H) {
      mx_scales_there(s[0], s[1], p.H, kb);
      mx_scales_there(s[2], s[3], p.H, kb);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ag = mx_mac<DT>(ag, x[j], cg[j], mx_block_scale<DT>(s[0], s[1], j));
      au = mx_mac<DT>(au, x[j], cu[j], mx_block_scale<DT>(s[2], s[3], j));
      if (DT != FP8K_BF16) SB();
    }
    SB();
  };
  // the sums of a tile of a strip
  auto finish = [&](int strip, int tile) __attribute__((always_inline)) {
    if (w < NW - 1) {
      red[w][0][lane] = ag;
      red[w][1][lane] = au;
    }
    lds_barrier();  // requests stay in flight
    if (w == NW - 1) {
      v4f g = red[0][0][lane], u = red[0][1][lane];
#pragma unroll
      for (int k = 1; k < NW; ++k) {
        const v4f a = k < NW - 1 ? red[k < NW - 1 ? k : 0][0][lane] : ag, b = k < NW - 1 ? red[k < NW - 1 ? k : 0][1][lane] : au;
#pragma unroll
        for (int i = 0; i < 4; ++i) { g[i] += a[i]; u[i] += b[i]; }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = kq * 4 + i, k = tile * RX + row;
        if (row >= RX || k >= total) continue;
        const int s = list[k];
        if (p.on_input) {
          g[i] *= p.topk_w[s];
          u[i] *= p.topk_w[s];
        }
        const float v = (GELU ? gelu_f32(g[i]) : silu_f32(g[i])) * u[i];
        // the first part stays finite, so that an infinity is left to the second
        constexpr float kMost = 3.3895313892515355e38f;
        const u16 hi = (u16)f32_to_bf16_bits(v > kMost ? kMost : v < -kMost ? -kMost : v);
        const float left = v - __uint_as_float((uint32_t)hi << 16);
        u16* const to = (u16*)p.h + (int64_t)s * 2 * p.I + (strip0 + strip) * 16 + r;
        to[0] = hi;
        to[p.I] = (u16)f32_to_bf16_bits(left);
      }
    }
    lds_barrier();
    ag = au = v4f{0.f, 0.f, 0.f, 0.f};
  };

  if (nb == 0) {
    for (int k = 0; k < nstrips * ntiles; ++k) finish(k / ntiles, k % ntiles);
    return;
  }
  request();
  const int all = nstrips * ntiles * nb;
  int ci = 0, ctile = 0, cstrip = 0;
  for (int q = 0; q < all; ++q) {
    block(w + NW * ci, q + 1 < all);
    if (++ci == nb) {
      finish(cstrip, ctile);
      ci = 0;
      if (++ctile == ntiles) { ctile = 0; ++cstrip; }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Second launch, grid H / 16: a workgroup owns 16 output columns and goes through all tiles of the table.  The K blocks of all tiles are
// one list, which the waves share out in runs; a wave adds a tile's results, times the routed weights, to sums of its own in LDS ([T][16]
// floats), and the sets are added in order at the end: no atomics between waves, so results do not depend on timing.
//
// Everything a K block needs - the lines of 16 weight rows, their scale words, the activations of the tile's RX slots - goes straight to
// the wave's LDS slot, requested as soon as the operands of the block before are out of it, and no other load stands in the loop.
// (Activations in operand form straight to registers, eight loads a block of which a few lanes are used, took 28 us for the 62 MB of one
// token where this takes 15.)  A slot's pair is two neighbouring rows of the operand, of whose sixteen few are used anyway: it costs LDS and
// the fetch, no product.  As many waves as there is room for, one LDS slot each: eight and two workgroups to a CU beat four waves with three
// slots each, 363 against 394 us (64 tokens, 256 experts of 7168 x 2048, h not in pairs); fourteen of one workgroup take 400 there, twelve 408;
// up to one strip per CU sixteen waves, 13.0 against 14.5 us (13 tokens, 128 of 4096 x 256).
// Sums of several workgroups per strip, added up by the last one to come, cost more than they balance: a release to the whole device
// writes its L2 back (13 tokens 16 -> 38 us).
// ------------------------------------------------------------------------------------------------
// waves of a workgroup: as many as the LDS has room for, up to one strip per CU (`wide`); else two workgroups to a CU if they fit
constexpr int mx_down_waves(int rx, int tc, bool wide) {
  if (tc > 64) return 8;
  if (tc > 32) return rx == 8 ? 10 : 14;
  return rx == 8 ? 12 : wide ? 16 : 8;
}
constexpr int mx_down_places(int tc) { return tc <= 16 ? 512 : kMxMaxSlots; }  // (token, choice) pairs

template <int DT, int TC, int RX, int NW>  // DT: of the result; TC: tokens that the sums have room for; RX: slots of a tile; NW: waves
__global__ __launch_bounds__(NW * 64, RX == 4 && TC <= 32 ? 4 : (NW + 3) / 4) void mx_experts_down_kernel(const MxExpertArgs p) {
  constexpr int kSlot = 2048 + RX * 1024 + 128, kX = 2048, kS = 2048 + RX * 1024;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NW * kSlot];
  __shared__ __attribute__((aligned(16))) float sums[NW * TC * 16];  // [NW][T][16]
  __shared__ int tiles[mx_down_places(TC)];
  __shared__ float weights[mx_down_places(TC)];
  __shared__ u16 order[mx_down_places(TC)];
  __shared__ uint8_t token[mx_down_places(TC)];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  float* const mine = sums + w * p.T * 16;

  const int ntiles = p.ntiles[0];
  for (int i = tid; i < p.slots; i += NW * 64) {  // what lies behind the tiles and the valid slots is not used below
    tiles[i] = p.tiles[i];
    const int slot = p.order[i];
    order[i] = (u16)slot;
    token[i] = (uint8_t)(slot / p.topk);
    weights[i] = p.on_input ? 1.f : p.weights[i];
  }
  for (int i = lane; i < p.T * 16; i += 64) mine[i] = 0.f;
  __syncthreads();

  const int row_bytes = p.I >> 1, words = (p.I + 127) >> 7, kbs = (p.I + kMxStep - 1) / kMxStep;
  const int all = ntiles * kbs, per = (all + NW - 1) / NW;
  const int b0 = w * per, nb = max(min(all, b0 + per) - b0, 0);
  const rsrc_t rH = make_rsrc(p.h, (uint32_t)((int64_t)p.slots * p.I * 4));
  const int rl = lane >> 3, cp = lane & 7;
  const uint32_t vo0 = (uint32_t)((n0 + rl) * row_bytes + (cp ^ (rl >> 1)) * 16), vo1 = (uint32_t)((n0 + rl + 8) * row_bytes + (cp ^ (4 + (rl >> 1))) * 16);
  const uint32_t voS = (uint32_t)((n0 + r) * p.s2_n * 4);
  uint8_t* const own = smem + w * kSlot;
  const MxCodes codes(lane);

  // ---- requests: block by block through the wave's run.  What a tile's requests need is formed when the run comes to it, from its entry
  // and its slots, which were read from LDS one tile earlier (the entry two): a request never waits for LDS.
  int rt = 0, rkb = 0, left = nb;  // tile, its K block, blocks to come
  rsrc_t rW = make_rsrc(p.w2, 0), rS = make_rsrc(p.s2, 0);
  uint32_t xoff[RX];               // of the activations that the lane fetches: a load brings slot i's pair, rows 2 i and 2 i + 1 of the
  int count = 0;                   // operand; 16-byte piece c of row m lies at position c ^ (4 (m & 3)), so that reads spread over the banks
  int entry1 = 0, entry2 = 0;      // of tiles rt + 1 (here, when it becomes rt) and rt + 2
  int slots1[RX];
  auto read_entry = [&](int t) { return tiles[min(t, ntiles - 1)]; };
  auto read_slots = [&](int entry) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RX; ++i) slots1[i] = order[min(((entry >> 4) & 1023) + i, p.slots - 1)];
  };
  auto enter_tile = [&] __attribute__((always_inline)) {  // entry1 and slots1 are those of tile rt
    const int t = __builtin_amdgcn_readfirstlane(entry1);
    const int64_t e = t >> 14;
    count = (t & 15) + 1;
    rW = make_rsrc(p.w2 + e * p.w2_e, (uint32_t)(p.H * row_bytes));
    rS = mx_scale_rsrc(p.s2 + e * p.s2_e * 4, 0, p.H, words, p.s2_n, p.s2_w);
#pragma unroll
    for (int i = 0; i < RX; ++i)
      xoff[i] = (uint32_t)(slots1[i] * 2 + (lane >> 5)) * (uint32_t)(p.I * 2) + (uint32_t)(((lane & 31) ^ (((2 * i + (lane >> 5)) & 3) << 2)) * 16);
    entry1 = entry2;
    read_slots(entry2);
    entry2 = read_entry(rt + 2);
  };
  auto request = [&] __attribute__((always_inline)) {
    const uint32_t ko = (uint32_t)rkb * kMxStepBytes;
    buf_load16_to_lds<true>(rW, vo0 + ko, 0, own);
    buf_load16_to_lds<true>(rW, vo1 + ko, 0, own + 1024);
#pragma unroll
    for (int i = 0; i < RX; ++i) {
      if (i >= count) break;  // what is left in the rows behind makes results that nobody takes
      const int k = rkb * kMxStep + ((lane & 31) ^ (((2 * i + (lane >> 5)) & 3) << 2)) * 8;
      buf_load16_to_lds(rH, k < p.I ? xoff[i] + (uint32_t)(rkb * kMxStep * 2) : kOutOfRange, 0, own + kX + i * 1024);
    }
    if (lane < 32)  // scale words 0 and 1 of the 16 rows
      buf_load4_to_lds(rS, voS + (uint32_t)min(2 * rkb + kq, words - 1) * (uint32_t)(p.s2_w * 4), 0, own + kS);
    SB();
    --left;
    if (++rkb == kbs) {
      rkb = 0;
      ++rt;
      if (left > 0) enter_tile();
    }
  };

  v4f acc = {0.f, 0.f, 0.f, 0.f}, odd = acc;
  if (nb > 0) {
    rt = b0 / kbs;
    rkb = b0 - rt * kbs;
    int ct = rt, ckb = rkb;
    entry1 = read_entry(rt);
    read_slots(entry1);
    entry2 = read_entry(rt + 1);
    enter_tile();
    request();
    const uint32_t xrd = (uint32_t)(kX + (r & (2 * RX - 1)) * 512);
    const int xkey = (r & 3) << 2;
    for (int b = 0; b < nb; ++b) {
      wait_vm<0>();
      uint32_t c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = codes.get(own, j);
      uint32_t s0 = *reinterpret_cast<const uint32_t*>(own + kS + r * 4), s1 = *reinterpret_cast<const uint32_t*>(own + kS + 64 + r * 4);
      v4i x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const v4i*>(own + xrd + (((j * 4 + kq) ^ xkey) << 4));
      SB();
      if (ckb * kMxStep + kMxStep > p.I) mx_scales_there(s0, s1, p.I, ckb);
      // two chains of products: one result waits for the one before it
      acc = mx_mac<FP8K_BF16>(acc, x[0], c[0], mx_block_scale<FP8K_BF16>(s0, s1, 0));
      odd = mx_mac<FP8K_BF16>(odd, x[1], c[1], mx_block_scale<FP8K_BF16>(s0, s1, 1));
      SB();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // everything is out of its slot
      if (b + 1 < nb) request();
#pragma unroll
      for (int j = 2; j < 8; j += 2) {
        acc = mx_mac<FP8K_BF16>(acc, x[j], c[j], mx_block_scale<FP8K_BF16>(s0, s1, j));
        odd = mx_mac<FP8K_BF16>(odd, x[j + 1], c[j + 1], mx_block_scale<FP8K_BF16>(s0, s1, j + 1));
      }
      SB();
      if (++ckb == kbs || b == nb - 1) {
        const int t = __builtin_amdgcn_readfirstlane(tiles[ct]), first = (t >> 4) & 1023, count = (t & 15) + 1;
        int to[2];
        float by[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = first + min(kq * 2 + i, count - 1);
          to[i] = token[at] * 16 + r;
          by[i] = weights[at];
        }
        // the lane's rows are the pairs of two slots.  Two slots of a tile may be of one token: LDS atomics, whose order within the wave
        // is fixed.
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (kq * 2 + i < count) unsafeAtomicAdd(&mine[to[i]], (acc[2 * i] + odd[2 * i] + (acc[2 * i + 1] + odd[2 * i + 1])) * by[i]);
        acc = odd = v4f{0.f, 0.f, 0.f, 0.f};
        ckb = 0;
        ++ct;
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < p.T * 16; i += NW * 64) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) v += sums[k * p.T * 16 + i];
    v *= p.scaling;
    ((u16*)p.out)[(int64_t)(i >> 4) * p.H + n0 + (i & 15)] = (u16)(DT == FP8K_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
  }
}

}  // namespace fp8k
