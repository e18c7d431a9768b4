// A whole mixture-of-experts layer on MXFP4 weights for a few tokens, in two launches (gfx950).
//
//   h[slot]  = round16(act(g) * u),  (g, u) = x[token] . W1[expert]^T        mx_experts_up_kernel
//   y[token] = round16(f * sum over its slots of weight * h[slot] . W2[expert]^T)   mx_experts_down_kernel
//
// A slot is one (token, choice) pair.  With few tokens the layer is a stream of the chosen experts' weights, so activations stay in 16
// bits: quantising them would move no byte less.  The codes become exact 16-bit floats in registers (v_cvt_scalef32_pk_*_fp4, two a
// instruction), and a product of 32 along K is one block of the scales.
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
// acc += a . (codes of a weight row * scale), 32 values along K that share the scale.  Eight codes to a lane become eight 16-bit floats.
// bfloat16 has float32's exponents, so that code * scale is exact and the products add up in place.  float16 does not: its codes stay
// unscaled, and the result of the 32 is multiplied (four more multiplications per product).
template <int DT>
__device__ __forceinline__ v4f mx_mac(v4f acc, v4i a, uint32_t c, float scale) {
  v4i b;
  if (DT == FP8K_BF16) {
    b[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
    b[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
    b[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
    b[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
    return mfma16<DT>(a, b, acc);
  }
  b[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 0));
  b[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 1));
  b[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 2));
  b[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, 1.0f, 3));
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
  void* h;              // [slots, I] 16-bit: the workspace, as are the four arrays of the table
  int32_t* tiles;       // [slots] tile t: up to 16 slots of one expert (mx_tile below)
  int32_t* order;       // [slots] slots sorted by expert
  float* weights;       // [slots] their routed weights, in that order
  int32_t* ntiles;
  int T, topk, E, H, I, slots;
  int ids64, on_input;
  int run;              // mx_experts_up_kernel: strips of a workgroup
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
__device__ __forceinline__ float mx_block_scale(uint32_t lo, uint32_t hi, int j) { return e8m0_f32(((j < 4 ? lo : hi) >> ((j & 3) * 8)) & 255u); }

// The table of the second launch: slots sorted by expert (and by their number within one), cut into tiles of up to 16 slots of one
// expert.  One workgroup of 512 threads; keys: LDS for kMxMaxSlots words, aux: for 64.
__device__ __forceinline__ void mx_sort_slots(const MxExpertArgs& p, int* keys, int* sorted, int* aux) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  constexpr int kNone = 0x7fffffff;
  const int padded = (p.slots + 3) & ~3;
  for (int s = tid; s < padded; s += 512) {
    const int e = s < p.slots ? mx_expert_of(p, s) : -1;
    keys[s] = e < 0 ? kNone : (e << 10) | s;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = j * 512 + tid;
    const int key = s < p.slots ? keys[s] : kNone;
    int at = 0;
#pragma unroll 4
    for (int o = 0; o < padded; o += 4) {
      const int4 k = *reinterpret_cast<const int4*>(keys + o);
      at += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
    }
    if (key != kNone) {
      sorted[at] = key;
      p.order[at] = s;
      p.weights[at] = p.topk_w[s];
    }
  }
  if (tid < 16) aux[tid] = -1;
  int valid = 0;
#pragma unroll 4
  for (int o = 0; o < padded; o += 4) {
    const int4 k = *reinterpret_cast<const int4*>(keys + o);
    valid += (k.x != kNone) + (k.y != kNone) + (k.z != kNone) + (k.w != kNone);
  }
  __syncthreads();
  // places 64 (8 j + w) + lane: the first of an expert; a place's rank is its distance to the last of those at or before it
  const uint64_t upto = (2ull << lane) - 1;
  int rank[2];
  uint64_t starts[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int at = j * 512 + tid;
    const uint64_t heads = __ballot(at < valid && (at == 0 || (sorted[at - 1] >> 10) != (sorted[at] >> 10)));
    rank[j] = (heads & upto) ? 63 - __clzll((long long)(heads & upto)) : -1;
    if (lane == 0 && heads) aux[j * 8 + w] = (j * 8 + w) * 64 + 63 - __clzll((long long)heads);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int at = j * 512 + tid, chunk = j * 8 + w;
    int head = rank[j] >= 0 ? chunk * 64 + rank[j] : -1;
    for (int c = 0; c < 16; ++c)
      if (rank[j] < 0 && c < chunk && aux[c] >= 0) head = aux[c];
    starts[j] = __ballot(at < valid && (at - head) % 16 == 0);
    if (lane == 0) aux[16 + chunk] = __popcll(starts[j]);
  }
  __syncthreads();
  int total = 0;
  for (int c = 0; c < 16; ++c) total += aux[16 + c];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int at = j * 512 + tid, chunk = j * 8 + w;
    if (!((starts[j] >> lane) & 1)) continue;
    int t = __popcll(starts[j] & (upto >> 1));
    for (int c = 0; c < chunk; ++c) t += aux[16 + c];
    int n = 1;
    while (n < 16 && at + n < valid && (sorted[at + n] >> 10) == (sorted[at] >> 10)) ++n;
    p.tiles[t] = mx_tile(sorted[at] >> 10, at, n);
  }
  if (tid == 0) p.ntiles[0] = total;
}

// ------------------------------------------------------------------------------------------------
// First launch.  Grid (runs of strips + 1, units).  Units are slots (the first slot of an expert does the work, the others end at once)
// or experts, whichever are fewer; the workgroup behind the last run of unit 0 makes the table of the second launch.
//
// A workgroup takes a run of strips of 16 columns of h: 16 gate and 16 up rows, all of K, for the expert's slots, 16 at a time.  Its eight
// waves take every eighth K block each.  A wave's requests - whole lines of its 32 rows straight to an LDS slot of its own and their scale
// words two blocks ahead, the slots' activations to registers one block ahead - run on across the strips of the run.  The eight sums meet in LDS;
// the last wave, which has the fewest blocks, adds them up, applies the activation and writes h, while the others go on.
// Bound: the weights' bytes.  80 KB of LDS and 128 registers: two workgroups share a CU.
// ------------------------------------------------------------------------------------------------
template <int DT, bool GELU>
__global__ __launch_bounds__(512, 4) void mx_experts_up_kernel(const MxExpertArgs p) {
  constexpr int kSlot = 2 * 2048, kWave = 2 * kSlot;
  constexpr int kOps = 4 + 4;  // loads of a wave per K block beside the activations: scale words, lines
  __shared__ __attribute__((aligned(1024))) uint8_t smem[8 * kWave];
  __shared__ __attribute__((aligned(16))) v4f red[7][2][64];
  __shared__ u16 list[kMxMaxSlots];

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
  bool mine[2];
  uint64_t masks[2];
  const int expert = __builtin_amdgcn_readfirstlane(by_slot ? mx_expert_of(p, blockIdx.y) : (int)blockIdx.y);
  if (expert < 0) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = j * 512 + tid;
    mine[j] = s < p.slots && mx_expert_of(p, s) == expert;
    masks[j] = __ballot(mine[j]);
    if (lane == 0) scratch[j * 8 + w] = __popcll(masks[j]);
  }
  __syncthreads();
  int total = 0;
  for (int k = 0; k < 16; ++k) total += scratch[k];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int at = __popcll(masks[j] & ((1ull << lane) - 1));
    for (int k = 0; k < j * 8 + w; ++k) at += scratch[k];
    if (mine[j]) list[at] = (u16)(j * 512 + tid);
  }
  total = __builtin_amdgcn_readfirstlane(total);
  __syncthreads();
  if (total == 0 || (by_slot && list[0] != (int)blockIdx.y)) return;

  const int row_bytes = p.H >> 1, words = (p.H + 127) >> 7, kbs = (p.H + kMxStep - 1) / kMxStep;
  const int strip0 = blockIdx.x * p.run, nstrips = min(p.run, strips - strip0), ntiles = (total + 15) >> 4;
  const int nb = kbs > w ? (kbs - w + 7) >> 3 : 0;  // blocks of the wave: w, w + 8, ..
  const rsrc_t rW = make_rsrc(p.w1 + (int64_t)expert * p.w1_e, (uint32_t)(2 * p.I * row_bytes));
  const rsrc_t rS = mx_scale_rsrc(p.s1 + (int64_t)expert * p.s1_e * 4, 0, 2 * p.I, words, p.s1_n, p.s1_w);
  const rsrc_t rX = make_rsrc(p.x, (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2));
  const int rl = lane >> 3, cp = lane & 7;
  const uint32_t vo0 = (uint32_t)(rl * row_bytes + (cp ^ (rl >> 1)) * 16), vo1 = (uint32_t)((rl + 8) * row_bytes + (cp ^ (4 + (rl >> 1))) * 16);
  const uint32_t voS = (uint32_t)(r * p.s1_n * 4), up_rows = (uint32_t)(p.I * row_bytes), up_scales = (uint32_t)(p.I * p.s1_n * 4);
  uint8_t* const own = smem + w * kWave;
  const MxCodes codes(lane);

  // a position in the wave's list of work: strips, tiles of a strip, blocks of a tile
  struct At { int strip, tile, i; };
  auto advance = [&](At& a) {
    if (++a.i < nb) return;
    a.i = 0;
    if (++a.tile < ntiles) return;
    a.tile = 0;
    ++a.strip;
  };
  auto row_of = [&](int tile) -> uint32_t {  // byte offset of the activations of the lane's slot
    const int k = tile * 16 + r;
    return k < total ? (uint32_t)((list[k] / p.topk) * p.ldx * 2) + kq * 16 : kOutOfRange;
  };
  uint32_t sc[2][4];
  v4i x[8];
  At ahead{0, 0, 0}, now{0, 0, 0};
  uint32_t xrow = row_of(0);
  auto request_x = [&](const At& a, int j) __attribute__((always_inline)) {
    const int k = (w + 8 * a.i) * kMxStep + j * 32;
    x[j] = buf_load16(rX, xrow != kOutOfRange && k + kq * 8 < p.H ? xrow + (uint32_t)k * 2 : kOutOfRange);
  };
  auto request = [&](int slot) __attribute__((always_inline)) {  // what `ahead` stands at; behind the end nothing is in range
    const bool in = ahead.strip < nstrips;
    const int kb = w + 8 * ahead.i, c0 = (strip0 + ahead.strip) * 16;
    const uint32_t ko = (uint32_t)kb * kMxStepBytes + (uint32_t)(c0 * row_bytes);
    const uint32_t so = voS + (uint32_t)(c0 * p.s1_n * 4);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t wo = (uint32_t)min(2 * kb + j, words - 1) * (uint32_t)(p.s1_w * 4);
      sc[slot][j] = buf_load4(rS, in ? so + wo : kOutOfRange);
      sc[slot][2 + j] = buf_load4(rS, in ? so + up_scales + wo : kOutOfRange);
    }
    uint8_t* const to = own + slot * kSlot;
    buf_load16_to_lds<true>(rW, in ? vo0 + ko : kOutOfRange, 0, to);
    buf_load16_to_lds<true>(rW, in ? vo1 + ko : kOutOfRange, 0, to + 1024);
    buf_load16_to_lds<true>(rW, in ? vo0 + ko + up_rows : kOutOfRange, 0, to + 2048);
    buf_load16_to_lds<true>(rW, in ? vo1 + ko + up_rows : kOutOfRange, 0, to + 3072);
    SB();
    if (in) advance(ahead);
  };

  v4f ag = {0.f, 0.f, 0.f, 0.f}, au = {0.f, 0.f, 0.f, 0.f};
  auto block = [&](int slot) __attribute__((always_inline)) {
    wait_vm<kOps>();  // younger than the block's activations: the lines of the block behind this one
    const uint8_t* const from = own + slot * kSlot;
    uint32_t cg[8], cu[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { cg[j] = codes.get(from, j); cu[j] = codes.get(from + 2048, j); }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every code is out of its slot
    At next = now;
    advance(next);
    if (next.tile != now.tile) xrow = row_of(next.tile);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ag = mx_mac<DT>(ag, x[j], cg[j], mx_block_scale(sc[slot][0], sc[slot][1], j));
      au = mx_mac<DT>(au, x[j], cu[j], mx_block_scale(sc[slot][2], sc[slot][3], j));
      request_x(next, j);  // of the block behind this one
      SB();
    }
    request(slot);
  };
  // the sums of a tile of a strip
  auto finish = [&](int strip, int tile) {
    if (w < 7) {
      red[w][0][lane] = ag;
      red[w][1][lane] = au;
    }
    lds_barrier();  // requests stay in flight
    if (w == 7) {
      v4f g = red[0][0][lane], u = red[0][1][lane];
#pragma unroll 1
      for (int k = 1; k < 7; ++k) {
        const v4f a = red[k][0][lane], b = red[k][1][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) { g[i] += a[i]; u[i] += b[i]; }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { g[i] += ag[i]; u[i] += au[i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = tile * 16 + kq * 4 + i;
        if (k >= total) continue;
        const int s = list[k];
        if (p.on_input) {
          g[i] *= p.topk_w[s];
          u[i] *= p.topk_w[s];
        }
        const float v = (GELU ? gelu_f32(g[i]) : silu_f32(g[i])) * u[i];
        ((u16*)p.h)[(int64_t)s * p.I + (strip0 + strip) * 16 + r] = (u16)(DT == FP8K_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
      }
    }
    lds_barrier();
    ag = au = v4f{0.f, 0.f, 0.f, 0.f};
  };

  if (nb == 0) {
    for (int k = 0; k < nstrips * ntiles; ++k) finish(k / ntiles, k % ntiles);
    return;
  }
  request(0);
#pragma unroll
  for (int j = 0; j < 8; ++j) request_x(now, j);
  SB();
  request(1);
  const int all = nstrips * ntiles * nb;
  for (int q = 0; q < all; q += 2) {
#pragma unroll
    for (int slot = 0; slot < 2; ++slot) {
      if (q + slot >= all) break;
      const At at = now;
      block(slot);
      advance(now);
      if (now.i == 0) finish(at.strip, at.tile);
    }
  }
  wait_vm0();  // requests behind the end moved nothing, but still point at the slots
}

// ------------------------------------------------------------------------------------------------
// Second launch, grid H / 16: a workgroup owns 16 output columns and goes through all tiles of the table.  The K blocks of all tiles are
// one list, which the waves share out in runs; a wave adds a tile's results, times the routed weights, to sums of its own in LDS ([T][16]
// floats), and the eight sets are added in order at the end: no atomics between waves, so results do not depend on timing.
// Lines go to LDS slots of the wave ST blocks ahead, the activations to registers two blocks ahead.
// ------------------------------------------------------------------------------------------------
constexpr int mx_down_slots(int tc) { return tc <= 16 ? 4 : 2; }       // K blocks in flight per wave
constexpr int mx_down_places(int tc) { return tc <= 16 ? 512 : kMxMaxSlots; }  // (token, choice) pairs

template <int DT, int TC>  // TC: tokens that the sums have room for
__global__ __launch_bounds__(512, 4) void mx_experts_down_kernel(const MxExpertArgs p) {
  constexpr int ST = mx_down_slots(TC), kWave = ST * 2048;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[8 * kWave];
  __shared__ __attribute__((aligned(16))) float sums[8 * TC * 16];  // [8][T][16]
  __shared__ int tiles[mx_down_places(TC)];
  __shared__ float weights[mx_down_places(TC)];
  __shared__ u16 order[mx_down_places(TC)];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  float* const mine = sums + w * p.T * 16;

  const int ntiles = p.ntiles[0];
  for (int i = tid; i < p.slots; i += 512) {  // what lies behind the tiles and valid slots is not read below
    tiles[i] = p.tiles[i];
    order[i] = (u16)p.order[i];
    weights[i] = p.on_input ? 1.f : p.weights[i];
  }
  for (int i = lane; i < p.T * 16; i += 64) mine[i] = 0.f;
  __syncthreads();

  const int row_bytes = p.I >> 1, words = (p.I + 127) >> 7, kbs = (p.I + kMxStep - 1) / kMxStep;
  const int all = ntiles * kbs, per = (all + 7) >> 3;
  const int b0 = w * per, b1 = min(all, b0 + per);
  const rsrc_t rH = make_rsrc(p.h, (uint32_t)((int64_t)p.slots * p.I * 2));
  const int rl = lane >> 3, cp = lane & 7;
  const uint32_t vo0 = (uint32_t)((n0 + rl) * row_bytes + (cp ^ (rl >> 1)) * 16), vo1 = (uint32_t)((n0 + rl + 8) * row_bytes + (cp ^ (4 + (rl >> 1))) * 16);
  const uint32_t voS = (uint32_t)((n0 + r) * p.s2_n * 4);
  uint8_t* const own = smem + w * kWave;
  const MxCodes codes(lane);

  struct At { int tile, kb; };
  auto entry = [&](int tile) { return __builtin_amdgcn_readfirstlane(tiles[min(tile, ntiles - 1)]); };
  auto advance = [&](At& a) {
    if (++a.kb == kbs) { a.kb = 0; ++a.tile; }
  };
  // lines of block `wa` into slot `slot`, its scale words into sc[slot]
  uint32_t sc[ST][2];
  auto request_w = [&](int slot, At& a, int left) __attribute__((always_inline)) {
    const bool in = left > 0;
    const int64_t e = entry(a.tile) >> 14;
    const rsrc_t rW = make_rsrc(p.w2 + e * p.w2_e, (uint32_t)(p.H * row_bytes));
    const rsrc_t rS = mx_scale_rsrc(p.s2 + e * p.s2_e * 4, 0, p.H, words, p.s2_n, p.s2_w);
    const uint32_t ko = (uint32_t)a.kb * kMxStepBytes;
#pragma unroll
    for (int j = 0; j < 2; ++j) sc[slot][j] = buf_load4(rS, in ? voS + (uint32_t)min(2 * a.kb + j, words - 1) * (uint32_t)(p.s2_w * 4) : kOutOfRange);
    buf_load16_to_lds<true>(rW, in ? vo0 + ko : kOutOfRange, 0, own + slot * 2048);
    buf_load16_to_lds<true>(rW, in ? vo1 + ko : kOutOfRange, 0, own + slot * 2048 + 1024);
    SB();
    advance(a);
  };
  v4i x[2][8];
  auto request_x = [&](int slot, At& a, int left) __attribute__((always_inline)) {
    const int t = entry(a.tile), first = (t >> 4) & 1023, count = left > 0 ? (t & 15) + 1 : 0;
    const uint32_t row = r < count ? (uint32_t)order[first + r] * (uint32_t)(p.I * 2) + kq * 16 : kOutOfRange;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = a.kb * kMxStep + j * 32;
      x[slot][j] = buf_load16(rH, r < count && k + kq * 8 < p.I ? row + (uint32_t)k * 2 : kOutOfRange);
    }
    SB();
    advance(a);
  };
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  At now{0, 0};
  if (b0 < b1) {
    now = At{b0 / kbs, b0 % kbs};
    At wa = now, xa = now;
    int wleft = b1 - b0, xleft = wleft;
    // the order of the loop: a block's activations, then the lines of the block ST - 2 behind it
#pragma unroll
    for (int s = 0; s < ST - 2; ++s) request_w(s, wa, wleft--);
    request_x(0, xa, xleft--);
    request_w(ST - 2, wa, wleft--);
    request_x(1, xa, xleft--);
    request_w(ST - 1, wa, wleft--);
    auto block = [&](int ws, int xs, bool last) __attribute__((always_inline)) {
      // younger than the block's activations and lines: the next block's activations, and the lines behind the two
      wait_vm<(ST > 2 ? 16 : 12)>();
      const uint8_t* const from = own + ws * 2048;
      uint32_t c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = codes.get(from, j);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every code is out of its slot
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc = mx_mac<DT>(acc, x[xs][j], c[j], mx_block_scale(sc[ws][0], sc[ws][1], j));
        SB();
      }
      request_x(xs, xa, xleft--);
      request_w(ws, wa, wleft--);
      const At at = now;
      advance(now);
      if (now.kb == 0 || last) {
        const int t = entry(at.tile), first = (t >> 4) & 1023, count = (t & 15) + 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = kq * 4 + i;
          // two slots of a tile may be of one token: an LDS atomic, whose order within the wave is fixed
          if (row < count) atomicAdd(&mine[(order[first + row] / p.topk) * 16 + r], acc[i] * weights[first + row]);
          acc[i] = 0.f;
        }
      }
    };
    for (int b = b0; b < b1; b += ST) {
#pragma unroll
      for (int k = 0; k < ST; ++k) {
        if (b + k >= b1) break;
        block(k, k & 1, b + k == b1 - 1);
      }
    }
  }
  wait_vm0();
  __syncthreads();
  for (int i = tid; i < p.T * 16; i += 512) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += sums[k * p.T * 16 + i];
    v *= p.scaling;
    ((u16*)p.out)[(int64_t)(i >> 4) * p.H + n0 + (i & 15)] = (u16)(DT == FP8K_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
  }
}

}  // namespace fp8k
