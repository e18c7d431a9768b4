// Absorbed latent attention of a few new tokens over the paged cache, gfx950.
//
// A request has M = queries x heads rows that all read the same cached rows: keys of 576, values their first 512.  With r over its tokens
//   s[m, r] = scale * q[m] . row[r],   p = exp(s - max s),   o[m] = sum p[r] row[r, :512] / sum p[r]
//
// The scores are formed transposed, S^T = K . Q^T, so that a lane holds scores of one query row, and what it holds is the operand of
// O^T = V^T . P^T as it lies: the order of the tokens inside a product is free, as long as V^T, read from LDS by transposed reads,
// has the same.  P never goes through LDS, and the rescaling factors of O are a lane's own.
//
// A workgroup is eight waves (four with WM = 1).  WM of them split the R = 16 WM query rows, the other factor splits the tokens of a step of the
// loop; each has its own running maximum and sum, and waves that share rows are joined through LDS at the end.  A wave holds its 16 rows' queries and
// all 512 columns of O, 200 registers.  With WM = 1 a wave reads nothing but the 16 rows that it fetched itself, and the loop has no barrier.
//
// LDS: a step of T rows is 9 blocks of [T rows][64 numbers], filled by global_load_lds with per-lane addresses (pages lie anywhere, beyond 4 GB
// too).  Few rows (WM = 1, 2) are bound by the bytes: T = 64, two stages.  Many (WM = 4, 8) by the matrix cores and LDS: T = 32, four stages, and
// one barrier to a step.  A wave-load is 8 rows of a block, so a lane fetches from one row of a step (WM = 1: two), at multiples of 128 bytes.  The
// 16-byte chunk c of row r of a block sits at c ^ swizzle(r), which keeps both the operand reads (16 rows, one chunk) and the transposed
// ones (8 rows, two chunks) off each other's banks.  8-bit rows are fetched to stages of half the size, 16 rows x 64 bytes to a wave-load, and
// widened into one 16-bit tile (WM = 4, 8: two by turns, the next one beside the products).  The entries of the page table come the same way, some steps
// ahead of the rows: no load into a register is waited for in the loop, which would wait for the rows behind it too.
//
// Work: the tiles (64 tokens) of all requests in a row are cut into equal runs, one to a workgroup, from the lengths on the device: a captured graph
// needs no plan.  A run that holds all of a request writes its result; others write normalised float32 partials and the base-2
// logarithm of their sums, which mla_join_kernel adds up.
//
// Measured (page 64, lengths from a third of the most to the most): one request of 8000 tokens, 128 heads, bf16 19 us and 4 for the join, latency; 64 of
// 8192, 2 x 16 heads, fp16 85 + 6 us, 4.5 TB/s with everything, 6.1 TB/s in the loop (128 of 16000, 16 heads); 128 of 6000, 128 heads, 8 bits 193 + 18 us back to back,
// 0.67 PFLOP/s with everything, 0.90 in the loop, where the matrix cores and LDS are busy half the time each.  Of the rest the most are the partials: 100 MB
// written at the end of all runs at once, and read by the join.
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
  float *part, *part_lse;  // [slots, M, 512], [slots, M]: mla_slots(B, walkers) of them
  v2i* spans;              // [B]: the first run that holds tokens of a request, and how many do (none: it has no tokens)
  int B, n, H, M;
  int page_size, pages, max_len;
  int page_shift;  // log2 of page_size, or -1
  int walkers, mblocks;
  float sm_scale;
};

constexpr int kMlaTile = 64;         // tokens of a tile
constexpr int kMlaMinRun = 2;        // tiles that a run has at least
// What beginning a request costs beside its tiles (pages, then rows, then queries to be waited for, and a result to be written), in tiles: a run with a new
// request in it gets as many fewer.  us with 0 / 4 / 8: 64 requests of up to 4000 tokens, 128 heads 102 / 91 / 92; 200 of 300, 16 heads 30 / 25.5 / 24;
// 64 of 8192, 2 x 16 heads 96 / 92 / 94; one of 32000, 128 heads 42.6 / 43 / 43.
constexpr int kMlaNew = 4;

// Places of partials.  A run leaves at most two: of the request that it goes on with, at the run's number, and of one that begins in it and does not
// end in it, behind those, at the request's number or the run's, whichever are fewer.
__host__ __device__ __forceinline__ int64_t mla_slots(int64_t B, int64_t walkers) { return walkers + (B < walkers ? B : walkers); }
__device__ __forceinline__ int mla_slot(const MlaDecodeArgs& p, int walker, int b, bool begins) {
  return begins ? p.walkers + (p.B < p.walkers ? b : walker) : walker;
}

__device__ __forceinline__ int mla_len(const MlaDecodeArgs& p, int b) { return min(max(p.lens[b], 0), p.max_len); }
__device__ __forceinline__ int mla_tiles(int len) { return (len + kMlaTile - 1) / kMlaTile; }
__device__ __forceinline__ int mla_units(int tiles) { return tiles ? tiles + kMlaNew : 0; }
// units of a run, from all requests' units
__device__ __forceinline__ int mla_run(int total, int walkers) { return max((total + walkers - 1) / walkers, kMlaMinRun); }
// Units of all requests, by a workgroup of NW waves; every thread returns the total.  Thread t counts requests [t * per, + per): `before`
// is what lies in front of them, `mine` their own, `len` the last one's tokens.  `note`: requests without tokens, which no run meets, get their spans.
template <int NW>
__device__ __forceinline__ int mla_scan(const MlaDecodeArgs& p, int per, int& before, int& mine, int& len, int* lds, bool note) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int sum = 0;
  len = 0;
  for (int b = tid * per; b < min((tid + 1) * per, p.B); ++b) {
    len = mla_len(p, b);
    if (note && len == 0) p.spans[b] = v2i{0, 0};
    sum += mla_units(mla_tiles(len));
  }
  int run = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(run, d);
    if (lane >= d) run += v;
  }
  if (lane == 63) lds[w] = run;
  lds_only_barrier();
  int total = 0, base = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    if (i < w) base += lds[i];
    total += lds[i];
  }
  before = base + run - sum;
  mine = sum;
  return total;
}

// position of a row's 16-byte chunks in a block: c ^ swizzle(r).  Rows are 128 bytes: neighbours use different halves of the banks already.  Of the
// linear maps of bits 1 .. 3 of r, those with full rate for either kind of read (operand reads 225 bytes a clock and CU, transposed ones 161; (r >> 1) & 7
// does as well for the first alone, its rotation has half the rate there).
__device__ __forceinline__ int mla_swizzle(int r) { return ((r & 2) ? 6 : 0) ^ ((r & 4) ? 5 : 0) ^ ((r & 8) ? 4 : 0); }

template <int DT, bool FP8, int WM>
__global__ __launch_bounds__(WM == 1 ? 256 : 512) void mla_decode_kernel(const MlaDecodeArgs p) {
  constexpr int NW = WM == 1 ? 4 : 8, WT = NW / WM, R = 16 * WM;
  constexpr int TT = WM >= 4 ? 32 : 64, NT = TT / WT / 16;  // tokens of a step of the loop, 16-token tiles of a wave
  constexpr bool kDeep = TT == 32;
  constexpr int kBlock = TT * 128;                         // bytes of a block of 64 numbers of a step's rows
  constexpr int kTileBytes = 9 * kBlock, kStageBytes = FP8 ? kTileBytes / 2 : kTileBytes;
  constexpr int kTiles = FP8 ? (kDeep ? 2 : 1) : 0;        // 16-bit tiles beside the stages, for 8-bit rows
  constexpr int kStageCount = kDeep ? 4 : 2;
  constexpr int kRow = FP8 ? kLatentRow : 2 * kLatentRow;  // bytes of a cached row
  // A wave fetches from kRowsOfWave rows, kRowsOfLane to a lane; kSharers waves share rows, by blocks: kMost of them the first, kLeast the others.
  constexpr int kRowsOfWave = FP8 || NW == 4 ? 16 : 8, kRowsOfLane = !FP8 && NW == 4 ? 2 : 1;
  constexpr int kSharers = NW * kRowsOfWave / TT, kLeast = 9 / kSharers, kMost = 9 - (kSharers - 1) * kLeast;
  constexpr int kPageSlots = 8;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kTiles * kTileBytes + kStageCount * kStageBytes];
  __shared__ int found[3], scan[NW], pages[kPageSlots][NW][16];
  __shared__ float join_m[NW][16], join_l[NW][16];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w % WM, wt = w / WM, l15 = lane & 15, g = lane >> 4;
  // the workgroups of a run's row blocks read the same rows: on one XCD (workgroup i runs on XCD i % 8), side by side
  const int per8 = p.mblocks * 8;
  const int walker = (int)(blockIdx.x / per8) * 8 + (int)(blockIdx.x % 8), mblk = (int)(blockIdx.x % per8) / 8;
  if (walker >= p.walkers) return;

  const int per = (p.B + NW * 64 - 1) / (NW * 64);
  int before, mine, mine_len;
  const int total = mla_scan<NW>(p, per, before, mine, mine_len, scan, walker == 0 && mblk == 0);
  const int run = mla_run(total, p.walkers);
  if ((int64_t)walker * run >= total) return;
  const int first = walker * run, last = min(first + run, total);
  // Lengths are read again from here on.  Should they have changed (a caller that overwrites them under the call gets no result to rely on), both walks over
  // the requests still end at the last one.
  if (first >= before && first < before + mine) {  // this thread counted the request that the run begins in
    int b = tid * per, at = before, len = per > 1 ? mla_len(p, b) : mine_len;
    const int end = min((tid + 1) * per, p.B) - 1;
    for (int t = mla_units(mla_tiles(len)); b < end && first >= at + t; t = mla_units(mla_tiles(len))) {
      at += t;
      len = mla_len(p, ++b);
    }
    found[0] = b;
    found[1] = at;
    found[2] = len;
  }
  lds_only_barrier();
  int b = __builtin_amdgcn_readfirstlane(found[0]), at = __builtin_amdgcn_readfirstlane(found[1]), len = __builtin_amdgcn_readfirstlane(found[2]);

  const float kscale = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(FP8 && p.scale ? *p.scale : 1.0f)));
  // at least the smallest number: with a product that is no number above zero any more, what is masked would be 0 times -inf
  const float c = fmaxf(p.sm_scale * kLog2e * kscale, 0x1p-149f);

  const int row = mblk * R + wm * 16 + l15;  // this lane's, of the M of a request

  for (int next_len; at < last && b < p.B; ++b, len = next_len) {
    next_len = b + 1 < p.B ? mla_len(p, b + 1) : 0;
    const int tiles = mla_tiles(len), tiles_at = at + kMlaNew, t_begin = max(first - tiles_at, 0), t_end = min(last - tiles_at, tiles);
    at += mla_units(tiles);
    if (t_begin >= t_end) continue;
    if (t_begin == 0 && mblk == 0 && tid == 0) p.spans[b] = v2i{walker, (at - 1) / run - walker + 1};

    // ---- fetching.  Steps are counted from the segment's first.  Tokens past the end are the last one's row again (masked).
    const int base = t_begin * kMlaTile, steps = min((t_end - t_begin) * (kMlaTile / TT), (len - base + TT - 1) / TT);
    const int group = w % (NW / kSharers), share = w / (NW / kSharers), first_row = kRowsOfWave * group;
    // What follows from the lane is computed anew for every step: kept across the loop, it goes to scratch memory, and a load from there waits for the
    // rows that are on their way.
    auto fresh_lane = [&] {
      int x = lane;
      asm volatile("" : "+v"(x));
      return x;
    };
    // The pages of a step's rows go to LDS as well, some steps ahead, so that no load into a register is ever waited for.  Always made, so that
    // loads can be counted; past the end for the last row again.
    const int32_t* const pages_of = p.table + b * p.table_stride;
    const uint32_t pages_to = lds_address(&pages[0][w][0]);
    auto page_of = [&](uint32_t tok) { return p.page_shift >= 0 ? tok >> p.page_shift : tok / (uint32_t)p.page_size; };
    auto fetch_pages = [&](int t) {
      const int lane = fresh_lane();
      const uint32_t tok = min(base + t * TT + first_row + lane, len - 1);
      if (lane < kRowsOfWave) load4_to_lds(pages_of + page_of(tok), pages_to + (t % kPageSlots) * (NW * 64));
    };
    auto fetch = [&](int t, uint32_t to) {  // to: of the stage
      const int lane = fresh_lane();
      const uint8_t* from[kRowsOfLane];
#pragma unroll
      for (int k = 0; k < kRowsOfLane; ++k) {
        const int r = FP8 ? lane >> 2 : 8 * k + (lane >> 3);  // of the wave's
        const uint32_t tok = min(base + t * TT + first_row + r, len - 1), place = tok - page_of(tok) * (uint32_t)p.page_size;
        const uint32_t page = min(max(pages[t % kPageSlots][w][r], 0), p.pages - 1);
        from[k] = p.cache + (uint64_t)page * (uint32_t)(p.page_size * kRow) + (place * kRow + (FP8 ? (lane & 3) : (lane & 7) ^ mla_swizzle(first_row + r)) * 16);
      }
#pragma unroll
      for (int k = 0; k < kRowsOfLane; ++k) {
        constexpr int kStep = FP8 ? 64 : 128, kToStep = FP8 ? 1024 : kBlock;
        const uint32_t place = FP8 ? to + group * 9 * 1024 : to + (first_row + 8 * k) * 128;
        if (kSharers == 1 || share == 0) load_blocks_to_lds<kStep, kToStep, 0, kMost>(from[k], place);
        else if (kSharers == 2 || share == 1) load_blocks_to_lds<kStep, kToStep, kMost, kMost + kLeast>(from[k], place);
        else if (share == 2) load_blocks_to_lds<kStep, kToStep, kMost + kLeast, kMost + 2 * kLeast>(from[k], place);
        else load_blocks_to_lds<kStep, kToStep, kMost + 2 * kLeast, 9>(from[k], place);
      }
    };
    // all loads but the youngest: FETCHES steps' rows and PAGES steps' pages
    auto wait_but = [&](auto fetches, auto page_loads) {
      constexpr int kF = decltype(fetches)::value, kP = decltype(page_loads)::value;
      if (kSharers == 1 || share == 0) wait_loads<kF * kMost * kRowsOfLane + kP>();
      else wait_loads<kF * kLeast * kRowsOfLane + kP>();
    };
    // 8-bit rows of a stage, as this wave fetched them: to registers, and from there as 16 bits to a tile
    const int first_block = share == 0 ? 0 : kMost + (share - 1) * kLeast;
    struct Raw {
      v4i x[kMost];
    };
    auto raw_of = [&](const uint8_t* stage) {
      const uint8_t* const from = stage + (group * 9 + first_block) * 1024 + fresh_lane() * 16;
      Raw raw;
#pragma unroll
      for (int j = 0; j < kMost; ++j)
        if (j < kLeast || share == 0) raw.x[j] = *(const v4i*)(from + j * 1024);
      return raw;
    };
    auto widen = [&](const Raw& raw, uint8_t* tile) {
      const int lane = fresh_lane();
      uint8_t* const to = tile + first_block * kBlock + (first_row + (lane >> 2)) * 128;
      const int at0 = ((2 * (lane & 3)) ^ mla_swizzle(lane >> 2)) << 4;
#pragma unroll
      for (int j = 0; j < kMost; ++j)
        if (j < kLeast || share == 0) {
          const v4i x = raw.x[j];
          *(v4i*)(to + j * kBlock + at0) = v4i{(int)fp8_to_16bit<DT, false>(x[0]), (int)fp8_to_16bit<DT, true>(x[0]),
                                               (int)fp8_to_16bit<DT, false>(x[1]), (int)fp8_to_16bit<DT, true>(x[1])};
          *(v4i*)(to + j * kBlock + (at0 ^ 16)) = v4i{(int)fp8_to_16bit<DT, false>(x[2]), (int)fp8_to_16bit<DT, true>(x[2]),
                                                      (int)fp8_to_16bit<DT, false>(x[3]), (int)fp8_to_16bit<DT, true>(x[3])};
        }
    };

    constexpr int kStagesAt = kTiles * kTileBytes;
    const uint32_t lds0 = lds_address(smem) + kStagesAt;
    auto to_stage = [&](int t) { return lds0 + t % kStageCount * kStageBytes; };
    auto stage_of = [&](int t) { return smem + kStagesAt + t % kStageCount * kStageBytes; };

    // Rows are asked for kRun steps before their step, pages kPagesRun steps before the rows.
    //   two stages:  the rows of step t + 1 (8 bits: t + 2) while step t is waited for, which takes two barriers, or none (WM = 1)
    //   four stages: the rows of step t + 3 (8 bits: t + 5) while those of t + 1 and t + 2 (8 bits: t + 2 .. t + 4) are on their way; one barrier
    constexpr int kRun = kStageCount - 1 + (FP8 ? (kDeep ? 2 : 1) : 0), kPagesRun = kDeep ? (FP8 ? 4 : 2) : 1;
    auto ask = [&](int t) {  // one step's rows, and the pages of a later one's
      fetch_pages(t + kPagesRun);
      fetch(t, to_stage(t));
    };
    constexpr int kFirst = FP8 ? kStageCount : kRun;  // steps asked for at first, with pages that have come already
#pragma unroll
    for (int t = 0; t < kFirst + (kDeep ? 0 : 1); ++t) fetch_pages(t);

    wait_loads<0>();
#pragma unroll
    for (int t = 0; t < kFirst; ++t)
      if (t < steps) ask(t);

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

    if constexpr (FP8 && kDeep) {  // the first tile, and the rows that take its stage
      wait_loads<0>();
      widen(raw_of(stage_of(0)), smem);
      wait_lds();
      if (kStageCount < steps) ask(kStageCount);
    }
    wait_loads<0>();  // the queries: waited for here, not in the loop
    for (int t = 0; t < steps; ++t) {
      const int lane = fresh_lane(), l15 = lane & 15, g = lane >> 4;
      const uint8_t* tile;
      Raw raw;
      if constexpr (!kDeep) {
        if (WM > 1) lds_only_barrier();  // nobody reads the step before any more
        else wait_lds();
        if constexpr (!FP8) {
          if (t + 1 < steps) {
            ask(t + 1);
            wait_but(Const<1>{}, Const<0>{});
          } else wait_loads<0>();
          tile = stage_of(t);
        } else {
          if (t + 1 < steps) wait_but(Const<1>{}, Const<0>{});
          else wait_loads<0>();
          const Raw raw = raw_of(stage_of(t));
          wait_lds();
          if (t + 2 < steps) ask(t + 2);
          widen(raw, smem);
          tile = smem;
        }
        if (WM > 1) lds_only_barrier();  // everybody's part of the step is there
      } else if constexpr (!FP8) {
        if (t + 2 < steps) wait_but(Const<2>{}, Const<1>{});
        else wait_loads<0>();
        lds_only_barrier();  // everybody's part of the step is there, and nobody reads the step before any more
        tile = stage_of(t);
      } else {
        lds_only_barrier();  // this step's tile is whole, and nobody reads the other any more
        if (t + 1 < steps) {
          if (t + 4 < steps) wait_but(Const<3>{}, Const<3>{});
          else wait_loads<0>();
          raw = raw_of(stage_of(t + 1));
        }
        tile = smem + t % 2 * kTileBytes;
      }

      // ---- S^T = K . Q^T: kAhead operand reads run ahead of the products.  With one tile of tokens, two sums by turns: a product waits for the
      // one before it in its sum.
      constexpr int kSums = NT == 1 ? 2 : NT, kAhead = NW == 4 ? 8 : kDeep && FP8 ? 3 : 6;
      v4f s[kSums];
#pragma unroll
      for (int i = 0; i < kSums; ++i) s[i] = v4f{0, 0, 0, 0};
      {
        // row l15 of a 16-token tile, chunk 4 ks + g
        const int k_off = (wt * NT * 16 + l15) * 128 + ((g ^ mla_swizzle(l15)) << 4);
        const uint8_t* const even = tile + k_off;
        const uint8_t* const odd = tile + (k_off ^ 64);
        auto read = [&](int i) {
          const int ks = i / NT, nt = i % NT;
          return *(const v4i*)((ks & 1 ? odd : even) + (ks >> 1) * kBlock + nt * 16 * 128);
        };
        v4i ring[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = read(i);
#pragma unroll
        for (int i = 0; i < 18 * NT; ++i) {
          s[i % kSums] = mfma16<DT>(ring[i % kAhead], q[i / NT], s[i % kSums]);
          if (i + kAhead < 18 * NT) ring[i % kAhead] = read(i + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (NT == 1) s[0] += s[1];
      // what has to be done for later steps, beside the last products
      if constexpr (kDeep && !FP8) {
        if (t + 3 < steps) ask(t + 3);
      }
      if constexpr (kDeep && FP8) {
        if (t + 1 < steps) {
          wait_lds();  // the stage has been read
          if (t + 5 < steps) ask(t + 5);
          widen(raw, smem + (t + 1) % 2 * kTileBytes);
        }
      }

      // ---- softmax: a lane's scores are those of query row l15, tokens 16 nt + 4 g + i
      const int tok0 = base + t * TT + wt * NT * 16 + 4 * g;
      const bool masked = base + (t + 1) * TT > len - (p.n - 1);
      float top = -INFINITY;
      if (__builtin_expect(masked, 0)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tok0 + nt * 16 + i >= lim) s[nt][i] = -INFINITY;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[nt][i]);
      // c > 0.  The row's maximum, over four lanes, is asked for only when one of them has passed the old one by far.
      if (__builtin_expect(__any(top * c > m + kMaxSlack), 0)) {
        top = max_across32(max_across16(top)) * c;
        const float raised = top > m + kMaxSlack ? top : m;
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
          e[i] = __builtin_amdgcn_exp2f(fmaf(s[nt][i], c, -shift));
          l += e[i];
        }
        // weights rounded to the 16-bit type, as the matrix core takes them; their sum is of the unrounded ones
        pk[nt][0] = pack2<DT>(e[0], e[1]);
        pk[nt][1] = pack2<DT>(e[2], e[3]);
      }

      // ---- O^T += V^T . P^T, reads ahead of the products likewise; columns in the inner loop, so that a product waits for no other
      {
        const int v_row = 4 * g + (l15 >> 2);
        const int v_off = (wt * NT * 16 + v_row) * 128 + ((((l15 & 3) >> 1) ^ mla_swizzle(v_row)) << 4) + ((l15 & 1) << 3);
        const uint8_t* v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = tile + (v_off ^ (i << 5));
        constexpr int kSteps = NT == 1 ? 32 : 16 * NT, kVAhead = NW == 4 ? 8 : NT == 1 ? 6 : 5;
        v2i ring[kVAhead][2];
        auto read = [&](int i, v2i* to) {
          const int dt = i & 31, nt = (i >> 5) * 2;
          const uint8_t* const at = v[dt & 3] + (dt >> 2) * kBlock + nt * 16 * 128;
          to[0] = lds_read_transposed(at);
          if (NT > 1) to[1] = lds_read_transposed(at + 16 * 128);
        };
#pragma unroll
        for (int i = 0; i < kVAhead; ++i) read(i, ring[i]);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int dt = i & 31, nt = (i >> 5) * 2;
          const v2i* const a = ring[i % kVAhead];
          if constexpr (NT == 1) o[dt] = mfma16_half<DT>(a[0], v2i{(int)pk[0][0], (int)pk[0][1]}, o[dt]);
          else o[dt] = mfma16<DT>(v4i{a[0][0], a[0][1], a[1][0], a[1][1]}, v4i{(int)pk[nt][0], (int)pk[nt][1], (int)pk[nt + 1][0], (int)pk[nt + 1][1]}, o[dt]);
          if (i + kVAhead < kSteps) read(i + kVAhead, ring[i % kVAhead]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }

    // ---- join the waves that share rows, normalise, write
    const bool whole = t_end - t_begin == tiles;
    const int64_t slot = mla_slot(p, walker, b, t_begin == 0);
    l = sum_across32(sum_across16(l));
    if (g == 0) {
      join_m[w][l15] = m;
      join_l[w][l15] = l;
    }
    wait_loads<0>();     // pages that nobody needed
    lds_only_barrier();  // and nobody reads a tile any more
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
    if constexpr (WT == 1) {
      if (row < p.M) {
        const int64_t to = (whole ? (int64_t)b * p.M + row : slot * p.M + row) * kLatent + 4 * g;
        if (whole) {
#pragma unroll
          for (int dt = 0; dt < 32; ++dt) *(v2i*)((u16*)p.out + to + dt * 16) = v2i{(int)pack2<DT>(o[dt][0], o[dt][1]), (int)pack2<DT>(o[dt][2], o[dt][3])};
        } else {
#pragma unroll
          for (int dt = 0; dt < 32; ++dt) *(v4f*)(p.part + to + dt * 16) = o[dt];
        }
      }
    } else {
      // a quarter of the 512 columns at a time through LDS: [WT][R] rows of 128 floats (and 4 of padding)
      constexpr int kLd = 132;
      float* const buf = (float*)smem;
#pragma unroll
      for (int quarter = 0; quarter < 4; ++quarter) {
        if (quarter) lds_only_barrier();
#pragma unroll
        for (int d = 0; d < 8; ++d) *(v4f*)(buf + (wt * R + wm * 16 + l15) * kLd + d * 16 + 4 * g) = o[quarter * 8 + d];
        lds_only_barrier();
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
      }
    }
    lds_only_barrier();  // before the next request's rows come
  }
}

// Adds up the partials of requests that several runs share, in the order of their tokens, and gives requests without tokens their zeros.
// WAVES waves of a workgroup of four share a row: one where there are many rows with few partials each, four where there are few rows with many.
// A wave takes every WAVES-th partial, eight columns to a lane.
template <int DT, int WAVES>
__global__ __launch_bounds__(256) void mla_join_kernel(const MlaDecodeArgs p) {
  __shared__ v4f parts[WAVES == 1 ? 1 : 3 * 128];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) % WAVES);
  const int b = blockIdx.y, r = (int)blockIdx.x * (4 / WAVES) + (int)(threadIdx.x >> 6) / WAVES;
  if (r >= p.M) return;  // whole workgroups, with WAVES = 4
  // The cut is that of the first launch, whatever becomes of the lengths meanwhile; held within the runs, so that no partial outside the workspace is
  // read even if lengths that changed under that launch left a span that nobody wrote.
  v2i span = p.spans[b];
  span[0] = min(max(span[0], 0), p.walkers - 1);
  const int n = min(span[1], p.walkers - span[0]);
  const int64_t row = (int64_t)b * p.M + r;
  u16* const out = (u16*)p.out + row * kLatent + 4 * lane;
  if (n <= 0) {
    if (w == 0) {
      *(v2i*)out = v2i{0, 0};
      *(v2i*)(out + 256) = v2i{0, 0};
      if (lane == 0 && p.lse) p.lse[row] = -INFINITY;
    }
    return;
  }
  if (n == 1) return;
  const int beginning = mla_slot(p, span[0], b, true);
  auto slot_of = [&](int i) -> int64_t { return i ? span[0] + i : beginning; };
  // The partials are asked for before their weights are known, a batch of up to 64 at a time (n <= 256): a logarithm to a lane, and
  // kEach partials to a wave at once.
  constexpr int kEach = WAVES == 1 ? 4 : 16;
  v4f x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
  float top = -INFINITY, sum = 0.0f;
  const float* const from = p.part + (int64_t)r * kLatent + 4 * lane;
  for (int at = 0; at < n; at += kEach * WAVES) {
    const int count = min(n - at, kEach * WAVES);  // at most 64
    const float lse = lane < count ? p.part_lse[slot_of(at + lane) * p.M + r] : -INFINITY;
    v4f u[kEach], v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      u[i] = v[i] = v4f{0, 0, 0, 0};
      if (i * WAVES + w < count) {
        const float* const part = from + slot_of(at + i * WAVES + w) * p.M * kLatent;
        u[i] = *(const v4f*)part;
        v[i] = *(const v4f*)(part + 256);
      }
    }
    float most = lse;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    most = fmaxf(most, top);
    const float before = __builtin_amdgcn_exp2f(top - shift_of(most));  // 0 at first
    const float weight = __builtin_amdgcn_exp2f(lse - shift_of(most));
    top = most;
    float s = weight;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    sum = sum * before + s;
    x *= before;
    y *= before;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (i * WAVES + w >= count) break;
      const float f = __shfl(weight, i * WAVES + w);
      x += f * u[i];
      y += f * v[i];
    }
  }
  const float shift = shift_of(top);
  if constexpr (WAVES > 1) {
    if (w) {
      parts[(w - 1) * 128 + lane] = x;
      parts[(w - 1) * 128 + 64 + lane] = y;
    }
    lds_only_barrier();
    if (w) return;
#pragma unroll
    for (int i = 0; i < WAVES - 1; ++i) {
      x += parts[i * 128 + lane];
      y += parts[i * 128 + 64 + lane];
    }
  }
  const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
  x *= f;
  y *= f;
  *(v2i*)out = v2i{(int)pack2<DT>(x[0], x[1]), (int)pack2<DT>(x[2], x[3])};
  *(v2i*)(out + 256) = v2i{(int)pack2<DT>(y[0], y[1]), (int)pack2<DT>(y[2], y[3])};
  if (lane == 0 && p.lse) p.lse[row] = sum == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(sum) + shift) * kLn2;
}

}  // namespace fp8k
