// 256(n) x 256(m) x 256(k) workgroup tiles of the MXFP4 product for large batches, gfx950: 8 wavefronts (2 along n x 4 along m), wave tile
// 128 x 64 = 8 x 4 products of 16 x 16, a K block being one 128-byte line of a row (256 values, two products of 128).
//
// Bound: issue, at a clock that the power limit sets.  4096 x 18432 x 7168: 252 - 262 us, 4.1 - 4.3 PFLOP/s; the same 455 thousand clocks take 208 -
// 217 us on zeros, the data lowers the clock from 2.3 to 1.9 GHz.  The matrix cores are 57 % busy in either; a wave issues in 39 % of its
// clocks, waits for an issue slot in 34 % and at barriers or for memory in 26 % (two waves to a SIMD).  The LDS is busy with reads in 24 %,
// 4 % of those in bank conflicts.  (A bare loop of e2m1 products reaches 6.2 PFLOP/s on quantised normal data, 8.8 on zeros.)  Moving the
// activation requests of a block apart changed nothing.
//
// Stages, walk and write-out are those of gemm_tile256_kernel: three weight stages and two activation stages of 256 rows x 128 B, filled
// by buffer_load ... lds with the whole offset in the range-checked per-lane operand, 16-byte chunk c of row r at position
// c ^ ((r >> 1) & 7); one barrier per K block in front of its last quarter, with a wave's four youngest loads - weights - still in
// flight; both rings run on across the tiles of a workgroup's walk, so that a tile opens with its operands in LDS.  In this kernel the
// products accumulate in place, and a lane takes chunks kq and 4 + kq of a line, bytes kq of the two scale words of a K block.  The words
// of 64 rows are one coalesced load (six a K block; they are older than the block's weight loads, so the wait at the barrier covers them)
// and are handed to the lanes of their rows by lane swaps.
//
// RAGGED: K is no multiple of 256.  Chunks of the activations past the end of a row are out of range for their lane and arrive as zeros;
// what the weights have there (bytes of the next row) is multiplied by them: e2m1 has neither infinities nor NaN.
#pragma once

#include "mx_common.h"

namespace fp8k {

template <int OUT_DT, int BIAS_DT, bool RAGGED>
__global__ __launch_bounds__(512, 1) void mx_tile256_kernel(const MxArgs p) {
  constexpr int kWStage = 256 * kMxStepBytes, kXStage = 256 * kMxStepBytes, kXBase = 3 * kWStage;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[3 * kWStage + 2 * kXStage];

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wn = w & 1, wm = w >> 1;

  const int bid = blockIdx.x;
  // ---- this workgroup's items: the whole tiles of its walk, then at most one half tile of the last, partial round
  int walk_next = 0, walk_step = 1, walk_first = 0, walk_end = 0;
  if (bid < p.walkers) {
    const int per_xcd = (p.tail_first + 7) >> 3;
    walk_next = bid >> 3;
    walk_step = p.walkers >> 3;
    walk_first = (bid & 7) * per_xcd;
    walk_end = min(walk_first + per_xcd, p.tail_first);
  }
  int tail_unit = p.tail_shared ? bid : bid - p.walkers;
  if (tail_unit >= (p.tiles_m * p.tiles_n - p.tail_first) * 2) tail_unit = -1;
  struct Item { int t, half; bool is_half; };
  auto next_item = [&](Item& it) -> bool {
    if (walk_first + walk_next < walk_end) {
      it = Item{walk_first + walk_next, 0, false};
      walk_next += walk_step;
      return true;
    }
    if (tail_unit >= 0) {
      it = Item{p.tail_first + (tail_unit >> 1), tail_unit & 1, true};
      tail_unit = -1;
      return true;
    }
    return false;
  };
  Item item;
  if (!next_item(item)) return;

  const int row_bytes = p.K >> 1, words = (p.K + 127) >> 7, nkb = (p.K + kMxStep - 1) / kMxStep;
  // K block b of an item sits in weight stage (gw0 + b) % 3 and activation stage (gx0 + b) & 1; loads behind an item's last block fetch
  // the first blocks of the next item.  `pref`: the item before requested activation block 0 and weight blocks 0 and 1.
  int gw0 = 0, gx0 = 0;
  bool pref = false;
  for (;;) {
    const int t = item.t, half = item.half;
    const bool is_half = item.is_half;
    // the lane constants are derived anew for every tile from a lane id the compiler cannot see through: hoisted out of the tile loop
    // they would stay live across it
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int rl = ln >> 3, cp = ln & 7;
    uint32_t voW[2], voX[2];
#pragma unroll
    for (int par = 0; par < 2; ++par) {
      const int c = cp ^ ((par << 2) + (rl >> 1));
      voW[par] = (uint32_t)(rl * p.ldw + c * 16);
      voX[par] = (uint32_t)(rl * p.ldx + c * 16);
    }
    const uint32_t soW = (uint32_t)(w * 32 * p.ldw), soX = (uint32_t)(w * 32 * p.ldx);
    const uint32_t stepW = (uint32_t)(8 * p.ldw), stepX = (uint32_t)(8 * p.ldx);
    const int lr = ln & 15, kq = ln >> 4;
    const uint32_t fa0 = (uint32_t)(lr * kMxStepBytes + ((kq ^ ((lr >> 1) & 7)) << 4)), fa1 = fa0 ^ 64u;

    rsrc_t rW = make_rsrc(p.W, 0), rX = make_rsrc(p.X, 0);
    rsrc_t rWn = make_rsrc(p.W, 0), rXn = make_rsrc(p.X, 0);  // the item after this one (empty: every load is a no-op)
    auto tile_rsrcs = [&](rsrc_t& dW, rsrc_t& dX, int tile, int hf, bool halved) {
      int tm, tn;
      tile_coords(tile, p.tiles_m, p.tiles_n, tm, tn);
      const int mm = tm * 256 + hf * 128, nn = tn * 256;
      const int rowsW = min(256, p.N - nn), rowsX = min(halved ? 128 : 256, p.M - mm);
      dW = make_rsrc(p.W + (int64_t)nn * p.ldw, rowsX > 0 ? (uint32_t)((rowsW - 1) * p.ldw + row_bytes) : 0u);
      dX = make_rsrc(p.X + (int64_t)mm * p.ldx, rowsX > 0 ? (uint32_t)((rowsX - 1) * p.ldx + row_bytes) : 0u);
    };

    int tile_m, tile_n;
    tile_coords(t, p.tiles_m, p.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * 256 + half * 128, n0 = tile_n * 256;
    if (m0 >= p.M) {  // upper half of a tile past the last row
      wait_vm0();     // requests of the item before may still point at the stages
      return;
    }
    const int nrows = is_half ? min(p.M, m0 + 128) : p.M;  // exclusive bound of a valid output row

    tile_rsrcs(rW, rX, t, half, is_half);
    Item next;
    const bool has_next = next_item(next);
    const bool stream = has_next && nkb >= 3;  // its first blocks are requested by this item's last trips
    if (has_next) tile_rsrcs(rWn, rXn, next.t, next.half, next.is_half);
    const rsrc_t rWs = stream ? rWn : make_rsrc(p.W, 0), rXs = stream ? rXn : make_rsrc(p.X, 0);
    auto LW = [&](int j, int kstep, int ws) {
      const bool nx = kstep >= nkb;
      buf_load16_to_lds(nx ? rWs : rW, voW[j & 1] + (soW + j * stepW + (uint32_t)(nx ? kstep - nkb : kstep) * kMxStepBytes), 0,
                        smem + ws * kWStage + w * 4096 + j * 1024);
    };
    // activations of K block kb: `step` its number in the item the descriptor belongs to
    auto load_x = [&](const rsrc_t& r, int j, int step, int xst) {
      uint32_t off = voX[j & 1] + (soX + j * stepX + (uint32_t)step * kMxStepBytes);
      if (RAGGED) {
        const int c = cp ^ (((j & 1) << 2) + (rl >> 1));
        if (step * kMxStepBytes + c * 16 >= row_bytes) off = kOutOfRange;
      }
      buf_load16_to_lds(r, off, 0, smem + kXBase + xst * kXStage + w * 4096 + j * 1024);
    };
    auto LX = [&](int j, int kstep, int xst) {
      const bool nx = kstep >= nkb;
      load_x(nx ? rXs : rX, j, nx ? kstep - nkb : kstep, xst);
    };
    auto wst = [&](int b) -> int { return (gw0 + b) % 3; };
    auto xst = [&](int b) -> int { return (gx0 + b) & 1; };

    // ---- scales: lane l fetches the words of rows l and l + 64 of the wave's 128 weight rows and of row l of its 64 activation rows, both
    // words of a K block; spread_rows hands a word to the lanes of its row, and a byte permute leaves each the two bytes of its chunks
    const int rowsSW = min(128, p.N - n0 - wn * 128), rowsSX = min(64, nrows - m0 - wm * 64);
    const rsrc_t rSW = mx_scale_rsrc(p.sw, n0 + wn * 128, rowsSW, words, p.sw_n, p.sw_w);
    const rsrc_t rSX = mx_scale_rsrc(p.sx, m0 + wm * 64, rowsSX, words, p.sx_m, p.sx_w);
    // a valid row for lanes past the end: in a strided layout the range of the descriptor does not end with the rows
    const uint32_t voSW0 = (uint32_t)(max(min(ln, rowsSW - 1), 0) * p.sw_n * 4), voSW1 = (uint32_t)(max(min(ln + 64, rowsSW - 1), 0) * p.sw_n * 4);
    const uint32_t voSX = (uint32_t)(max(min(ln, rowsSX - 1), 0) * p.sx_m * 4);
    const uint32_t kSW = (uint32_t)(p.sw_w * 4), kSX = (uint32_t)(p.sx_w * 4);
    const uint32_t sel = (uint32_t)(kq | ((4 + kq) << 8));
    uint32_t sqw[2][2], sqx[2], scw[8], scx[4];
    auto request_scales = [&](int b) {
      const uint32_t word = 2 * min(b, nkb - 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t wd = RAGGED ? min(word + j, (uint32_t)words - 1) : word + j;  // a word past the row: multiplied by zero codes
        sqw[0][j] = buf_load4(rSW, voSW0 + wd * kSW);
        sqw[1][j] = buf_load4(rSW, voSW1 + wd * kSW);
        sqx[j] = buf_load4(rSX, voSX + wd * kSX);
      }
    };
    auto take_scales = [&] {
      uint32_t a[4], b[4];
#pragma unroll
      for (int h = 0; h < 3; ++h) {
        spread_rows(h < 2 ? sqw[h][0] : sqx[0], a);
        spread_rows(h < 2 ? sqw[h][1] : sqx[1], b);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t& to = h < 2 ? scw[h * 4 + g] : scx[g];
          to = __builtin_amdgcn_perm(b[g], a[g], sel);
          asm volatile("" : "+v"(to));  // formed here, in front of the next request
        }
      }
    };

    v4f acc[8][4];
#pragma unroll
    for (int ns = 0; ns < 8; ++ns)
#pragma unroll
      for (int ms = 0; ms < 4; ++ms) acc[ns][ms] = v4f{0.f, 0.f, 0.f, 0.f};

    // X[ms]: the activation fragments of a K block; W[ns & 3]: the weight fragments of two pairs of 16-row groups.  A K block is walked as
    // four pairs of 16 products: per weight group the four activation groups with the first chunks, then with the second ones, so
    // that an accumulator is used again four products later.  The weights of a pair are fetched during the pair before, X is refilled
    // behind its last use of a block.
    v4i X[4][2], W[4][2];
    auto RW = [&](const uint8_t* st, int ns) {
      const uint8_t* const g = st + (wn * 128 + ns * 16) * kMxStepBytes;
      W[ns & 3][0] = *reinterpret_cast<const v4i*>(g + fa0);
      W[ns & 3][1] = *reinterpret_cast<const v4i*>(g + fa1);
    };
    auto RX = [&](const uint8_t* st, int ms, int c) {
      X[ms][c] = *reinterpret_cast<const v4i*>(st + (wm * 64 + ms * 16) * kMxStepBytes + (c ? fa1 : fa0));
    };
    auto pair = [&](int pr, auto&& between) {  // between(i) comes behind product i of the pair
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int ns = pr * 2 + (i >> 3), ms = i & 3;
        if ((i >> 2) & 1) acc[ns][ms] = mfma_fp4<1>(W[ns & 3][1], X[ms][1], acc[ns][ms], (int)scw[ns], (int)scx[ms]);
        else acc[ns][ms] = mfma_fp4<0>(W[ns & 3][0], X[ms][0], acc[ns][ms], (int)scw[ns], (int)scx[ms]);
        SB();
        between(i);
        SB();
      }
    };

    if (is_half && wm >= 2) {
      // half tile (always a workgroup's last item): the waves of the upper 128 rows issue their share of the weight loads and keep the
      // barriers; their activation rows are out of range and nobody reads them
      if (!pref) {
#pragma unroll
        for (int j = 0; j < 4; ++j) LW(j, 0, wst(0));
#pragma unroll
        for (int j = 0; j < 4; ++j) LW(j, 1, wst(1));
      }
      wait_vm0();
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) LW(j, 2, wst(2));
      int w_ld = wst(0), w_rd = wst(1);
      for (int it = 0; it < nkb - 1; ++it) {
        lds_barrier<4>();
        SB();
#pragma unroll
        for (int j = 0; j < 4; ++j) LW(j, it + 3, w_ld);
        w_ld = w_rd;
        w_rd = w_rd == 2 ? 0 : w_rd + 1;
      }
      wait_vm0();
      lds_barrier();  // the others' barrier in front of the write-out
      return;
    }
    // ---- prologue: blocks 0 and 1 into their stages, the first three pairs of block 0
    if (!pref) {
#pragma unroll
      for (int j = 0; j < 4; ++j) LX(j, 0, xst(0));
#pragma unroll
      for (int j = 0; j < 4; ++j) LW(j, 0, wst(0));
#pragma unroll
      for (int j = 0; j < 4; ++j) LW(j, 1, wst(1));
    }
    request_scales(0);
    wait_vm0();
    __syncthreads();
    take_scales();
    SB();
#pragma unroll
    for (int j = 0; j < 4; ++j) LX(j, 1, xst(1));
    request_scales(1);
    SB();
#pragma unroll
    for (int j = 0; j < 4; ++j) LW(j, 2, wst(2));
    {
      const uint8_t* const stW = smem + wst(0) * kWStage;
      const uint8_t* const stX = smem + kXBase + xst(0) * kXStage;
      RW(stW, 0); RW(stW, 1);
#pragma unroll
      for (int ms = 0; ms < 4; ++ms) { RX(stX, ms, 0); RX(stX, ms, 1); }
      SB();
#pragma unroll
      for (int pr = 0; pr < 3; ++pr)
        pair(pr, [&](int i) {
          if (i == 2) RW(stW, 2 * pr + 2);
          if (i == 6) RW(stW, 2 * pr + 3);
        });
    }

    int w_ld = wst(0), w_rd = wst(1);  // weight stages: the one block it left (refilled with block it+3), the one of block it+1
    for (int it = 0; it < nkb - 1; ++it) {
      const uint8_t* const stW = smem + w_rd * kWStage;  // block it+1
      const uint8_t* const stX = smem + kXBase + xst(it + 1) * kXStage;
      const int xl = xst(it);                            // activation stage block it left
      lds_barrier<4>();  // block it+1 has landed; the weights of block it+2 may still be on their way
      SB();
      // of the two waves that share a SIMD the one that is behind goes first
      __builtin_amdgcn_s_setprio(3);
      pair(3, [&](int i) {
        if (i == 0) RW(stW, 0);
        if (i == 4) RW(stW, 1);
        if (i < 8 && (i & 1)) LX(i >> 1, it + 2, xl);
        if (i >= 8 && i < 12) RX(stX, i - 8, 0);
        if (i >= 12) RX(stX, i - 12, 1);
      });
      __builtin_amdgcn_s_setprio(2);
      take_scales();
      SB();
      pair(0, [&](int i) {
        if (i == 0) request_scales(it + 2);
        if (i == 2) RW(stW, 2);
        if (i == 6) RW(stW, 3);
        if (i == 4 || i == 8 || i == 12) LW(i / 4 - 1, it + 3, w_ld);
      });
      __builtin_amdgcn_s_setprio(1);
      pair(1, [&](int i) {
        if (i == 0) LW(3, it + 3, w_ld);
        if (i == 2) RW(stW, 4);
        if (i == 6) RW(stW, 5);
      });
      __builtin_amdgcn_s_setprio(0);
      pair(2, [&](int i) {
        if (i == 2) RW(stW, 6);
        if (i == 6) RW(stW, 7);
      });
      w_ld = w_rd;
      w_rd = w_rd == 2 ? 0 : w_rd + 1;
    }
    pair(3, [](int) {});

    // Finished tiles leave through LDS so that every store instruction writes whole 256-byte row segments: each wave re-lays its 64 x 128
    // block out, 32 rows at a time, in an 8 KB slot of the stages of the item's last block, while the others receive the next item.
    const bool wide = (p.ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(p.C) & 15) == 0;
    lds_barrier();
    const int ews = wst(nkb - 1), exs = xst(nkb - 1);
    if (has_next && !stream) {
      SB();
#pragma unroll
      for (int j = 0; j < 4; ++j) load_x(rXn, j, 0, xst(nkb));
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          buf_load16_to_lds(rWn, voW[j & 1] + (soW + j * stepW + (uint32_t)b * kMxStepBytes), 0, smem + wst(nkb + b) * kWStage + w * 4096 + j * 1024);
      SB();
    }

    const auto col_of = [&](int ns) { return n0 + wn * 128 + ns * 16 + kq * 4; };
    // the 16 lanes of a row (equal kq) own the same 32 columns: each fetches the bias of two, which a broadcast along the row hands round
    float biasv[2] = {0.f, 0.f};
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < 2; ++j) biasv[j] = load_scalar<BIAS_DT>(p.bias, min(col_of(j * 4 + (lr >> 2)) + (lr & 3), p.N - 1));
    }
    auto out_pair = [&](auto ns_c, int ms) -> uint2 {
      constexpr int ns = decltype(ns_c)::value;
      v4f v = acc[ns][ms];
      if (p.bias) {
        const float b = biasv[ns >> 2];
        constexpr int l0 = (ns & 3) * 4;
        v[0] += row_broadcast<l0>(b); v[1] += row_broadcast<l0 + 1>(b); v[2] += row_broadcast<l0 + 2>(b); v[3] += row_broadcast<l0 + 3>(b);
      }
      return pack4<OUT_DT>(v[0], v[1], v[2], v[3]);
    };
    if (wide) {
      uint8_t* ep = smem + (w < 4 ? ews * kWStage + w * 8192 : kXBase + exs * kXStage + (w - 4) * 8192);  // 32 rows x 256 B per pass
#pragma unroll
      for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
          static_for<8>([&](auto ns) {
            *reinterpret_cast<uint2*>(ep + (g * 16 + lr) * 256 + (((ns * 2 + (kq >> 1)) ^ lr) << 4) + (kq & 1) * 8) = out_pair(ns, pass * 2 + g);
          });
        __builtin_amdgcn_wave_barrier();  // one wave's LDS accesses complete in order
        const int rr = ln >> 4, pc = ln & 15;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + rr;
          const uint4 o = *reinterpret_cast<const uint4*>(ep + r * 256 + ((pc ^ (r & 15)) << 4));
          const int m = m0 + wm * 64 + pass * 32 + r, n = n0 + wn * 128 + (pc << 3);
          if (m < nrows && n < p.N) *reinterpret_cast<uint4*>((u16*)p.C + (int64_t)m * p.ldc + n) = o;
        }
        __builtin_amdgcn_wave_barrier();
      }
    } else {
#pragma unroll
      for (int ms = 0; ms < 4; ++ms) {
        const int m = m0 + wm * 64 + ms * 16 + lr;
        static_for<8>([&](auto ns) {
          const int n = col_of(ns);
          const uint2 o = out_pair(ns, ms);  // by all lanes: its broadcasts read lanes that store nothing
          if (m < nrows && n < p.N) *reinterpret_cast<uint2*>((u16*)p.C + (int64_t)m * p.ldc + n) = o;
        });
      }
    }
    if (!has_next) {
      wait_vm0();  // requests that moved nothing still point at the stages: let them retire before the LDS goes back
      return;
    }
    item = next;
    pref = true;
    gw0 = wst(nkb);
    gx0 = xst(nkb);
  }
}

}  // namespace fp8k
