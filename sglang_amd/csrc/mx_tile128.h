// 128(n) x TM(m) tiles of the MXFP4 product, TM = 128 or 64, gfx950: products between the weight stream and the 256x256 tiles.
//
// The structure is gemm_tile128_kernel's: 8 wavefronts, 2 along n x 4 along m (64 x 32 each) or 4 x 2 (32 x 32), five LDS stages of a K
// block (a 128-byte line of every row, 256 values), one barrier per block that waits for loads only, operands of block `it` fetched
// into one register set while the products of block it-1 are issued from the other.  What bounds it is the chain of a block - barrier,
// LDS, issue - more than any unit's throughput: 0.385 us a block with 64 activation rows and 0.62 with 128, for 0.17 and 0.34 us of the
// matrix cores.  256 x 7168 x 7168: 13.5 us with 64 (64x64 tiles 15.3, 256x256 29), 512 x 4096 x 4096 9.9 (14.7, 20).
//
// The scales of a block travel with its operands, three blocks ahead in registers: one load for the 32 activation rows (lanes 0 .. 31 the
// first word, the others the second) and one or two for the weight rows; lane swaps hand them to the lanes of their rows and a byte
// permute picks those of the lane's chunks kq and 4 + kq.
//
// RAGGED: K is no multiple of 256; chunks of the activations past the end of a row arrive as zeros.
#pragma once

#include "mx_common.h"

namespace fp8k {

template <int OUT_DT, int BIAS_DT, int TM, bool RAGGED>
__global__ __launch_bounds__(512, 1) void mx_tile128_kernel(const MxArgs p) {
  static_assert(TM == 64 || TM == 128, "activation rows of a tile");
  constexpr int NST = 5, kStage = (128 + TM) * kMxStepBytes, kXOff = 128 * kMxStepBytes;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NST * kStage];
  constexpr int NWN = TM == 128 ? 2 : 4, NT = 128 / NWN / 16, MT = 2, NP = NT * MT * 2;  // waves along n, groups of a wave, products of a block
  constexpr int WS = NT / 2;                         // weight scale loads of a block
  constexpr int XL = TM / 64, LPB = 2 + XL, SL = WS + 1;  // loads of a wave per block: operands, scales

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wn = w % NWN, wm = w / NWN;
  const int wrow = wn * (NT * 16), xrow = wm * 32;

  int t;
  {  // each XCD (workgroup id mod 8) walks a contiguous run of the tiles
    const int total = p.tiles_m * p.tiles_n, per_xcd = (total + 7) >> 3;
    t = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per_xcd || t >= total) return;
  }
  int tile_m, tile_n;
  tile_coords(t, p.tiles_m, p.tiles_n, tile_m, tile_n);
  const int m0 = tile_m * TM, n0 = tile_n * 128;
  const int row_bytes = p.K >> 1, words = (p.K + 127) >> 7, nkb = (p.K + kMxStep - 1) / kMxStep;

  // ---- global -> LDS: wave w brings rows [16w, 16w+16) of W and [8 XL w, 8 XL (w+1)) of X, 1 KB (8 rows) a load
  const int rowsW = min(128, p.N - n0), rowsX = min(TM, p.M - m0);
  const rsrc_t rW = make_rsrc(p.W + (int64_t)n0 * p.ldw, (uint32_t)((rowsW - 1) * p.ldw + row_bytes));
  const rsrc_t rX = make_rsrc(p.X + (int64_t)m0 * p.ldx, (uint32_t)((rowsX - 1) * p.ldx + row_bytes));
  const int rl = lane >> 3, cp = lane & 7;
  uint32_t voW[2], voX[XL];
  int xc[XL];
#pragma unroll
  for (int j = 0; j < 2; ++j) voW[j] = (uint32_t)((w * 16 + j * 8 + rl) * p.ldw + (cp ^ ((j << 2) + (rl >> 1))) * 16);
#pragma unroll
  for (int j = 0; j < XL; ++j) {  // chunk c of row r at position c ^ ((r >> 1) & 7)
    const int r = (w * XL + j) * 8 + rl;
    xc[j] = (cp ^ ((r >> 1) & 7)) * 16;
    voX[j] = (uint32_t)(r * p.ldx + xc[j]);
  }
  auto load_block = [&](int stage, int kb, int j) {  // j: 0, 1 weights; 2 .. LPB-1 activations
    const uint32_t ko = (uint32_t)kb * kMxStepBytes;
    if (j < 2) {
      buf_load16_to_lds(rW, voW[j] + ko, 0, smem + stage + w * 2048 + j * 1024);
    } else {
      const bool ok = !RAGGED || (int)ko + xc[j - 2] < row_bytes;
      buf_load16_to_lds(rX, ok ? voX[j - 2] + ko : kOutOfRange, 0, smem + stage + kXOff + (w * XL + j - 2) * 1024);
    }
  };

  const int lr = lane & 15, kq = lane >> 4;
  const uint32_t fa0 = (uint32_t)(lr * kMxStepBytes + ((kq ^ ((lr >> 1) & 7)) << 4)), fa1 = fa0 ^ 64u;

  // ---- scales.  64 weight rows of a wave: lane = row, a load for each word.  32 rows: lane % 32 = row, lane / 32 = word.
  const rsrc_t rSW = mx_scale_rsrc(p.sw, n0 + wrow, min(NT * 16, p.N - n0 - wrow), words, p.sw_n, p.sw_w);
  const rsrc_t rSX = mx_scale_rsrc(p.sx, m0 + xrow, min(32, p.M - m0 - xrow), words, p.sx_m, p.sx_w);
  const int h = lane >> 5;
  const uint32_t voSW = (uint32_t)(max(min(NT == 4 ? lane : lane & 31, p.N - n0 - wrow - 1), 0) * p.sw_n * 4);
  const uint32_t voSX = (uint32_t)(max(min(lane & 31, p.M - m0 - xrow - 1), 0) * p.sx_m * 4);
  const uint32_t kSW = (uint32_t)(p.sw_w * 4), kSX = (uint32_t)(p.sx_w * 4), sel = (uint32_t)(kq | ((4 + kq) << 8));
  struct Scales { uint32_t w[WS], x; };
  Scales ring[4];  // of block b in ring[b % 4]
  auto request_scales = [&](Scales& c, int kb) {
    const int word = 2 * min(kb, nkb - 1);
#pragma unroll
    for (int j = 0; j < WS; ++j) c.w[j] = buf_load4(rSW, voSW + (uint32_t)min(word + (WS == 2 ? j : h), words - 1) * kSW);
    c.x = buf_load4(rSX, voSX + (uint32_t)min(word + h, words - 1) * kSX);
  };
  uint32_t sw[NT], sx[MT];
  auto take_scales = [&](const Scales& c) {
    uint32_t a[4], b[4];
    spread_rows(c.x, a);  // groups 0, 1 of the first word, then of the second
#pragma unroll
    for (int g = 0; g < MT; ++g) { sx[g] = __builtin_amdgcn_perm(a[2 + g], a[g], sel); asm volatile("" : "+v"(sx[g])); }
    spread_rows(c.w[0], a);
    if (WS == 2) spread_rows(c.w[WS - 1], b);
#pragma unroll
    for (int g = 0; g < NT; ++g) { sw[g] = __builtin_amdgcn_perm(WS == 2 ? b[g] : a[2 + g], a[g], sel); asm volatile("" : "+v"(sw[g])); }
  };

  v4f acc[NT][MT];
#pragma unroll
  for (int ns = 0; ns < NT; ++ns)
#pragma unroll
    for (int ms = 0; ms < MT; ++ms) acc[ns][ms] = v4f{0.f, 0.f, 0.f, 0.f};

  struct Operands { v4i W[NT][2], X[MT][2]; };  // of one K block
  Operands oa, ob;
  // the products of a block; between(k) comes behind product k.  An accumulator is used again four products later.
  auto compute = [&](const Operands& o, auto&& between) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int ns = (k >> 3) * 2 + ((k >> 1) & 1), ms = k & 1;
      if ((k >> 2) & 1) acc[ns][ms] = mfma_fp4<1>(o.W[ns][1], o.X[ms][1], acc[ns][ms], (int)sw[ns], (int)sx[ms]);
      else acc[ns][ms] = mfma_fp4<0>(o.W[ns][0], o.X[ms][0], acc[ns][ms], (int)sw[ns], (int)sx[ms]);
      SB();
      between(k);
      SB();
    }
  };
  // fragment f of a block: the activation groups' halves, then the weight groups'
  auto read_frag = [&](Operands& o, const uint8_t* st, int f) {
    const int c = f & 1, g = f >> 1;
    const uint32_t at = c ? fa1 : fa0;
    if (g < MT) o.X[g][c] = *reinterpret_cast<const v4i*>(st + kXOff + (xrow + g * 16) * kMxStepBytes + at);
    else o.W[g - MT][c] = *reinterpret_cast<const v4i*>(st + (wrow + (g - MT) * 16) * kMxStepBytes + at);
  };
  constexpr int NF = 2 * (MT + NT), FPP = (NF + NP / 2 - 1) / (NP / 2);  // fragments of a block; fetched behind one product
  int st_rd = 0, st_fill = (NST - 2) * kStage;  // stage of block `it`, stage that block it + NST - 2 goes to
  auto next = [&](int st) { return st == (NST - 1) * kStage ? 0 : st + kStage; };
  // trip `it` (u = it % 4): block `it` has landed everywhere; its operands from LDS into `rd`, the products of block it-1 from `use`, and the
  // loads of block it + 3 into the stage of block it-2, whose operands every wave has used by now.  The trips behind the loop (u = 1 .. 3)
  // request nothing and count the operand loads alone: a request whose result is never used is dropped by the compiler, and a wait that
  // counted it would let a block's own loads pass.
  auto trip = [&](auto u_c, auto tail_c, int it, Operands& rd, const Operands& use) {
    constexpr int u = decltype(u_c)::value;
    constexpr bool tail = decltype(tail_c)::value;
    const uint8_t* const st = smem + st_rd;
    const int kf = it + NST - 2, fill = st_fill;
    SB();
    vm_barrier<tail ? (NST - 2 - u) * LPB : (NST - 3) * (LPB + SL)>();  // younger than block it's loads: those of the two blocks behind it
    take_scales(ring[(u + 3) & 3]);
    SB();
    if (!tail) request_scales(ring[(u + 3) & 3], kf);  // kf % 4 == (it - 1) % 4
    SB();
    compute(use, [&](int i) {
#pragma unroll
      for (int f = 0; f < FPP; ++f)
        if (i * FPP + f < NF) read_frag(rd, st, i * FPP + f);
      if (!tail && i >= NP / 2 && i - NP / 2 < LPB) load_block(fill, kf, i - NP / 2);
    });
    st_rd = next(st_rd);
    st_fill = next(st_fill);
  };
  const std::false_type loop{};
  const std::true_type tail{};
  const std::integral_constant<int, 0> c0{};
  const std::integral_constant<int, 1> c1{};
  const std::integral_constant<int, 2> c2{};
  const std::integral_constant<int, 3> c3{};

  // ---- prologue: blocks 0 .. 2 and one more into their stages, block 0's operands into `oa`
#pragma unroll
  for (int s = 0; s < NST - 2; ++s) {
    request_scales(ring[s], s);
    SB();
#pragma unroll
    for (int j = 0; j < LPB; ++j) load_block(s * kStage, s, j);
    SB();
  }
  vm_barrier<(NST - 3) * (LPB + SL)>();
  request_scales(ring[NST - 2], NST - 2);
  SB();
#pragma unroll
  for (int j = 0; j < LPB; ++j) load_block((NST - 2) * kStage, NST - 2, j);
#pragma unroll
  for (int f = 0; f < NF; ++f) read_frag(oa, smem, f);
  st_rd = kStage;
  st_fill = (NST - 1) * kStage;
  // ---- block b is fetched in trip b and multiplied in trip b+1; even blocks live in `oa`, odd ones in `ob`
  auto nothing = [](int) {};
  int it = 1;
  for (; it + 3 < nkb; it += 4) {
    trip(c1, loop, it, ob, oa);
    trip(c2, loop, it + 1, oa, ob);
    trip(c3, loop, it + 2, ob, oa);
    trip(c0, loop, it + 3, oa, ob);
  }
  if (it >= nkb) {
    take_scales(ring[0]);
    compute(oa, nothing);
  } else {
    trip(c1, tail, it, ob, oa);
    if (it + 1 >= nkb) {
      take_scales(ring[1]);
      compute(ob, nothing);
    } else {
      trip(c2, tail, it + 1, oa, ob);
      if (it + 2 >= nkb) {
        take_scales(ring[2]);
        compute(oa, nothing);
      } else {
        trip(c3, tail, it + 2, ob, oa);
        take_scales(ring[3]);
        compute(ob, nothing);
      }
    }
  }

  const auto col_of = [&](int ns) { return n0 + wrow + ns * 16 + kq * 4; };
  if (p.bias) {
    float b[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) load_bias4<BIAS_DT>(p.bias, min(col_of(j), p.N - 4), b[j]);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int ms = 0; ms < MT; ++ms)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[j][ms][q] += b[j][q];
  }
  auto out_quad = [&](int ns, int ms) -> uint2 { return pack4<OUT_DT>(acc[ns][ms][0], acc[ns][ms][1], acc[ns][ms][2], acc[ns][ms][3]); };

  // Finished tiles leave through LDS so that a store instruction writes whole 128- or 64-byte row segments: each wave re-lays its 32 rows
  // out in a private slot, 16-byte chunks XOR-swizzled by the row.
  const bool wide = (p.ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(p.C) & 15) == 0;
  if (wide) {
    wait_vm0_lgkm0();                // own stray loads have landed ...
    __builtin_amdgcn_s_barrier();    // ... and so have everyone's; every wave has taken its last operands
    asm volatile("" ::: "memory");
    constexpr int CPR = NT * 2, RPI = 64 / CPR;  // 16-byte chunks of a row, rows per store instruction
    const int rr = lane / CPR, pc = lane % CPR;
    uint8_t* const ep = smem + w * (32 * CPR * 16);
#pragma unroll
    for (int ms = 0; ms < MT; ++ms)
#pragma unroll
      for (int ns = 0; ns < NT; ++ns)
        *reinterpret_cast<uint2*>(ep + (ms * 16 + lr) * (CPR * 16) + (((ns * 2 + (kq >> 1)) ^ (lr & (CPR - 1))) << 4) + (kq & 1) * 8) = out_quad(ns, ms);
    __builtin_amdgcn_wave_barrier();  // one wave's LDS accesses complete in order
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int r = i * RPI + rr;
      const uint4 o = *reinterpret_cast<const uint4*>(ep + r * (CPR * 16) + ((pc ^ (r & (CPR - 1))) << 4));
      const int m = m0 + xrow + r, n = n0 + wrow + (pc << 3);
      if (m < p.M && n < p.N) *reinterpret_cast<uint4*>((u16*)p.C + (int64_t)m * p.ldc + n) = o;
    }
    return;
  }
  wait_vm0();
#pragma unroll
  for (int ms = 0; ms < MT; ++ms)
#pragma unroll
    for (int ns = 0; ns < NT; ++ns) {
      const int m = m0 + xrow + ms * 16 + lr, n = col_of(ns);
      if (m < p.M && n < p.N) *reinterpret_cast<uint2*>((u16*)p.C + (int64_t)m * p.ldc + n) = out_quad(ns, ms);
    }
}

}  // namespace fp8k
