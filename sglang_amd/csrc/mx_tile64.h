// 64(n) x 64(m) tiles of the MXFP4 product, gfx950: batches whose larger tiles leave most of the chip idle.
//
// The structure is gemm_tile64_kernel's: one workgroup of four waves per tile, each on every fourth K block (a 128-byte line of every
// row, 256 values) of the whole tile, its loads going to two LDS slots that nobody else touches; no barrier stands in the K loop, and
// the four sums meet in LDS at the end, in ascending order.  A block is 32 products of 16x16x128 for 16 KB of operands.  Bound: the one
// wave of a SIMD.  128 x 7168 x 16384: 16.5 us (224 tiles, 62 MB of weights; 10.2 at 6.4 TB/s), in which a wave issues in 46 % of its clocks,
// waits for an issue slot in 31 % and for memory in 23 %; the matrix cores are 24 % busy.
// 64 x 4608 x 7168 takes 10.1.  Eight waves with one slot each were no faster: there 10.1 -> 10.2 us, with 1 GB of weights in turn 18.2 ->
// 19.7, 64 x 64 x 16384 12.3 -> 14.0.
//
// Scales: one load each of the two words of a block for 64 weight rows and 64 activation rows (lane = row), handed to the lanes of a row
// by lane swaps, a byte permute picking those of the lane's chunks kq and 4 + kq.
//
// RAGGED: K is no multiple of 256; chunks of the activations past the end of a row arrive as zeros.
#pragma once

#include "gemm_tile64.h"
#include "mx_common.h"

namespace fp8k {

template <int OUT_DT, int BIAS_DT, bool RAGGED>
__global__ __launch_bounds__(512) void mx_tile64_kernel(const MxArgs p) {  // 256 threads; the bound keeps it within 256 registers
  constexpr int kOps = 64 * kMxStepBytes;
  constexpr int kSlot = 2 * kOps;  // weights, then activations
  constexpr int kWave = 2 * kSlot;
  constexpr uint32_t kPast = 0x80000000u;  // past every descriptor's range (64 rows of less than 8 MiB), and so with any offset added
  constexpr int kScaleLoads = 4;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * kWave];

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  int t;
  {  // each XCD (workgroup id mod 8) walks a contiguous run of the tiles
    const int total = p.tiles_m * p.tiles_n, per_xcd = (total + 7) >> 3;
    t = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per_xcd || t >= total) return;
  }
  int tile_m, tile_n;
  tile_coords(t, p.tiles_m, p.tiles_n, tile_m, tile_n);
  const int m0 = tile_m * 64, n0 = tile_n * 64;
  const int row_bytes = p.K >> 1, words = (p.K + 127) >> 7, nkb = (p.K + kMxStep - 1) / kMxStep;

  const int rowsW = min(64, p.N - n0), rowsX = min(64, p.M - m0);
  const rsrc_t rW = make_rsrc(p.W + (int64_t)n0 * p.ldw, (uint32_t)((rowsW - 1) * p.ldw + row_bytes));
  const rsrc_t rX = make_rsrc(p.X + (int64_t)m0 * p.ldx, (uint32_t)((rowsX - 1) * p.ldx + row_bytes));
  uint8_t* const own = smem + w * kWave;
  const int rl = lane >> 3, cp = lane & 7;
  uint32_t voW[2], voX[2];
  int xc[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // chunk c of row r at position c ^ ((r >> 1) & 7)
    const int c = cp ^ ((j << 2) + (rl >> 1));
    voW[j] = (uint32_t)((j * 8 + rl) * p.ldw + c * 16);
    voX[j] = (uint32_t)((j * 8 + rl) * p.ldx + c * 16);
    xc[j] = c * 16;
  }
  const uint32_t stW = (uint32_t)(16 * p.ldw), stX = (uint32_t)(16 * p.ldx);
  auto load = [&](uint8_t* slot, int kb, int g) {  // load g of block kb's sixteen: weights, then activations
    const uint32_t ko = kb < nkb ? (uint32_t)kb * kMxStepBytes : kPast;
    if (g < 8) {
      buf_load16_to_lds(rW, voW[g & 1] + (ko + (g >> 1) * stW), 0, slot + g * 1024);
    } else {
      uint32_t off = voX[g & 1] + (ko + ((g - 8) >> 1) * stX);
      if (RAGGED && kb * kMxStepBytes + xc[g & 1] >= row_bytes) off = kPast;
      buf_load16_to_lds(rX, off, 0, slot + g * 1024);
    }
  };
  const int lr = lane & 15, kq = lane >> 4;
  const uint32_t fa0 = (uint32_t)(lr * kMxStepBytes + ((kq ^ ((lr >> 1) & 7)) << 4)), fa1 = fa0 ^ 64u;

  const rsrc_t rSW = mx_scale_rsrc(p.sw, n0, rowsW, words, p.sw_n, p.sw_w), rSX = mx_scale_rsrc(p.sx, m0, rowsX, words, p.sx_m, p.sx_w);
  const uint32_t voSW = (uint32_t)(min(lane, rowsW - 1) * p.sw_n * 4), voSX = (uint32_t)(min(lane, rowsX - 1) * p.sx_m * 4);
  const uint32_t kSW = (uint32_t)(p.sw_w * 4), kSX = (uint32_t)(p.sx_w * 4), sel = (uint32_t)(kq | ((4 + kq) << 8));
  struct Scales { uint32_t w[2], x[2]; } sa, sb;
  auto load_scales = [&](Scales& c, int kb) {
    const uint32_t word = 2 * min(kb, nkb - 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t wd = RAGGED ? min(word + j, (uint32_t)words - 1) : word + j;
      c.w[j] = buf_load4(rSW, voSW + wd * kSW);
      c.x[j] = buf_load4(rSX, voSX + wd * kSX);
    }
  };

  v4f acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  v4i W[4][2], X[4][2];
  auto read_w = [&](const uint8_t* slot, int i) {
    W[i][0] = *reinterpret_cast<const v4i*>(slot + i * 2048 + fa0);
    W[i][1] = *reinterpret_cast<const v4i*>(slot + i * 2048 + fa1);
  };
  auto read_x = [&](const uint8_t* slot, int i, int c) { X[i][c] = *reinterpret_cast<const v4i*>(slot + kOps + i * 2048 + (c ? fa1 : fa0)); };
  // The products of block kb, whose operands are in W and X.  Its slot takes block kb + 8, the operand registers, as they fall free, block
  // kb + 4 out of the other one.
  auto trip = [&](uint8_t* slot, const uint8_t* other, Scales& c, int kb) {
    uint32_t s[2][4], a[4], b[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      spread_rows(h ? c.x[0] : c.w[0], a);
      spread_rows(h ? c.x[1] : c.w[1], b);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        s[h][g] = __builtin_amdgcn_perm(b[g], a[g], sel);
        asm volatile("" : "+v"(s[h][g]));
      }
    }
    SB();
    load_scales(c, kb + 8);
    SB();
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const int ns = k >> 3, ms = k & 3;
      if ((k >> 2) & 1) acc[ns][ms] = mfma_fp4<1>(W[ns][1], X[ms][1], acc[ns][ms], (int)s[0][ns], (int)s[1][ms]);
      else acc[ns][ms] = mfma_fp4<0>(W[ns][0], X[ms][0], acc[ns][ms], (int)s[0][ns], (int)s[1][ms]);
      SB();
      if (k == 3) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every operand is out of its slot
      if (k >= 3 && k < 19) load(slot, kb + 8, k - 3);
      SB();
      if (k == 18) wait_vm<kScaleLoads + 16>();  // block kb + 4 has landed: younger are this trip's requests
      if (k == 19) read_w(other, 0);
      if (k == 20) read_w(other, 1);
      if (k == 23) read_w(other, 2);
      if (k >= 24) read_x(other, k & 3, (k >> 2) & 1);
      if (k == 31) read_w(other, 3);
      SB();
    }
  };
  // ---- wave w works on K blocks w, w + 4, ..
  load_scales(sa, w);
  SB();
#pragma unroll
  for (int g = 0; g < 16; ++g) load(own, w, g);
  SB();
  load_scales(sb, w + 4);
  SB();
#pragma unroll
  for (int g = 0; g < 16; ++g) load(own + kSlot, w + 4, g);
  SB();
  wait_vm<kScaleLoads + 16>();
#pragma unroll
  for (int i = 0; i < 4; ++i) { read_x(own, i, 0); read_x(own, i, 1); read_w(own, i); }
  SB();
  for (int kb = w; kb < nkb; kb += 8) {
    trip(own, own + kSlot, sa, kb);
    if (kb + 4 < nkb) trip(own + kSlot, own, sb, kb + 4);
  }
  wait_vm0_lgkm0();  // requests past the last block must not land on the sums

  // ---- the K shares meet in LDS: [wave][row 64][16-byte chunk c at c ^ (row & 15)]
  asm volatile("" ::: "memory");
#pragma unroll
  for (int ms = 0; ms < 4; ++ms)
#pragma unroll
    for (int ns = 0; ns < 4; ++ns) *reinterpret_cast<v4f*>(own + (ms * 16 + lr) * 256 + (((ns * 4 + kq) ^ lr) << 4)) = acc[ns][ms];
  __syncthreads();
  // wave w finishes rows 16 w .. 16 w + 15, eight at a time: lane -> row lane / 8, eight columns
  const int pc = lane & 7, n = n0 + pc * 8;
  const bool wide = (p.ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(p.C) & 15) == 0;
  float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (p.bias && n < p.N) load_bias8<BIAS_DT>(p.bias, n, bias);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = w * 16 + half * 8 + (lane >> 3), m = m0 + row;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint8_t* const q = smem + k * kWave + row * 256;
      const v4f lo = *reinterpret_cast<const v4f*>(q + (((2 * pc) ^ (row & 15)) << 4));
      const v4f hi = *reinterpret_cast<const v4f*>(q + (((2 * pc + 1) ^ (row & 15)) << 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] += lo[i]; v[4 + i] += hi[i]; }
    }
    if (m >= p.M || n >= p.N) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += bias[i];
    u16* const o = (u16*)p.C + (int64_t)m * p.ldc + n;
    const uint2 ol = pack4<OUT_DT>(v[0], v[1], v[2], v[3]), oh = pack4<OUT_DT>(v[4], v[5], v[6], v[7]);
    if (wide) {
      *reinterpret_cast<uint4*>(o) = make_uint4(ol.x, ol.y, oh.x, oh.y);
    } else {
      *reinterpret_cast<uint2*>(o) = ol;
      *reinterpret_cast<uint2*>(o + 4) = oh;
    }
  }
}

}  // namespace fp8k
