// Products of two MXFP4 operands, gfx950: C = A . B^T with both operands' block scales applied by the matrix core
// (v_mfma_scale_f32_16x16x128_f8f6f4), float32 sums, one rounding.
//
// The matrix core sums over K, so the order of a row's blocks inside a line is free as long as both operands agree: lane (row, kq)
// takes the 32 bytes from 32 kq on, two consecutive blocks, whose scale bytes lie next to each other in a scale word.  One 16-bit
// load fetches both, and the instruction's byte select picks the one of its product: no lane exchange, no shifts.
#pragma once

#include "mx_common.h"

namespace fp8k {

// ------------------------------------------------------------------------------------------------
// The weight stream for few activation rows: a workgroup owns 16 * NW weight rows; its 8 waves are NW along n and KS = 8 / NW along
// k.  A wave streams whole 128-byte lines of its weight rows through registers and a 2 KB LDS slot of its own into operand form and
// takes the activation operands straight from memory.  The sums of the K ranges meet in LDS in ascending order.
// ------------------------------------------------------------------------------------------------
template <int MS, int OUT_DT, int BIAS_DT>
__global__ __launch_bounds__(512, 1) void mx_stream_kernel(const MxArgs p) {
  constexpr int D = MS == 4 ? 2 : 4;  // K blocks in flight per wave
  __shared__ __attribute__((aligned(16))) uint8_t wl[8][16 * kMxStepBytes];
  __shared__ __attribute__((aligned(16))) float red[8][MS][64][4];

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r = lane & 15, kq = lane >> 4;
  const int NW = p.nw, nw = w % NW, ks = w / NW;
  const int n0w = (blockIdx.x * NW + nw) * 16, m0 = blockIdx.y * (16 * MS);
  const int row_bytes = p.K >> 1, words = (p.K + 127) >> 7;
  const int kb0 = ks * p.kb_per_wave;
  const int nkb = n0w < p.N ? max(min((p.K + kMxStep - 1) / kMxStep, kb0 + p.kb_per_wave) - kb0, 0) : 0;

  const int rowsW = min(16, p.N - n0w), rowsX = min(16 * MS, p.M - m0);
  const rsrc_t rW = make_rsrc(p.W + (int64_t)n0w * p.ldw, nkb > 0 ? (uint32_t)((rowsW - 1) * p.ldw + row_bytes) : 0u);
  const rsrc_t rX = make_rsrc(p.X + (int64_t)m0 * p.ldx, (uint32_t)((rowsX - 1) * p.ldx + row_bytes));
  const rsrc_t rSW = mx_scale_rsrc(p.sw, n0w, nkb > 0 ? rowsW : 0, words, p.sw_n, p.sw_w);
  const rsrc_t rSX = mx_scale_rsrc(p.sx, m0, rowsX, words, p.sx_m, p.sx_w);

  // load j of a K block: row j*8 + lane/8, chunk lane%8; chunk c of row i sits at position c ^ ((i>>1)&7) in LDS
  const int wrow = lane >> 3, wc = lane & 7;
  const uint32_t voW0 = (uint32_t)(wrow * p.ldw) + wc * 16, voW1 = (uint32_t)((wrow + 8) * p.ldw) + wc * 16;
  uint8_t* const wslot = wl[w];
  const uint32_t wst0 = (uint32_t)(wrow * kMxStepBytes + ((wc ^ ((wrow >> 1) & 7)) << 4));
  const uint32_t wst1 = (uint32_t)((wrow + 8) * kMxStepBytes + ((wc ^ (((wrow + 8) >> 1) & 7)) << 4));
  const uint32_t wrd0 = (uint32_t)(r * kMxStepBytes + (((2 * kq) ^ ((r >> 1) & 7)) << 4)), wrd1 = wrd0 ^ 16u;
  const uint32_t voSW = (uint32_t)((r * p.sw_n + (kq >> 1) * p.sw_w) * 4) + (kq & 1) * 2;
  uint32_t voX[MS], voSX[MS];
#pragma unroll
  for (int ms = 0; ms < MS; ++ms) {
    const int m = ms * 16 + r;
    voX[ms] = m < rowsX ? (uint32_t)(m * p.ldx) + kq * 32 : kOutOfRange;
    voSX[ms] = m < rowsX ? (uint32_t)((m * p.sx_m + (kq >> 1) * p.sx_w) * 4) + (kq & 1) * 2 : kOutOfRange;
  }

  v4i wreg[D][2], xreg[D][MS][2];
  uint32_t sw[D], sx[D][MS];
  auto issue = [&](int slot, int kb) {
    const bool in = kb < nkb;
    const uint32_t ko = (uint32_t)(kb0 + kb) * kMxStepBytes;
    const bool okw = in && (int)ko + wc * 16 < row_bytes;
    wreg[slot][0] = buf_load16_stream(rW, okw ? voW0 + ko : kOutOfRange);
    wreg[slot][1] = buf_load16_stream(rW, okw ? voW1 + ko : kOutOfRange);
    const bool ok0 = in && (int)ko + kq * 32 < row_bytes, ok1 = in && (int)ko + kq * 32 + 16 < row_bytes;
    // words past the last one hold no block of the row; what is read there is multiplied by zero codes, so it must not be a NaN
    const bool oks = in && 2 * (kb0 + kb) + (kq >> 1) < words;
    sw[slot] = buf_load_u16(rSW, oks ? voSW + (uint32_t)((kb0 + kb) * 2 * p.sw_w * 4) : kOutOfRange);
#pragma unroll
    for (int ms = 0; ms < MS; ++ms) {
      const bool row = voX[ms] != kOutOfRange;
      xreg[slot][ms][0] = buf_load16(rX, ok0 && row ? voX[ms] + ko : kOutOfRange);
      xreg[slot][ms][1] = buf_load16(rX, ok1 && row ? voX[ms] + ko + 16 : kOutOfRange);
      sx[slot][ms] = buf_load_u16(rSX, oks && row ? voSX[ms] + (uint32_t)((kb0 + kb) * 2 * p.sx_w * 4) : kOutOfRange);
    }
  };

  v4f acc[MS];
#pragma unroll
  for (int ms = 0; ms < MS; ++ms) acc[ms] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D; ++d) issue(d, d);
  for (int k0 = 0; k0 < nkb; k0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      *reinterpret_cast<v4i*>(wslot + wst0) = wreg[d][0];
      *reinterpret_cast<v4i*>(wslot + wst1) = wreg[d][1];
      const v4i a0 = *reinterpret_cast<const v4i*>(wslot + wrd0), a1 = *reinterpret_cast<const v4i*>(wslot + wrd1);
#pragma unroll
      for (int ms = 0; ms < MS; ++ms) {
        acc[ms] = mfma_fp4<0>(a0, xreg[d][ms][0], acc[ms], (int)sw[d], (int)sx[d][ms]);
        acc[ms] = mfma_fp4<1>(a1, xreg[d][ms][1], acc[ms], (int)sw[d], (int)sx[d][ms]);
      }
      issue(d, k0 + d + D);
    }
  }

#pragma unroll
  for (int ms = 0; ms < MS; ++ms) *reinterpret_cast<v4f*>(red[w][ms][lane]) = acc[ms];
  __syncthreads();
  if (ks != 0) return;
  const int n = n0w + kq * 4, KS = 8 / NW;
  if (n >= p.N) return;
#pragma unroll
  for (int ms = 0; ms < MS; ++ms) {
    const int m = m0 + ms * 16 + r;
    if (m >= p.M) continue;
    v4f s = acc[ms];
    for (int k = 1; k < KS; ++k) {
      const v4f o = *reinterpret_cast<const v4f*>(red[k * NW + nw][ms][lane]);
      s[0] += o[0]; s[1] += o[1]; s[2] += o[2]; s[3] += o[3];
    }
    float v[4] = {s[0], s[1], s[2], s[3]};
    if (p.bias) {
      float b[4];
      load_bias4<BIAS_DT>(p.bias, n, b);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += b[i];
    }
    store4<OUT_DT>(p.C, (int64_t)m * p.ldc + n, v[0], v[1], v[2], v[3]);
  }
}

}  // namespace fp8k
