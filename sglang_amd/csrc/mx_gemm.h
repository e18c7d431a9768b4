// Products of two MXFP4 operands for few activation rows, gfx950: C = A . B^T with both operands' block scales applied by the matrix core
// (v_mfma_scale_f32_16x16x128_f8f6f4), float32 sums, one rounding.  Decode linears with the quantisation inside.
//
// The matrix core sums over K, so the order of a row's blocks inside a line is free as long as both operands agree: lane (row, kq)
// takes the 32 bytes from 32 kq on, two consecutive blocks, whose scale bytes lie next to each other in a scale word.  One 16-bit
// load fetches both, and the instruction's byte select picks the one of its product: no lane exchange, no shifts.
#pragma once

#include "gemm_tile64.h"
#include "mx_common.h"

namespace fp8k {

// what a workgroup quantises for itself: at most kMxFuse elements whose codes and scale bytes fit these two areas, with which two
// workgroups of strips up to 32 rows share a CU
constexpr int kMxFuse = 28672, kMxFuseRows = 15424, kMxFuseScales = 960;
__host__ __device__ constexpr int mx_fuse_stride(int kbs) { return kbs * kMxStepBytes + 16; }  // the rows of an operand fall into different banks

// ------------------------------------------------------------------------------------------------
// A workgroup owns a strip of 16 NS weight rows over all of K; its 8 waves take every eighth K block (a 128-byte line of every row) each,
// for all 16 MS activation rows.  A wave's loads go straight to LDS slots of its own, whole lines, ST blocks ahead; no barrier stands in
// the K loop.  The eight sums meet in LDS at the end, in ascending order.
//
// FUSE (MS = 1): x holds 16-bit activations, at most kMxFuse of them.  Every workgroup quantises all of them for itself while its first
// weight lines travel - mx_quant_kernel's arithmetic - and keeps codes and scales in LDS.
//
// Bound: weight bytes out of HBM; for the smallest, launch and first-load latency: 1 x 4608 x 7168 with the quantisation 5.3 - 6.4 us for
// 17.5 MB (2.7 at 6.4 TB/s), 32 x 4096 x 4096 4.0 - 4.4, 24 x 7168 x 18432 23 (11.0).
// RAGGED: K is no multiple of 256; the activations are zero past the end of a row, what the weights have there does not matter.
// ------------------------------------------------------------------------------------------------
constexpr int mx_strip_slots(int ms, int ns, bool fuse) { return fuse ? (ns == 1 ? 4 : 2) : (ms == 1 && ns == 1 ? 4 : 2); }

template <int MS, int NS, bool FUSE, int OUT_DT, int BIAS_DT, bool RAGGED>
__global__ __launch_bounds__(512, 4) void mx_strip_kernel(const MxArgs p) {
  static_assert(!FUSE || MS == 1, "a few rows only");
  constexpr int XG = FUSE ? 0 : MS, ST = mx_strip_slots(MS, NS, FUSE);
  constexpr int kSlot = (NS + XG) * 2048, kWave = ST * kSlot;
  constexpr int kLoads = 3 * (NS + XG);  // of a wave per K block: two for the codes of 16 rows, one for their scales
  static_assert(kWave >= MS * NS * 1024, "the sums of a wave take the place of its slots");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[8 * kWave];
  __shared__ __attribute__((aligned(16))) uint8_t xs[FUSE ? kMxFuseRows : 16];
  __shared__ __attribute__((aligned(16))) uint8_t xsc[FUSE ? kMxFuseScales : 16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * (16 * NS), m0 = blockIdx.y * (16 * MS);
  const int row_bytes = p.K >> 1, words = (p.K + 127) >> 7, nkb = (p.K + kMxStep - 1) / kMxStep;
  const int rowsW = min(16 * NS, p.N - n0), rowsX = min(16 * MS, p.M - m0);

  // ---- FUSE: the 16-bit activations are requested first; piece q is 8 elements, four pieces a block
  constexpr int P = (kMxFuse / 8 + 511) / 512;
  const int per_row = p.K >> 3, pieces = p.M * per_row;
  const float inv = 1.0f / (float)per_row;
  Raw8<OUT_DT> raw[FUSE ? P : 1];
  auto row_of = [&](int q) { return (int)(((float)q + 0.5f) * inv); };  // q / per_row, exact: q < 2^12
  if (FUSE) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (j * 512 + w * 64 >= pieces) break;
      const int q = min(j * 512 + tid, pieces - 1), m = row_of(q);
      raw[j].load(p.X, (int64_t)m * p.ldx + (q - m * per_row) * 8);
    }
    SB();
  }

  const rsrc_t rW = make_rsrc(p.W + (int64_t)n0 * p.ldw, (uint32_t)((rowsW - 1) * p.ldw + row_bytes));
  const rsrc_t rX = FUSE ? rW : make_rsrc(p.X + (int64_t)m0 * p.ldx, (uint32_t)((rowsX - 1) * p.ldx + row_bytes));
  const rsrc_t rSW = mx_scale_rsrc(p.sw, n0, rowsW, words, p.sw_n, p.sw_w);
  const rsrc_t rSX = FUSE ? rSW : mx_scale_rsrc(p.sx, m0, rowsX, words, p.sx_m, p.sx_w);
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
  uint32_t voSW[NS], voSX[XG + 1];  // a valid row for lanes past the end: a strided layout does not end the descriptor's range with the rows
  const int wd = kq >> 1;
#pragma unroll
  for (int g = 0; g < NS; ++g) voSW[g] = (uint32_t)(min(g * 16 + lr, rowsW - 1) * p.sw_n * 4) + (kq & 1) * 2;
#pragma unroll
  for (int g = 0; g < XG; ++g) voSX[g] = (uint32_t)(min(g * 16 + lr, rowsX - 1) * p.sx_m * 4) + (kq & 1) * 2;
  uint8_t* const own = smem + w * kWave;
  uint32_t sw[ST][NS], sx[ST][XG + 1];
  auto request = [&](int slot, int kb) {
    const uint32_t ko = (uint32_t)kb * kMxStepBytes, word = (uint32_t)min(2 * kb + wd, words - 1);
#pragma unroll
    for (int g = 0; g < NS; ++g) sw[slot][g] = buf_load_u16(rSW, voSW[g] + word * (uint32_t)(p.sw_w * 4));
#pragma unroll
    for (int g = 0; g < XG; ++g) sx[slot][g] = buf_load_u16(rSX, voSX[g] + word * (uint32_t)(p.sx_w * 4));
    SB();
#pragma unroll
    for (int g = 0; g < 2 * NS; ++g) buf_load16_to_lds<true>(rW, voW[g & 1] + (ko + (g >> 1) * stW), 0, own + slot * kSlot + g * 1024);
#pragma unroll
    for (int g = 0; g < 2 * XG; ++g) {
      const bool ok = !RAGGED || (int)ko + xc[g & 1] < row_bytes;
      buf_load16_to_lds(rX, ok ? voX[g & 1] + (ko + (g >> 1) * stX) : kOutOfRange, 0, own + slot * kSlot + (2 * NS + g) * 1024);
    }
    SB();
  };
#pragma unroll
  for (int s = 0; s < ST; ++s)
    if (w + 8 * s < nkb) request(s, w + 8 * s);

  const int xstride = mx_fuse_stride(nkb), sstride = nkb * 8;
  if (FUSE) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (j * 512 + w * 64 >= pieces) break;
      const int q = j * 512 + tid;
      const int m = row_of(min(q, pieces - 1)), c = q - m * per_row;
      float v[8];
      raw[j].unpack(v);
      uint32_t byte;
      const uint32_t codes = mx_quant8(v, byte);
      if (q < pieces) {
        *reinterpret_cast<uint32_t*>(xs + m * xstride + c * 4) = codes;
        if ((c & 3) == 0) xsc[m * sstride + (c >> 2)] = (uint8_t)byte;
      }
    }
    if (RAGGED) {  // zeros behind the rows
      const int rest = nkb * 32 - per_row;  // 4-byte pieces, at most 28
      for (int i = tid; i < p.M * rest; i += 512) {
        const int m = i / rest, c = per_row + i - m * rest;
        *reinterpret_cast<uint32_t*>(xs + m * xstride + c * 4) = 0;
        if ((c & 3) == 0) xsc[m * sstride + (c >> 2)] = 0;
      }
    }
    lds_barrier();  // the weight loads stay in flight
  }

  // ---- K loop
  v4f acc[NS][MS];
#pragma unroll
  for (int ns = 0; ns < NS; ++ns)
#pragma unroll
    for (int ms = 0; ms < MS; ++ms) acc[ns][ms] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint32_t fa0 = (uint32_t)(lr * kMxStepBytes + (((2 * kq) ^ ((lr >> 1) & 7)) << 4)), fa1 = fa0 ^ 16u;
  const int xrow = FUSE ? min(lr, p.M - 1) : 0;  // rows past M repeat the last one: their results are not stored
  const uint8_t* const xrd = xs + xrow * xstride + kq * 32;
  const uint8_t* const srd = xsc + xrow * sstride + kq * 2;
  for (int k0 = w; k0 < nkb; k0 += 8 * ST) {
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      const int kb = k0 + 8 * s;
      if (kb >= nkb) break;
      // the blocks behind this one that have been requested, at most ST - 1, are younger than its loads
      const int behind = min((nkb - 1 - kb) >> 3, ST - 1);
      if (behind >= 3) wait_vm<(ST > 3 ? 3 : 0) * kLoads>();
      else if (behind == 2) wait_vm<(ST > 2 ? 2 : 0) * kLoads>();
      else if (behind == 1) wait_vm<kLoads>();
      else wait_vm<0>();
      const uint8_t* const slot = own + s * kSlot;
      v4i W[NS][2], X[MS][2];
#pragma unroll
      for (int g = 0; g < NS; ++g) {
        W[g][0] = *reinterpret_cast<const v4i*>(slot + g * 2048 + fa0);
        W[g][1] = *reinterpret_cast<const v4i*>(slot + g * 2048 + fa1);
      }
      int sxk[MS], swk[NS];
#pragma unroll
      for (int g = 0; g < MS; ++g) {
        if (FUSE) {
          X[g][0] = *reinterpret_cast<const v4i*>(xrd + kb * kMxStepBytes);
          X[g][1] = *reinterpret_cast<const v4i*>(xrd + kb * kMxStepBytes + 16);
          sxk[g] = *reinterpret_cast<const u16*>(srd + kb * 8);
        } else {
          X[g][0] = *reinterpret_cast<const v4i*>(slot + (NS + g) * 2048 + fa0);
          X[g][1] = *reinterpret_cast<const v4i*>(slot + (NS + g) * 2048 + fa1);
          sxk[g] = (int)sx[s][g];
        }
        asm volatile("" : "+v"(sxk[g]));
      }
#pragma unroll
      for (int g = 0; g < NS; ++g) { swk[g] = (int)sw[s][g]; asm volatile("" : "+v"(swk[g])); }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every operand is out of its slot
      SB();
      if (kb + 8 * ST < nkb) request(s, kb + 8 * ST);
#pragma unroll
      for (int ns = 0; ns < NS; ++ns)
#pragma unroll
        for (int ms = 0; ms < MS; ++ms) acc[ns][ms] = mfma_fp4<0>(W[ns][0], X[ms][0], acc[ns][ms], swk[ns], sxk[ms]);
#pragma unroll
      for (int ns = 0; ns < NS; ++ns)
#pragma unroll
        for (int ms = 0; ms < MS; ++ms) acc[ns][ms] = mfma_fp4<1>(W[ns][1], X[ms][1], acc[ns][ms], swk[ns], sxk[ms]);
    }
  }

  // ---- the K shares meet: [wave][group pair][lane], four results of a lane together
#pragma unroll
  for (int ns = 0; ns < NS; ++ns)
#pragma unroll
    for (int ms = 0; ms < MS; ++ms) *reinterpret_cast<v4f*>(own + (ns * MS + ms) * 1024 + lane * 16) = acc[ns][ms];
  __syncthreads();
  for (int i = tid; i < MS * NS * 64; i += 512) {
    const int pair = i >> 6, l = i & 63, ns = pair / MS, ms = pair % MS;
    const int m = m0 + ms * 16 + (l & 15), n = n0 + ns * 16 + (l >> 4) * 4;
    if (m >= p.M || n >= p.N) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const v4f o = *reinterpret_cast<const v4f*>(smem + k * kWave + i * 16);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += o[q];
    }
    if (p.bias) {
      float b[4];
      load_bias4<BIAS_DT>(p.bias, n, b);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += b[q];
    }
    store4<OUT_DT>(p.C, (int64_t)m * p.ldc + n, v[0], v[1], v[2], v[3]);
  }
}

}  // namespace fp8k
