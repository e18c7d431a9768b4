// Device helpers of the 4-bit (MXFP4) kernels, gfx950.
//
// The format: 32 e2m1 values along K share one e8m0 scale 2^(byte - 127) (byte 255: NaN).  Two codes to a byte, the even element in
// the low half; four scale bytes (blocks 4j .. 4j+3 of a row) to an int32 word, words addressed by (row stride, word stride).
#pragma once

#include "gemm_direct.h"
#include "quant_math.h"

namespace fp8k {

constexpr int kMxBlock = 32;     // values that share a scale
constexpr int kMxStep = 256;     // values of a K block of the kernels: one 128-byte line of a row
constexpr int kMxStepBytes = 128;

// 2^(byte - 127) as a float, exact for every byte (0 is a subnormal); 255 is NaN
__device__ __forceinline__ float e8m0_f32(uint32_t byte) {
  const uint32_t bits = byte == 255u ? 0x7fc00000u : byte << 23;
  return __uint_as_float(byte == 0u ? 0x00400000u : bits);
}

// The 16 bytes of a row that a lane hands to one product are the 32 values of one block; the instruction reads four registers of the
// eight that its operand type has.
__device__ __forceinline__ v8i fp4_operand(v4i a) {
  v8i r;
  r[0] = a[0]; r[1] = a[1]; r[2] = a[2]; r[3] = a[3];
  r[4] = r[5] = r[6] = r[7] = 0;
  return r;
}
// 16 x 16 x 128 with e2m1 operands: lane (row lane & 15, lane >> 4) holds one block of its row of either operand, and byte S of
// scale_a / scale_b is that block's scale.  Result: column lane & 15 (of b), rows (lane >> 4) * 4 + i (of a).
template <int S>
__device__ __forceinline__ v4f mfma_fp4(v4i a, v4i b, v4f c, int scale_a, int scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(a), fp4_operand(b), c, 4, 4, S, scale_a, S, scale_b);
}

__device__ __forceinline__ uint32_t buf_load_u16(rsrc_t r, uint32_t voff) {
  return (uint32_t)(u16)__builtin_amdgcn_raw_buffer_load_b16(r, (int)voff, 0, 0);
}

// Quantises the 8 values of each of four neighbouring lanes, which make a block: the lane's eight codes, and the block's scale byte.
// The scale's exponent is that of the largest magnitude after a rounding to one fraction bit (the codes' own), minus the 2 of the
// largest code 6 = 1.5 * 2^2: 3.5 <= |largest| / scale < 7, and what lies above 6 becomes 6.  The values times 2^-exponent (exact) are
// rounded to nearest, ties to the even code, by v_cvt_scalef32_pk_fp4_f32.  An infinity or a NaN makes the byte 255 and the codes zero.
__device__ __forceinline__ uint32_t mx_quant8(const float (&v)[8], uint32_t& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);  // NaN above infinity above every number
  m = dpp_umax<kDppXor1>(m);
  m = dpp_umax<kDppXor2>(m);
  const bool finite = m < 0x7f800000u;
  const int e = min((int)((m + 0x200000u) >> 23), 254) - 2;
  byte = finite ? (uint32_t)max(e, 0) : 255u;
  const float to = finite ? __uint_as_float((254u - byte) << 23) : 0.f;  // 2^(127 - byte)
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0] * to, v[1] * to, 1.0f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2] * to, v[3] * to, 1.0f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4] * to, v[5] * to, 1.0f, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6] * to, v[7] * to, 1.0f, 3);
  return finite ? codes : 0u;
}

__device__ __forceinline__ uint32_t buf_load4(rsrc_t r, uint32_t voff) {
  return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, 0, 0);
}

struct MxArgs {
  const uint8_t* X;   // [M, K/2] codes of the activations
  const uint8_t* W;   // [N, K/2] codes of the weight
  const uint8_t* sx;  // int32 words of scales: row m, word w at byte (m * sx_m + w * sx_w) * 4
  const uint8_t* sw;
  const void* bias;   // [N], may be null; added in float32 before the only rounding
  void* C;            // [M, N]
  int M, N, K;
  int64_t ldx, ldw;   // bytes (16-bit activations: elements)
  int64_t ldc;        // elements
  int64_t sx_m, sx_w, sw_n, sw_w;  // int32 words
  int tiles_m, tiles_n;
  int walkers;        // mx_tile256_kernel: workgroups [0, walkers) walk the whole tiles (a multiple of 8)
  int tail_first;     // mx_tile256_kernel: tiles from here on are computed as two 128-row halves
  int tail_shared;    // mx_tile256_kernel: half u belongs to workgroup u (after its walk), else to workgroup walkers + u
};

// descriptor of the scale words of `rows` rows from row `row0` on
__device__ __forceinline__ rsrc_t mx_scale_rsrc(const uint8_t* s, int64_t row0, int rows, int words, int64_t s_row, int64_t s_word) {
  return make_rsrc(s + row0 * s_row * 4, rows > 0 ? (uint32_t)(((rows - 1) * s_row + (words - 1) * s_word + 1) * 4) : 0u);
}

}  // namespace fp8k
