// Shared pieces of the latent-attention kernels (gfx950): matrix products of 16-bit operands, transposed LDS reads, LDS fills, lane
// exchange, and the softmax's elementary steps.
#pragma once

#include "fp8k_common.h"

namespace fp8k {

constexpr int kLatent = 512, kRope = 64, kLatentRow = kLatent + kRope;  // numbers of a cached row
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// a number as an argument's type
template <int N>
struct Const {
  static constexpr int value = N;
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4v __attribute__((__vector_size__(8)));

// D += A . B, A [16, 32] with lane l holding row l % 16, columns 8 (l / 16) .. + 7; B [32, 16] likewise by columns; D [16, 16] with lane l
// holding rows 4 (l / 16) .. + 3 of column l % 16
template <int DT>
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
  if constexpr (DT == FP8K_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// the same over 16 columns of A: lane l holds columns 4 (l / 16) .. + 3
template <int DT>
__device__ __forceinline__ v4f mfma16_half(v2i a, v2i b, v4f c) {
  if constexpr (DT == FP8K_BF16) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
// D += A . B, A [32, 16]: lane l holds row l % 32, columns 8 (l / 32) .. + 7; D [32, 32]: element i of lane l is row 8 (i / 4) + 4 (l / 32) + i % 4
// of column l % 32
template <int DT>
__device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
  if constexpr (DT == FP8K_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == FP8K_BF16) return pack_bf16x2(lo, hi);
  else {
    const v2f v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  }
}
// the two halves of a word of 16-bit numbers
template <int DT>
__device__ __forceinline__ v2f unpack2(uint32_t w) {
  if constexpr (DT == FP8K_BF16) return v2f{bf16_lo(w), bf16_hi(w)};
  else return v2f{f16_bits_to_f32(w & 0xffffu), f16_bits_to_f32(w >> 16)};
}
// two e4m3 bytes (the low or high half of w) as 16-bit numbers: exact in either type
template <int DT, bool HIGH>
__device__ __forceinline__ uint32_t fp8_to_16bit(uint32_t w) {
  if constexpr (DT == FP8K_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
}

__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }
// 16 bytes from every lane's own address p + OFFSET to LDS at `to` + 16 * lane (to: the wave's, one value).  In assembly, as the compiler
// waits for all such loads that it knows of before any transposed read; this one writes no register, and whoever reads the LDS waits
// for vmcnt himself.  The instruction's offset counts on both sides, hence the subtraction.  Non-temporal, for rows that are read once.
template <int OFFSET = 0>
__device__ __forceinline__ void load16_to_lds(const void* p, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:%2 nt" ::"v"(p), "s"(to - OFFSET), "n"(OFFSET) : "m0", "memory");
}
// the same from base + every lane's own offset, cached; base is the wave's.  (Five wait states in front: a scalar register that a vector instruction
// has just written - the compiler's own spills - is not ready for a vector load before.)
__device__ __forceinline__ void load16_to_lds(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to) : "m0", "memory");
}
// 4 bytes likewise, to `to` + 4 * lane
__device__ __forceinline__ void load4_to_lds(const void* p, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(to) : "m0", "memory");
}
// FIRST .. LAST - 1 of a row of such loads: the lanes' addresses p + STEP * j to `to` + TO_STEP * j + 16 * lane
template <int STEP, int TO_STEP, int FIRST, int LAST>
__device__ __forceinline__ void load_blocks_to_lds(const uint8_t* p, uint32_t to) {
  load16_to_lds<STEP * FIRST>(p, to + TO_STEP * FIRST);
  if constexpr (FIRST + 1 < LAST) load_blocks_to_lds<STEP, TO_STEP, FIRST + 1, LAST>(p, to);
}
// Transposed read: within 16 lanes, lane i names the 8 bytes of row i / 4, numbers 4 (i % 4) .. + 3, of a block of 4 rows x 16 16-bit
// numbers, and receives the four rows' number i.
__device__ __forceinline__ v2i lds_read_transposed(const uint8_t* p) {
  return __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4v*)p));
}

// v of lane l ^ 32, l ^ 16 combined with one's own
__device__ __forceinline__ float max_across32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_across16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_across16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What an exponent is shifted by: the running maximum, or 0 while a row has seen nothing (-inf minus -inf is no number).
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }

// A row's maximum is raised (and what has been summed rescaled) only when a score passes it by more than this, in powers of two: up to
// there the exponentials stay below 2^8, which float32 sums and 16-bit weights hold as exactly as those below 1.
constexpr float kMaxSlack = 8.0f;

// The wave's LDS reads and writes are done, and all but the youngest N of its vector loads.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// All waves of the workgroup have come here; their LDS traffic before it is done, their loads go on.
__device__ __forceinline__ void lds_only_barrier() {
  wait_lds();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace fp8k
