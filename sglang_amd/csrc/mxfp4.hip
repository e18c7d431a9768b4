// MXFP4 (4-bit, block-scaled) operators: quantisation, dequantisation, the product of two quantised operands, whole linears and an
// expert layer for a few tokens.  The format is described in mx_common.h.
#include <algorithm>

#include "../../include/fp8k_tune.h"
#include "mx_common.h"
#include "mx_gemm.h"
#include "mx_moe.h"
#include "mx_tile128.h"
#include "mx_tile256.h"
#include "mx_tile64.h"

namespace fp8k {

// ------------------------------------------------------------------------------------------------
// Quantisation.  amax over 32 values; the scale's exponent is that of amax after a rounding to one fraction bit (the codes' own),
// minus the 2 of the largest code 6 = 1.5 * 2^2: 3.5 <= |largest| / scale < 7, and what lies above 6 becomes 6.  The values times
// 2^-exponent (exact) are rounded to nearest, ties to the even code, by v_cvt_scalef32_pk_fp4_f32.  A block with an infinity or a NaN
// gets scale 255 (NaN) and zero codes.
//
// Memory bound: 2 bytes read and 17/32 written per 16-bit element.  A wave takes 512 columns of four rows, 8 values to a lane, four
// lanes to a block and sixteen to a scale word; the words of four rows lie side by side in memory and leave as one 16-byte store.
// 4096 x 9216 with silu_and_mul from bfloat16: 34 us, 5.1 TB/s read and written; 32 x 7168: 3 us, a launch.
// ------------------------------------------------------------------------------------------------
template <int DT, bool FUSE>
__global__ __launch_bounds__(256) void mx_quant_kernel(const void* x, uint8_t* q, int32_t* s, int M, int K, int64_t ldx, int64_t s_m, int64_t s_w) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int m0 = (blockIdx.y * 4 + w) * 4;
  const int c = blockIdx.x * 512 + lane * 8;
  const bool in = c < K;
  Raw8<DT> a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i].zero();
    if (FUSE) b[i].zero();
    if (in && m0 + i < M) {
      a[i].load(x, (int64_t)(m0 + i) * ldx + c);
      if (FUSE) b[i].load(x, (int64_t)(m0 + i) * ldx + K + c);
    }
  }
  uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
    a[i].unpack(v);
    if (FUSE) {
      float u[8];
      b[i].unpack(u);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = silu_f32(v[k]) * u[k];
    }
    uint32_t byte;
    const uint32_t codes = mx_quant8(v, byte);
    if (in && m0 + i < M) *reinterpret_cast<uint32_t*>(q + (int64_t)(m0 + i) * (K >> 1) + (c >> 1)) = codes;
    // the four bytes of a word: one per quad of lanes; past the end of the row zero
    uint32_t word = in ? byte << (((lane >> 2) & 3) * 8) : 0u;
    word |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)word, kDppHalfMirror, 0xf, 0xf, true);
    word |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)word, kDppMirror, 0xf, 0xf, true);
    words[i] = word;
  }
  if ((lane & 15) != 0 || !in) return;
  int32_t* const to = s + (int64_t)(c >> 7) * s_w + (int64_t)m0 * s_m;
  if (s_m == 1 && m0 + 4 <= M && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
    *reinterpret_cast<uint4*>(to) = make_uint4(words[0], words[1], words[2], words[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (m0 + i < M) to[i * s_m] = (int32_t)words[i];
  }
}

// Values of codes and scales: float32, exact, then one rounding to the output type.  A lane takes 8 codes of four rows, whose loads are
// on their way together; 16 bytes a lane leave.  Bound by memory, mostly the writes: 7168 x 18432 to bfloat16 58 us, 5.8 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void mx_dequant_kernel(const uint8_t* q, const int32_t* s, void* out, int N, int K, int64_t s_e, int64_t s_n, int64_t s_w) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n0 = (blockIdx.y * 4 + w) * 4;
  const int c = blockIdx.x * 512 + lane * 8;
  if (c >= K) return;
  const int64_t e = blockIdx.z;
  uint32_t codes[4], words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n0 + i < N) {
      codes[i] = *reinterpret_cast<const uint32_t*>(q + ((e * N + n0 + i) * K + c) / 2);
      words[i] = (uint32_t)s[e * s_e + (n0 + i) * s_n + (c >> 7) * s_w];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n0 + i >= N) break;
    const uint32_t byte = (words[i] >> (((lane >> 2) & 3) * 8)) & 255u;
    const float f = byte == 255u ? __uint_as_float(0x7fc00000u) : 1.0f;
    const int ex = (int)byte - 127;
    float v[8];
    const v2f p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 1);
    const v2f p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 3);
    v[0] = p0[0]; v[1] = p0[1]; v[2] = p1[0]; v[3] = p1[1]; v[4] = p2[0]; v[5] = p2[1]; v[6] = p3[0]; v[7] = p3[1];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __builtin_amdgcn_ldexpf(v[k] * f, ex);
    const int64_t at = (e * N + n0 + i) * K + c;
    if (DT == FP8K_F32) {
      *reinterpret_cast<float4*>((float*)out + at) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>((float*)out + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      const uint2 lo = pack4<DT>(v[0], v[1], v[2], v[3]), hi = pack4<DT>(v[4], v[5], v[6], v[7]);
      *reinterpret_cast<uint4*>((u16*)out + at) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  }
}

namespace {

bool is_float_type(int dt) { return dt == FP8K_F32 || dt == FP8K_F16 || dt == FP8K_BF16; }
bool is_half_type(int dt) { return dt == FP8K_F16 || dt == FP8K_BF16; }
int64_t words_of(int64_t K) { return (K + 127) / 128; }
int64_t up_to(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// the byte offsets of a tensor of scale words, as the kernels form them in 32 bits
bool scales_fit(int64_t rows, int64_t words, int64_t s_row, int64_t s_word) {
  constexpr int64_t kMost = 0x7fffffff;
  if (s_row < 0 || s_word < 0 || s_row > kMost / 4 || s_word > kMost / 4) return false;
  return ((rows - 1) * s_row + (words - 1) * s_word + 1) * 4 <= kMost;
}

int check_scales(const char* what, const void* s, int64_t rows, int64_t words, int64_t s_row, int64_t s_word) {
  FP8K_REQUIRE(s && aligned(s, 4), "%s: scales must be aligned int32 words", what);
  FP8K_REQUIRE(scales_fit(rows, words, s_row, s_word), "%s: scale strides out of range", what);
  return FP8K_OK;
}

int quant(const void* x, void* q, void* s, int64_t M, int64_t K, int64_t ldx, int64_t s_m, int64_t s_w, int dt, bool fuse, hipStream_t st) {
  const dim3 grid((unsigned)((K + 511) / 512), (unsigned)((M + 15) / 16));
#define MX_QUANT(DT, F) mx_quant_kernel<DT, F><<<grid, 256, 0, st>>>(x, (uint8_t*)q, (int32_t*)s, (int)M, (int)K, ldx, s_m, s_w)
  if (dt == FP8K_BF16) fuse ? MX_QUANT(FP8K_BF16, true) : MX_QUANT(FP8K_BF16, false);
  else if (dt == FP8K_F16) fuse ? MX_QUANT(FP8K_F16, true) : MX_QUANT(FP8K_F16, false);
  else fuse ? MX_QUANT(FP8K_F32, true) : MX_QUANT(FP8K_F32, false);
#undef MX_QUANT
  return check_launch("mxfp4 quant");
}

int check_quant(const void* x, const void* q, int64_t M, int64_t K, int64_t ldx, int dt, bool fuse) {
  FP8K_REQUIRE(is_float_type(dt), "mxfp4 quant: float32, float16 or bfloat16 input expected");
  FP8K_REQUIRE(M >= 0 && K > 0 && K % kMxBlock == 0, "mxfp4 quant: K must be a positive multiple of 32");
  FP8K_REQUIRE(M <= (1 << 19) && K <= (1 << 24), "mxfp4 quant: too many rows or columns");
  if (M == 0) return FP8K_OK;
  FP8K_REQUIRE(x && q, "mxfp4 quant: null pointer");
  FP8K_REQUIRE(ldx >= (fuse ? 2 * K : K) && ldx % 8 == 0, "mxfp4 quant: the row stride must be a multiple of 8 and not less than a row");
  FP8K_REQUIRE(aligned(x, 16) && aligned(q, 16), "mxfp4 quant: operands must be 16-byte aligned");
  return FP8K_OK;
}

// ------------------------------------------------------------------------------------------------ product
template <int O, int B>
void launch_tile256(MxArgs p, hipStream_t st) {
  p.tiles_m = (p.M + 255) / 256;
  p.tiles_n = (p.N + 255) / 256;
  const int tiles = p.tiles_m * p.tiles_n, cu = std::max(8, num_cu() / 8 * 8), rest = tiles % cu;
  // the last, partial round over the chip: as halves, one workgroup each, where they fill at most the chip
  p.tail_first = rest > 0 && 2 * rest <= cu ? tiles - rest : tiles;
  const int units = (tiles - p.tail_first) * 2;
  unsigned grid;
  if (p.tail_first >= cu) {
    p.walkers = cu;
    p.tail_shared = 1;
    grid = (unsigned)std::max(cu, units);
  } else {
    p.walkers = (p.tail_first + 7) / 8 * 8;
    p.tail_shared = 0;
    grid = (unsigned)(p.walkers + units);
  }
  if (p.K % kMxStep) mx_tile256_kernel<O, B, true><<<grid, 512, 0, st>>>(p);
  else mx_tile256_kernel<O, B, false><<<grid, 512, 0, st>>>(p);
}

template <int O, int B>
void launch_tile(MxArgs p, int tm, int tn, hipStream_t st) {
  p.tiles_m = (p.M + tm - 1) / tm;
  p.tiles_n = (p.N + tn - 1) / tn;
  const unsigned grid = (unsigned)(((int64_t)p.tiles_m * p.tiles_n + 7) / 8 * 8);
  const bool ragged = p.K % kMxStep != 0;
  if (tn == 64) ragged ? mx_tile64_kernel<O, B, true><<<grid, 256, 0, st>>>(p) : mx_tile64_kernel<O, B, false><<<grid, 256, 0, st>>>(p);
  else if (tm == 64) ragged ? mx_tile128_kernel<O, B, 64, true><<<grid, 512, 0, st>>>(p) : mx_tile128_kernel<O, B, 64, false><<<grid, 512, 0, st>>>(p);
  else ragged ? mx_tile128_kernel<O, B, 128, true><<<grid, 512, 0, st>>>(p) : mx_tile128_kernel<O, B, 128, false><<<grid, 512, 0, st>>>(p);
}

// strips of 16 NS weight rows: wider while that leaves two or more for every CU.  Products that are quantised already reach 16 columns a
// strip up to N = 16352 and 32 from there to the 16384 that plan_of gives them: 16 x 16384 x 7168 13.0 us (16 columns 17.2), 32 rows 15.1 (21.2).
// Their LDS (96 .. 160 KB) has room for one workgroup on a CU at a time; the quantising form's for two up to 32 columns, for one with 64.
int strip_groups(int64_t N, int m_blocks, int most) {
  int ns = 1;
  while (ns < most && (N + 32 * ns - 1) / (32 * ns) * m_blocks >= 2 * num_cu()) ns *= 2;
  return ns;
}
template <int MS, int NS, bool FUSE, int O, int B>
void launch_strip(const MxArgs& p, hipStream_t st) {
  const dim3 grid((unsigned)((p.N + 16 * NS - 1) / (16 * NS)), (unsigned)((p.M + 16 * MS - 1) / (16 * MS)));
  if (p.K % kMxStep) mx_strip_kernel<MS, NS, FUSE, O, B, true><<<grid, 512, 0, st>>>(p);
  else mx_strip_kernel<MS, NS, FUSE, O, B, false><<<grid, 512, 0, st>>>(p);
}
template <int O, int B>
void launch_strips(const MxArgs& p, hipStream_t st) {
  if (p.M <= 16) {
    if (strip_groups(p.N, 1, 2) == 1) launch_strip<1, 1, false, O, B>(p, st);
    else launch_strip<1, 2, false, O, B>(p, st);
  } else if (p.M <= 32) {
    if (strip_groups(p.N, 1, 2) == 1) launch_strip<2, 1, false, O, B>(p, st);
    else launch_strip<2, 2, false, O, B>(p, st);
  } else {
    launch_strip<4, 1, false, O, B>(p, st);
  }
}
// a whole linear of a few rows in one launch: p.X holds 16-bit activations, p.ldx their row stride in elements
bool fuses_quant(int64_t M, int64_t K) {
  if (M > 16 || M * K > kMxFuse) return false;
  const int64_t kbs = (K + kMxStep - 1) / kMxStep;
  return M * mx_fuse_stride((int)kbs) <= kMxFuseRows && M * kbs * 8 <= kMxFuseScales;
}
template <int O, int B>
int launch_fused(const MxArgs& p, hipStream_t st) {
  const int ns = strip_groups(p.N, 1, 4);
  if (ns == 1) launch_strip<1, 1, true, O, B>(p, st);
  else if (ns == 2) launch_strip<1, 2, true, O, B>(p, st);
  else launch_strip<1, 4, true, O, B>(p, st);
  return check_launch("mxfp4 linear");
}

thread_local int g_force = -1;  // fp8k_tune_force_mxfp4_plan

// which kernel a product takes: the tuning aid's numbers
enum { kPlanStrips = 0, kPlanTile64 = 1, kPlanTile128x64 = 2, kPlanTile128 = 3, kPlanTile256 = 4 };
// Up to 64 rows the strips, while they are one round over the chip or the rows are few; of the tiles the one with the shortest time
// by rounds * (start and write-out + K blocks * time of a block), the times as measured on products of 128 .. 4096 rows (weights
// out of HBM): 64x64 tiles 0.24 us a block, 128x64 0.385, 128x128 0.62, 256x256 1.1 while the tiles are computed in halves and 2.0 whole.
int plan_of(const MxArgs& p) {
  if (g_force >= 0) return g_force;
  const int64_t cu = num_cu();
  // 64 x 4096 x 4096: strips 6.5 us, 64x64 tiles 8.0; 64 x 4608 x 7168, a second round: 15.0 and 10.1
  if (p.M <= 64 && p.N <= 16 * cu) return kPlanStrips;
  // 24 x 7168 x 18432: strips 23.2, 64x64 tiles 26.3, 128x64 33.7; 32 x 28672 x 4096: 19.4, 19.7, 15.3; 16 rows: 16.8, 19.2, 15.0
  if (p.M <= 32 && p.N <= 64 * cu) return kPlanStrips;
  const double kbs = (p.K + kMxStep - 1) / kMxStep;
  const auto time = [&](int tm, int tn, double tile, double block) {
    const int64_t tiles = (int64_t)((p.M + tm - 1) / tm) * ((p.N + tn - 1) / tn);
    return (double)((tiles + cu - 1) / cu) * (tile + kbs * block);
  };
  const int64_t big = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256), rest = big % cu;
  const bool halves = rest > 0 && 2 * rest <= cu;
  const double t[] = {time(64, 64, 1.2, 0.24), time(64, 128, 1.3, 0.385), time(128, 128, 1.6, 0.62),
                      (double)((big + cu - 1) / cu - halves) * (4.0 + kbs * 2.0) + (halves ? 3.0 + kbs * 1.1 : 0.0)};
  constexpr int kind[] = {kPlanTile64, kPlanTile128x64, kPlanTile128, kPlanTile256};
  int best = 0;
  for (int i = 1; i < 4; ++i)
    if (t[i] < t[best]) best = i;
  return kind[best];
}

template <int O, int B>
int launch_gemm(const MxArgs& p, hipStream_t st) {
  switch (plan_of(p)) {
    case kPlanStrips: launch_strips<O, B>(p, st); break;
    case kPlanTile64: launch_tile<O, B>(p, 64, 64, st); break;
    case kPlanTile128x64: launch_tile<O, B>(p, 64, 128, st); break;
    case kPlanTile128: launch_tile<O, B>(p, 128, 128, st); break;
    default: launch_tile256<O, B>(p, st);
  }
  return check_launch("mxfp4 gemm");
}
int launch_gemm(const MxArgs& p, int out_dtype, int bias_dtype, hipStream_t st) {
  if (out_dtype == FP8K_BF16) return bias_dtype == FP8K_F32 ? launch_gemm<FP8K_BF16, FP8K_F32>(p, st) : launch_gemm<FP8K_BF16, FP8K_BF16>(p, st);
  return bias_dtype == FP8K_F32 ? launch_gemm<FP8K_F16, FP8K_F32>(p, st) : launch_gemm<FP8K_F16, FP8K_F16>(p, st);
}

int check_gemm(const char* what, int64_t M, int64_t N, int64_t K, int64_t ldb, int64_t ldc, const void* B, const void* C, const void* bias,
               int out_dtype, int bias_dtype) {
  FP8K_REQUIRE(is_half_type(out_dtype), "%s: the result must be Half or BFloat16", what);
  FP8K_REQUIRE(M >= 0 && N > 0 && K > 0, "%s: bad sizes", what);
  FP8K_REQUIRE(K % kMxBlock == 0, "%s: K must be a multiple of 32", what);
  FP8K_REQUIRE(N % 8 == 0, "%s: out must be multiple of 16 bytes for memory alignment (N %% 8)", what);
  FP8K_REQUIRE(M <= (1 << 20) && N <= (1 << 24) && K <= (1 << 22), "%s: too large", what);
  FP8K_REQUIRE(!bias || bias_dtype == out_dtype || bias_dtype == FP8K_F32, "%s: bias must have the result's type or be float32", what);
  FP8K_REQUIRE(!bias || aligned(bias, bias_dtype == FP8K_F32 ? 4 : 2), "%s: misaligned bias", what);
  if (M == 0) return FP8K_OK;
  FP8K_REQUIRE(B && C, "%s: null pointer", what);
  FP8K_REQUIRE(aligned(B, 16) && ldb % 16 == 0 && ldb >= K / 2 && ldb < (1 << 23), "%s: rows of codes must be 16-byte aligned", what);
  FP8K_REQUIRE(aligned(C, 8) && ldc % 4 == 0 && ldc >= N, "%s: rows of the result must be 8-byte aligned", what);
  return FP8K_OK;
}

int64_t experts_part(int64_t slots, int64_t I) { return up_to(slots * I * 4, 256); }

}  // namespace
}  // namespace fp8k

using namespace fp8k;

extern "C" void fp8k_tune_force_mxfp4_plan(int kind) { g_force = kind >= 0 && kind <= kPlanTile256 ? kind : -1; }

extern "C" int fp8k_mxfp4_quant(const void* x, void* q, void* s, int64_t M, int64_t K, int64_t ldx, int64_t s_stride_m, int64_t s_stride_w,
                                int in_dtype, int fuse_silu_and_mul, void* stream) {
  clear_error();
  if (const int rc = check_quant(x, q, M, K, ldx, in_dtype, fuse_silu_and_mul != 0)) return rc;
  if (M == 0) return FP8K_OK;
  if (const int rc = check_scales("mxfp4 quant", s, M, words_of(K), s_stride_m, s_stride_w)) return rc;
  FP8K_REQUIRE(s_stride_m > 0 && s_stride_w > 0, "mxfp4 quant: scale strides must be positive");
  return quant(x, q, s, M, K, ldx, s_stride_m, s_stride_w, in_dtype, fuse_silu_and_mul != 0, (hipStream_t)stream);
}

extern "C" int fp8k_mxfp4_dequant(const void* q, const void* s, void* out, int64_t E, int64_t N, int64_t K, int64_t s_stride_e,
                                  int64_t s_stride_n, int64_t s_stride_w, int out_dtype, void* stream) {
  clear_error();
  FP8K_REQUIRE(is_float_type(out_dtype), "mxfp4 dequant: float32, float16 or bfloat16 output expected");
  FP8K_REQUIRE(E >= 0 && N >= 0 && K > 0 && K % kMxBlock == 0, "mxfp4 dequant: K must be a positive multiple of 32");
  FP8K_REQUIRE(E <= 65535 && N <= (1 << 19) && K <= (1 << 24), "mxfp4 dequant: too large");
  if (E == 0 || N == 0) return FP8K_OK;
  FP8K_REQUIRE(q && out && aligned(q, 16) && aligned(out, 16), "mxfp4 dequant: operands must be 16-byte aligned");
  if (const int rc = check_scales("mxfp4 dequant", s, N, words_of(K), s_stride_n, s_stride_w)) return rc;
  FP8K_REQUIRE(s_stride_e >= 0, "mxfp4 dequant: scale strides out of range");
  const dim3 grid((unsigned)((K + 511) / 512), (unsigned)((N + 15) / 16), (unsigned)E);
  const hipStream_t st = (hipStream_t)stream;
#define MX_DEQUANT(DT) \
  mx_dequant_kernel<DT><<<grid, 256, 0, st>>>((const uint8_t*)q, (const int32_t*)s, out, (int)N, (int)K, s_stride_e, s_stride_n, s_stride_w)
  if (out_dtype == FP8K_BF16) MX_DEQUANT(FP8K_BF16);
  else if (out_dtype == FP8K_F16) MX_DEQUANT(FP8K_F16);
  else MX_DEQUANT(FP8K_F32);
#undef MX_DEQUANT
  return check_launch("mxfp4 dequant");
}

extern "C" int fp8k_mxfp4_gemm(const void* A, const void* B, const void* As, const void* Bs, const void* bias, void* C, int64_t M, int64_t N,
                               int64_t K, int64_t lda, int64_t ldb, int64_t as_stride_m, int64_t as_stride_w, int64_t bs_stride_n,
                               int64_t bs_stride_w, int64_t ldc, int out_dtype, int bias_dtype, void* stream) {
  clear_error();
  if (const int rc = check_gemm("mxfp4 gemm", M, N, K, ldb, ldc, B, C, bias, out_dtype, bias_dtype)) return rc;
  if (M == 0) return FP8K_OK;
  FP8K_REQUIRE(A && aligned(A, 16) && lda % 16 == 0 && lda >= K / 2 && lda < (1 << 23), "mxfp4 gemm: rows of codes must be 16-byte aligned");
  if (const int rc = check_scales("mxfp4 gemm", As, M, words_of(K), as_stride_m, as_stride_w)) return rc;
  if (const int rc = check_scales("mxfp4 gemm", Bs, N, words_of(K), bs_stride_n, bs_stride_w)) return rc;
  MxArgs p{};
  p.X = (const uint8_t*)A; p.W = (const uint8_t*)B; p.sx = (const uint8_t*)As; p.sw = (const uint8_t*)Bs;
  p.bias = bias; p.C = C; p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.ldx = lda; p.ldw = ldb; p.ldc = ldc;
  p.sx_m = as_stride_m; p.sx_w = as_stride_w; p.sw_n = bs_stride_n; p.sw_w = bs_stride_w;
  return launch_gemm(p, out_dtype, bias ? bias_dtype : FP8K_F32, (hipStream_t)stream);
}

extern "C" int64_t fp8k_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || fuses_quant(M, K)) return 0;
  return up_to(M * K / 2, 256) + up_to(words_of(K) * up_to(M, 4) * 4, 256);
}

extern "C" int fp8k_mxfp4_linear(const void* x, const void* B, const void* Bs, const void* bias, void* C, int64_t M, int64_t N, int64_t K,
                                 int64_t ldx, int64_t ldb, int64_t bs_stride_n, int64_t bs_stride_w, int64_t ldc, int dtype, int bias_dtype,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (const int rc = check_gemm("mxfp4 linear", M, N, K, ldb, ldc, B, C, bias, dtype, bias_dtype)) return rc;
  if (const int rc = check_quant(x, x, M, K, ldx, dtype, false)) return rc;
  if (M == 0) return FP8K_OK;
  if (const int rc = check_scales("mxfp4 linear", Bs, N, words_of(K), bs_stride_n, bs_stride_w)) return rc;
  const int64_t need = fp8k_mxfp4_linear_workspace_bytes(M, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
    return fail(FP8K_ERR_WORKSPACE, "mxfp4 linear: workspace of %lld bytes needed, 256-byte aligned", (long long)need);
  MxArgs p{};
  p.W = (const uint8_t*)B; p.sw = (const uint8_t*)Bs;
  p.bias = bias; p.C = C; p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.ldw = ldb; p.ldc = ldc;
  p.sw_n = bs_stride_n; p.sw_w = bs_stride_w;
  const hipStream_t st = (hipStream_t)stream;
  const int bt = bias ? bias_dtype : FP8K_F32;
  if (fuses_quant(M, K)) {
    p.X = (const uint8_t*)x;
    p.ldx = ldx;
    if (dtype == FP8K_BF16) return bt == FP8K_F32 ? launch_fused<FP8K_BF16, FP8K_F32>(p, st) : launch_fused<FP8K_BF16, FP8K_BF16>(p, st);
    return bt == FP8K_F32 ? launch_fused<FP8K_F16, FP8K_F32>(p, st) : launch_fused<FP8K_F16, FP8K_F16>(p, st);
  }
  uint8_t* const q = (uint8_t*)workspace;
  uint8_t* const s = q + up_to(M * K / 2, 256);
  const int64_t ld = up_to(M, 4);
  FP8K_REQUIRE(scales_fit(M, words_of(K), 1, ld), "mxfp4 linear: too many activations");
  if (const int rc = quant(x, q, s, M, K, ldx, 1, ld, dtype, false, st)) return rc;
  p.X = q; p.sx = s;
  p.ldx = K / 2;
  p.sx_m = 1; p.sx_w = ld;
  return launch_gemm(p, dtype, bt, st);
}

extern "C" int64_t fp8k_mxfp4_experts_workspace_bytes(int64_t T, int64_t topk, int64_t I) {
  if (T <= 0 || topk <= 0 || I <= 0) return 0;
  const int64_t slots = T * topk;
  return experts_part(slots, I) + 3 * up_to(slots * 4, 256) + 256;
}

extern "C" int fp8k_mxfp4_experts(const void* x, const void* w1, const void* w2, const void* s1, const void* s2, const float* topk_weights,
                                  const void* topk_ids, int ids_are_64bit, void* out, int64_t T, int64_t topk, int64_t E, int64_t H, int64_t I,
                                  int64_t ldx, int64_t w1_stride_e, int64_t w2_stride_e, int64_t s1_stride_e, int64_t s1_stride_n,
                                  int64_t s1_stride_w, int64_t s2_stride_e, int64_t s2_stride_n, int64_t s2_stride_w, int activation,
                                  int weight_on_input, float scaling, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  FP8K_REQUIRE(is_half_type(dtype), "mxfp4 experts: Half or BFloat16 activations expected");
  FP8K_REQUIRE(activation == FP8K_ACT_SILU || activation == FP8K_ACT_GELU, "mxfp4 experts: the activation must be silu or gelu");
  FP8K_REQUIRE(T >= 0 && topk > 0 && E > 0 && H > 0 && I > 0, "mxfp4 experts: bad sizes");
  FP8K_REQUIRE(H % kMxBlock == 0 && I % kMxBlock == 0, "mxfp4 experts: hidden and intermediate size must be multiples of 32");
  FP8K_REQUIRE(H <= (1 << 20) && I <= (1 << 19) && H * I < (1ll << 31) && E <= 65535, "mxfp4 experts: too large");
  FP8K_REQUIRE(T <= kMxMaxTokens && T * topk <= kMxMaxSlots, "mxfp4 experts: built for at most %d tokens and %d (token, choice) pairs, got %lld and %lld",
               kMxMaxTokens, kMxMaxSlots, (long long)T, (long long)(T * topk));
  if (T == 0) return FP8K_OK;
  FP8K_REQUIRE(x && w1 && w2 && topk_weights && topk_ids && out, "mxfp4 experts: null pointer");
  FP8K_REQUIRE(aligned(x, 16) && ldx % 8 == 0 && ldx >= H && ldx <= (1 << 22), "mxfp4 experts: rows of the activations must be 16-byte aligned");
  FP8K_REQUIRE(aligned(w1, 16) && aligned(w2, 16) && w1_stride_e % 16 == 0 && w2_stride_e % 16 == 0 && w1_stride_e >= 0 && w2_stride_e >= 0,
               "mxfp4 experts: weights must be 16-byte aligned");
  FP8K_REQUIRE(aligned(topk_weights, 4) && aligned(topk_ids, ids_are_64bit ? 8 : 4) && aligned(out, 4), "mxfp4 experts: misaligned operand");
  if (const int rc = check_scales("mxfp4 experts", s1, 2 * I, words_of(H), s1_stride_n, s1_stride_w)) return rc;
  if (const int rc = check_scales("mxfp4 experts", s2, H, words_of(I), s2_stride_n, s2_stride_w)) return rc;
  FP8K_REQUIRE(s1_stride_e >= 0 && s2_stride_e >= 0, "mxfp4 experts: scale strides out of range");
  const int64_t need = fp8k_mxfp4_experts_workspace_bytes(T, topk, I);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
    return fail(FP8K_ERR_WORKSPACE, "mxfp4 experts: workspace of %lld bytes needed, 256-byte aligned", (long long)need);
  const int64_t slots = T * topk;
  MxExpertArgs p{};
  p.x = x; p.w1 = (const uint8_t*)w1; p.w2 = (const uint8_t*)w2; p.s1 = (const uint8_t*)s1; p.s2 = (const uint8_t*)s2;
  p.topk_w = topk_weights; p.ids = topk_ids; p.out = out;
  uint8_t* at = (uint8_t*)workspace;
  p.h = at; at += experts_part(slots, I);
  p.tiles = (int32_t*)at; at += up_to(slots * 4, 256);
  p.order = (int32_t*)at; at += up_to(slots * 4, 256);
  p.weights = (float*)at; at += up_to(slots * 4, 256);
  p.ntiles = (int32_t*)at;
  p.T = (int)T; p.topk = (int)topk; p.E = (int)E; p.H = (int)H; p.I = (int)I; p.slots = (int)slots;
  p.ids64 = ids_are_64bit != 0; p.on_input = weight_on_input != 0; p.ldx = ldx;
  p.w1_e = w1_stride_e; p.w2_e = w2_stride_e;
  p.s1_e = s1_stride_e; p.s1_n = s1_stride_n; p.s1_w = s1_stride_w;
  p.s2_e = s2_stride_e; p.s2_n = s2_stride_n; p.s2_w = s2_stride_w;
  p.scaling = scaling;
  const hipStream_t st = (hipStream_t)stream;
  const bool gelu = activation == FP8K_ACT_GELU;
  // runs of strips: as long as leaves four workgroups for every CU (they are on it together), so that a workgroup's start - the list of
  // its slots, its first lines - comes once for several strips
  const int64_t units = std::min(slots, E), strips = I / 16;
  p.run = (int)std::min<int64_t>(8, std::max<int64_t>(1, units * strips / (4 * num_cu())));
  const dim3 grid1((unsigned)((strips + p.run - 1) / p.run + 1), (unsigned)units), grid2((unsigned)(H / 16));
  // slots that a workgroup of the first launch takes at a time (4 or 16), and those of a tile of the second (4 or 8: the operand has 16 rows):
  // few while an expert has no more on average.  (The first with 8, 64 experts of 7168 x 2048 and 6 slots to one: 280 us, with 16 246.)
  const bool few = slots <= 4 * units;
  p.tile = few ? 4 : 8;
  // up to one strip of columns per CU: sixteen waves to it, as far as their sums fit; else eight, two workgroups to a CU
  const bool wide = H <= 16 * num_cu();
#define MX_DOWN(DT, TC)                                                                                                        \
  do {                                                                                                                         \
    constexpr int kMany = mx_down_waves(8, TC, false), kFew = mx_down_waves(4, TC, false), kWide = mx_down_waves(4, TC, true); \
    if (!few) mx_experts_down_kernel<DT, TC, 8, kMany><<<grid2, kMany * 64, 0, st>>>(p);                                       \
    else if (wide) mx_experts_down_kernel<DT, TC, 4, kWide><<<grid2, kWide * 64, 0, st>>>(p);                                  \
    else mx_experts_down_kernel<DT, TC, 4, kFew><<<grid2, kFew * 64, 0, st>>>(p);                                              \
  } while (0)
#define MX_UP(DT, RX)                                                             \
  do {                                                                            \
    if (gelu) mx_experts_up_kernel<DT, true, RX><<<grid1, 256, 0, st>>>(p);       \
    else mx_experts_up_kernel<DT, false, RX><<<grid1, 256, 0, st>>>(p);           \
  } while (0)
#define MX_EXPERTS(DT)                                                     \
  do {                                                                     \
    if (few) MX_UP(DT, 4);                                                 \
    else MX_UP(DT, 16);                                                    \
    if (const int rc = check_launch("mxfp4 experts")) return rc;           \
    if (T <= 16 && slots <= mx_down_places(16)) MX_DOWN(DT, 16);           \
    else if (T <= 32) MX_DOWN(DT, 32);                                     \
    else if (T <= 64) MX_DOWN(DT, 64);                                     \
    else MX_DOWN(DT, kMxMaxTokens);                                        \
  } while (0)
  if (dtype == FP8K_BF16) MX_EXPERTS(FP8K_BF16);
  else MX_EXPERTS(FP8K_F16);
#undef MX_EXPERTS
#undef MX_UP
#undef MX_DOWN
  return check_launch("mxfp4 experts");
}
