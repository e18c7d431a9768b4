// Expanded latent attention over ragged sequences, gfx950: per-head keys of 128 numbers and a position part of 64 that all heads share,
// values of 128.
//
//   s[i, j] = scale * (q[i, :128] . k_nope[j] + q[i, 128:] . k_pe[j]),   o[i] = sum over j <= i + Lk - Lq of softmax(s[i])[j] v[j]
//
// A workgroup is four waves with 32 query rows each, on tiles of 64 keys; two workgroups share a CU, so that one's softmax runs beside the
// other's products.  Scores are formed transposed, S^T = K . Q^T, in 32x32x16 products: a lane holds 32 scores of one query row, a row's maximum is
// a lane's own and that of the lane 32 away, and what a lane holds is the operand of O^T = V^T . P^T as it lies, the order of the keys inside
// a product being free as long as V^T, read from LDS by transposed reads, has the same.
//
// LDS: two stages of k_nope [64, 128], k_pe [64, 64] and v [64, 128], filled by global_load_lds; the position part is read where it lies, once for
// each head, and never copied beside the keys.  16-byte chunks of a row are permuted by the row so that the operand reads (16 rows, one
// chunk) and the transposed ones (8 rows, two chunks) spread over all banks.
#pragma once

#include "mla_common.h"

namespace fp8k {

struct MlaPrefillArgs {
  const void *q, *k_nope, *k_pe, *v;
  int64_t q_t, q_h, kn_t, kn_h, kp_t, v_t, v_h;  // strides in elements
  const int32_t *cu_q, *cu_k;
  void* out;   // [Tq, H, 128]
  float* lse;  // [Tq, H] or null
  int B, H, Tq, Tk, blocks;  // blocks: of 128 queries that a sequence has at most
  int causal;
  float sm_scale;
};

constexpr int kPreRows = 128, kPreKeys = 64, kPreNope = 128, kPreValue = 128;

// position of the 16-byte chunks of a value's row of 256 bytes: c ^ swizzle(r), as the transposed reads of 16 rows x 32 bytes spread best
__device__ __forceinline__ int mla_value_swizzle(int r) { return ((r & 1) ? 12 : 0) ^ ((r & 2) ? 10 : 0) ^ ((r & 4) ? 6 : 0); }

template <int DT>
__global__ __launch_bounds__(256, 2) void mla_prefill_kernel(const MlaPrefillArgs p) {
  constexpr int kN = 0, kP = kPreKeys * 256, kV = kP + kPreKeys * 128, kStage = kV + kPreKeys * 256;  // 40960 bytes
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kStage];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, half = lane >> 5;
  // the blocks of a sequence's head follow each other on one XCD (workgroup i runs on XCD i % 8): they read the same keys; the last
  // queries, which have most keys, first
  const int unit = (int)(blockIdx.x / 8 / p.blocks) * 8 + (int)(blockIdx.x % 8);
  if (unit >= p.B * p.H) return;
  const int b = unit / p.H, h = unit - b * p.H, block = p.blocks - 1 - (int)(blockIdx.x / 8) % p.blocks;
  const int q_begin = min(max(p.cu_q[b], 0), p.Tq), q_end = min(max(p.cu_q[b + 1], q_begin), p.Tq), lq = q_end - q_begin;
  const int k_begin = min(max(p.cu_k[b], 0), p.Tk), k_end = min(max(p.cu_k[b + 1], k_begin), p.Tk), lk = k_end - k_begin;
  const int q0 = block * kPreRows;
  if (q0 >= lq) return;
  const int shift_k = lk - lq;  // query i is the key of place i + shift_k
  const int last_row = min(q0 + kPreRows, lq) - 1;
  const int keys = p.causal ? min(max(last_row + shift_k + 1, 0), lk) : lk;  // that any row of the workgroup sees
  const int tiles = (keys + kPreKeys - 1) / kPreKeys;

  const int row0 = q0 + w * 32, qi = min(row0 + l31, lq - 1);
  const int lim = p.causal ? min(qi + shift_k + 1, lk) : lk;  // keys that this lane's row sees
  const int wave_keys = p.causal ? min(min(row0 + 31, lq - 1) + shift_k + 1, lk) : lk, wave_free = p.causal ? min(row0 + shift_k + 1, lk) : lk;
  const float c = p.sm_scale * kLog2e;

  v4i q[12];
  {
    const u16* const from = (const u16*)p.q + (int64_t)(q_begin + qi) * p.q_t + h * p.q_h + 8 * half;
#pragma unroll
    for (int ks = 0; ks < 12; ++ks) q[ks] = *(const v4i*)(from + 16 * ks);
  }

  // a wave fetches 16 rows of each part of a stage: four wave-loads of k_nope, two of k_pe, four of v
  auto fetch = [&](int t, uint32_t stage) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = w * 16 + j * 4 + (lane >> 4), at = lane & 15;
      const int64_t row = k_begin + min(t * kPreKeys + r, lk - 1);
      load16_to_lds((const u16*)p.k_nope + row * p.kn_t + h * p.kn_h + ((at ^ (r & 15)) << 3), stage + kN + (w * 16 + j * 4) * 256);
      load16_to_lds((const u16*)p.v + row * p.v_t + h * p.v_h + ((at ^ mla_value_swizzle(r)) << 3), stage + kV + (w * 16 + j * 4) * 256);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = w * 16 + j * 8 + (lane >> 3), at = lane & 7;
      const int64_t row = k_begin + min(t * kPreKeys + r, lk - 1);
      load16_to_lds((const u16*)p.k_pe + row * p.kp_t + ((at ^ ((r >> 1) & 7)) << 3), stage + kP + (w * 16 + j * 8) * 128);
    }
  };

  // LDS offsets of a lane: row l31 of a 32-key tile, chunk 2 ks + half; transposed reads of v
  const int n_off = kN + l31 * 256, n_sw = l31 & 15, p_off = kP + l31 * 128, p_sw = (l31 >> 1) & 7;
  const int v_row = 4 * half + ((lane & 15) >> 2), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int v_off = kV + v_row * 256 + ((lane & 1) << 3), v_sw = mla_value_swizzle(v_row);

  v16f o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  const uint32_t lds0 = lds_address(smem);
  if (tiles > 0) fetch(0, lds0);
  for (int t = 0; t < tiles; ++t) {
    const uint8_t* const stage = smem + (t & 1) * kStage;
    wait_loads<0>();
    lds_only_barrier();  // this tile has arrived, and nobody reads the one before any more
    if (t + 1 < tiles) fetch(t + 1, lds0 + ((t + 1) & 1) * kStage);
    if (t * kPreKeys >= wave_keys) continue;  // nothing that this wave's rows see

    v16f s[2];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[nt][i] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < 12; ++ks) {
        const uint8_t* const at = ks < 8 ? stage + n_off + nt * 32 * 256 + (((2 * ks + half) ^ n_sw) << 4)
                                         : stage + p_off + nt * 32 * 128 + (((2 * (ks - 8) + half) ^ p_sw) << 4);
        s[nt] = mfma32<DT>(*(const v4i*)at, q[ks], s[nt]);
      }
    }

    // a lane's scores are those of query row l31, keys 32 nt + 8 (i / 4) + 4 half + i % 4
    const int key0 = t * kPreKeys + 4 * half;
    if (__builtin_expect((t + 1) * kPreKeys > wave_free, 0)) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + nt * 32 + 8 * (i >> 2) + (i & 3) >= lim) s[nt][i] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[nt][i]);
    // c > 0.  The row's maximum, over two lanes, is asked for only when one of them has passed the old one by far.
    if (__builtin_expect(__any(top * c > m + kMaxSlack), 0)) {
      top = max_across32(top) * c;
      const float raised = top > m + kMaxSlack ? top : m;
      const float alpha = raised != m ? __builtin_amdgcn_exp2f(m - raised) : 1.0f;
      m = raised;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
    }
    const float shift = shift_of(m);
    uint32_t pk[2][8];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[nt][i], c, -shift)), e1 = __builtin_amdgcn_exp2f(fmaf(s[nt][i + 1], c, -shift));
        l += e0;
        l += e1;
        // weights rounded to the 16-bit type, as the matrix core takes them; their sum is of the unrounded ones
        pk[nt][i >> 1] = pack2<DT>(e0, e1);
      }

#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const v4i pb = {(int)pk[nt][4 * ks], (int)pk[nt][4 * ks + 1], (int)pk[nt][4 * ks + 2], (int)pk[nt][4 * ks + 3]};
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          const uint8_t* const at = stage + v_off + (nt * 32 + ks * 16) * 256 + (((4 * dt + v_chunk) ^ v_sw) << 4);
          const v2i a0 = lds_read_transposed(at), a1 = lds_read_transposed(at + 8 * 256);
          o[dt] = mfma32<DT>(v4i{a0[0], a0[1], a1[0], a1[1]}, pb, o[dt]);
        }
      }
  }

  l = sum_across32(l);
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (row0 + l31 < lq) {
    const int64_t row = (int64_t)(q_begin + row0 + l31) * p.H + h;
    u16* const to = (u16*)p.out + row * kPreValue + 4 * half;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *(v2i*)(to + dt * 32 + k * 8) = v2i{(int)pack2<DT>(o[dt][4 * k] * f, o[dt][4 * k + 1] * f), (int)pack2<DT>(o[dt][4 * k + 2] * f, o[dt][4 * k + 3] * f)};
    if (half == 0 && p.lse) p.lse[row] = l == 0.0f ? -INFINITY : (__builtin_amdgcn_logf(l) + shift_of(m)) * kLn2;
  }
}

}  // namespace fp8k
