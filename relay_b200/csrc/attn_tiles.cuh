// Pieces the attention kernels on mma.sync tiles share (attention.cu, shared_prefix.cu): the base-2
// exponential, page addressing, and the two products of a 16-key tile.
#pragma once

#include "common.cuh"

namespace rb200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (x, y) as two pairs of halves, x = hi + lo to 2^-22 of x (2^-25 where lo is subnormal). With hi alone
// the rounding of q would cost an attention output about as much as its own rounding to fp16.
__device__ __forceinline__ void split_half2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 b = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack_half2(x - b.x, y - b.y);
}

// Halves from the start of one layer's pool to row `key` of KV head `kvh`.
// `table` is indexed by absolute block number of the sequence minus `first_block`.
__device__ __forceinline__ long long key_offset(const int* table, int first_block, int key, int bs, int bs_shift,
                                                int kv_heads, int kvh, int D) {
  int blk_i, slot;
  if (bs_shift >= 0) {
    blk_i = key >> bs_shift;
    slot = key & (bs - 1);
  } else {
    blk_i = key / bs;
    slot = key - blk_i * bs;
  }
  const long long blk = table[blk_i - first_block];
  return ((blk * kv_heads + kvh) * bs + slot) * static_cast<long long>(D);
}

// Scores of 16 query rows against 16 keys.
// s[0] covers keys 0-7 of the tile, s[1] keys 8-15; ktile is [16][D] halves, swizzled.
template <int D>
__device__ __forceinline__ void qk_16x16(float (&s)[2][4], const uint32_t (&qf)[D / 16][4], uint32_t ktile, int lane) {
  constexpr int CH = D / 8;
  const int row = (lane & 7) + ((lane >> 4) << 3);
  const int csel = (lane >> 3) & 1;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    uint32_t kb[4];
    ldmatrix_x4(kb, ktile + swz<CH>(row, 2 * kk + csel) * 16);
    mma_f16(s[0], qf[kk], kb[0], kb[1]);
    mma_f16(s[1], qf[kk], kb[2], kb[3]);
  }
}

// O(16 x D) += P(16 x 16 keys) V(16 keys x D); vtile is [16][D] halves, swizzled.
template <int D>
__device__ __forceinline__ void pv_16x16(float (&o)[D / 8][4], const uint32_t (&pa)[4], uint32_t vtile, int lane) {
  constexpr int CH = D / 8;
  const int row = (lane & 7) + (((lane >> 3) & 1) << 3);
  const int csel = lane >> 4;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    uint32_t vb[4];
    ldmatrix_x4_trans(vb, vtile + swz<CH>(row, 2 * j + csel) * 16);
    mma_f16(o[2 * j], pa, vb[0], vb[1]);
    mma_f16(o[2 * j + 1], pa, vb[2], vb[3]);
  }
}

inline int shift_of(int bs) {
  if (bs <= 0 || (bs & (bs - 1)) != 0) return -1;
  int s = 0;
  while ((1 << s) < bs) ++s;
  return s;
}

}  // namespace rb200
