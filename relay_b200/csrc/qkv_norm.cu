// Norms of the query and key heads, rotation and paged append in one pass over the projection's
// output (qkv_post_kernel of small_ops.cu for models that normalise their heads first).
//
//   y = x * rsqrt(mean(x^2) + eps) * w      per head, x = projection + bias, sums in float32
//   (a, b) -> (a cos - b sin, b cos + a sin)  on the pairs (i, i + rot/2) of y
//
// Every value is read once and written once: 4 (Q + 2 KV) bytes of a token come in, 4 Q + 4 KV go
// out, so the kernel is bound by memory, and by latency for a few tokens.
#include "kernels.h"

namespace rb200 {

namespace {

constexpr int kQnWarps = 8;

// cos and sin of pos * inv_freq. The product is exact in float64 and reduced there: its float32
// rounding alone would be off by 4e-3 rad at position 131072. What is left, at most pi, rounds to
// float32 within 2^-23.
__device__ __forceinline__ void rotation(int pos, float inv_freq, float& c, float& s) {
  constexpr double kTwoPi = 6.283185307179586476925;
  const double a = static_cast<double>(pos) * static_cast<double>(inv_freq);
  const double r = fma(-rint(a * (1.0 / kTwoPi)), kTwoPi, a);
  sincosf(static_cast<float>(r), &s, &c);
}

// One CTA per token, one warp per head at a time; the head's values pass through the warp's own
// shared row, because the partner of a rotated value is rot/2 away.
__global__ void __launch_bounds__(kQnWarps * 32)
qkv_norm_post_kernel(const float* qkv, const float* __restrict__ bias, const float* __restrict__ q_norm,
                     const float* __restrict__ k_norm, float eps, const float* __restrict__ inv_freq, int rot, TokenMeta m,
                     float* q_out, __half* __restrict__ kc, __half* __restrict__ vc, int heads, int kv_heads, int D, int bs,
                     int qkv_stride, int q_stride) {
  extern __shared__ float sm[];  // [rot/2] cos, [rot/2] sin, [warps][D] rows
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, half = rot >> 1;
  const int seq = m.seq[t], p = m.pos[t];
  if (seq < 0 || p < 0) return;  // padding
  for (int i = threadIdx.x; i < half; i += blockDim.x) rotation(p, inv_freq[i], sm[i], sm[half + i]);
  const long long block = m.tables[m.table_off[seq] + p / bs];
  const int slot = p % bs;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* row = sm + rot + warp * D;
  const float* src0 = qkv + static_cast<long long>(t) * qkv_stride;
  for (int h = warp; h < heads + 2 * kv_heads; h += kQnWarps) {
    const float* src = src0 + h * D;
    const bool is_v = h >= heads + kv_heads;
    const float* w = h < heads ? q_norm : (is_v ? nullptr : k_norm);
    float ss = 0.0f;
    for (int d = lane; d < D; d += 32) {
      float x = src[d];
      if (bias) x += bias[h * D + d];
      row[d] = x;
      ss += x * x;
    }
    const float scale = w ? 1.0f / sqrtf(warp_sum(ss) / static_cast<float>(D) + eps) : 1.0f;
    __syncwarp();
    const int kvh = is_v ? h - heads - kv_heads : h - heads;
    const long long off = ((block * kv_heads + kvh) * bs + slot) * D;
    for (int d = lane; d < D; d += 32) {
      float y = row[d];
      if (w) y = y * scale * w[d];
      if (!is_v && d < rot) {
        const int i = d < half ? d : d - half, e = d < half ? d + half : d - half;
        float z = row[e];
        if (w) z = z * scale * w[e];
        y = d < half ? y * sm[i] - z * sm[half + i] : y * sm[i] + z * sm[half + i];
      }
      if (h < heads) q_out[static_cast<long long>(t) * q_stride + h * D + d] = y;
      else (is_v ? vc : kc)[off + d] = __float2half_rn(y);
    }
    __syncwarp();
  }
}

}  // namespace

void launch_qkv_norm_post(const float* qkv, int qkv_stride, const float* bias, const float* q_norm, const float* k_norm, float eps,
                          const float* inv_freq, int rot, const TokenMeta& m, int T, float* q_out, int q_stride, __half* kc,
                          __half* vc, int heads, int kv_heads, int D, int block_size, cudaStream_t st) {
  if (T == 0) return;
  count_launch();
  const size_t smem = (static_cast<size_t>(rot) + kQnWarps * D) * sizeof(float);
  launch_pdl(qkv_norm_post_kernel, dim3(T), dim3(kQnWarps * 32), smem, st, qkv, bias, q_norm, k_norm, eps, inv_freq, rot, m, q_out,
             kc, vc, heads, kv_heads, D, block_size, qkv_stride, q_stride);
}

}  // namespace rb200

using namespace rb200;

extern "C" int rb200_qkv_norm_post(const float* qkv, int qkv_stride, const float* bias, const float* q_norm, const float* k_norm,
                                   float eps, const float* inv_freq, int rot_dim, const rb200_token_meta* m, int T, float* q_out,
                                   int q_stride, void* k_pool, void* v_pool, int heads, int kv_heads, int head_dim, int block_size,
                                   void* stream) {
  return guarded([&] {
    RB_REQUIRE(T >= 0 && heads > 0 && kv_heads > 0 && block_size > 0, "qkv_norm_post: bad shape");
    RB_REQUIRE(head_dim > 0 && head_dim % 2 == 0 && head_dim <= 256, "qkv_norm_post: head_dim must be even and at most 256");
    RB_REQUIRE(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= head_dim, "qkv_norm_post: rot_dim must be even and at most head_dim");
    const long long q_dim = static_cast<long long>(heads) * head_dim, row = q_dim + 2LL * kv_heads * head_dim;
    RB_REQUIRE(qkv_stride >= row && q_stride >= q_dim, "qkv_norm_post: row strides too small");
    RB_REQUIRE(eps >= 0.0f, "qkv_norm_post: eps must not be negative");
    if (T == 0) return 0;
    RB_REQUIRE(qkv && q_out && k_pool && v_pool && m && m->pos && m->seq && m->table_off && m->tables && (rot_dim == 0 || inv_freq),
               "qkv_norm_post: null argument");
    RB_REQUIRE(static_cast<const void*>(qkv) != q_out || qkv_stride == q_stride, "qkv_norm_post: q in place needs the same stride");
    launch_qkv_norm_post(qkv, qkv_stride, bias, q_norm, k_norm, eps, inv_freq, rot_dim,
                         TokenMeta{m->pos, m->seq, m->table_off, m->tables}, T, q_out, q_stride, static_cast<__half*>(k_pool),
                         static_cast<__half*>(v_pool), heads, kv_heads, head_dim, block_size, as_stream(stream));
    RB_CUDA(cudaGetLastError());
    return 0;
  });
}
