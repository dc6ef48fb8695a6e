// Norms of the query and key heads, rotation and paged append in one pass over the projection's
// output (qkv_post_kernel of small_ops.cu for models that normalise their heads first).
//
//   y = x * rsqrt(mean(x^2) + eps) * w      per head, x = projection + bias, sums in float32
//   (a, b) -> (a cos - b sin, b cos + a sin)  on the pairs (i, i + rot/2) of y
//
// Every value is read once and written once: 4 (Q + 2 KV) bytes of a token come in, 4 Q + 4 KV go
// out, so the kernels are bound by memory, and by latency for a few tokens. Heads of 32, 64, 128 or 256 values
// that are rotated whole or by half take qkv_norm_pair_kernel; other heads whose rows are whole 16-byte
// vectors qkv_norm_vec_kernel; the rest (head_dim not a multiple of 4, rot_dim not of 8, unaligned rows)
// qkv_norm_post_kernel.
#include "kernels.h"

namespace rb200 {

namespace {

constexpr int kQnWarps = 8;       // of qkv_norm_post_kernel
constexpr int kQnRounds = 4;      // rounds of a warp in flight in qkv_norm_vec_kernel
constexpr int kQnPairRounds = 2;  // and in qkv_norm_pair_kernel

// cos and sin of pos * inv_freq. The product is taken in float64 (exact below position 2^29) and reduced there, in
// units of pi: its float32 rounding alone would be off by 4e-3 rad at position 131072. What is left, at most 1,
// rounds to float32 within 2^-24 of itself.
__device__ __forceinline__ void rotation(int pos, float inv_freq, float& c, float& s) {
  constexpr double kInvTwoPi = 0.15915494309189533577;
  const double turns = static_cast<double>(pos) * static_cast<double>(inv_freq) * kInvTwoPi;
  sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
}

// The values of a vector as two pairs, the operands of packed fp32 instructions.
struct Pair2 {
  float2 a, b;
};
__device__ __forceinline__ Pair2 pairs(const float4& v) { return {make_float2(v.x, v.y), make_float2(v.z, v.w)}; }
__device__ __forceinline__ Pair2 mul(const Pair2& x, const Pair2& y) { return {__fmul2_rn(x.a, y.a), __fmul2_rn(x.b, y.b)}; }
__device__ __forceinline__ Pair2 fma(const Pair2& x, const Pair2& y, const Pair2& z) {
  return {__ffma2_rn(x.a, y.a, z.a), __ffma2_rn(x.b, y.b, z.b)};
}
__device__ __forceinline__ Pair2 add(const Pair2& x, const Pair2& y) { return {__fadd2_rn(x.a, y.a), __fadd2_rn(x.b, y.b)}; }
__device__ __forceinline__ Pair2 all(float v) { return {make_float2(v, v), make_float2(v, v)}; }

// Heads of 8 LPH values. LPH lanes hold one, lane l its vectors l and l + LPH: rotated whole, a vector's partner is
// in the same lane; rotated by half, all that turns is in the first vectors and the partner LPH / 2 lanes
// away. A warp takes 32 / LPH heads at a time and has kQnPairRounds such rounds in flight. A CTA goes through
// tokens a grid apart: a token's position and page (three dependent loads) are looked up while the one before
// it is at work, its angles are computed under its row's loads. What kept a first form of this kernel (a
// head in 32 lanes, 126 instructions a head) at 139 us for 8 x 2048 tokens was instruction issue; hence
// two vectors a lane and packed arithmetic.
template <int LPH, bool HALF>
__global__ void __launch_bounds__(512, 2)
qkv_norm_pair_kernel(const float* qkv, const float* __restrict__ bias, const float* __restrict__ q_norm,
                     const float* __restrict__ k_norm, float eps, const float* __restrict__ inv_freq, TokenMeta m, int T, float* q_out,
                     __half* __restrict__ kc, __half* __restrict__ vc, int heads, int kv_heads, int bs, int qkv_stride, int q_stride) {
  constexpr int D = 8 * LPH, HPW = 32 / LPH, U = kQnPairRounds, kAngles = HALF ? D / 4 : D / 2;
  __shared__ __align__(16) float s_cos[2][kAngles], s_sin[2][kAngles];  // tokens in turn
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int sub = lane / LPH, l = lane % LPH, step = warps * HPW, total = heads + 2 * kv_heads;
  int t = blockIdx.x, seq = m.seq[t], p = m.pos[t], turn = 0;
  int block = seq >= 0 && p >= 0 ? m.tables[m.table_off[seq] + p / bs] : 0;
  while (true) {
    const int t_next = t + gridDim.x;
    const int seq_next = t_next < T ? m.seq[t_next] : -1, p_next = t_next < T ? m.pos[t_next] : -1;
    const bool next = seq_next >= 0 && p_next >= 0;
    int entry_next = -1;  // of the next token's page in the tables
    if (seq >= 0 && p >= 0) {  // else padding
      const float* src = qkv + static_cast<long long>(t) * qkv_stride + l * 4;
      float* dst = q_out + static_cast<long long>(t) * q_stride + l * 4;
      const long long page = (static_cast<long long>(block) * kv_heads * bs + p % bs) * D + l * 4;  // the slot in KV head 0
      Pair2 c, s, ns;  // this lane's cos, sin and -sin
      for (int h0 = warp * HPW + sub; h0 - sub < total; h0 += step * U) {
        float4 x[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = min(h0 + u * step, total - 1);  // behind the last head: read, not written
          x[u][0] = *reinterpret_cast<const float4*>(src + h * D);
          x[u][1] = *reinterpret_cast<const float4*>(src + h * D + D / 2);
        }
        if (h0 < step) {  // the first time round, which every warp makes
          for (int i = threadIdx.x; i < kAngles; i += blockDim.x) rotation(p, inv_freq[i], s_cos[turn][i], s_sin[turn][i]);
          __syncthreads();
          const int i = (HALF ? l & (LPH / 2 - 1) : l) * 4;
          c = pairs(*reinterpret_cast<const float4*>(&s_cos[turn][i]));
          s = pairs(*reinterpret_cast<const float4*>(&s_sin[turn][i]));
          ns = mul(s, all(-1.0f));
          if (HALF && l < LPH / 2) s = ns;  // what turns with the partner: -sin in the first half, sin in the second
          if (next) entry_next = m.table_off[seq_next] + p_next / bs;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * step;
          if (h - sub >= total) break;  // no head of this warp
          const bool is_q = h < heads, is_v = h >= heads + kv_heads;
          Pair2 y0 = pairs(x[u][0]), y1 = pairs(x[u][1]);
          if (bias && h < total) {
            y0 = add(y0, pairs(*reinterpret_cast<const float4*>(bias + h * D + l * 4)));
            y1 = add(y1, pairs(*reinterpret_cast<const float4*>(bias + h * D + D / 2 + l * 4)));
          }
          const float* w = is_q ? q_norm : (is_v ? nullptr : k_norm);
          if (HPW > 1 ? (q_norm || k_norm) : w != nullptr) {
            const Pair2 sq = fma(y1, y1, mul(y0, y0));
            float ss = (sq.a.x + sq.a.y) + (sq.b.x + sq.b.y);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (w) {
              const Pair2 scale = all(rsqrtf(ss * (1.0f / D) + eps));
              y0 = mul(y0, mul(scale, pairs(reinterpret_cast<const float4*>(w)[l])));
              y1 = mul(y1, mul(scale, pairs(reinterpret_cast<const float4*>(w)[l + LPH])));
            }
          }
          if constexpr (HALF) {
            Pair2 z;
            z.a.x = __shfl_xor_sync(0xffffffffu, y0.a.x, LPH / 2), z.a.y = __shfl_xor_sync(0xffffffffu, y0.a.y, LPH / 2);
            z.b.x = __shfl_xor_sync(0xffffffffu, y0.b.x, LPH / 2), z.b.y = __shfl_xor_sync(0xffffffffu, y0.b.y, LPH / 2);
            if (!is_v) y0 = fma(z, s, mul(y0, c));
          } else if (!is_v) {
            const Pair2 z = y0;
            y0 = fma(y1, ns, mul(y0, c));
            y1 = fma(z, s, mul(y1, c));
          }
          if (h >= total) continue;
          if (is_q) {
            *reinterpret_cast<float4*>(dst + h * D) = make_float4(y0.a.x, y0.a.y, y0.b.x, y0.b.y);
            *reinterpret_cast<float4*>(dst + h * D + D / 2) = make_float4(y1.a.x, y1.a.y, y1.b.x, y1.b.y);
          } else {
            __half* to = (is_v ? vc : kc) + page + static_cast<long long>(is_v ? h - heads - kv_heads : h - heads) * bs * D;
            *reinterpret_cast<uint2*>(to) = make_uint2(pack_half2(y0.a.x, y0.a.y), pack_half2(y0.b.x, y0.b.y));
            *reinterpret_cast<uint2*>(to + D / 2) = make_uint2(pack_half2(y1.a.x, y1.a.y), pack_half2(y1.b.x, y1.b.y));
          }
        }
      }
      turn ^= 1;
    }
    if (t_next >= T) break;
    if (next && entry_next < 0) entry_next = m.table_off[seq_next] + p_next / bs;  // this token was padding
    block = next ? m.tables[entry_next] : 0;
    t = t_next, seq = seq_next, p = p_next;
  }
}

// One CTA per token. A head is held by LPH lanes, lane l with the vectors (4 values) l and, with NV = 2,
// l + LPH; a warp takes 32 / LPH heads at a time and has U such rounds in flight, so that a token's
// whole row is under way before anything waits. The rotation angles and the page lookup (three
// dependent loads) run under those loads. The partner of a rotated vector is rot/8 vectors away, in
// another lane: it comes by shuffle.
template <int LPH, int NV>
__global__ void __launch_bounds__(512, 2)
qkv_norm_vec_kernel(const float* qkv, const float* __restrict__ bias, const float* __restrict__ q_norm,
                    const float* __restrict__ k_norm, float eps, const float* __restrict__ inv_freq, int rot, TokenMeta m,
                    float* q_out, __half* __restrict__ kc, __half* __restrict__ vc, int heads, int kv_heads, int D, int bs,
                    int qkv_stride, int q_stride) {
  constexpr int HPW = 32 / LPH, U = kQnRounds / NV;
  extern __shared__ float sm[];  // [rot/2] cos, [rot/2] -sin, [rot/2] sin
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, half = rot >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int sub = lane / LPH, l = lane % LPH, step = warps * HPW;
  const int vecs = D >> 2, h4 = rot >> 3;  // vectors of a head; how far a rotated vector's partner is
  const int total = heads + 2 * kv_heads;
  const int seq = m.seq[t], p = m.pos[t];
  const float* src = qkv + static_cast<long long>(t) * qkv_stride + l * 4;
  float* dst = q_out + static_cast<long long>(t) * q_stride + l * 4;
  const float inv_d = 1.0f / static_cast<float>(D);
  long long page = 0;       // first value of the token's slot in KV head 0
  float4 cs[NV], sn[NV];    // this lane's angles: y = x cos + partner * (-sin or sin)
  for (int h0 = warp * HPW + sub; h0 - sub < total; h0 += step * U) {
    float4 x[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * step;
#pragma unroll
      for (int n = 0; n < NV; ++n)
        x[u][n] = h < total && l + n * LPH < vecs ? *reinterpret_cast<const float4*>(src + h * D + n * LPH * 4)
                                                            : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (h0 < step) {  // the first time round, which every warp makes
      if (seq < 0 || p < 0) return;  // padding; looked at only here so that the row's loads do not wait for it
      for (int i = threadIdx.x; i < half; i += blockDim.x) {
        float c, s;
        rotation(p, inv_freq[i], c, s);
        sm[i] = c;
        sm[half + i] = -s;
        sm[2 * half + i] = s;
      }
      const int entry = p / bs;
      page = (static_cast<long long>(m.tables[m.table_off[seq] + entry]) * kv_heads * bs + (p - entry * bs)) * D;
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int v = l + n * LPH;
        cs[n] = make_float4(1.f, 1.f, 1.f, 1.f), sn[n] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (v < 2 * h4) {
          const int i = (v < h4 ? v : v - h4) * 4;
          cs[n] = *reinterpret_cast<const float4*>(sm + i);
          sn[n] = *reinterpret_cast<const float4*>(sm + (v < h4 ? half : 2 * half) + i);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * step;
      if (h - sub >= total) break;  // no head of this warp
      const bool is_q = h < heads, is_v = h >= heads + kv_heads, there = h < total;
      if (bias && there) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
          if (l + n * LPH < vecs) {
            const float4 b = *reinterpret_cast<const float4*>(bias + h * D + (l + n * LPH) * 4);
            x[u][n].x += b.x, x[u][n].y += b.y, x[u][n].z += b.z, x[u][n].w += b.w;
          }
      }
      if (HPW > 1 || !is_v) {  // with one head to a warp the branch is the warp's
        const float* w = is_q ? q_norm : (is_v ? nullptr : k_norm);
        if (q_norm || k_norm) {
          float ss = 0.f;
#pragma unroll
          for (int n = 0; n < NV; ++n)
            ss += x[u][n].x * x[u][n].x + x[u][n].y * x[u][n].y + x[u][n].z * x[u][n].z + x[u][n].w * x[u][n].w;
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if (w) {
            const float scale = rsqrtf(ss * inv_d + eps);
#pragma unroll
            for (int n = 0; n < NV; ++n)
              if (l + n * LPH < vecs) {
                const float4 g = reinterpret_cast<const float4*>(w)[l + n * LPH];
                x[u][n].x *= scale * g.x, x[u][n].y *= scale * g.y, x[u][n].z *= scale * g.z, x[u][n].w *= scale * g.w;
              }
          }
        }
        float4 z[NV];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          // the partner of vector v: v + h4 for the first h4 vectors, v - h4 for the next h4
          const int v = l + n * LPH, pv = v < h4 ? v + h4 : v - h4;
          const int from = sub * LPH + (pv & (LPH - 1));
          z[n].x = __shfl_sync(0xffffffffu, x[u][0].x, from), z[n].y = __shfl_sync(0xffffffffu, x[u][0].y, from);
          z[n].z = __shfl_sync(0xffffffffu, x[u][0].z, from), z[n].w = __shfl_sync(0xffffffffu, x[u][0].w, from);
          if constexpr (NV == 2) {
            const float4 z1 = make_float4(__shfl_sync(0xffffffffu, x[u][1].x, from), __shfl_sync(0xffffffffu, x[u][1].y, from),
                                          __shfl_sync(0xffffffffu, x[u][1].z, from), __shfl_sync(0xffffffffu, x[u][1].w, from));
            if (pv >= LPH) z[n] = z1;
          }
        }
        if (!is_v) {
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            if (l + n * LPH >= 2 * h4) continue;  // passes: its "partner" may hold anything
            x[u][n].x = x[u][n].x * cs[n].x + z[n].x * sn[n].x, x[u][n].y = x[u][n].y * cs[n].y + z[n].y * sn[n].y;
            x[u][n].z = x[u][n].z * cs[n].z + z[n].z * sn[n].z, x[u][n].w = x[u][n].w * cs[n].w + z[n].w * sn[n].w;
          }
        }
      }
      if (!there) continue;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        if (l + n * LPH >= vecs) continue;
        if (is_q) {
          *reinterpret_cast<float4*>(dst + h * D + n * LPH * 4) = x[u][n];
        } else {
          const int kvh = is_v ? h - heads - kv_heads : h - heads;
          *reinterpret_cast<uint2*>((is_v ? vc : kc) + page + static_cast<long long>(kvh) * bs * D + (l + n * LPH) * 4) =
              make_uint2(pack_half2(x[u][n].x, x[u][n].y), pack_half2(x[u][n].z, x[u][n].w));
        }
      }
    }
  }
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
  auto aligned = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (D % 4 == 0 && rot % 8 == 0 && qkv_stride % 4 == 0 && q_stride % 4 == 0 && aligned(qkv, 16) && aligned(q_out, 16) &&
      aligned(bias, 16) && aligned(q_norm, 16) && aligned(k_norm, 16) && aligned(kc, 8) && aligned(vc, 8)) {
    // A few tokens: as many warps as have the whole row in flight, the shortest way through. Many: fewer, with the
    // rounds even among them, so that more tokens are under way on an SM. At 32 + 2 x 8 heads of 128, 8 x 2048
    // tokens take 113 us with six warps, 118 with eight, 126 with four.
    const bool many = T > 2 * sm_count();
    auto warps_for = [&](int per_warp, int in_flight, int most) {
      const int turns = div_up(heads + 2 * kv_heads, per_warp * in_flight);  // of one warp, for the whole row
      return many ? div_up(turns, div_up(turns, most)) : std::min(16, turns);
    };
    if ((D == 32 || D == 64 || D == 128 || D == 256) && (rot == D || rot == D / 2)) {
      const bool half = rot != D;
      auto kernel = D == 256   ? (half ? qkv_norm_pair_kernel<32, true> : qkv_norm_pair_kernel<32, false>)
                    : D == 128 ? (half ? qkv_norm_pair_kernel<16, true> : qkv_norm_pair_kernel<16, false>)
                    : D == 64  ? (half ? qkv_norm_pair_kernel<8, true> : qkv_norm_pair_kernel<8, false>)
                               : (half ? qkv_norm_pair_kernel<4, true> : qkv_norm_pair_kernel<4, false>);
      const int warps = warps_for(256 / D, kQnPairRounds, 6);
      const int ctas = many ? std::min(T, sm_count() * (1024 / (warps * 32))) : T;  // what 64 registers a thread let an SM hold
      launch_pdl(kernel, dim3(ctas), dim3(warps * 32), 0, st, qkv, bias, q_norm, k_norm, eps, inv_freq, m, T, q_out, kc, vc, heads, kv_heads,
                 block_size, qkv_stride, q_stride);
      return;
    }
    const int lanes = D > 64 ? 32 : (D > 32 ? 16 : 8), nv = D > 128 ? 2 : 1;
    const int warps = warps_for(32 / lanes, kQnRounds / nv, 8);
    auto kernel = nv == 2       ? qkv_norm_vec_kernel<32, 2>
                  : lanes == 32 ? qkv_norm_vec_kernel<32, 1>
                  : lanes == 16 ? qkv_norm_vec_kernel<16, 1>
                                : qkv_norm_vec_kernel<8, 1>;
    launch_pdl(kernel, dim3(T), dim3(warps * 32), rot / 2 * 3 * sizeof(float), st, qkv, bias, q_norm, k_norm, eps, inv_freq, rot, m, q_out, kc,
               vc, heads, kv_heads, D, block_size, qkv_stride, q_stride);
    return;
  }
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
    // a single row has no stride: torch, for one, reports a row's own width for a one-row view of wider rows
    RB_REQUIRE(static_cast<const void*>(qkv) != q_out || qkv_stride == q_stride || T == 1, "qkv_norm_post: q in place needs the same stride");
    launch_qkv_norm_post(qkv, qkv_stride, bias, q_norm, k_norm, eps, inv_freq, rot_dim,
                         TokenMeta{m->pos, m->seq, m->table_off, m->tables}, T, q_out, q_stride, static_cast<__half*>(k_pool),
                         static_cast<__half*>(v_pool), heads, kv_heads, head_dim, block_size, as_stream(stream));
    RB_CUDA(cudaGetLastError());
    return 0;
  });
}
