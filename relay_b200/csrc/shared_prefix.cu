// Decode attention for groups of sequences whose contexts begin with the same keys. With P shared
// keys and s_i keys of its own, token i's output is
//
//   o_i = (e^(m_p - M) l_p o_p + e^(m_s - M) l_s o_s) / (e^(m_p - M) l_p + e^(m_s - M) l_s),  M = max(m_p, m_s)
//
// with (m, l, o) the running maximum, sum and output of the softmax over the P shared keys and over
// the s_i own ones. The shared part has the same keys for every token of the group, so it is a
// product of matrices: (tokens x heads of a KV head) rows against P keys, each key read once per row
// tile instead of once per token. Two kernels:
//
//  * umma_prefix_kernel (umma_prefix.cu; head sizes 64 and 128, block sizes that are multiples of 16) or
//    prefix_mma_kernel (the other layouts): a CTA takes 128 or 64 rows (token, head) of one group and
//    KV head and a slice of the shared keys, and leaves a partial (m, l, o) per row;
//  * suffix_kernel: a CTA takes one token and KV head (or a slice of its own keys, the slices
//    as one cluster), streams the keys behind the prefix, adds the partials of the prefix and writes
//    the output. It starts under the tail of the first kernel and waits for it only ahead of the join.
//
// Scores take q in full (two fp16 halves, split_half2); the weights round to fp16 for the second product.
#include "attn_tiles.cuh"
#include "kernels.h"
#include "prefix_groups.cuh"
#include "tcgen05.cuh"

namespace rb200 {

namespace {

// ---------------------------------------------------------------------------------------
// The shared keys
// ---------------------------------------------------------------------------------------

constexpr int kPxRows = 64;  // rows of a CTA, 16 to a warp
constexpr int kPxKeys = 64;  // keys per shared-memory stage, two stages

template <int D>
constexpr size_t prefix_smem_bytes() {
  return static_cast<size_t>(2) * 2 * kPxKeys * D * sizeof(__half);
}

template <int D>
__global__ void __launch_bounds__(128)
prefix_mma_kernel(const float* __restrict__ q, TokenMeta m, Groups gr, const __half* __restrict__ kc, const __half* __restrict__ vc,
                  Partials part, int heads, int kv_heads, int bs, int bs_shift, int q_stride, float scale_log2e) {
  constexpr int CH = D / 8;
  constexpr int STAGE_HALVES = 2 * kPxKeys * D;  // K tile then V tile
  extern __shared__ __align__(128) unsigned char smem_raw[];
  const uint32_t smem0 = smem_u32(smem_raw);
  pdl_wait();
  pdl_trigger();  // behind the wait: what suffix_kernel reads early is then complete
  const int G = heads / kv_heads, kvh = blockIdx.y;
  int g = 0, tile = 0, lo, hi;
  if (!find_tile(gr, G, kPxRows, blockIdx.x, g, tile)) return;
  group_bounds(gr, g, lo, hi);
  const Prefix px = prefix_of(gr, m, g, lo, hi);
  const int slice = slice_of(px.keys, part.parts);
  const int k0 = blockIdx.z * slice;
  if (px.keys == 0 || k0 >= px.keys) return;
  const int k1 = min(px.keys, k0 + slice);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t4 = lane & 3;
  // This thread's two rows: entry and head, and how many of the shared keys its context holds.
  int entry[2], head[2], limit[2];
  const float* qrow[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int idx = tile * kPxRows + warp * 16 + gid + 8 * r;
    entry[r] = lo + idx / G;
    head[r] = kvh * G + idx % G;
    const int tok = entry[r] < hi ? gr.decode_tokens[entry[r]] : -1;
    limit[r] = tok >= 0 ? min(px.keys, m.pos[tok] + 1) : 0;
    if (tok < 0) entry[r] = -1;
    qrow[r] = q + static_cast<long long>(max(tok, 0)) * q_stride + head[r] * D;
  }
  uint32_t qf[D / 16][4], ql[D / 16][4];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const int d0 = kk * 16 + 2 * t4;
    float2 v[2][2] = {};
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (entry[r] >= 0) {
        v[r][0] = *reinterpret_cast<const float2*>(qrow[r] + d0);
        v[r][1] = *reinterpret_cast<const float2*>(qrow[r] + d0 + 8);
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) split_half2(v[e & 1][e >> 1].x, v[e & 1][e >> 1].y, qf[kk][e], ql[kk][e]);
  }

  auto load_stage = [&](int kt, int stage) {
    const uint32_t kdst = smem0 + static_cast<uint32_t>(stage) * STAGE_HALVES * 2;
    const uint32_t vdst = kdst + kPxKeys * D * 2;
    const int key0 = k0 + kt * kPxKeys;
    for (int idx = threadIdx.x; idx < kPxKeys * CH; idx += blockDim.x) {
      const int row = idx / CH, c = idx % CH;
      const bool ok = key0 + row < k1;
      const long long base = ok ? key_offset(px.table, 0, key0 + row, bs, bs_shift, kv_heads, kvh, D) : 0;
      const int bytes = ok ? 16 : 0;
      const uint32_t off = static_cast<uint32_t>(swz<CH>(row, c)) * 16;
      cp_async16_zfill(kdst + off, kc + base + c * 8, bytes);
      cp_async16_zfill(vdst + off, vc + base + c * 8, bytes);
    }
  };

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

  const int nkt = (k1 - k0 + kPxKeys - 1) / kPxKeys;
  load_stage(0, 0);
  cp_async_commit();
  for (int kt = 0; kt < nkt; ++kt) {
    if (kt + 1 < nkt) load_stage(kt + 1, (kt + 1) & 1);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t ktile = smem0 + static_cast<uint32_t>(kt & 1) * STAGE_HALVES * 2;
    const uint32_t vtile = ktile + kPxKeys * D * 2;
    const int key0 = k0 + kt * kPxKeys;
    float s[kPxKeys / 8][4];
#pragma unroll
    for (int kp = 0; kp < kPxKeys / 16; ++kp) {
      float s2[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      qk_16x16<D>(s2, qf, ktile + kp * 16 * D * 2, lane);
      qk_16x16<D>(s2, ql, ktile + kp * 16 * D * 2, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[2 * kp][e] = s2[0][e];
        s[2 * kp + 1][e] = s2[1][e];
      }
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
    const int see0 = min(limit[0], k1), see1 = min(limit[1], k1);
#pragma unroll
    for (int nt = 0; nt < kPxKeys / 8; ++nt) {
      const int ka = key0 + nt * 8 + 2 * t4;
      s[nt][0] = ka < see0 ? s[nt][0] * scale_log2e : -INFINITY;
      s[nt][1] = ka + 1 < see0 ? s[nt][1] * scale_log2e : -INFINITY;
      s[nt][2] = ka < see1 ? s[nt][2] * scale_log2e : -INFINITY;
      s[nt][3] = ka + 1 < see1 ? s[nt][3] * scale_log2e : -INFINITY;
      mx0 = fmaxf(mx0, fmaxf(s[nt][0], s[nt][1]));
      mx1 = fmaxf(mx1, fmaxf(s[nt][2], s[nt][3]));
    }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    // a row that has seen no key yet keeps the maximum -inf; its exponents then refer to 0
    const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
    const float r0 = n0 == -INFINITY ? 0.f : n0, r1 = n1 == -INFINITY ? 0.f : n1;
    const float c0 = fast_exp2(m0 - r0), c1 = fast_exp2(m1 - r1);
    m0 = n0;
    m1 = n1;
    float sum0 = 0.f, sum1 = 0.f;
    uint32_t pa[kPxKeys / 16][4];
#pragma unroll
    for (int kp = 0; kp < kPxKeys / 16; ++kp) {
      const float a0 = fast_exp2(s[2 * kp][0] - r0), a1 = fast_exp2(s[2 * kp][1] - r0);
      const float b0 = fast_exp2(s[2 * kp][2] - r1), b1 = fast_exp2(s[2 * kp][3] - r1);
      const float a2 = fast_exp2(s[2 * kp + 1][0] - r0), a3 = fast_exp2(s[2 * kp + 1][1] - r0);
      const float b2 = fast_exp2(s[2 * kp + 1][2] - r1), b3 = fast_exp2(s[2 * kp + 1][3] - r1);
      sum0 += (a0 + a1) + (a2 + a3);
      sum1 += (b0 + b1) + (b2 + b3);
      // P is rounded to fp16 for the tensor cores: at most 2^-11 of each weight, all of them in [0, 1]
      pa[kp][0] = pack_half2(a0, a1);
      pa[kp][1] = pack_half2(b0, b1);
      pa[kp][2] = pack_half2(a2, a3);
      pa[kp][3] = pack_half2(b2, b3);
    }
    l0 = l0 * c0 + sum0;
    l1 = l1 * c1 + sum1;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      o[i][0] *= c0;
      o[i][1] *= c0;
      o[i][2] *= c1;
      o[i][3] *= c1;
    }
#pragma unroll
    for (int kp = 0; kp < kPxKeys / 16; ++kp) pv_16x16<D>(o, pa[kp], vtile + kp * 16 * D * 2, lane);
    __syncthreads();
  }

  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (entry[r] < 0) continue;
    const long long at = (static_cast<long long>(entry[r]) * heads + head[r]) * part.parts + blockIdx.z;
    float* dst = part.o + at * D + 2 * t4;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    if (t4 == 0) *reinterpret_cast<float2*>(part.ml + at * 2) = r == 0 ? make_float2(m0, l0) : make_float2(m1, l1);
  }
}

// ---------------------------------------------------------------------------------------
// Each sequence's own keys, and the join
// ---------------------------------------------------------------------------------------

constexpr int kSxWarps = 4;   // independent tile workers per CTA
constexpr int kSxStages = 3;  // 16-key tiles in flight per warp

template <int D>
constexpr size_t suffix_smem_bytes() {
  return static_cast<size_t>(kSxWarps) * kSxStages * 2 * 16 * D * sizeof(__half);
}

// CONTIG: block_size is a multiple of 16, so an aligned 16-key tile is one contiguous run of a page.
// WIDE: more than 8 query heads per KV head (rows 8..15 of the M tile are real heads).
// gridDim.z CTAs share the token's own keys as one cluster and join through distributed shared memory.
template <int D, bool CONTIG, bool WIDE>
__global__ void __launch_bounds__(kSxWarps * 32, 2)
suffix_kernel(const float* __restrict__ q, TokenMeta m, Groups gr, const __half* __restrict__ kc, const __half* __restrict__ vc,
              Partials px, __half* __restrict__ out, int heads, int kv_heads, int bs, int bs_shift, int q_stride, int o_stride,
              float scale_log2e, int early) {
  constexpr int CH = D / 8;
  constexpr int TILE_HALVES = 16 * D;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ float s_m[kSxWarps][16], s_l[kSxWarps][16];
  __shared__ float j_m[16], j_l[16];  // this CTA's (max, sum) per head

  pdl_trigger();
  // `early`: the kernel ahead is a prefix kernel, all of whose CTAs have waited for what came before them, so
  // the metadata, q and the pages are complete (read from L2); only its partials have to be waited for.
  if (!early) pdl_wait();
  const int di = blockIdx.x, kvh = blockIdx.y, slices = gridDim.z, rank = blockIdx.z;
  const int tok = __ldcg(gr.decode_tokens + di);
  const int g = group_of(gr, di);
  if (tok < 0 || g < 0) {  // padding: the whole cluster leaves
    pdl_wait();
    return;
  }
  int lo, hi;
  group_bounds(gr, g, lo, hi);
  const int P = prefix_of(gr, m, g, lo, hi).keys;
  const int ctx = max(__ldcg(m.pos + tok) + 1, 0), start = min(P, ctx);
  // Tiles start at multiples of 16 where a tile has to be a run of a page; keys before `start` are masked.
  const int base = CONTIG ? start & ~15 : start;
  const int per = ((ctx - base + slices - 1) / slices + 15) & ~15;
  const int k0 = min(base + rank * per, ctx), k1 = min(k0 + per, ctx);
  const int ntiles = (k1 - k0 + 15) >> 4;
  const int* table = ctx > 0 ? m.tables + __ldcg(m.table_off + __ldcg(m.seq + tok)) : nullptr;

  const int G = heads / kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, t4 = lane & 3;

  // The heads' queries as A fragments: rows 0..7 hi of heads 0..7; rows 8..15 hi of heads 8..15 (then the lo
  // halves need fragments of their own) or, with up to 8 heads, their lo, so that one product makes both.
  uint32_t qf[D / 16][4], ql[WIDE ? D / 16 : 1][4];
  {
    const float* q0 = q + static_cast<long long>(tok) * q_stride + (kvh * G) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d0 = kk * 16 + 2 * t4 + 8 * e;
        float2 a = make_float2(0.f, 0.f), b = a;
        if (gid < G) a = __ldcg(reinterpret_cast<const float2*>(q0 + gid * D + d0));
        if constexpr (WIDE) {
          if (gid + 8 < G) b = __ldcg(reinterpret_cast<const float2*>(q0 + (gid + 8) * D + d0));
          split_half2(a.x, a.y, qf[kk][2 * e], ql[kk][2 * e]);
          split_half2(b.x, b.y, qf[kk][2 * e + 1], ql[kk][2 * e + 1]);
        } else {
          split_half2(a.x, a.y, qf[kk][2 * e], qf[kk][2 * e + 1]);
        }
      }
    }
  }

  __half* ring = reinterpret_cast<__half*>(smem_raw) + static_cast<size_t>(warp) * kSxStages * 2 * TILE_HALVES;
  const uint32_t ring_u32 = smem_u32(ring);
  // Tiles warp, warp + 4, ... of the slice belong to this warp. Where a tile lies in one page, its
  // block id waits in a register: 32 tiles' ids at a time, one per lane, the next 32 on their way.
  const int my_tiles = ntiles > warp ? (ntiles - warp + kSxWarps - 1) / kSxWarps : 0;
  auto fetch_ids = [&](int j0) {
    const int j = j0 + lane, key = k0 + (warp + j * kSxWarps) * 16;
    return CONTIG && j < my_tiles ? __ldcg(table + (bs_shift >= 0 ? key >> bs_shift : key / bs)) : 0;
  };
  int ids = fetch_ids(0), ids_next = fetch_ids(32);
  auto load_tile = [&](int j) {
    const uint32_t kdst = ring_u32 + static_cast<uint32_t>(j % kSxStages) * 2 * TILE_HALVES * 2;
    const uint32_t vdst = kdst + TILE_HALVES * 2;
    const int key0 = k0 + (warp + j * kSxWarps) * 16;
    const int nvalid = min(16, k1 - key0);
    if constexpr (CONTIG) {
      if (j > 0 && (j & 31) == 0) {
        ids = ids_next;
        ids_next = fetch_ids(j + 32);
      }
      const long long block = __shfl_sync(0xffffffffu, ids, j & 31);
      const int slot = bs_shift >= 0 ? key0 & (bs - 1) : key0 % bs;
      const long long at = ((block * kv_heads + kvh) * bs + slot) * D;
#pragma unroll
      for (int idx = lane; idx < 16 * CH; idx += 32) {
        const int row = idx / CH, c = idx % CH;
        const int bytes = row < nvalid ? 16 : 0;
        const uint32_t off = static_cast<uint32_t>(swz<CH>(row, c)) * 16;
        cp_async16_zfill(kdst + off, kc + at + (bytes ? idx * 8 : 0), bytes);
        cp_async16_zfill(vdst + off, vc + at + (bytes ? idx * 8 : 0), bytes);
      }
    } else {
#pragma unroll
      for (int idx = lane; idx < 16 * CH; idx += 32) {
        const int row = idx / CH, c = idx % CH;
        const bool ok = row < nvalid;
        const long long at = ok ? key_offset(table, 0, key0 + row, bs, bs_shift, kv_heads, kvh, D) : 0;
        const int bytes = ok ? 16 : 0;
        const uint32_t off = static_cast<uint32_t>(swz<CH>(row, c)) * 16;
        cp_async16_zfill(kdst + off, kc + at + c * 8, bytes);
        cp_async16_zfill(vdst + off, vc + at + c * 8, bytes);
      }
    }
  };

#pragma unroll
  for (int s = 0; s < kSxStages - 1; ++s) {
    if (s < my_tiles) load_tile(s);
    cp_async_commit();
  }

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float mr[2] = {-INFINITY, -INFINITY}, lr[2] = {0.f, 0.f};  // rows gid and gid + 8, log2 domain

  for (int j = 0; j < my_tiles; ++j) {
    cp_async_wait<kSxStages - 2>();
    __syncwarp();
    if (j + kSxStages - 1 < my_tiles) load_tile(j + kSxStages - 1);
    cp_async_commit();

    const uint32_t ktile = ring_u32 + static_cast<uint32_t>(j % kSxStages) * 2 * TILE_HALVES * 2;
    const uint32_t vtile = ktile + TILE_HALVES * 2;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    qk_16x16<D>(s, qf, ktile, lane);
    if constexpr (WIDE) {
      qk_16x16<D>(s, ql, ktile, lane);
    } else {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        s[nt][0] += s[nt][2];
        s[nt][1] += s[nt][3];
      }
    }

    const int key0 = k0 + (warp + j * kSxWarps) * 16 + 2 * t4;
    float corr[2];
    uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int r = 0; r < (WIDE ? 2 : 1); ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + (e >> 1) * 8 + (e & 1);
        float& x = s[e >> 1][2 * r + (e & 1)];
        x = key >= start && key < k1 ? x * scale_log2e : -INFINITY;
        mx = fmaxf(mx, x);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(mr[r], mx);
      const float ref = mn == -INFINITY ? 0.f : mn;  // only masked keys so far
      corr[r] = fast_exp2(mr[r] - ref);
      mr[r] = mn;
      const float p0 = fast_exp2(s[0][2 * r] - ref), p1 = fast_exp2(s[0][2 * r + 1] - ref);
      const float p2 = fast_exp2(s[1][2 * r] - ref), p3 = fast_exp2(s[1][2 * r + 1] - ref);
      lr[r] = lr[r] * corr[r] + ((p0 + p1) + (p2 + p3));
      pa[r] = pack_half2(p0, p1);
      pa[r + 2] = pack_half2(p2, p3);
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      o[i][0] *= corr[0];
      o[i][1] *= corr[0];
      if constexpr (WIDE) {
        o[i][2] *= corr[1];
        o[i][3] *= corr[1];
      }
    }
    pv_16x16<D>(o, pa, vtile, lane);
  }
  cp_async_wait<0>();
  __syncwarp();

  // The warps' (m, l, o) meet in shared memory (each warp reuses its own ring).
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    lr[r] += __shfl_xor_sync(0xffffffffu, lr[r], 1);
    lr[r] += __shfl_xor_sync(0xffffffffu, lr[r], 2);
    if (t4 == 0) {
      s_m[warp][gid + 8 * r] = mr[r];
      s_l[warp][gid + 8 * r] = lr[r];
    }
  }
  float* os = reinterpret_cast<float*>(ring);  // [16][D] floats = 64 D bytes <= the ring's 192 D
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    *reinterpret_cast<float2*>(os + gid * D + i * 8 + 2 * t4) = make_float2(o[i][0], o[i][1]);
    if constexpr (WIDE) *reinterpret_cast<float2*>(os + (gid + 8) * D + i * 8 + 2 * t4) = make_float2(o[i][2], o[i][3]);
  }
  if (early) pdl_wait();
  __syncthreads();

  const float* os_all = reinterpret_cast<const float*>(smem_raw);
  constexpr int WARP_FLOATS = kSxStages * TILE_HALVES;  // ring size of one warp in floats
  float* own = reinterpret_cast<float*>(smem_raw) + 16 * D;  // behind warp 0's own partial, where nothing is read any more
  const int n_px = min(px.parts, P > 0 ? (P + slice_of(P, px.parts) - 1) / slice_of(P, px.parts) : 0);
  // Adds the prefix's partials of head r, value d, in the order of the slices, and divides.
  auto finish = [&](int r, int d, float M, float L, float acc) {
    const long long at = (static_cast<long long>(di) * heads + kvh * G + r) * px.parts;
    float top = M;
    for (int p = 0; p < n_px; ++p) top = fmaxf(top, px.ml[(at + p) * 2]);
    if (top == -INFINITY) top = 0.f;  // no key at all: the sums below are 0
    const float e = fast_exp2(M - top);
    acc *= e;
    L *= e;
    for (int p = 0; p < n_px; ++p) {
      const float2 ml = *reinterpret_cast<const float2*>(px.ml + (at + p) * 2);
      const float w = fast_exp2(ml.x - top);
      acc += w * px.o[(at + p) * D + d];
      L += w * ml.y;
    }
    out[static_cast<long long>(tok) * o_stride + (kvh * G + r) * D + d] = __float2half_rn(L == 0.f ? 0.f : acc / L);
  };
  for (int idx = threadIdx.x; idx < G * D; idx += blockDim.x) {
    const int r = idx / D, d = idx - r * D;
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kSxWarps; ++w) M = fmaxf(M, s_m[w][r]);
    const float ref = M == -INFINITY ? 0.f : M;
    float acc = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < kSxWarps; ++w) {
      const float e = fast_exp2(s_m[w][r] - ref);
      acc += e * os_all[w * WARP_FLOATS + r * D + d];
      L += e * s_l[w][r];
    }
    if (slices == 1) {
      finish(r, d, M, L, acc);
    } else {
      own[idx] = acc;
      if (d == 0) {
        j_m[r] = M;
        j_l[r] = L;
      }
    }
  }
  if (slices > 1) {
    // CTA `rank` of the cluster finishes the heads r with r % slices == rank, reading the members in
    // rank order: the result is the same on every run.
    tc::cluster_sync_all();
    for (int idx = threadIdx.x; idx < G * D; idx += blockDim.x) {
      const int r = idx / D, d = idx - r * D;
      if (r % slices != rank) continue;
      float M = -INFINITY;
      for (int p = 0; p < slices; ++p) M = fmaxf(M, tc::ld_dsmem_f32(smem_u32(&j_m[r]), p));
      const float ref = M == -INFINITY ? 0.f : M;
      float acc = 0.f, L = 0.f;
      for (int p = 0; p < slices; ++p) {
        const float e = fast_exp2(tc::ld_dsmem_f32(smem_u32(&j_m[r]), p) - ref);
        acc += e * tc::ld_dsmem_f32(smem_u32(own + idx), p);
        L += e * tc::ld_dsmem_f32(smem_u32(&j_l[r]), p);
      }
      finish(r, d, M, L, acc);
    }
    tc::cluster_sync_all();  // nobody leaves while a peer may still read its shared memory
  }
}

// ---------------------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------------------

// At most this many row tiles of `rows` rows: a group rounds up by less than one tile.
long long row_tiles(const AttnShape& s, int n_decode, int n_groups, int rows) {
  return (static_cast<long long>(n_decode) * (s.heads / s.kv_heads) + static_cast<long long>(n_groups) * (rows - 1)) / rows;
}

// Into how many slices the longest prefix is cut: the number that keeps the last SM busy for the shortest
// time, a CTA costing its keys and as much as kSetupKeys more to start and to leave its partials.
constexpr int kSetupKeys = 256;
int prefix_parts(long long ctas, long long slots, int max_prefix) {
  int best = 1;
  long long least = -1;
  for (int p = 1; p <= 64 && (p == 1 || max_prefix > (p - 1) * 2 * kPrefixSlice); ++p) {
    const long long keys = (div_up(max_prefix, p) + kPrefixSlice - 1LL) / kPrefixSlice * kPrefixSlice;
    const long long cost = (ctas * p + slots - 1) / slots * (keys + kSetupKeys);
    if (least < 0 || cost < least) {
      least = cost;
      best = p;
    }
  }
  return best;
}

int prefix_rows(const AttnShape& s) { return umma_prefix_usable(s) ? kUmmaPrefixRows : kPxRows; }

// One CTA of the tcgen05 kernel fits an SM, two of the other.
int parts_of(const AttnShape& s, int n_decode, int n_groups, int max_prefix) {
  const long long ctas = row_tiles(s, n_decode, n_groups, prefix_rows(s)) * s.kv_heads;
  return prefix_parts(ctas, (umma_prefix_usable(s) ? 1LL : 2LL) * sm_count(), max_prefix);
}

template <int D, bool CONTIG, bool WIDE>
void launch_suffix(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const __half* kc, const __half* vc,
                   const Partials& px, __half* out, int slices, float scale_log2e, int early, cudaStream_t st) {
  static PerDeviceOnce once;
  auto kernel = suffix_kernel<D, CONTIG, WIDE>;
  if (once.first())
    RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(suffix_smem_bytes<D>())));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(gr.n_decode, s.kv_heads, slices);
  cfg.blockDim = dim3(kSxWarps * 32);
  cfg.dynamicSmemBytes = suffix_smem_bytes<D>();
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = slices;
  cfg.attrs = attr;
  cfg.numAttrs = slices > 1 ? 2 : 1;
  count_launch();
  const int heads = s.heads, kv_heads = s.kv_heads, bs = s.block_size, shift = shift_of(s.block_size), qs = s.q_stride, os = s.o_stride;
  RB_CUDA(cudaLaunchKernelEx(&cfg, kernel, q, m, gr, kc, vc, px, out, heads, kv_heads, bs, shift, qs, os, scale_log2e, early));
}

template <int D>
void launch_d(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, int max_prefix, int max_suffix,
              const __half* kc, const __half* vc, Partials px, __half* out, cudaStream_t st) {
  const float scale_log2e = kLog2e / sqrtf(static_cast<float>(D));
  const int early = max_prefix > 0;
  if (early) {
    const long long tiles = row_tiles(s, gr.n_decode, gr.n_groups, prefix_rows(s));
    if (umma_prefix_usable(s)) {
      launch_umma_prefix(s, q, m, gr, kc, vc, px, static_cast<int>(tiles), st);
    } else {
      static PerDeviceOnce once;
      auto kernel = prefix_mma_kernel<D>;
      if (once.first())
        RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(prefix_smem_bytes<D>())));
      count_launch();
      launch_pdl(kernel, dim3(static_cast<unsigned>(tiles), s.kv_heads, px.parts), dim3(128), prefix_smem_bytes<D>(), st, q, m, gr, kc, vc,
                 px, s.heads, s.kv_heads, s.block_size, shift_of(s.block_size), s.q_stride, scale_log2e);
    }
  }
  // A few tokens with many keys of their own: up to eight CTAs of at least 128 keys for each (token, KV head).
  const long long pairs = static_cast<long long>(gr.n_decode) * s.kv_heads;
  int slices = 1;
  while (slices < 8 && pairs * slices * 2 <= 2LL * sm_count() && max_suffix / (slices * 2) >= 128) slices *= 2;
  const bool contig = s.block_size % 16 == 0, wide = s.heads / s.kv_heads > 8;
  if (contig && !wide) launch_suffix<D, true, false>(s, q, m, gr, kc, vc, px, out, slices, scale_log2e, early, st);
  else if (contig) launch_suffix<D, true, true>(s, q, m, gr, kc, vc, px, out, slices, scale_log2e, early, st);
  else if (!wide) launch_suffix<D, false, false>(s, q, m, gr, kc, vc, px, out, slices, scale_log2e, early, st);
  else launch_suffix<D, false, true>(s, q, m, gr, kc, vc, px, out, slices, scale_log2e, early, st);
}

}  // namespace

size_t shared_prefix_scratch_bytes(const AttnShape& s, int n_decode, int n_groups, int max_prefix) {
  if (n_decode <= 0 || n_groups <= 0) return 0;
  return static_cast<size_t>(n_decode) * s.heads * parts_of(s, n_decode, n_groups, max_prefix) * (s.D + 2) * sizeof(float);
}

void launch_shared_prefix_attention(const AttnShape& s, const float* q, const TokenMeta& m, const int* decode_tokens, int n_decode,
                                    const int* group_off, const int* prefix_len, int n_groups, int max_prefix, int max_suffix,
                                    const __half* kc, const __half* vc, float* scratch, __half* out, cudaStream_t st) {
  if (n_decode == 0) return;
  const Groups gr{decode_tokens, group_off, max_prefix > 0 ? prefix_len : nullptr, n_decode, n_groups};
  Partials px;
  px.parts = parts_of(s, n_decode, n_groups, max_prefix);
  px.o = scratch;
  px.ml = scratch + static_cast<size_t>(n_decode) * s.heads * px.parts * s.D;
  switch (s.D) {
    case 16: launch_d<16>(s, q, m, gr, max_prefix, max_suffix, kc, vc, px, out, st); break;
    case 32: launch_d<32>(s, q, m, gr, max_prefix, max_suffix, kc, vc, px, out, st); break;
    case 64: launch_d<64>(s, q, m, gr, max_prefix, max_suffix, kc, vc, px, out, st); break;
    case 128: launch_d<128>(s, q, m, gr, max_prefix, max_suffix, kc, vc, px, out, st); break;
    default: fail(RB200_ERR_INVALID_ARGUMENT, "shared prefix attention: head_dim must be 16, 32, 64 or 128");
  }
}

}  // namespace rb200

using namespace rb200;

static AttnShape shape_of(const rb200_attn_shape* s) {
  return AttnShape{s->heads, s->kv_heads, s->head_dim, s->block_size, s->q_stride, s->o_stride};
}

extern "C" {

size_t rb200_shared_prefix_scratch_bytes(const rb200_attn_shape* s, int n_decode, int n_groups, int max_prefix) {
  if (!s || !fast_attention_supported(shape_of(s))) return 0;
  return shared_prefix_scratch_bytes(shape_of(s), n_decode, n_groups, max_prefix);
}

int rb200_shared_prefix_attention(const rb200_attn_shape* s, const float* q, const rb200_token_meta* m, const int32_t* decode_tokens,
                                  int n_decode, const int32_t* group_off, const int32_t* prefix_len, int n_groups, int max_prefix,
                                  int max_suffix, const void* k_pool, const void* v_pool, void* scratch, size_t scratch_bytes,
                                  void* out, void* stream) {
  return guarded([&] {
    RB_REQUIRE(s != nullptr, "shared prefix attention: null shape");
    const AttnShape sh = shape_of(s);
    RB_REQUIRE(sh.heads > 0 && sh.kv_heads > 0 && sh.heads % sh.kv_heads == 0 && sh.D > 0 && sh.block_size > 0,
               "shared prefix attention: bad head layout");
    RB_REQUIRE(static_cast<long long>(sh.q_stride) >= static_cast<long long>(sh.heads) * sh.D &&
                   static_cast<long long>(sh.o_stride) >= static_cast<long long>(sh.heads) * sh.D,
               "shared prefix attention: row strides too small");
    RB_REQUIRE(fast_attention_supported(sh), "shared prefix attention: head_dim must be 16/32/64/128 and heads/kv_heads <= 16");
    RB_REQUIRE(sh.q_stride % 4 == 0 && sh.o_stride % 8 == 0, "shared prefix attention: q_stride must be a multiple of 4, o_stride of 8");
    RB_REQUIRE(n_decode >= 0 && n_groups >= 0 && max_prefix >= 0 && max_suffix >= 0, "shared prefix attention: bad batch");
    if (n_decode == 0 || n_groups == 0) return 0;  // every entry is padding
    RB_REQUIRE(q && m && m->pos && m->seq && m->table_off && m->tables && decode_tokens && group_off && prefix_len && k_pool &&
                   v_pool && scratch && out,
               "shared prefix attention: null argument");
    for (const void* p : {static_cast<const void*>(q), k_pool, v_pool, static_cast<const void*>(scratch), static_cast<const void*>(out)})
      RB_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "shared prefix attention: q, the pools, scratch and out must be 16-byte aligned");
    RB_REQUIRE(scratch_bytes >= shared_prefix_scratch_bytes(sh, n_decode, n_groups, max_prefix),
               "shared prefix attention: scratch too small");
    launch_shared_prefix_attention(sh, q, TokenMeta{m->pos, m->seq, m->table_off, m->tables}, decode_tokens, n_decode, group_off,
                                   prefix_len, n_groups, max_prefix, max_suffix, static_cast<const __half*>(k_pool),
                                   static_cast<const __half*>(v_pool), static_cast<float*>(scratch), static_cast<__half*>(out),
                                   as_stream(stream));
    RB_CUDA(cudaGetLastError());
    return 0;
  });
}

}  // extern "C"
