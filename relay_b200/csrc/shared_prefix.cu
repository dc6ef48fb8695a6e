// Decode attention for groups of sequences whose contexts begin with the same keys. With P shared
// keys and s_i keys of its own, token i's output is
//
//   o_i = (e^(m_p - M) l_p o_p + e^(m_s - M) l_s o_s) / (e^(m_p - M) l_p + e^(m_s - M) l_s),  M = max(m_p, m_s)
//
// with (m, l, o) the running maximum, sum and output of the softmax over the P shared keys and over
// the s_i own ones. The shared part has the same keys for every token of the group, so it is a
// product of matrices: (tokens x heads of a KV head) rows against P keys, each key read once per row
// tile instead of once per token. Three kernels, each started under the one ahead:
//
//  * umma_prefix_kernel (umma_prefix.cu; head sizes 64 and 128, block sizes that are multiples of 16) or
//    prefix_mma_kernel (the other layouts): a CTA takes 128 or 64 rows (token, head) of one group and
//    KV head and a slice of the shared keys, and leaves a partial (m, l, o) per row. Bound by the
//    tensor cores where many tokens share, by memory where few do;
//  * suffix_kernel: a CTA takes one token and KV head and a slice of the token's own keys, and leaves a
//    partial per head. Bound by memory (alone, 256 tokens with 128 - 640 keys of 8 x 128: 407 MB in 70 us =
//    5.8 TB/s). Its keys need nothing of the first kernel: it runs beside it, on the SMs that one leaves free,
//    and in a small batch (`finish`) then waits for it and adds its partials;
//  * join_kernel, in larger batches: a warp takes one token and head and adds its partials. Bound by latency.
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
  pdl_trigger();  // behind the wait: what the kernels behind read early is then complete
  const int G = heads / kv_heads, kvh = blockIdx.y;
  const RowTile rt = find_tile(gr, G, kPxRows, blockIdx.x);
  if (rt.g < 0) return;
  const int lo = rt.lo, hi = rt.hi, tile = rt.tile;
  const Prefix px = prefix_of(gr, m, rt.g, lo, hi, true);
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
    const long long at = (static_cast<long long>(entry[r]) * heads + head[r]) * part.total + blockIdx.z;
    float* dst = part.o + at * D + 2 * t4;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
    if (t4 == 0) *reinterpret_cast<float2*>(part.ml + at * 2) = r == 0 ? make_float2(m0, l0) : make_float2(m1, l1);
  }
}

// ---------------------------------------------------------------------------------------
// Each sequence's own keys
// ---------------------------------------------------------------------------------------

// W warps to a CTA, each with a ring of S 16-key tiles: one at work, the others in flight. 4 and 2 (three CTAs to an SM)
// where there are CTAs enough to fill the GPU, 8 and 3 where each has an SM to itself.
template <int D, int W, int S>
constexpr size_t suffix_smem_bytes() {
  return static_cast<size_t>(W) * S * 2 * 16 * D * sizeof(__half);
}

// The transpose of an 8x8 matrix of halves, a row's pairs in four lanes.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The products run with the keys (then the head's dimensions) on the M axis of m16n8k16 and the query heads on
// its N axis, 8 at a time: S^T = K Q^T and O^T += V^T P^T. With the heads on M half of each product and of O's
// registers would be rows that no head fills.
// CONTIG: block_size is a multiple of 16, so an aligned 16-key tile is one contiguous run of a page.
// NT: groups of 8 query heads to a KV head (1 or 2). gridDim.z CTAs share the token's own keys.
template <int D, bool CONTIG, int NT, int W, int S>
__global__ void __launch_bounds__(W * 32, W == 8 ? 1 : NT == 1 ? 3 : 2)
suffix_kernel(const float* __restrict__ q, TokenMeta m, Groups gr, const __half* __restrict__ kc, const __half* __restrict__ vc,
              Partials part, __half* __restrict__ out, int heads, int kv_heads, int bs, int bs_shift, int q_stride, int o_stride,
              float scale_log2e, int first, int finish) {
  constexpr int CH = D / 8;
  constexpr int TILE_HALVES = 16 * D;
  constexpr int OS = D + 4;  // floats between heads in the exchange: they start on different banks
  static_assert(8 * NT * OS * 4 <= S * 2 * TILE_HALVES * 2, "a warp's ring holds its output");
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ float s_m[W][8 * NT], s_l[W][8 * NT];

  // Behind a prefix kernel, all of whose CTAs have waited for what came before them, the metadata, q and the
  // pages are complete (and read from L2): nothing is waited for until the keys are done. Then every CTA waits
  // for the shared part (`finish`) or only the grid's last one, so that this kernel is not complete before the one
  // ahead of it is. `first`: there is none.
  if (first) pdl_wait();
  pdl_trigger();
  const bool last = blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1;
  const int di = blockIdx.x, kvh = blockIdx.y, slices = gridDim.z, rank = blockIdx.z;
  const int tok = __ldcg(gr.decode_tokens + di);
  const RowTile rt = group_of(gr, di);
  if (tok < 0 || rt.g < 0) {  // padding
    if (last) pdl_wait();
    return;
  }
  const int pos = __ldcg(m.pos + tok), seq = __ldcg(m.seq + tok);
  const int P = prefix_of(gr, m, rt.g, rt.lo, rt.hi, false).keys;
  const int ctx = max(pos + 1, 0), start = min(P, ctx);
  const int* table = ctx > 0 ? m.tables + __ldcg(m.table_off + seq) : nullptr;
  // Tiles start at multiples of 16 where a tile has to be a run of a page; keys before `start` are masked.
  const int base = CONTIG ? start & ~15 : start;
  const int per = ((ctx - base + slices - 1) / slices + 15) & ~15;
  const int k0 = min(base + rank * per, ctx), k1 = min(k0 + per, ctx);
  const int ntiles = (k1 - k0 + 15) >> 4;

  const int G = heads / kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, t4 = lane & 3;

  __half* ring = reinterpret_cast<__half*>(smem_raw) + static_cast<size_t>(warp) * S * 2 * TILE_HALVES;
  const uint32_t ring_u32 = smem_u32(ring);
  // Tiles warp, warp + W, ... of the slice belong to this warp. Block ids wait in registers, read ahead of their use
  // and from L2: where a tile lies in one page 32 tiles' ids, one per lane, otherwise those of a tile's 16 keys.
  const int my_tiles = ntiles > warp ? (ntiles - warp + W - 1) / W : 0;
  auto fetch_ids = [&](int j0) {
    const int j = CONTIG ? j0 + lane : j0, key = k0 + (warp + j * W) * 16 + (CONTIG ? 0 : lane & 15);
    return j < my_tiles && key < k1 ? __ldcg(table + (bs_shift >= 0 ? key >> bs_shift : key / bs)) : 0;
  };
  int ids = fetch_ids(0), ids_next = fetch_ids(CONTIG ? 32 : 1);
  auto load_tile = [&](int j) {
    const uint32_t kdst = ring_u32 + static_cast<uint32_t>(j % S) * 2 * TILE_HALVES * 2;
    const uint32_t vdst = kdst + TILE_HALVES * 2;
    const int key0 = k0 + (warp + j * W) * 16;
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
      const int mine = ids;  // of this tile: tiles are loaded in order
      ids = ids_next;
      ids_next = fetch_ids(j + 2);
      const int my_slot = bs_shift >= 0 ? 0 : (key0 + (lane & 15)) % bs;
#pragma unroll
      for (int idx = lane; idx < 16 * CH; idx += 32) {
        const int row = idx / CH, c = idx % CH;
        const long long block = __shfl_sync(0xffffffffu, mine, row);
        const int slot = bs_shift >= 0 ? (key0 + row) & (bs - 1) : __shfl_sync(0xffffffffu, my_slot, row);
        const int bytes = row < nvalid ? 16 : 0;
        const long long at = bytes ? ((block * kv_heads + kvh) * bs + slot) * D + c * 8 : 0;
        const uint32_t off = static_cast<uint32_t>(swz<CH>(row, c)) * 16;
        cp_async16_zfill(kdst + off, kc + at, bytes);
        cp_async16_zfill(vdst + off, vc + at, bytes);
      }
    }
  };

#pragma unroll
  for (int st = 0; st < S - 1; ++st) {
    if (st < my_tiles) load_tile(st);
    cp_async_commit();
  }

  // The heads' queries as B fragments, hi and lo halves: head n * 8 + gid, dimensions 2 t4 and 2 t4 + 8 of each 16.
  uint32_t qh[NT][D / 16][2], ql[NT][D / 16][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int h = n * 8 + gid;
    const float* q0 = q + static_cast<long long>(tok) * q_stride + (kvh * G + min(h, G - 1)) * D + 2 * t4;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(q0 + kk * 16 + 8 * e));
        split_half2(h < G ? x.x : 0.f, h < G ? x.y : 0.f, qh[n][kk][e], ql[n][kk][e]);
      }
  }

  float o[NT][D / 16][4];  // O^T: dimensions 16 j + gid (then + 8), heads n * 8 + 2 t4 and + 1
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
  float mr[NT][2], lr[NT][2];  // heads n * 8 + 2 t4 and + 1, log2 domain; the sum is this lane's keys' own
#pragma unroll
  for (int n = 0; n < NT; ++n) mr[n][0] = mr[n][1] = -INFINITY, lr[n][0] = lr[n][1] = 0.f;

  for (int j = 0; j < my_tiles; ++j) {
    cp_async_wait<S - 2>();
    __syncwarp();
    if (j + S - 1 < my_tiles) load_tile(j + S - 1);
    cp_async_commit();

    const uint32_t ktile = ring_u32 + static_cast<uint32_t>(j % S) * 2 * TILE_HALVES * 2;
    const uint32_t vtile = ktile + TILE_HALVES * 2;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t ka[4];
      ldmatrix_x4(ka, ktile + swz<CH>((lane & 7) + ((lane >> 3) & 1) * 8, 2 * kk + (lane >> 4)) * 16);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_f16(s[n], ka, qh[n][kk][0], qh[n][kk][1]);
        mma_f16(s[n], ka, ql[n][kk][0], ql[n][kk][1]);
      }
    }

    const int key = k0 + (warp + j * W) * 16 + gid;  // of s[.][0], s[.][1]; 8 further on for the other two
    const bool see0 = key >= start && key < k1, see1 = key + 8 >= start && key + 8 < k1;
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float corr[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& x0 = s[n][e];
        float& x1 = s[n][e + 2];
        x0 = see0 ? x0 * scale_log2e : -INFINITY;
        x1 = see1 ? x1 * scale_log2e : -INFINITY;
        float mx = fmaxf(x0, x1);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(mr[n][e], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;  // only masked keys so far
        corr[e] = fast_exp2(mr[n][e] - ref);
        mr[n][e] = mn;
        x0 = fast_exp2(x0 - ref);
        x1 = fast_exp2(x1 - ref);
        lr[n][e] = lr[n][e] * corr[e] + (x0 + x1);
      }
      // weights of key gid (then gid + 8) -> weights of keys 2 t4, 2 t4 + 1 of head gid: the second product's B operand
      pb[n][0] = transpose_8x8(pack_half2(s[n][0], s[n][1]));
      pb[n][1] = transpose_8x8(pack_half2(s[n][2], s[n][3]));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[n][i][0] *= corr[0];
        o[n][i][1] *= corr[1];
        o[n][i][2] *= corr[0];
        o[n][i][3] *= corr[1];
      }
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t va[4];
      ldmatrix_x4_trans(va, vtile + swz<CH>((lane & 7) + (lane >> 4) * 8, 2 * i + ((lane >> 3) & 1)) * 16);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(o[n][i], va, pb[n][0], pb[n][1]);
    }
  }
  cp_async_wait<0>();
  __syncwarp();

  // The warps' (m, l, o) meet in shared memory (each warp reuses its own ring).
  float* os = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      lr[n][e] += __shfl_xor_sync(0xffffffffu, lr[n][e], 4);
      lr[n][e] += __shfl_xor_sync(0xffffffffu, lr[n][e], 8);
      lr[n][e] += __shfl_xor_sync(0xffffffffu, lr[n][e], 16);
      const int h = n * 8 + 2 * t4 + e;
      if (gid == 0) {
        s_m[warp][h] = mr[n][e];
        s_l[warp][h] = lr[n][e];
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        os[h * OS + i * 16 + gid] = o[n][i][e];
        os[h * OS + i * 16 + 8 + gid] = o[n][i][e + 2];
      }
    }
  }
  if (finish) pdl_wait();
  __syncthreads();

  const float* os_all = reinterpret_cast<const float*>(smem_raw);
  constexpr int WARP_FLOATS = S * TILE_HALVES;  // ring size of one warp in floats
  const int used = slices_used(P, part.parts);
  for (int idx = threadIdx.x; idx < G * D / 4; idx += blockDim.x) {
    const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, s_m[w][r]);
    const float ref = M == -INFINITY ? 0.f : M;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float e = fast_exp2(s_m[w][r] - ref);
      const float4 x = *reinterpret_cast<const float4*>(os_all + w * WARP_FLOATS + r * OS + d);
      acc.x += e * x.x, acc.y += e * x.y, acc.z += e * x.z, acc.w += e * x.w;
      L += e * s_l[w][r];
    }
    const long long at = (static_cast<long long>(di) * heads + kvh * G + r) * part.total;
    if (!finish) {
      *reinterpret_cast<float4*>(part.o + (at + part.parts + rank) * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(part.ml + (at + part.parts + rank) * 2) = make_float2(M, L);
      continue;
    }
    // the shared part's partials of this head, U at a time, in the order of the slices
    constexpr int U = 8;
    for (int p0 = 0; p0 < used; p0 += U) {
      float2 ml[U];
      float4 x[U];
      float top = M;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool there = p0 + u < used;
        ml[u] = there ? *reinterpret_cast<const float2*>(part.ml + (at + p0 + u) * 2) : make_float2(-INFINITY, 0.f);
        x[u] = there ? *reinterpret_cast<const float4*>(part.o + (at + p0 + u) * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, ml[u].x);
      const float to = top == -INFINITY ? 0.f : top, e = fast_exp2(M - to);
      acc.x *= e, acc.y *= e, acc.z *= e, acc.w *= e;
      L *= e;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = fast_exp2(ml[u].x - to);
        acc.x += w * x[u].x, acc.y += w * x[u].y, acc.z += w * x[u].z, acc.w += w * x[u].w;
        L += w * ml[u].y;
      }
      M = top;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;  // no key at all: zeros
    *reinterpret_cast<uint2*>(out + static_cast<long long>(tok) * o_stride + (kvh * G + r) * D + d) =
        make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  }
  if (last && !finish) pdl_wait();
}

// ---------------------------------------------------------------------------------------
// The join
// ---------------------------------------------------------------------------------------

constexpr int kMostParts = 64;  // slices of the shared keys, and of a token's own
constexpr int kJoinWarps = 4;

// out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p over the partials of a (token, head), one warp each. The
// lanes first hold the partials' weights, then D / 4 of them at a time a partial's values, 128 / D partials
// side by side; all in a fixed order.
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_kernel(TokenMeta m, Groups gr, Partials part, __half* __restrict__ out, int heads, int o_stride) {
  constexpr int LPD = D / 4, SIDE = 32 / LPD, CHUNKS = 2 * kMostParts / 32;
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pair = min(blockIdx.x * kJoinWarps + warp, gr.n_decode * heads - 1);
  const int di = pair / heads, head = pair - di * heads;
  const int tok = __ldcg(gr.decode_tokens + di);
  const RowTile rt = group_of(gr, di);
  const bool live = tok >= 0 && rt.g >= 0 && pair == blockIdx.x * kJoinWarps + warp;
  const int P = live ? prefix_of(gr, m, rt.g, rt.lo, rt.hi, false).keys : 0;
  const int used = slices_used(P, part.parts);
  pdl_wait();
  if (!live) return;
  const long long base = static_cast<long long>(pair) * part.total;
  float w[CHUNKS], top = -INFINITY, L = 0.f;
  float2 ml[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int p = c * 32 + lane;
    ml[c] = p < part.total && (p < used || p >= part.parts) ? *reinterpret_cast<const float2*>(part.ml + (base + p) * 2)
                                                            : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[c].x);
  }
  top = warp_max(top);
  if (top == -INFINITY) top = 0.f;  // no key at all: every sum is 0
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    w[c] = fast_exp2(ml[c].x - top);
    L += w[c] * ml[c].y;
  }
  L = warp_sum(L);
  const int side = lane / LPD, d = (lane % LPD) * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int n = min(part.total - c * 32, 32);
    constexpr int U = 8;  // loads in flight
#pragma unroll 1
    for (int p0 = 0; p0 < n; p0 += U * SIDE) {
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int p = c * 32 + p0 + u * SIDE + side;
        x[u] = p < part.total && (p < used || p >= part.parts) ? *reinterpret_cast<const float4*>(part.o + (base + p) * D + d)
                                                               : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float wp = __shfl_sync(0xffffffffu, w[c], (p0 + u * SIDE + side) & 31);
        const bool there = p0 + u * SIDE + side < 32;  // else the weight is another partial's
        acc.x += there ? wp * x[u].x : 0.f, acc.y += there ? wp * x[u].y : 0.f;
        acc.z += there ? wp * x[u].z : 0.f, acc.w += there ? wp * x[u].w : 0.f;
      }
    }
  }
#pragma unroll
  for (int o = LPD; o < 32; o <<= 1) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o), acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o), acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
  }
  if (side == 0) {
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<uint2*>(out + static_cast<long long>(tok) * o_stride + head * D + d) =
        make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  }
}

// ---------------------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------------------

// At most this many row tiles of `rows` rows: a group rounds up by less than one tile.
long long row_tiles(const AttnShape& s, int n_decode, int n_groups, int rows) {
  return (static_cast<long long>(n_decode) * (s.heads / s.kv_heads) + static_cast<long long>(n_groups) * (rows - 1)) / rows;
}

// How a call is split: row tiles, slices of the longest prefix and of a token's own keys.
//  * `parts` 0: nothing is read as shared. A few tokens behind a short prefix are done sooner when each reads all of its
//    keys, from L2 but for the first.
//  * `finish`: the suffix kernel joins the shared part itself, without a third kernel, where each (token, KV head) is one
//    CTA and all of them have a place beside the prefix kernel (two on an SM, where its CTAs of tcgen05 take both and the
//    others one): none that waits for the shared part keeps another from its keys. Measured: 32 tokens behind 4096 keys,
//    whose 256 CTAs do not fit beside it, 24.0 us against 20.6 with the third kernel; 48 tokens of 4 KV heads of 32 in two
//    groups of 777 and 300 keys 9.6 against 11.0.
//  * `wide`: CTAs of eight warps in the suffix kernel, where each has an SM to itself.
struct Plan {
  int rows, tiles, parts, slices;
  bool finish, wide;
};

// The own keys' partials stay in the CTA where it finishes.
int partials_of(const Plan& p) { return p.parts + (p.finish ? 0 : p.slices); }

size_t scratch_of(const AttnShape& s, int n_decode, const Plan& p) {
  return static_cast<size_t>(n_decode) * s.heads * partials_of(p) * (s.D + 2) * sizeof(float);
}

// The plan follows from estimates in us:
//  * a CTA of the prefix kernel takes kTileUs for every 128 keys and kStartUs besides, and the join kJoinUs; the own keys
//    (six tenths of the most) take their bytes at kBytesPerUs of the whole GPU, of which the SMs that the prefix kernel
//    leaves free get kBytesPerSmUs each until it ends. Measured at 32 + 2 x 8 heads of 128: 256 tokens behind 8192 keys
//    with 128 - 640 of their own, 105 us in one slice (64 CTAs beside the own keys) and 117 in two, which fill the
//    GPU; 32 tokens behind 4096 with 64 - 512: 24, 20.5, 25 and 28 us in 4, 8, 11 and 16 slices;
//  * the suffix kernel takes kOwnStartUs and for every key of a slice 5 ns and 35 ps a value of the head (blocks that
//    16 keys do not divide: 2.5 ns more; measured with blocks of 8, 2 more at heads of 32, 4 at 64, 7 at 128), 0.6 of that
//    in CTAs of eight warps (`wide`); with x CTAs to an SM 0.65 + x / 2 times as much (heads of 64 and less: 0.65 + 0.35 x).
//    Slices take kOwnJoinUs more;
//  * a launch behind the first counts kLaunchUs, most of the 2.5 us of the caller's time for it, which a graph does
//    not spend.
// Measured over 400 batches of 1 - 512 tokens in 1 - 64 groups behind 64 - 3000 keys in five head layouts, where the plan
// takes at most 20 % or 2 us longer than the better of both ways: all keys as the tokens' own 5.1 us against 10.3 shared
// at 16 tokens of 8 KV heads of 128 behind 100 keys, 7.8 against 10.8 behind 500, 21 against 14 behind 3000; one
// token behind 500 keys 6.9 against 8.5 in CTAs of four warps.
constexpr double kTileUs = 1.3, kStartUs = 6.0, kJoinUs = 1.5, kBytesPerUs = 5.5e6, kBytesPerSmUs = 4.2e4;
constexpr double kOwnStartUs = 3.8, kOwnJoinUs = 2.0, kLaunchUs = 2.0;

double own_us(const AttnShape& s, long long pairs, double keys, int slices, bool wide) {
  const double key_us = (0.005 + 35e-6 * s.D + (s.block_size % 16 == 0 ? 0.0 : 0.0025)) * (wide ? 0.6 : 1.0);
  const double share = s.D == 128 ? 0.5 : 0.35, load = share * static_cast<double>(pairs * slices) / sm_count() + 0.65;
  return kOwnStartUs + keys / slices * key_us * std::max(1.0, load) + (slices > 1 ? kOwnJoinUs + kLaunchUs : 0.0);
}

Plan plan_of(const AttnShape& s, int n_decode, int n_groups, int max_prefix, int max_suffix) {
  const long long pairs = static_cast<long long>(n_decode) * s.kv_heads;
  // Slices of own keys: at least 128 keys each, two CTAs for every SM.
  auto most_slices = [&](double keys) {
    const double most = std::min<double>(2.0 * sm_count() / static_cast<double>(pairs), keys / 128.0);
    return static_cast<int>(std::max(1.0, std::min<double>(most, kMostParts)));
  };

  // every key as the token's own
  Plan alone{0, 0, 0, 1, true, false};
  const double keys = static_cast<double>(max_prefix) + max_suffix;
  double alone_us = -1.0;
  for (int n = 1; n <= most_slices(keys); ++n) {
    const bool wide = pairs * n <= sm_count();
    const double us = own_us(s, pairs, keys, n, wide);
    if (alone_us < 0.0 || us < alone_us) {
      alone_us = us;
      alone.slices = n;
      alone.finish = n == 1;
      alone.wide = wide;
    }
  }
  if (max_prefix == 0) return alone;

  Plan p{0, 0, 1, 1, false, false};
  // 64 rows where the average group has no more
  p.rows = umma_prefix_usable(s) && static_cast<long long>(n_decode) * (s.heads / s.kv_heads) > 64LL * n_groups ? 128 : 64;
  p.tiles = static_cast<int>(row_tiles(s, n_decode, n_groups, p.rows));
  const long long ctas = static_cast<long long>(p.tiles) * s.kv_heads;
  const long long slots = (umma_prefix_usable(s) ? 1LL : 2LL) * sm_count();
  const double suffix_us = 0.6 * 4.0 * max_suffix * s.D * static_cast<double>(pairs) / kBytesPerUs;
  // The time of n slices with `running` CTAs, and how much of the own keys' time that takes along.
  auto shared_us = [&](long long running, int n, double tile_us) {
    return static_cast<double>((running + slots - 1) / slots) * (div_up(div_up(max_prefix, n), kPrefixSlice) * tile_us + kStartUs);
  };
  auto beside_us = [&](long long running, double us) {
    const double idle = std::max<double>(0.0, 1.0 - static_cast<double>(running) / slots) * sm_count();
    return us * std::min(1.0, idle * kBytesPerSmUs / kBytesPerUs);
  };
  double least = -1.0, prefix_us = 0.0;
  for (int n = 1; n <= kMostParts && (n == 1 || max_prefix > (n - 1) * 2 * kPrefixSlice); ++n) {
    const double shared = shared_us(ctas * n, n, kTileUs);
    const double us = shared + std::max(0.0, suffix_us - beside_us(ctas * n, shared));
    if (least < 0.0 || us < least) {
      least = us;
      prefix_us = shared;
      p.parts = n;
    }
  }
  // own keys that one CTA of each pair reads beside the prefix kernel need no slices
  const bool beside = pairs <= 2LL * sm_count() - (umma_prefix_usable(s) ? 2 : 1) * ctas * p.parts;
  p.slices = beside && own_us(s, pairs, max_suffix, 1, false) <= prefix_us ? 1 : most_slices(max_suffix);
  p.finish = beside && p.slices == 1;

  // Both ways against each other, with as many row tiles as groups of one size have. Two CTAs of prefix_mma_kernel on an SM
  // take 1.6 times as long for their tiles.
  const long long rows = static_cast<long long>(n_decode) * (s.heads / s.kv_heads);
  const long long expected = n_groups * static_cast<long long>(div_up(rows, static_cast<long long>(n_groups) * p.rows));
  const long long running = std::min<long long>(p.tiles, expected) * s.kv_heads * p.parts;
  prefix_us = shared_us(running, p.parts, umma_prefix_usable(s) || running <= sm_count() ? kTileUs : 1.6 * kTileUs);
  const double own = std::max(suffix_us, own_us(s, pairs, max_suffix, 1, false));
  const double behind_us = std::max(0.0, own - beside_us(running, prefix_us));
  const double join_us = kJoinUs + 2.0 * static_cast<double>(scratch_of(s, n_decode, p)) / kBytesPerUs;
  return alone_us <= prefix_us + behind_us + join_us + (p.finish ? 1 : 2) * kLaunchUs ? alone : p;
}

template <int D, bool CONTIG, int NT, int W, int S>
void launch_suffix(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const __half* kc, const __half* vc,
                   const Partials& part, __half* out, const Plan& plan, cudaStream_t st) {
  static PerDeviceOnce once;
  auto kernel = suffix_kernel<D, CONTIG, NT, W, S>;
  once.run([&] {
    RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(suffix_smem_bytes<D, W, S>())));
  });
  count_launch();
  const int first = plan.parts == 0, finish = plan.finish;
  launch_pdl(kernel, dim3(gr.n_decode, s.kv_heads, plan.slices), dim3(W * 32), suffix_smem_bytes<D, W, S>(), st, q, m, gr, kc, vc, part,
             out, s.heads, s.kv_heads, s.block_size, shift_of(s.block_size), s.q_stride, s.o_stride, kLog2e / sqrtf(static_cast<float>(D)),
             first, finish);
}

template <int D>
void launch_d(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const Plan& plan, const __half* kc,
              const __half* vc, const Partials& part, __half* out, cudaStream_t st) {
  if (plan.parts > 0) {
    if (umma_prefix_usable(s)) {
      launch_umma_prefix(s, q, m, gr, kc, vc, part, plan.rows, plan.tiles, st);
    } else {
      static PerDeviceOnce once;
      auto kernel = prefix_mma_kernel<D>;
      once.run([&] {
        RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(prefix_smem_bytes<D>())));
      });
      count_launch();
      launch_pdl(kernel, dim3(plan.tiles, s.kv_heads, plan.parts), dim3(128), prefix_smem_bytes<D>(), st, q, m, gr, kc, vc, part, s.heads,
                 s.kv_heads, s.block_size, shift_of(s.block_size), s.q_stride, kLog2e / sqrtf(static_cast<float>(D)));
    }
  }
  const bool contig = s.block_size % 16 == 0, wide = s.heads / s.kv_heads > 8;
  auto launch = [&](auto contig_, auto nt) {
    constexpr bool CONTIG = decltype(contig_)::value;
    constexpr int NT = decltype(nt)::value;
    if (plan.wide) launch_suffix<D, CONTIG, NT, 8, 3>(s, q, m, gr, kc, vc, part, out, plan, st);
    else launch_suffix<D, CONTIG, NT, 4, 2>(s, q, m, gr, kc, vc, part, out, plan, st);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (contig && !wide) launch(std::true_type{}, One{});
  else if (contig) launch(std::true_type{}, Two{});
  else if (!wide) launch(std::false_type{}, One{});
  else launch(std::false_type{}, Two{});
  if (plan.finish) return;
  count_launch();
  launch_pdl(join_kernel<D>, dim3(div_up(static_cast<long long>(gr.n_decode) * s.heads, kJoinWarps)), dim3(kJoinWarps * 32), 0, st, m, gr,
             part, out, s.heads, s.o_stride);
}

}  // namespace

size_t shared_prefix_scratch_bytes(const AttnShape& s, int n_decode, int n_groups, int max_prefix, int max_suffix) {
  if (n_decode <= 0 || n_groups <= 0) return 0;
  return scratch_of(s, n_decode, plan_of(s, n_decode, n_groups, max_prefix, max_suffix));
}

void launch_shared_prefix_attention(const AttnShape& s, const float* q, const TokenMeta& m, const int* decode_tokens, int n_decode,
                                    const int* group_off, const int* prefix_len, int n_groups, int max_prefix, int max_suffix,
                                    const __half* kc, const __half* vc, float* scratch, size_t scratch_bytes, __half* out,
                                    cudaStream_t st) {
  if (n_decode == 0) return;
  const Plan plan = plan_of(s, n_decode, n_groups, max_prefix, max_suffix);
  const size_t need = scratch_of(s, n_decode, plan);
  RB_REQUIRE(scratch != nullptr || need == 0, "shared prefix attention: null scratch");
  RB_REQUIRE(scratch_bytes >= need, "shared prefix attention: scratch too small");
  if (umma_prefix_usable(s)) umma_status_word();  // allocated by the first call, whichever kernels that one takes
  const Groups gr{decode_tokens, group_off, plan.parts > 0 ? prefix_len : nullptr, n_decode, n_groups};
  Partials part;
  part.parts = plan.parts;
  part.total = partials_of(plan);
  part.o = scratch;
  part.ml = scratch + static_cast<size_t>(n_decode) * s.heads * part.total * s.D;
  switch (s.D) {
    case 16: launch_d<16>(s, q, m, gr, plan, kc, vc, part, out, st); break;
    case 32: launch_d<32>(s, q, m, gr, plan, kc, vc, part, out, st); break;
    case 64: launch_d<64>(s, q, m, gr, plan, kc, vc, part, out, st); break;
    case 128: launch_d<128>(s, q, m, gr, plan, kc, vc, part, out, st); break;
    default: fail(RB200_ERR_INVALID_ARGUMENT, "shared prefix attention: head_dim must be 16, 32, 64 or 128");
  }
}

}  // namespace rb200

using namespace rb200;

static AttnShape shape_of(const rb200_attn_shape* s) {
  return AttnShape{s->heads, s->kv_heads, s->head_dim, s->block_size, s->q_stride, s->o_stride};
}

extern "C" {

size_t rb200_shared_prefix_scratch_bytes(const rb200_attn_shape* s, int n_decode, int n_groups, int max_prefix, int max_suffix) {
  if (!s || !fast_attention_supported(shape_of(s)) || max_prefix < 0 || max_suffix < 0) return 0;
  return shared_prefix_scratch_bytes(shape_of(s), n_decode, n_groups, max_prefix, max_suffix);
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
    RB_REQUIRE(static_cast<long long>(n_decode) * sh.heads <= 0x7fffffff, "shared prefix attention: bad batch (too many entries)");
    if (n_decode == 0 || n_groups == 0) return 0;  // every entry is padding
    RB_REQUIRE(q && m && m->pos && m->seq && m->table_off && m->tables && decode_tokens && group_off && prefix_len && k_pool &&
                   v_pool && out,
               "shared prefix attention: null argument");
    for (const void* p : {static_cast<const void*>(q), k_pool, v_pool, static_cast<const void*>(scratch), static_cast<const void*>(out)})
      RB_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "shared prefix attention: q, the pools, scratch and out must be 16-byte aligned");
    launch_shared_prefix_attention(sh, q, TokenMeta{m->pos, m->seq, m->table_off, m->tables}, decode_tokens, n_decode, group_off,
                                   prefix_len, n_groups, max_prefix, max_suffix, static_cast<const __half*>(k_pool),
                                   static_cast<const __half*>(v_pool), static_cast<float*>(scratch), scratch_bytes,
                                   static_cast<__half*>(out), as_stream(stream));
    RB_CUDA(cudaGetLastError());
    return 0;
  });
}

}  // extern "C"
