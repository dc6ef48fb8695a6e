// The shared keys of the shared-prefix decode attention (shared_prefix.cu) on tcgen05 tensor cores, for
// head sizes 64 and 128 and block sizes that are multiples of 16.
//
// One CTA takes 128 rows (64 where groups are small), a row being one query head of one token: tokens of
// one group, heads of one KV head, so every row sees the same keys. It runs over a slice of the group's shared keys in tiles
// of 128, the even tiles and the odd ones as two streams of their own: while the softmax warps of one
// stream work on its scores, the tensor cores make the products of the other. For a tile of stream h:
//   S_h = Q K^T   A = Q in shared memory as two fp16 halves (q = hi + lo, exact to 2^-22 of q: with hi
//                 alone the rounding of q would cost as much as that of the output), B = the K tile,
//                 D = S_h in TMEM (128 lanes x 128 columns);
//   softmax       the stream's four warps, a thread per row: the row's maximum, then P = exp2(.) as fp16
//                 over the columns of S_h that have been read;
//   O_h += P V    A = P from TMEM, B = the V tile, D = O_h in TMEM, rescaled only when a row's maximum
//                 outgrew its reference by 2^8. S_h is free for the stream's next tile behind it.
// At the end a row's two streams are joined and (maximum, sum, O) is left as the row's partial result.
// Rows without a token cost nothing but their share of the products: a warp without any skips the softmax.
//
// K and V tiles pass through one ring of slots in the order K0 V0 K1 V1 ..., each slot with its own
// pair of barriers: a K slot is free again once its scores are made, long before V of the same tile.
// Every wait is bounded; one that gives up records a code in the device's status word.
//
// Measured at head_dim 128: with 128 rows a tile takes 2300 - 2700 cycles (64 CTAs of 64 tiles: 96 us, tensor
// pipe 64 % active), a stream's chain of Q K^T (1330, half of it for lo), softmax (2200) and P V (790) against
// the other's. With 40 rows and 144 CTAs it reads 268 MB of keys in 53 us = 5.1 TB/s. Tried
// and left out: one stream with the halves of a tile as separate softmax states (20 % slower), P kept in
// registers for one pass over S (spills), sixteen softmax warps (no faster).
#include <cuda.h>

#include "attn_tiles.cuh"
#include "kernels.h"
#include "prefix_groups.cuh"
#include "tcgen05.cuh"

namespace rb200 {

using namespace tc;

namespace {

constexpr int kKeys = 128;
constexpr int kRows = 128;  // of the products; a tile fills 64 or all of them
constexpr int kThreads = 384;  // two loader warps, the MMA issuer, a third loader, eight softmax warps
// ROWS: rows of a tile. With 64 the products' other rows read what lies behind the queries and are not looked at;
// the room goes to another slot of the ring, which a few rows, bound by memory, have more use for.
template <int D, int ROWS>
struct Smem {
  static constexpr int kQBytes = ROWS * D * 2;  // one half of q
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kSlots = D == 64 ? 10 : (ROWS == 64 ? 6 : 5);
  static constexpr int kBarBytes = 256;
  static constexpr size_t kTotal = 2 * kQBytes + static_cast<size_t>(kSlots) * kTileBytes + kBarBytes + 1024;
  static_assert(kTotal <= 232448, "shared memory of one CTA");
  static constexpr int kParkStride = D + 4;  // floats; rows start on different banks
  static_assert(static_cast<size_t>(kSlots) * kTileBytes >= static_cast<size_t>(kParkStride + 3) * ROWS * 4, "the streams meet in the ring");
};

__device__ __forceinline__ void softmax_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D, int ROWS>
__global__ void __launch_bounds__(kThreads, 1)
umma_prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __half* __restrict__ kc,
                   const __half* __restrict__ vc, const float* __restrict__ q, TokenMeta m, Groups gr, Partials part, int heads,
                   int kv_heads, int bs, int q_stride, float scale_log2e, int* __restrict__ status) {
  using S = Smem<D, ROWS>;
  constexpr int NS = S::kSlots;
  constexpr float kGrow = 8.f;  // how far (log2) a row's maximum may outgrow its reference before O is rescaled
  // TMEM columns: S (then P, over its first half) of the two streams 0..127 and 128..255, then their O.
  constexpr uint32_t kTmemCols = 512;
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  unsigned char* gen = smem_dyn + (base - smem_u32(smem_dyn));
  const uint32_t sQ = base;
  const uint32_t sKV = sQ + 2 * S::kQBytes;
  const uint32_t bars = sKV + NS * S::kTileBytes;
  const uint32_t full = bars, empty = bars + 80;             // NS (<= 10) x 8 bytes each
  const uint32_t s_ready = bars + 160, p_ready = bars + 176, pv_done = bars + 192;  // one per stream
  const uint32_t q_ready = bars + 208, tmem_slot = bars + 216;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_ready + 8 * s, 1);
      mbar_init(p_ready + 8 * s, 4);
      mbar_init(pv_done + 8 * s, 1);
    }
    mbar_init(q_ready, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 1 && lane == 0) {
    prefetch_map(&map_k);
    prefetch_map(&map_v);
  }
  // Everything, the group metadata too, may come from the kernel ahead. TMEM is taken behind the wait (a CTA that
  // holds it and waits could keep the kernel ahead from getting its own) and the trigger comes last, so
  // that whatever the kernels behind this one read early is complete by the time they start.
  pdl_wait();
  if (warp == 2) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(gen + (tmem_slot - base));

  const int G = heads / kv_heads, kvh = blockIdx.y;
  const RowTile rt = find_tile(gr, G, ROWS, blockIdx.x);
  const int lo = rt.lo, hi = rt.hi, tile = rt.tile;
  if (warp >= 4 && rt.g >= 0) {
    // The rows' queries -> hi + lo -> swizzled A operands, before anything about the keys is known: a warp takes an
    // eighth of the rows, a row's values side by side in D / 4 lanes.
    constexpr int kLanes = D / 4, kSide = 32 / kLanes, kMine = ROWS / 8;
    const int row0 = (warp - 4) * kMine;
    const int entry = lo + (tile * ROWS + row0 + (lane & (kMine - 1))) / G;  // of row row0 + lane
    const int token = entry < hi ? __ldcg(gr.decode_tokens + entry) : -1;
    const int d = (lane % kLanes) * 4, c = d / 8;
    constexpr int kBatch = kMine / kSide;  // loads in flight
    {
      float4 x[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = i * kSide + lane / kLanes;
        const int t = __shfl_sync(0xffffffffu, token, r);
        const int head = kvh * G + (tile * ROWS + row0 + r) % G;
        x[i] = t >= 0 ? *reinterpret_cast<const float4*>(q + static_cast<long long>(t) * q_stride + head * D + d)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int r = row0 + i * kSide + lane / kLanes;
        uint2 hv, lv;
        split_half2(x[i].x, x[i].y, hv.x, lv.x);
        split_half2(x[i].z, x[i].w, hv.y, lv.y);
        unsigned char* dst = gen + (sQ - base) + (c / 8) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4) + (d & 4) * 2;
        *reinterpret_cast<uint2*>(dst) = hv;
        *reinterpret_cast<uint2*>(dst + S::kQBytes) = lv;
      }
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_ready);
  }
  const Prefix px = rt.g >= 0 ? prefix_of(gr, m, rt.g, lo, hi, warp < 4) : Prefix{0, nullptr};
  const int slice = slice_of(px.keys, part.parts);
  const int k0 = blockIdx.z * slice, k1 = min(px.keys, k0 + slice);
  const int ntiles = (k1 - k0 + kKeys - 1) / kKeys;  // 0 or less: nothing to do

  bool ok = true;
  if (ntiles <= 0) {
    // no such tile or slice
  } else if (warp < 2 || warp == 3) {
    // ---- loaders: a tile's keys come from 8 pages of 16 keys; one box per page and 64-wide slice of the
    //      head, dealt round-robin to the lanes of three warps. Page rows are looked up 32 at a time (four
    //      tiles), one per lane, a group ahead of their use. Pages that the slice does not fill are
    //      written by warp 0 with plain copies, zeros for the missing keys of V (whatever the pool
    //      or the slot holds there must not meet a weight of 0; missing keys of K are masked). ----
    constexpr int kAtoms = D / 64;
    constexpr int kBoxes = 8 * kAtoms;
    const int li = warp == 3 ? 2 : warp;
    const int box = li + 3 * lane;
    const bool has_box = box < kBoxes;
    const int box_pg = box & 7, box_atom = box >> 3;
    auto load_group = [&](int t4) {  // first pool row ([block][kv head][slot]) of this lane's page
      const int key = k0 + (t4 * 4 + lane / 8) * kKeys + (lane % 8) * 16;
      return key < k1 ? (px.table[key / bs] * kv_heads + kvh) * bs + key % bs : 0;
    };
    int tab_cur = 0, tab_next = load_group(0);
    for (int j = 0; j < ntiles && ok; ++j) {
      if (j % 4 == 0) {
        tab_cur = tab_next;
        tab_next = load_group(j / 4 + 1);
      }
      const int keys = min(kKeys, k1 - k0 - j * kKeys);
      const int whole = keys / 16;  // pages that are there in full
      const int row = __shfl_sync(0xffffffffu, tab_cur, (j % 4) * 8 + box_pg);
      const int last_row = __shfl_sync(0xffffffffu, tab_cur, (j % 4) * 8 + min(whole, 7));
      for (int kv = 0; kv < 2; ++kv) {
        const int u = 2 * j + kv, s = u % NS;
        ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ((u / NS) & 1) ^ 1));
        if (!ok) break;
        const uint32_t dst = sKV + s * S::kTileBytes;
        if (warp == 0 && whole < 8) {
          constexpr int CH = D / 8;  // 16-byte chunks per row
          const __half* src = (kv ? vc : kc) + static_cast<long long>(last_row) * D;
          const int first = whole * 16, end = kv ? kKeys : keys;
          for (int i = lane; i < (end - first) * CH; i += 32) {
            const int r = first + i / CH, c = i % CH;
            const int bytes = r < keys ? 16 : 0;
            cp_async16_zfill(dst + (c / 8) * (kKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                             src + (bytes ? (r - first) * D + c * 8 : 0), bytes);
          }
          cp_async_commit();
          cp_async_wait<0>();
          fence_async_smem();
          __syncwarp();
        }
        if (warp == 0 && lane == 0) mbar_expect_tx(full + 8 * s, whole * kAtoms * 2048);
        if (has_box && box_pg < whole)
          tma_load_2d(dst + box_atom * (kKeys * 128) + box_pg * 2048, kv ? &map_v : &map_k, box_atom * 64, row, full + 8 * s);
      }
    }
    if (!ok && lane == 0) atomicExch(status, 21);
  } else if (warp == 2) {
    // ---- MMA issuer: P V of a tile when its P arrives, then Q K^T of the stream's next tile, whose S lies over that
    //      P. The other stream is in its softmax meanwhile. ----
    if (elect_one()) {
      constexpr uint32_t idesc_qk = umma_idesc(kRows, kKeys);
      constexpr uint32_t idesc_pv = umma_idesc(kRows, D) | (1u << 16);  // B (V) is MN-major
      auto issue_qk = [&](int j) {
        const int u = 2 * j, s = u % NS;
        if (!mbar_wait(full + 8 * s, (u / NS) & 1)) return false;
        tc_fence_after();
        const uint32_t kt = sKV + s * S::kTileBytes;
#pragma unroll
        for (int part_q = 0; part_q < 2; ++part_q)
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = (k % 4) * 32;  // 64-wide atoms, 32 bytes per 16 dims
            umma_f16(tmem_base + (j & 1) * kKeys, smem_desc_sw128(sQ + part_q * S::kQBytes + (k / 4) * (ROWS * 128) + at),
                     smem_desc_sw128(kt + (k / 4) * (kKeys * 128) + at), idesc_qk, part_q != 0 || k != 0);
          }
        umma_commit(s_ready + 8 * (j & 1));
        umma_commit(empty + 8 * s);
        return true;
      };
      ok = mbar_wait(q_ready, 0) && issue_qk(0) && (ntiles == 1 || issue_qk(1));
      for (int j = 0; j < ntiles && ok; ++j) {
        const int h = j & 1, u = 2 * j + 1, s = u % NS;
        ok = mbar_wait(full + 8 * s, (u / NS) & 1) && mbar_wait(p_ready + 8 * h, (j >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t vt = sKV + s * S::kTileBytes, pa = tmem_base + h * kKeys;
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          umma_f16_ta(tmem_base + 2 * kKeys + h * D, pa + 8 * k, smem_desc_mn_sw128(vt + k * 2048, kKeys * 128), idesc_pv,
                      (j > 1) || (k != 0));
        umma_commit(pv_done + 8 * h);
        umma_commit(empty + 8 * s);
        if (j + 2 < ntiles) ok = mbar_wait(pv_done + 8 * h, (j >> 1) & 1) && issue_qk(j + 2);
      }
      if (!ok) atomicExch(status, 22);
    }
  } else if (warp >= 4) {
    // ---- softmax and epilogue ----
    const int h = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int idx = tile * ROWS + row;
    const int entry = lo + idx / G, head = kvh * G + idx % G;
    const int tok = row < ROWS && entry < hi ? __ldcg(gr.decode_tokens + entry) : -1;
    // Keys of the slice that this row sees end here. A row without a token may see anything: it is not looked at.
    const int limit = tok >= 0 ? min(k1, m.pos[tok] + 1) : k1;
    const bool live = __any_sync(0xffffffffu, tok >= 0);       // some row of the warp belongs to a token
    float m_ref = -INFINITY, l_run = 0.f;  // the maximum that the exponents refer to (log2 domain)
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tmem_s = tmem_base + h * kKeys + lane_sel, tmem_o = tmem_base + 2 * kKeys + h * D + lane_sel;
    const int steps = (ntiles - h + 1) >> 1;  // tiles of this stream
    for (int i = 0; i < steps && ok; ++i) {
      // Q K^T of this tile was issued behind the stream's last P V: O_h is at rest, too
      ok = __all_sync(0xffffffffu, mbar_wait(s_ready + 8 * h, i & 1));
      if (!ok) break;
      tc_fence_after();
      if (live) {
        const int key0 = k0 + (2 * i + h) * kKeys;
        const bool masked = __any_sync(0xffffffffu, key0 + kKeys > limit);
        auto hide = [&](uint32_t (&v)[32], int key) {
          if (!masked) return;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (key + e >= limit) v[e] = __float_as_uint(-INFINITY);
        };
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          uint32_t va[32], vb[32];
          tmem_ld32(tmem_s + c * 32, va);
          tmem_ld32(tmem_s + c * 32 + 32, vb);
          tmem_ld_wait();
          hide(va, key0 + c * 32);
          hide(vb, key0 + c * 32 + 32);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            mx4[e & 3] = fmaxf(mx4[e & 3], fmaxf(__uint_as_float(va[e]), __uint_as_float(vb[e])));
        }
        const float m_cand = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2e;
        if (__any_sync(0xffffffffu, m_cand > m_ref + kGrow)) {  // always on a row's first visible tile
          const float m_new = fmaxf(m_ref, m_cand);
          const float corr = m_new == -INFINITY ? 1.f : fast_exp2(m_ref - m_new);
          if (i > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(tmem_o + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st16(tmem_o + c * 16, o);
            }
          }
          l_run *= corr;
          m_ref = m_new;
        }
        const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;  // a row without a visible key yet: all -inf, all weights 0
        const float2 sc2 = make_float2(scale_log2e, scale_log2e), nm2 = make_float2(neg_m, neg_m);
        float2 sum2[2] = {{0.f, 0.f}, {0.f, 0.f}};
        // 32 scores -> 16 pairs of weights, over columns of S that have been read: 16 c + 15 < 32 (c + 1)
        auto weigh = [&](uint32_t (&v)[32], int c) {
          uint32_t pk[16];
          hide(v, key0 + c * 32);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), sc2, nm2);
            const float2 w = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            sum2[e & 1] = __fadd2_rn(sum2[e & 1], w);
            pk[e] = pack_half2(w.x, w.y);  // fp16 for the tensor cores: 2^-11 of each weight
          }
          tmem_st16(tmem_s + c * 16, pk);
        };
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          uint32_t va[32], vb[32];
          tmem_ld32(tmem_s + c * 32, va);
          tmem_ld32(tmem_s + c * 32 + 32, vb);
          tmem_ld_wait();
          weigh(va, c);
          weigh(vb, c + 1);
        }
        const float2 st = __fadd2_rn(sum2[0], sum2[1]);
        l_run += st.x + st.y;
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready + 8 * h);
    }
    if (ok && steps > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(pv_done + 8 * h, (steps - 1) & 1));
      tc_fence_after();
    }
    if (!ok) atomicExch(status, 23);
    // The second stream parks (m, l, O) in the ring, idle now that both streams are done, the first joins the two
    // there, and all eight warps store the rows.
    float* park = reinterpret_cast<float*>(gen + (sKV - base));
    float* park_m = park + ROWS * S::kParkStride;
    float* park_l = park_m + ROWS;
    int* park_at = reinterpret_cast<int*>(park_l + ROWS);  // the row's (entry, head), or -1
    float* mine = park + row * S::kParkStride;
    softmax_bar();
    if (h == 1 && live) {
      park_m[row] = m_ref;
      park_l[row] = l_run;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32] = {};
        if (steps > 0) {  // else nothing has been accumulated, and TMEM may hold anything
          tmem_ld32(tmem_o + c * 32, v);
          tmem_ld_wait();
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(mine + c * 32 + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
      }
    }
    softmax_bar();
    if (h == 0 && row < ROWS) {
      park_at[row] = ok && tok >= 0 ? entry * heads + head : -1;
      if (live) {
        const float m_b = park_m[row], l_b = park_l[row];
        const float M = fmaxf(m_ref, m_b), ref = M == -INFINITY ? 0.f : M;
        const float wa = fast_exp2(m_ref - ref), wb = fast_exp2(m_b - ref);
        const long long at = (static_cast<long long>(entry) * heads + head) * part.total + blockIdx.z;
        if (ok && tok >= 0) *reinterpret_cast<float2*>(part.ml + at * 2) = make_float2(M, wa * l_run + wb * l_b);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[32];
          tmem_ld32(tmem_o + c * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float4 x = *reinterpret_cast<const float4*>(mine + c * 32 + e);
            x.x = wa * __uint_as_float(v[e]) + wb * x.x, x.y = wa * __uint_as_float(v[e + 1]) + wb * x.y;
            x.z = wa * __uint_as_float(v[e + 2]) + wb * x.z, x.w = wa * __uint_as_float(v[e + 3]) + wb * x.w;
            *reinterpret_cast<float4*>(mine + c * 32 + e) = x;
          }
        }
      }
    }
    softmax_bar();
    constexpr int kLanes = D / 4, kSide = 32 / kLanes;  // lanes to a row, rows to a warp's store
    const int d = (lane % kLanes) * 4;
#pragma unroll 4
    for (int r = (warp - 4) * kSide + lane / kLanes; r < ROWS; r += 8 * kSide) {
      const long long at = park_at[r];
      if (at >= 0)
        *reinterpret_cast<float4*>(part.o + (at * part.total + blockIdx.z) * D + d) =
            *reinterpret_cast<const float4*>(park + r * S::kParkStride + d);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int D, int ROWS>
void launch_d(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const __half* kc, const __half* vc,
              const Partials& px, int tiles, cudaStream_t st) {
  using S = Smem<D, ROWS>;
  static PerDeviceOnce once;
  auto kernel = umma_prefix_kernel<D, ROWS>;
  once.run([&] {
    RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kTotal)));
  });
  // The pool as rows of D halves, box = one 16-key page x 64 dims. The row count only limits the
  // coordinates: the kernel asks for no row that the block table does not name.
  const CUtensorMap mk = make_map(kc, 2, 1LL << 31, D, D, 16, 64, true);
  const CUtensorMap mv = make_map(vc, 2, 1LL << 31, D, D, 16, 64, true);
  count_launch();
  launch_pdl(kernel, dim3(tiles, s.kv_heads, px.parts), dim3(kThreads), S::kTotal, st, mk, mv, kc, vc, q, m, gr, px, s.heads, s.kv_heads,
             s.block_size, s.q_stride, kLog2e / sqrtf(static_cast<float>(D)), status_word());
}

}  // namespace

bool umma_prefix_usable(const AttnShape& s) { return (s.D == 64 || s.D == 128) && s.block_size % 16 == 0; }

void launch_umma_prefix(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const __half* kc, const __half* vc,
                        const Partials& px, int rows, int tiles, cudaStream_t st) {
  if (s.D == 64 && rows == 64) launch_d<64, 64>(s, q, m, gr, kc, vc, px, tiles, st);
  else if (s.D == 64) launch_d<64, 128>(s, q, m, gr, kc, vc, px, tiles, st);
  else if (rows == 64) launch_d<128, 64>(s, q, m, gr, kc, vc, px, tiles, st);
  else launch_d<128, 128>(s, q, m, gr, kc, vc, px, tiles, st);
}

}  // namespace rb200
