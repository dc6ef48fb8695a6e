// The shared keys of the shared-prefix decode attention (shared_prefix.cu) on tcgen05 tensor cores, for
// head sizes 64 and 128 and block sizes that are multiples of 16.
//
// One CTA takes 128 rows, a row being one query head of one token: tokens of one group, heads of one
// KV head, so every row sees the same keys. It runs over a slice of the group's shared keys in tiles
// of 128:
//   S = Q K^T    A = Q in shared memory as two fp16 halves (q = hi + lo, exact to 2^-22 of q: with hi
//                alone the rounding of q would cost as much as that of the output), B = the K tile,
//                D = S in TMEM (128 lanes x 128 columns). One buffer, released as soon as the softmax
//                warps hold it in registers;
//   softmax      eight warps, two threads per row, one per 64-key half of the tile, each with its own
//                running (reference maximum, sum); P = exp2(.) as fp16 into one of two buffers in TMEM;
//   O_h += P_h V_h   one product per half, A = P_h from TMEM, B = the half's V rows, D = O_h in TMEM,
//                rescaled only when a row's maximum outgrew its reference by 2^8.
// At the end the halves of a row are joined and (maximum, sum, O) is left as the row's partial result.
// Rows without a token cost nothing but their share of the products: a warp without any skips the softmax.
//
// K and V tiles pass through one ring of slots in the order K0 V0 K1 V1 ..., each slot with its own
// pair of barriers: a K slot is free again once its scores are made, long before V of the same tile.
// Every wait is bounded; one that gives up records a code in the device's status word.
#include <cuda.h>

#include "attn_tiles.cuh"
#include "kernels.h"
#include "prefix_groups.cuh"
#include "tcgen05.cuh"

namespace rb200 {

using namespace tc;

namespace {

constexpr int kKeys = 128;
constexpr int kRows = kUmmaPrefixRows;
constexpr int kThreads = 384;  // two loader warps, the MMA issuer, a third loader, eight softmax warps
template <int D>
struct Smem {
  static constexpr int kQBytes = kRows * D * 2;  // one half of q
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kSlots = D == 64 ? 10 : 5;
  static constexpr int kBarBytes = 256;
  static constexpr size_t kTotal = 2 * kQBytes + static_cast<size_t>(kSlots) * kTileBytes + kBarBytes + 1024;
  static_assert(kTotal <= 232448, "shared memory of one CTA");
  static_assert(static_cast<size_t>(kSlots) * kTileBytes >= static_cast<size_t>(2 + D) * kRows * 4, "the halves meet in the ring");
};

__device__ __forceinline__ void softmax_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
umma_prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __half* __restrict__ kc,
                   const __half* __restrict__ vc, const float* __restrict__ q, TokenMeta m, Groups gr, Partials part, int heads,
                   int kv_heads, int bs, int q_stride, float scale_log2e, int* __restrict__ status) {
  using S = Smem<D>;
  constexpr int NS = S::kSlots;
  constexpr float kGrow = 8.f;  // how far (log2) a row's maximum may outgrow its reference before O is rescaled
  // TMEM columns: S 0..127, P of even tiles 128..191 and of odd tiles 192..255, then O of the two halves.
  constexpr uint32_t kTmemCols = 512;
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  unsigned char* gen = smem_dyn + (base - smem_u32(smem_dyn));
  const uint32_t sQ = base;
  const uint32_t sKV = sQ + 2 * S::kQBytes;
  const uint32_t bars = sKV + NS * S::kTileBytes;
  const uint32_t full = bars, empty = bars + 80;             // NS (<= 10) x 8 bytes each
  const uint32_t s_ready = bars + 160, s_free = bars + 168;
  const uint32_t p_ready = bars + 176, pv_done = bars + 192;  // one per half
  const uint32_t q_ready = bars + 208, tmem_slot = bars + 216;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    mbar_init(s_ready, 1);
    mbar_init(s_free, 8);
    for (int s = 0; s < 2; ++s) {
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
  const int G = heads / kv_heads, kvh = blockIdx.y;
  const RowTile rt = find_tile(gr, G, kRows, blockIdx.x);
  const int lo = rt.lo, hi = rt.hi, tile = rt.tile;
  const Prefix px = rt.g >= 0 ? prefix_of(gr, m, rt.g, lo, hi) : Prefix{0, nullptr};
  const int slice = slice_of(px.keys, part.parts);
  const int k0 = blockIdx.z * slice, k1 = min(px.keys, k0 + slice);
  const int ntiles = (k1 - k0 + kKeys - 1) / kKeys;  // 0 or less: nothing to do
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(gen + (tmem_slot - base));

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
    // ---- MMA issuer: Q K^T of tile j + 1 as soon as the softmax warps hold the scores of tile j, then
    //      P V of tile j when P arrives ----
    if (elect_one()) {
      constexpr uint32_t idesc_qk = umma_idesc(kRows, kKeys);
      constexpr uint32_t idesc_pv = umma_idesc(kRows, D) | (1u << 16);  // B (V) is MN-major
      auto issue_qk = [&](int j) {
        const int s = (2 * j) % NS;
        const uint32_t kt = sKV + s * S::kTileBytes;
#pragma unroll
        for (int part_q = 0; part_q < 2; ++part_q)
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k / 4) * (kRows * 128) + (k % 4) * 32;  // 64-wide atom, then 32 bytes per 16 dims
            umma_f16(tmem_base, smem_desc_sw128(sQ + part_q * S::kQBytes + off), smem_desc_sw128(kt + off), idesc_qk,
                     part_q != 0 || k != 0);
          }
        umma_commit(s_ready);
        umma_commit(empty + 8 * s);
      };
      ok = mbar_wait(q_ready, 0) && mbar_wait(full, 0);
      if (ok) {
        tc_fence_after();
        issue_qk(0);
      }
      for (int j = 0; j < ntiles && ok; ++j) {
        if (j + 1 < ntiles) {
          const int u = 2 * j + 2;
          ok = mbar_wait(s_free, j & 1) && mbar_wait(full + 8 * (u % NS), (u / NS) & 1);
          if (!ok) break;
          tc_fence_after();
          issue_qk(j + 1);
        }
        const int u = 2 * j + 1, s = u % NS;
        ok = mbar_wait(full + 8 * s, (u / NS) & 1);
        if (!ok) break;
        const uint32_t vt = sKV + s * S::kTileBytes;
#pragma unroll 1
        for (int h = 0; h < 2 && ok; ++h) {
          ok = mbar_wait(p_ready + 8 * h, j & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t pa = tmem_base + kKeys + (j & 1) * 64 + h * 32;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ta(tmem_base + 2 * kKeys + h * D, pa + 8 * k, smem_desc_mn_sw128(vt + (h * 4 + k) * 2048, kKeys * 128),
                        idesc_pv, (j > 0) || (k != 0));
          umma_commit(pv_done + 8 * h);
        }
        if (!ok) break;
        umma_commit(empty + 8 * s);
      }
      if (!ok) atomicExch(status, 22);
    }
  } else if (warp >= 4) {
    // ---- softmax and epilogue ----
    const int half = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int idx = tile * kRows + row;
    const int entry = lo + idx / G, head = kvh * G + idx % G;
    const int tok = entry < hi ? gr.decode_tokens[entry] : -1;
    const int limit = tok >= 0 ? min(k1, m.pos[tok] + 1) : 0;  // keys of the slice that this row sees end here
    const bool live = __any_sync(0xffffffffu, tok >= 0);       // some row of the warp belongs to a token
    {  // q row -> hi + lo -> swizzled A operands (each half converts half of the row's chunks)
      const float* src = q + static_cast<long long>(max(tok, 0)) * q_stride + head * D;
#pragma unroll
      for (int cc = 0; cc < D / 16; ++cc) {
        const int c = half * (D / 16) + cc;
        float x[8] = {};
        if (tok >= 0) {
          const float4 a = *reinterpret_cast<const float4*>(src + c * 8), b = *reinterpret_cast<const float4*>(src + c * 8 + 4);
          x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        }
        uint32_t hv[4], lv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_half2(x[2 * i], x[2 * i + 1], hv[i], lv[i]);
        unsigned char* dst = gen + (sQ - base) + (c / 8) * (kRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(dst) = make_uint4(hv[0], hv[1], hv[2], hv[3]);
        *reinterpret_cast<uint4*>(dst + S::kQBytes) = make_uint4(lv[0], lv[1], lv[2], lv[3]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    float m_ref = -INFINITY, l_run = 0.f;  // the maximum that the exponents refer to (log2 domain)
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tmem_o = tmem_base + 2 * kKeys + half * D + lane_sel;
    for (int j = 0; j < ntiles && ok; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(s_ready, j & 1));
      if (!ok) break;
      tc_fence_after();
      const int key0 = k0 + j * kKeys + half * 64;
      const uint32_t tmem_s = tmem_base + lane_sel + half * 64;
      const uint32_t tmem_p = tmem_base + kKeys + (j & 1) * 64 + half * 32 + lane_sel;
      uint32_t sv[64], pk[32];
      if (live) {
        tmem_ld32(tmem_s, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
        tmem_ld32(tmem_s + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
        tmem_ld_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      if (live) {
        if (__any_sync(0xffffffffu, key0 + 64 > limit)) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (key0 + i >= limit) sv[i] = __float_as_uint(-INFINITY);
        }
        // Exponentials against the current reference with the maximum gathered in the same pass; only when a
        // row outgrew its reference (always on its first visible tile) the pass is repeated.
        float sum = 0.f, mx = 0.f;
        auto exp_pass = [&](float neg_m) {
          float2 sum2[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          const float2 sc2 = make_float2(scale_log2e, scale_log2e), nm2 = make_float2(neg_m, neg_m);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float2 sp = make_float2(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1]));
            const float2 x = __ffma2_rn(sp, sc2, nm2);
            const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            mx4[i & 3] = fmaxf(mx4[i & 3], fmaxf(sp.x, sp.y));
            sum2[i & 3] = __fadd2_rn(sum2[i & 3], e);
            pk[i] = pack_half2(e.x, e.y);  // fp16 for the tensor cores: 2^-11 of each weight
          }
          const float2 st = __fadd2_rn(__fadd2_rn(sum2[0], sum2[1]), __fadd2_rn(sum2[2], sum2[3]));
          sum = st.x + st.y;
          mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        };
        exp_pass(m_ref == -INFINITY ? 0.f : -m_ref);
        const float m_cand = mx * scale_log2e;
        if (__any_sync(0xffffffffu, m_cand > m_ref + kGrow)) {
          const float m_new = fmaxf(m_ref, m_cand);
          const float corr = m_new == -INFINITY ? 1.f : fast_exp2(m_ref - m_new);
          if (j > 0) {
            ok = __all_sync(0xffffffffu, mbar_wait(pv_done + 8 * half, (j - 1) & 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t v[32];
              tmem_ld32(tmem_o + c * 32, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
              tmem_st32(tmem_o + c * 32, v);
            }
          }
          l_run *= corr;
          m_ref = m_new;
          exp_pass(m_ref == -INFINITY ? 0.f : -m_ref);
        }
        l_run += sum;
      }
      // Arrive for tile j only once this half's product of tile j - 1 is done (a half that arrived twice
      // while the issuer waits for the other would complete a phase unobserved); the product of tile
      // j - 2, the last reader of this P buffer, is done then too.
      if (j > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(pv_done + 8 * half, (j - 1) & 1));
        if (!ok) break;
      }
      if (live) {
        tmem_st32(tmem_p, pk);
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready + 8 * half);
    }
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_wait(pv_done + 8 * half, (ntiles - 1) & 1));
      tc_fence_after();
    }
    if (!ok) atomicExch(status, 23);
    // The second half parks (m, l, O) in the idle ring as [value][row], the first half joins and stores.
    float* park = reinterpret_cast<float*>(gen + (sKV - base));
    if (half == 1 && ok && live) {
      park[row] = m_ref;
      park[kRows + row] = l_run;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        tmem_ld32(tmem_o + c * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) park[(2 + c * 32 + i) * kRows + row] = __uint_as_float(v[i]);
      }
    }
    softmax_bar();
    if (half == 0 && ok && live) {
      const float m_b = park[row], l_b = park[kRows + row];
      const float M = fmaxf(m_ref, m_b), ref = M == -INFINITY ? 0.f : M;
      const float wa = fast_exp2(m_ref - ref), wb = fast_exp2(m_b - ref);
      const long long at = (static_cast<long long>(entry) * heads + head) * part.total + blockIdx.z;
      if (tok >= 0) *reinterpret_cast<float2*>(part.ml + at * 2) = make_float2(M, wa * l_run + wb * l_b);
      float* dst = part.o + at * D;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        tmem_ld32(tmem_o + c * 32, v);  // every lane takes part in the load
        tmem_ld_wait();
        if (tok >= 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = wa * __uint_as_float(v[i + e]) + wb * park[(2 + c * 32 + i + e) * kRows + row];
            *reinterpret_cast<float4*>(dst + c * 32 + i) = make_float4(o[0], o[1], o[2], o[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int D>
void launch_d(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const __half* kc, const __half* vc,
              const Partials& px, int tiles, cudaStream_t st) {
  using S = Smem<D>;
  static PerDeviceOnce once;
  auto kernel = umma_prefix_kernel<D>;
  if (once.first())
    RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kTotal)));
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
                        const Partials& px, int tiles, cudaStream_t st) {
  if (s.D == 64) launch_d<64>(s, q, m, gr, kc, vc, px, tiles, st);
  else launch_d<128>(s, q, m, gr, kc, vc, px, tiles, st);
}

}  // namespace rb200
