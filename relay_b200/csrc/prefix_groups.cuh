// What the kernels of the shared-prefix decode attention (shared_prefix.cu, umma_prefix.cu) share: the
// group geometry, the layout of the shared part's partial results, and the walk from a row tile or
// a decode token to its group.
#pragma once

#include "kernels.h"

// The loads of the group and batch metadata here go to L2: the suffix and join kernels make them ahead of a
// dependency wait, when they are complete in memory (the first kernel of the call has waited for
// them ahead of its trigger) but nothing has been said about this SM's L1.

namespace rb200 {

constexpr int kPrefixSlice = 128;  // slices of the shared keys are multiples of this

// The group geometry on the device.
struct Groups {
  const int* decode_tokens;
  const int* off;         // [n_groups + 1]
  const int* prefix_len;  // [n_groups]; null: nothing is shared
  int n_decode, n_groups;
};

// Partial results, `total` to a (token, head): o [n_decode * heads][total][D], then (maximum in log2 units, sum)
// [n_decode * heads][total]. The first `parts` are the slices of the shared keys: slice p of a prefix of
// P keys starts at p * slice_of(P, parts), and one that starts at or behind P is neither written nor
// read. The others are the slices of the token's own keys.
struct Partials {
  float* o;
  float* ml;
  int parts, total;
};

__device__ __forceinline__ int slice_of(int P, int parts) { return (((P + parts - 1) / parts) + kPrefixSlice - 1) / kPrefixSlice * kPrefixSlice; }

// How many of them a prefix of P keys fills.
__device__ __forceinline__ int slices_used(int P, int parts) {
  if (P <= 0) return 0;
  const int slice = slice_of(P, parts);
  return (P + slice - 1) / slice;
}

// How many keys the entries [lo, hi) of group g share, and (`with_table`) the block table that names them.
struct Prefix {
  int keys;
  const int* table;
};
__device__ __forceinline__ Prefix prefix_of(const Groups& gr, const TokenMeta& m, int g, int lo, int hi, bool with_table) {
  if (gr.prefix_len == nullptr || lo >= hi) return {0, nullptr};
  const int len = __ldcg(gr.prefix_len + g);
  int tok = __ldcg(gr.decode_tokens + lo);
  for (int i = lo + 1; i < hi && tok < 0; ++i) tok = __ldcg(gr.decode_tokens + i);  // the first entry that is not padding
  if (tok < 0) return {0, nullptr};
  const int pos = __ldcg(m.pos + tok), seq = with_table ? __ldcg(m.seq + tok) : 0;
  const int keys = min(len, pos + 1);
  if (keys <= 0) return {0, nullptr};
  return {keys, with_table ? m.tables + __ldcg(m.table_off + seq) : nullptr};
}

// A row tile: group g, its entries [lo, hi), and the tile's number in the group.
struct RowTile {
  int g, lo, hi, tile;
};

// The x-th row tile over all groups, a group of n entries having ceil(n * G / rows) of them. Called by whole
// warps; every lane gets the answer. g = -1 behind the last tile. Bounds that do not fit the batch are cut to it.
__device__ __forceinline__ RowTile find_tile(const Groups& gr, int G, int rows, int x) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < gr.n_groups; g0 += 32) {
    const int g = min(g0 + lane, gr.n_groups - 1);
    const int lo = max(__ldcg(gr.off + g), 0), hi = min(__ldcg(gr.off + g + 1), gr.n_decode);
    const int n = g0 + lane < gr.n_groups ? (max(hi - lo, 0) * G + rows - 1) / rows : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + incl > x);
    if (past) {
      const int src = __ffs(past) - 1;
      return {g0 + src, __shfl_sync(0xffffffffu, lo, src), __shfl_sync(0xffffffffu, hi, src),
              x - before - __shfl_sync(0xffffffffu, incl - n, src)};
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return {-1, 0, 0, 0};
}

// The group that entry di belongs to and the group's entries; g = -1 for padding. Called by whole warps.
__device__ __forceinline__ RowTile group_of(const Groups& gr, int di) {
  const int lane = threadIdx.x & 31;
  int n = 0, lo = 0, hi = gr.n_decode;  // n: offsets at or before di; lo the last of them, hi the first behind
  for (int j0 = 0; j0 <= gr.n_groups; j0 += 32) {
    const int off = __ldcg(gr.off + min(j0 + lane, gr.n_groups));
    const unsigned in = __ballot_sync(0xffffffffu, j0 + lane <= gr.n_groups && off <= di);
    n += __popc(in);
    if (in) lo = __shfl_sync(0xffffffffu, off, 31 - __clz(in));
    if (in != 0xffffffffu) {
      hi = __shfl_sync(0xffffffffu, off, __ffs(~in) - 1);
      break;
    }
  }
  return {n >= 1 && n <= gr.n_groups ? n - 1 : -1, max(lo, 0), min(hi, gr.n_decode), 0};
}

// umma_prefix.cu: the shared keys on tcgen05 tensor cores, for head sizes 64 and 128 and block sizes that are
// multiples of 16; `tiles` bounds the row tiles of `rows` rows (64 or 128).
bool umma_prefix_usable(const AttnShape& s);
void launch_umma_prefix(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const __half* kc, const __half* vc,
                        const Partials& px, int rows, int tiles, cudaStream_t st);

}  // namespace rb200
