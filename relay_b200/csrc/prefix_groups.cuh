// What the kernels of the shared-prefix decode attention (shared_prefix.cu, umma_prefix.cu) share: the
// group geometry, the layout of the shared part's partial results, and the walk from a row tile or
// a decode token to its group.
#pragma once

#include "kernels.h"

// The loads of the group and batch metadata here go to L2: the suffix kernel makes them ahead of its
// dependency wait, when they are complete in memory (the kernel in front of it has waited for them)
// but nothing has been said about this SM's L1.

namespace rb200 {

constexpr int kPrefixSlice = 128;     // slices of the shared keys are multiples of this
constexpr int kUmmaPrefixRows = 128;  // rows (token, head) of a CTA of umma_prefix_kernel

// The group geometry on the device.
struct Groups {
  const int* decode_tokens;
  const int* off;         // [n_groups + 1]
  const int* prefix_len;  // [n_groups]; null: nothing is shared
  int n_decode, n_groups;
};

// Partial results of the shared part: o [n_decode * heads][parts][D], then (max in log2 units, sum)
// [n_decode * heads][parts]. Slice p of a prefix of P keys starts at p * slice_of(P, parts); slices
// that start at or behind P are neither written nor read.
struct Partials {
  float* o;
  float* ml;
  int parts;
};

__device__ __forceinline__ int slice_of(int P, int parts) { return (((P + parts - 1) / parts) + kPrefixSlice - 1) / kPrefixSlice * kPrefixSlice; }

// How many keys the group [lo, hi) shares, and the block table that names them.
struct Prefix {
  int keys;
  const int* table;
};
__device__ __forceinline__ Prefix prefix_of(const Groups& gr, const TokenMeta& m, int g, int lo, int hi) {
  int tok = -1;
  for (int i = lo; i < hi && tok < 0; ++i) tok = __ldcg(gr.decode_tokens + i);  // the first entry that is not padding
  if (tok < 0 || gr.prefix_len == nullptr) return {0, nullptr};
  const int keys = min(__ldcg(gr.prefix_len + g), __ldcg(m.pos + tok) + 1);
  if (keys <= 0) return {0, nullptr};
  return {keys, m.tables + __ldcg(m.table_off + __ldcg(m.seq + tok))};
}

// Entries [lo, hi) of group g; bounds that do not fit the batch are cut to it.
__device__ __forceinline__ void group_bounds(const Groups& gr, int g, int& lo, int& hi) {
  lo = max(__ldcg(gr.off + g), 0);
  hi = min(__ldcg(gr.off + g + 1), gr.n_decode);
}

// The x-th row tile over all groups, a group of n entries having ceil(n * G / rows) of them. Called by
// whole warps; every lane gets the answer. False behind the last tile.
__device__ __forceinline__ bool find_tile(const Groups& gr, int G, int rows, int x, int& g, int& tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < gr.n_groups; g0 += 32) {
    int n = 0;
    if (g0 + lane < gr.n_groups) {
      int lo, hi;
      group_bounds(gr, g0 + lane, lo, hi);
      n = (max(hi - lo, 0) * G + rows - 1) / rows;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + incl > x);
    if (past) {
      const int src = __ffs(past) - 1;
      g = g0 + src;
      tile = x - before - __shfl_sync(0xffffffffu, incl - n, src);
      return true;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// The group that entry di belongs to, or -1.
__device__ __forceinline__ int group_of(const Groups& gr, int di) {
  const int lane = threadIdx.x & 31;
  int n = 0;  // offsets at or before di
  for (int j0 = 0; j0 <= gr.n_groups; j0 += 32)
    n += __popc(__ballot_sync(0xffffffffu, j0 + lane <= gr.n_groups && __ldcg(gr.off + min(j0 + lane, gr.n_groups)) <= di));
  return n >= 1 && n <= gr.n_groups ? n - 1 : -1;
}

// umma_prefix.cu: the shared keys on tcgen05 tensor cores, for head sizes 64 and 128 and block sizes that are
// multiples of 16; `tiles` bounds the row tiles of kUmmaPrefixRows rows.
bool umma_prefix_usable(const AttnShape& s);
void launch_umma_prefix(const AttnShape& s, const float* q, const TokenMeta& m, const Groups& gr, const __half* kc, const __half* vc,
                        const Partials& px, int tiles, cudaStream_t st);

}  // namespace rb200
