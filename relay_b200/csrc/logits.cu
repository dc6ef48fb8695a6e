// What a request asks of its logits ahead of the sampler: penalties for tokens that occur in its
// history, biases, and a grammar's mask, in one pass over the row.
//
// A CTA owns a segment of one row's vocabulary. It counts the history's tokens of that segment in
// shared memory (integer atomics: the counts do not depend on their order) while the segment's
// logits are on their way into registers, then adjusts and stores them. The few biases follow as a
// correction of what was stored, with the counters' memory now holding the last entry of each biased
// token. 8 bytes per logit move, plus one bit of mask: the kernel is bound by memory, and by latency
// for a few rows.
#include "kernels.h"

namespace rb200 {

namespace {

constexpr int kLgThreads = 512;
constexpr uint32_t kSeen = 0x80000000u;  // the token occurs; the bits below count the generated ones

struct LogitArgs {
  const float* logits;
  float* out;
  const rb200_penalties* penalties;
  const int *history, *history_len, *prompt_len, *bias_ids;
  const float* bias_values;
  const int* bias_len;
  const uint32_t* mask;
  int ld_logits, ld_out, V, ld_history, ld_bias, ld_mask;
};

__device__ __forceinline__ float adjusted(float x, uint32_t c, const rb200_penalties& pen) {
  if (c) {
    x = x > 0.0f ? x / pen.repetition : x * pen.repetition;
    const uint32_t times = c & ~kSeen;
    if (times) x -= pen.frequency * static_cast<float>(times) + pen.presence;
  }
  return x;
}

__device__ __forceinline__ bool allowed(const uint32_t* mask, int v) { return mask == nullptr || ((mask[v >> 5] >> (v & 31)) & 1u); }

// NV vectors of 4 logits per thread: a segment of 2048 NV tokens. Segments are cut on the 16-byte grid of the
// row's memory, so the row's first `shift` (0..3) places of segment 0 lie ahead of the row.
template <int NV>
__global__ void __launch_bounds__(kLgThreads)
adjust_logits_kernel(const LogitArgs a) {
  constexpr int kSegment = kLgThreads * 4 * NV;
  extern __shared__ uint32_t count[];  // [kSegment]
  pdl_trigger();
  pdl_wait();
  const long long r = blockIdx.y;
  const float* x = a.logits + r * a.ld_logits;
  float* o = a.out + r * a.ld_out;
  const uint32_t* mask = a.mask ? a.mask + r * a.ld_mask : nullptr;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  const bool same_grid = static_cast<int>((reinterpret_cast<uintptr_t>(o) >> 2) & 3) == shift;
  const int V = a.V, v0 = static_cast<int>(blockIdx.x) * kSegment - shift;  // token at place 0
  if (v0 >= V) return;
  const int room = min(kSegment, V - v0);  // places behind the row's end count nothing

  float4 val[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int v = v0 + (n * kLgThreads + static_cast<int>(threadIdx.x)) * 4;
    if (v >= 0 && v + 4 <= V) {
      val[n] = *reinterpret_cast<const float4*>(x + v);
    } else {
      val[n].x = v >= 0 && v < V ? x[v] : 0.0f;
      val[n].y = v + 1 >= 0 && v + 1 < V ? x[v + 1] : 0.0f;
      val[n].z = v + 2 >= 0 && v + 2 < V ? x[v + 2] : 0.0f;
      val[n].w = v + 3 >= 0 && v + 3 < V ? x[v + 3] : 0.0f;
    }
  }

  rb200_penalties pen{1.0f, 0.0f, 0.0f, 0.0f};
  bool counted = false;  // some token of the row is penalised: the same answer in every thread
  if (a.penalties) {
    pen = a.penalties[r];
    const int len = min(a.history_len[r], a.ld_history);
    counted = len > 0 && !(pen.repetition == 1.0f && pen.presence == 0.0f && pen.frequency == 0.0f);
    if (counted) {
      uint4* zero = reinterpret_cast<uint4*>(count);
#pragma unroll
      for (int n = 0; n < NV; ++n) zero[n * kLgThreads + threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      const int prompt = a.prompt_len ? a.prompt_len[r] : 0;
      const int* h = a.history + r * a.ld_history;
      constexpr int U = 8;
      for (int i0 = threadIdx.x; i0 < len; i0 += U * kLgThreads) {
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = i0 + u * kLgThreads < len ? h[i0 + u * kLgThreads] : -1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = id[u] - v0;  // ids below 0 are passed over first: the difference then fits
          if (id[u] >= 0 && at >= 0 && at < room) {
            if (i0 + u * kLgThreads < prompt) atomicOr(&count[at], kSeen);
            else atomicAdd(&count[at], 1u);
          }
        }
      }
      __syncthreads();
    }
  }

#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int at = (n * kLgThreads + static_cast<int>(threadIdx.x)) * 4, v = v0 + at;
    float y[4] = {val[n].x, val[n].y, val[n].z, val[n].w};
    if (counted) {
      const uint4 c = *reinterpret_cast<const uint4*>(count + at);
      if (c.x | c.y | c.z | c.w) {
        y[0] = adjusted(y[0], c.x, pen), y[1] = adjusted(y[1], c.y, pen);
        y[2] = adjusted(y[2], c.z, pen), y[3] = adjusted(y[3], c.w, pen);
      }
    }
    if (v >= 0 && v + 4 <= V) {
      if (mask) {
        if (shift == 0) {
          const uint32_t bits = mask[v >> 5] >> (v & 31);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((bits >> e) & 1u)) y[e] = -INFINITY;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!allowed(mask, v + e)) y[e] = -INFINITY;
        }
      }
      if (same_grid) {
        *reinterpret_cast<float4*>(o + v) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[v + e] = y[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v + e >= 0 && v + e < V) o[v + e] = allowed(mask, v + e) ? y[e] : -INFINITY;
    }
  }

  if (a.bias_ids == nullptr) return;
  const int len = min(a.bias_len[r], a.ld_bias);
  if (len <= 0) return;
  const int* ids = a.bias_ids + r * a.ld_bias;
  const float* values = a.bias_values + r * a.ld_bias;
  auto place = [&](int i) {  // of entry i in the segment, or -1
    const int id = ids[i], at = id - v0;
    return id >= 0 && at >= 0 && at < room ? at : -1;
  };
  __syncthreads();  // the counters are read, the segment is stored
  for (int i = threadIdx.x; i < len; i += kLgThreads) {
    const int at = place(i);
    if (at >= 0) count[at] = 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < len; i += kLgThreads) {
    const int at = place(i);
    if (at >= 0) atomicMax(&count[at], static_cast<uint32_t>(i));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < len; i += kLgThreads) {
    const int at = place(i);
    if (at >= 0 && count[at] == static_cast<uint32_t>(i) && allowed(mask, v0 + at)) o[v0 + at] += values[i];
  }
}

template <int NV>
void launch_segments(const LogitArgs& a, int R, cudaStream_t st) {
  constexpr int kSegment = kLgThreads * 4 * NV;
  static PerDeviceOnce once;
  auto kernel = adjust_logits_kernel<NV>;
  if (once.first())
    RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSegment * 4));
  count_launch();
  launch_pdl(kernel, dim3(div_up(a.V + 3LL, kSegment), R), dim3(kLgThreads), kSegment * 4, st, a);
}

}  // namespace

void launch_adjust_logits(const float* logits, int ld_logits, float* out, int ld_out, int R, int V, const rb200_penalties* penalties,
                          const int* history, int ld_history, const int* history_len, const int* prompt_len, const int* bias_ids,
                          const float* bias_values, int ld_bias, const int* bias_len, const uint32_t* mask, int ld_mask,
                          cudaStream_t st) {
  if (R == 0) return;
  const LogitArgs a{logits, out, penalties, history, history_len, prompt_len, bias_ids, bias_values, bias_len, mask,
                    ld_logits, ld_out, V, ld_history, ld_bias, ld_mask};
  // Every segment reads its row's whole history, so segments are as long as leaves two CTAs for every SM.
  const long long places = V + 3LL, want = 2LL * sm_count();
  if (R * (places / (kLgThreads * 32)) >= want) launch_segments<8>(a, R, st);
  else if (R * (places / (kLgThreads * 16)) >= want) launch_segments<4>(a, R, st);
  else launch_segments<1>(a, R, st);
}

}  // namespace rb200

using namespace rb200;

extern "C" int rb200_adjust_logits(const float* logits, int ld_logits, float* out, int ld_out, int R, int V,
                                   const rb200_penalties* penalties, const int32_t* history, int ld_history,
                                   const int32_t* history_len, const int32_t* prompt_len, const int32_t* bias_ids,
                                   const float* bias_values, int ld_bias, const int32_t* bias_len, const uint32_t* mask, int ld_mask,
                                   void* stream) {
  return guarded([&] {
    RB_REQUIRE(R >= 0 && R <= 65535 && V > 0, "adjust_logits: bad shape (1 to 65535 rows)");
    RB_REQUIRE(ld_logits >= V && ld_out >= V, "adjust_logits: rows shorter than the vocabulary");
    if (R == 0) return 0;
    RB_REQUIRE(logits && out, "adjust_logits: null argument");
    RB_REQUIRE(logits != out || ld_logits == ld_out, "adjust_logits: in place needs the same stride");
    RB_REQUIRE(ld_history >= 0 && ld_bias >= 0, "adjust_logits: negative leading dimension");
    if (ld_history == 0) penalties = nullptr;  // no token of any row is penalised
    RB_REQUIRE(!penalties || (history && history_len), "adjust_logits: penalties need a history");
    if (ld_bias == 0) bias_ids = nullptr;
    RB_REQUIRE(!bias_ids || (bias_values && bias_len), "adjust_logits: bias ids need values and lengths");
    RB_REQUIRE(!mask || ld_mask >= div_up(V, 32), "adjust_logits: mask rows shorter than the vocabulary");
    launch_adjust_logits(logits, ld_logits, out, ld_out, R, V, penalties, history, ld_history, history_len, prompt_len, bias_ids,
                         bias_values, ld_bias, bias_len, mask, ld_mask, as_stream(stream));
    RB_CUDA(cudaGetLastError());
    return 0;
  });
}
