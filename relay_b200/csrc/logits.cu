// What a request asks of its logits ahead of the sampler: penalties for tokens that occur in its
// history, biases, and a grammar's mask, in one pass over the row.
//
// A CTA owns a segment of one row's vocabulary. It counts the history's tokens of the segment in shared memory
// (integer atomics, so the counts do not depend on their order) and reads which logits the mask leaves; then each
// of these is read, adjusted and stored (a vector of four that the mask takes whole is not read), while
// other CTAs of the SM are at their counts. The few biases follow as a correction of what was stored, with the
// counters' memory now holding the last entry of each biased token. At most 8 bytes per logit move, plus one
// bit of mask: the kernel is bound by memory, and by latency for a few rows.
#include <climits>

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

// x / repetition for x > 0 without a division (56 us instead of 53.9 for 256 rows of 128256 logits; the product with the
// reciprocal alone, 52, would be rounded twice). With repetition * scale in [1/2, 1) for a power of two `scale` (in
// [2^-23, 1) where the repetition is subnormal) the quotient is z / (repetition * scale), z = x * scale. Its product with
// the reciprocal is within 1.5 steps, and one residual step (Markstein's: r = z - q b in one rounding, q + r / b) brings
// it to the nearest float32 but for 2^-22 of a step. Where r could underflow or q overflow the product stands.
struct Repetition {
  float value, scale, scaled, inverse;
  __device__ __forceinline__ explicit Repetition(float repetition) : value(repetition) {
    const int biased = 253 - static_cast<int>(__float_as_uint(repetition) >> 23 & 255u);  // exponent of the scale
    scale = biased > 0 ? __uint_as_float(static_cast<uint32_t>(biased) << 23) : biased == 0 ? 0x1p-127f : 0x1p-128f;
    scaled = repetition * scale;
    inverse = 1.0f / scaled;
  }
  __device__ __forceinline__ float divides(float x) const {
    const float z = x * scale, q = z * inverse, y = __fmaf_rn(__fmaf_rn(-q, scaled, z), inverse, q);
    return z > 0x1p-100f && z < 0x1p100f ? y : q;
  }
};

__device__ __forceinline__ float adjusted(float x, uint32_t c, const rb200_penalties& pen, const Repetition& rep) {
  const float times = static_cast<float>(c & ~kSeen);
  const float less = times > 0.0f ? pen.frequency * times + pen.presence : 0.0f;
  return c ? (x > 0.0f ? rep.divides(x) : x * rep.value) - less : x;
}

__device__ __forceinline__ bool allowed(const uint32_t* mask, int v) { return mask == nullptr || ((mask[v >> 5] >> (v & 31)) & 1u); }

// NV vectors of 4 logits per thread: a segment of 4 kLgThreads NV tokens. Segments are cut on the 16-byte grid
// of the row's memory, so the row's first `shift` (0..3) places of segment 0 lie ahead of the row.
template <int NV>
__global__ void __launch_bounds__(kLgThreads, 3)
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
  const bool in_place = x == o;
  const int V = a.V, v0 = static_cast<int>(blockIdx.x) * kSegment - shift;  // token at place 0
  if (v0 >= V) return;
  const int room = min(kSegment, V - v0);  // places behind the row's end count nothing
  const int tid = static_cast<int>(threadIdx.x);

  // What is small and decides what follows: all of it under way before anything waits.
  rb200_penalties pen{1.0f, 0.0f, 0.0f, 0.0f};
  int len = 0, prompt = 0, biases = 0;  // the same in every thread
  if (a.penalties) {
    pen = a.penalties[r];
    len = a.history_len[r];
    if (a.prompt_len) prompt = a.prompt_len[r];
  }
  if (a.bias_ids) biases = a.bias_len[r];

  // Which values are in the row and pass the mask, four bits for each vector. A segment that lies inside the row on the
  // mask's own grid needs no look at the row's ends.
  const bool inside = shift == 0 && v0 + kSegment <= V;
  uint32_t keep = 0;
  if (inside) {
    uint32_t word[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) word[n] = mask ? mask[(v0 >> 5) + n * (kLgThreads / 8) + (tid >> 3)] : 0xffffffffu;
#pragma unroll
    for (int n = 0; n < NV; ++n) keep |= (word[n] >> ((tid & 7) * 4) & 15u) << (4 * n);
  } else {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int v = v0 + (n * kLgThreads + tid) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v + e >= 0 && v + e < V && allowed(mask, v + e)) keep |= 1u << (4 * n + e);
    }
  }

  // The place in the segment of a token id, or -1.
  auto place = [&](int id) {
    const int at = id - v0;  // ids below 0 are passed over first: for the others the difference fits
    return id >= 0 && at >= 0 && at < room ? at : -1;
  };
  len = min(len, a.ld_history);
  if (pen.repetition == 1.0f && pen.presence == 0.0f && pen.frequency == 0.0f) len = 0;
  const bool counted = len > 0;
  if (counted) {
    const int* h = a.history + r * a.ld_history;
    uint4* zero = reinterpret_cast<uint4*>(count);
#pragma unroll
    for (int n = 0; n < NV; ++n) zero[n * kLgThreads + tid] = make_uint4(0u, 0u, 0u, 0u);
    constexpr int U = 8;
    for (int i0 = tid; i0 - tid < len; i0 += U * kLgThreads) {
      int id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = i0 + u * kLgThreads < len ? h[i0 + u * kLgThreads] : INT_MIN;
      if (i0 == tid) __syncthreads();  // the counters are zero
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // one comparison: an id below 0 is out of reach, or a place ahead of the row, whose count nobody reads
        const uint32_t at = static_cast<uint32_t>(id[u]) - static_cast<uint32_t>(v0);
        if (at >= static_cast<uint32_t>(room)) continue;
        if (i0 + u * kLgThreads < prompt) atomicOr(&count[at], kSeen);
        else atomicAdd(&count[at], 1u);
      }
    }
    __syncthreads();
  }

  // The values, B vectors of a thread at a time. (All of them on their way ahead of the count leave registers for two CTAs
  // to an SM instead of three: 63 us for 256 rows of 128256 logits against 51, measured with a reciprocal in place of the
  // quotient. The first B ahead of it spill: 69.)
  const Repetition rep(pen.repetition);
  constexpr int B = NV < 4 ? NV : 4;
#pragma unroll
  for (int n0 = 0; n0 < NV; n0 += B) {
    float4 val[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int n = n0 + j, v = v0 + (n * kLgThreads + tid) * 4;
      const uint32_t bits = keep >> (4 * n) & 15u;
      val[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (inside || (v >= 0 && v + 4 <= V)) {
        if (bits) val[j] = *reinterpret_cast<const float4*>(x + v);
      } else {
        if (bits & 1u) val[j].x = x[v];
        if (bits & 2u) val[j].y = x[v + 1];
        if (bits & 4u) val[j].z = x[v + 2];
        if (bits & 8u) val[j].w = x[v + 3];
      }
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int n = n0 + j, at = (n * kLgThreads + tid) * 4, v = v0 + at;
      const uint32_t bits = keep >> (4 * n) & 15u;
      bool changed = !in_place || bits != 15u;
      if (counted && bits) {
        const uint4 c = *reinterpret_cast<const uint4*>(count + at);
        if (c.x | c.y | c.z | c.w) {
          changed = true;
          val[j].x = adjusted(val[j].x, c.x, pen, rep), val[j].y = adjusted(val[j].y, c.y, pen, rep);
          val[j].z = adjusted(val[j].z, c.z, pen, rep), val[j].w = adjusted(val[j].w, c.w, pen, rep);
        }
      }
      if (!changed) continue;
      const float y[4] = {bits & 1u ? val[j].x : -INFINITY, bits & 2u ? val[j].y : -INFINITY, bits & 4u ? val[j].z : -INFINITY,
                          bits & 8u ? val[j].w : -INFINITY};
      if (same_grid && (inside || (v >= 0 && v + 4 <= V))) {
        *reinterpret_cast<float4*>(o + v) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v + e >= 0 && v + e < V) o[v + e] = y[e];
      }
    }
  }

  biases = min(biases, a.ld_bias);
  if (biases <= 0) return;
  const int* ids = a.bias_ids + r * a.ld_bias;
  const float* values = a.bias_values + r * a.ld_bias;
  bool any = false;
  for (int i = tid; i < biases; i += kLgThreads) any |= place(ids[i]) >= 0;
  if (!__syncthreads_or(any)) return;  // also: the counters are read, the segment is stored
  for (int i = tid; i < biases; i += kLgThreads) {
    const int at = place(ids[i]);
    if (at >= 0) count[at] = 0u;
  }
  __syncthreads();
  for (int i = tid; i < biases; i += kLgThreads) {
    const int at = place(ids[i]);
    if (at >= 0) atomicMax(&count[at], static_cast<uint32_t>(i));
  }
  __syncthreads();
  for (int i = tid; i < biases; i += kLgThreads) {
    const int at = place(ids[i]);
    if (at >= 0 && count[at] == static_cast<uint32_t>(i) && allowed(mask, v0 + at)) o[v0 + at] += values[i];
  }
}

template <int NV>
void launch_segments(const LogitArgs& a, int R, cudaStream_t st) {
  constexpr int kSegment = kLgThreads * 4 * NV;
  static PerDeviceOnce once;
  auto kernel = adjust_logits_kernel<NV>;
  once.run([&] {
    RB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSegment * 4));
  });
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
  // Every segment reads its row's whole history, so segments are as long as leaves the GPU busy: three CTAs for every SM
  // in segments of 16384, two in 8192, one in 4096, otherwise 2048. Measured at 128256 logits and histories of 8192:
  // 256 rows 59, 72, 99 and 153 us in 16384, 8192, 4096 and 2048; 32 rows 13.5 in 8192, 15.0 in 4096; 16 rows 9.8 and 9.2;
  // 8 rows 7.3 in 4096, 7.4 in 2048; one row with 800 tokens 4.3 and 3.8.
  // (Clusters that read a history once and count in the owner's shared memory: 119 us for 256 rows; a list of the counted
  // tokens, whose values alone are adjusted once the others are stored: 77, against 51 then, with histories of 40 - 8192.)
  const long long places = V + 3LL, sms = sm_count();
  if (R * (places / (kLgThreads * 32)) >= 3 * sms) launch_segments<8>(a, R, st);
  else if (R * (places / (kLgThreads * 16)) >= 2 * sms) launch_segments<4>(a, R, st);
  else if (R * (places / (kLgThreads * 8)) >= sms) launch_segments<2>(a, R, st);
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
    RB_REQUIRE(R >= 0 && R <= 65535 && V > 0 && V <= (1 << 30), "adjust_logits: bad shape (at most 65535 rows of 2^30)");
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
