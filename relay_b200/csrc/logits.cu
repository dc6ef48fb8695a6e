// What a request asks of its logits ahead of the sampler: penalties for tokens that occur in its
// history, biases, and a grammar's mask, in one pass over the row.
//
// A CTA owns a segment of one row's vocabulary. It counts the history's tokens of that segment in
// shared memory (integer atomics: the counts do not depend on their order), notes the last bias
// entry of each token the same way, and then passes once over the segment's logits. 8 bytes per
// logit move, plus one bit of mask: the kernel is bound by memory, and by latency for a few rows.
#include "kernels.h"

namespace rb200 {

namespace {

constexpr int kLgThreads = 512;
constexpr int kLgSegment = 4096;
constexpr uint32_t kSeen = 0x80000000u;  // the token occurs; the bits below count the generated ones

__global__ void __launch_bounds__(kLgThreads)
adjust_logits_kernel(const float* logits, int ld_logits, float* out, int ld_out, int V, const rb200_penalties* __restrict__ penalties,
                     const int* __restrict__ history, int ld_history, const int* __restrict__ history_len,
                     const int* __restrict__ prompt_len, const int* __restrict__ bias_ids, const float* __restrict__ bias_values,
                     int ld_bias, const int* __restrict__ bias_len, const uint32_t* __restrict__ mask, int ld_mask) {
  __shared__ uint32_t count[kLgSegment];
  __shared__ int last[kLgSegment];
  pdl_trigger();
  pdl_wait();
  const long long r = blockIdx.y;
  const int v0 = blockIdx.x * kLgSegment, n = min(kLgSegment, V - v0);
  for (int i = threadIdx.x; i < n; i += kLgThreads) {
    count[i] = 0;
    last[i] = -1;
  }
  __syncthreads();
  rb200_penalties pen{1.0f, 0.0f, 0.0f, 0.0f};
  if (penalties) {
    pen = penalties[r];
    const int len = min(history_len[r], ld_history), prompt = prompt_len ? prompt_len[r] : 0;
    const int* h = history + r * ld_history;
    for (int i = threadIdx.x; i < len; i += kLgThreads) {
      const uint32_t v = static_cast<uint32_t>(h[i]) - static_cast<uint32_t>(v0);
      if (v < static_cast<uint32_t>(n)) {
        if (i < prompt) atomicOr(&count[v], kSeen);
        else atomicAdd(&count[v], 1u);
      }
    }
  }
  const float* bv = bias_values + r * ld_bias;
  if (bias_ids) {
    const int len = min(bias_len[r], ld_bias);
    const int* b = bias_ids + r * ld_bias;
    for (int i = threadIdx.x; i < len; i += kLgThreads) {
      const uint32_t v = static_cast<uint32_t>(b[i]) - static_cast<uint32_t>(v0);
      if (v < static_cast<uint32_t>(n)) atomicMax(&last[v], i);
    }
  }
  __syncthreads();
  const float* x = logits + r * ld_logits + v0;
  float* o = out + r * ld_out + v0;
  const uint32_t* mk = mask ? mask + r * ld_mask : nullptr;
  for (int i = threadIdx.x; i < n; i += kLgThreads) {
    float y = x[i];
    const uint32_t c = count[i];
    if (c) {
      y = y > 0.0f ? y / pen.repetition : y * pen.repetition;
      const uint32_t times = c & ~kSeen;
      if (times) y -= pen.frequency * static_cast<float>(times) + pen.presence;
    }
    if (last[i] >= 0) y += bv[last[i]];
    if (mk && !((mk[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u)) y = -INFINITY;
    o[i] = y;
  }
}

}  // namespace

void launch_adjust_logits(const float* logits, int ld_logits, float* out, int ld_out, int R, int V, const rb200_penalties* penalties,
                          const int* history, int ld_history, const int* history_len, const int* prompt_len, const int* bias_ids,
                          const float* bias_values, int ld_bias, const int* bias_len, const uint32_t* mask, int ld_mask,
                          cudaStream_t st) {
  if (R == 0) return;
  count_launch();
  launch_pdl(adjust_logits_kernel, dim3(div_up(V, kLgSegment), R), dim3(kLgThreads), 0, st, logits, ld_logits, out, ld_out, V, penalties,
             history, ld_history, history_len, prompt_len, bias_ids, bias_values, ld_bias, bias_len, mask, ld_mask);
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
