// Log probabilities of given tokens, with each row's entropy and its most likely tokens, from [T, V] logits.
//
// Beside probs_from_logits (nanovllm/layers/spec_sampler.py:65-69), which writes all T * V probabilities; a server that
// answers with log probabilities needs a few numbers a row.  With x = logit / temperature, m = max x:
//   S = sum e^(x - m),  log p_t = x_t - m - log S,  H = log S - (sum (x - m) e^(x - m)) / S   (both terms >= 0).
// The alternatives are the num_top largest logits (ties to the lowest index, NaN above all) with their log p.
//
// First form: one CTA a row, a pass for the maximum, one for the sums, one for each alternative.
#include "common.cuh"

#include <math.h>

namespace specdec {
namespace logprobs {

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;
constexpr int kErrToken = 8;

// Ranks logits: larger first, the two zeros equal, NaN above all (but below the all-ones sentinel), ties to the lower index.
__device__ __forceinline__ unsigned long long rank_key(float f, unsigned index) {
  const unsigned high = f != f ? 0xfffffffeu : ordered_key(f == 0.0f ? 0.0f : f);
  return (static_cast<unsigned long long>(high) << 32) | (0xffffffffu - index);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const T* logits, long long row_stride, int V,
                                                            const long long* tokens, const float* temps, int num_top,
                                                            float* lp, float* entropy, long long* top_ids, float* top_lp,
                                                            int* err) {
  __shared__ float redf[2][kThreads / 32];
  __shared__ unsigned long long redk[kThreads / 32];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = logits + row * row_stride;
  const long long token = tokens[row];
  if (token < 0) {
    if (tid == 0) lp[row] = entropy[row] = 0.0f;
    for (int i = tid; i < num_top; i += kThreads) {
      top_ids[(long long)row * num_top + i] = -1;
      top_lp[(long long)row * num_top + i] = 0.0f;
    }
    return;
  }
  const float temp = temps ? temps[row] : 1.0f;
  float m = -INFINITY;
  for (int i = tid; i < V; i += kThreads) m = fmaxf(m, to_f32(x[i]));
  m = warp_max_f32(m);
  if (lane == 0) redf[0][warp] = m;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, redf[0][w]);
  __syncthreads();
  float s = 0.0f, e = 0.0f;
  for (int i = tid; i < V; i += kThreads) {
    const float d = (to_f32(x[i]) - m) / temp;
    const float p = expf(d);
    s += p;
    e += d == -INFINITY ? 0.0f : d * p;
  }
  s = warp_sum_f32(s);
  e = warp_sum_f32(e);
  if (lane == 0) {
    redf[0][warp] = s;
    redf[1][warp] = e;
  }
  __syncthreads();
  s = e = 0.0f;
  for (int w = 0; w < kThreads / 32; ++w) {
    s += redf[0][w];
    e += redf[1][w];
  }
  const float log_s = logf(s);
  if (tid == 0) {
    if (token >= V) {
      atomicCAS(err, 0, kErrToken);
      lp[row] = NAN;
    } else {
      lp[row] = (to_f32(x[token]) - m) / temp - log_s;
    }
    entropy[row] = log_s - e / s;
  }
  unsigned long long prev = ~0ull;
  for (int n = 0; n < num_top; ++n) {
    unsigned long long best = 0;
    for (int i = tid; i < V; i += kThreads) {
      const unsigned long long k = rank_key(to_f32(x[i]), i);
      if (k < prev && k > best) best = k;
    }
    best = warp_max_u64(best);
    __syncthreads();
    if (lane == 0) redk[warp] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) best = redk[w] > best ? redk[w] : best;
    prev = best;
    if (tid == 0) {
      top_ids[(long long)row * num_top + n] = argmax_key_index(best);
      top_lp[(long long)row * num_top + n] = (key_to_float((unsigned)(best >> 32)) - m) / temp - log_s;
    }
  }
}

}  // namespace logprobs
}  // namespace specdec

using namespace specdec;

extern "C" {

int specdec_token_logprobs(const void* logits, int dtype, long long T, long long V, long long row_stride,
                           const long long* tokens, const float* temperatures, int num_top, float* logprobs,
                           float* entropy, long long* top_ids, float* top_logprobs, int* err, void* stream) {
  namespace L = specdec::logprobs;
  SPECDEC_CHECK_ARG(dtype_ok(dtype), "dtype code %d", dtype);
  SPECDEC_CHECK_ARG(T >= 0 && T <= 65535 && V >= 1 && V <= (1 << 24) && row_stride >= V, "bad sizes: %lld rows of %lld", T, V);
  SPECDEC_CHECK_ARG(num_top >= 0 && num_top <= L::kMaxTop && num_top <= V, "num_top %d: 0 to %d and at most V", num_top,
                    L::kMaxTop);
  if (T == 0) return kOk;
  SPECDEC_CHECK_ARG(logits && tokens && logprobs && entropy && err && (num_top == 0 || (top_ids && top_logprobs)),
                    "null pointer argument");
  SPECDEC_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype) == 0, "logits not aligned to their type");
  const dim3 grid((unsigned)T);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == kF32)
    L::logprobs_kernel<float><<<grid, L::kThreads, 0, s>>>(static_cast<const float*>(logits), row_stride, (int)V, tokens,
                                                           temperatures, num_top, logprobs, entropy, top_ids, top_logprobs, err);
  else if (dtype == kBF16)
    L::logprobs_kernel<__nv_bfloat16><<<grid, L::kThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(logits), row_stride,
                                                                   (int)V, tokens, temperatures, num_top, logprobs,
                                                                   entropy, top_ids, top_logprobs, err);
  else
    L::logprobs_kernel<__half><<<grid, L::kThreads, 0, s>>>(static_cast<const __half*>(logits), row_stride, (int)V, tokens,
                                                            temperatures, num_top, logprobs, entropy, top_ids,
                                                            top_logprobs, err);
  SPECDEC_LAUNCH_CHECK();
  return kOk;
}

}  // extern "C"
