// Log probabilities of given tokens, with the entropy of each row and its most probable tokens
// (the reference's sampler returns token ids only, mini_vllm/layers/sampler.py:12-25):
//   m = max_i x_i, Z = sum_i e^(x_i - m)
//   logprob = x_t - m - ln Z,   entropy = ln Z - (1/Z) sum_i e^(x_i - m) (x_i - m)
//   top: the top_n tokens by (logit descending, index ascending) and their log probabilities.
// Sums are fp32.  A masked token (-inf) has probability 0 and adds nothing to the entropy; a row
// with nothing but -inf has log probabilities -inf and entropy 0; a token id outside [0, vocab) has
// log probability -inf; a NaN or +inf makes the row's results NaN, and a NaN ranks below -inf.
#include "hl_common.cuh"

namespace hl {
namespace {

constexpr int kLpThreads = 1024;
constexpr int kMaxTop = 32;

__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_logit(const float* p) { return *p; }

// Whole numbers in the order of the logits: NaN lowest, then -inf ... +inf; -0 and +0 alike.  Never 0.
__device__ __forceinline__ uint32_t logit_key(float x) {
  if (x != x) return 1u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Unique over a row: larger for a larger logit, and for a lower index among equals.
__device__ __forceinline__ uint64_t entry_key(float x, int i) {
  return (uint64_t(logit_key(x)) << 32) | uint32_t(~i);
}

template <typename T>
__device__ T block_max(T v, T* shared) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const T w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < kLpThreads / 32; ++w) v = shared[w] > v ? shared[w] : v;
  return v;
}

__device__ float block_sum(float v, float* shared) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < kLpThreads / 32; ++w) v += shared[w];
  return v;
}

// One thread block per row, three passes and one more per alternative.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(
    const T* __restrict__ logits, int64_t row_stride, int vocab, const int64_t* __restrict__ tokens, int top_n,
    float* __restrict__ logprobs, float* __restrict__ entropies, int64_t* __restrict__ top_tokens,
    float* __restrict__ top_logprobs) {
  __shared__ uint64_t s64[32];
  __shared__ float sf[32];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * row_stride;
  uint64_t best = 0;
  float nan = 0.f;
  for (int i = threadIdx.x; i < vocab; i += kLpThreads) {
    const float v = load_logit(x + i);
    const uint64_t k = entry_key(v, i);
    best = k > best ? k : best;
    if (v != v) nan = v;
  }
  best = block_max(best, s64);
  const float m = load_logit(x + int(~uint32_t(best)));
  float z = nan, s = 0.f;
  for (int i = threadIdx.x; i < vocab; i += kLpThreads) {
    const float v = load_logit(x + i);
    if (v == -INFINITY) continue;
    const float e = expf(v - m);
    z += e;
    s += e * (v - m);
  }
  z = block_sum(z, sf);
  s = block_sum(s, sf);
  const float log_z = z != z ? z : (m == -INFINITY ? INFINITY : logf(z));
  if (threadIdx.x == 0) {
    const int64_t t = tokens[row];
    const float xt = t >= 0 && t < vocab ? load_logit(x + t) : -INFINITY;
    logprobs[row] = (xt == -INFINITY && log_z == log_z) ? -INFINITY : xt - m - log_z;
    entropies[row] = m == -INFINITY && z == z ? 0.f : log_z - s / z;
  }
  for (int r = 0; r < top_n; ++r) {
    if (r > 0) {
      uint64_t next = 0;
      for (int i = threadIdx.x; i < vocab; i += kLpThreads) {
        const uint64_t k = entry_key(load_logit(x + i), i);
        if (k < best && k > next) next = k;
      }
      best = block_max(next, s64);
    }
    if (threadIdx.x == 0) {
      const int i = int(~uint32_t(best));
      const float v = load_logit(x + i);
      top_tokens[row * top_n + r] = i;
      top_logprobs[row * top_n + r] = (v == -INFINITY && log_z == log_z) ? -INFINITY : v - m - log_z;
    }
  }
}

}  // namespace
}  // namespace hl

using namespace hl;

extern "C" int hl_token_logprobs(const void* logits, int logits_fp32, int64_t row_stride, int64_t rows, int vocab,
                                 const int64_t* token_ids, int top_n, float* logprobs, float* entropies,
                                 int64_t* top_tokens, float* top_logprobs, void* stream) {
  clear_error();
  HL_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff && vocab > 0 && row_stride >= vocab,
               "hl_token_logprobs: bad logits shape");
  HL_CHECK_ARG(top_n >= 0 && top_n <= kMaxTop && top_n <= vocab, "hl_token_logprobs: top_n not in [0, min(%d, vocab)]",
               kMaxTop);
  if (rows == 0) return HL_OK;
  HL_CHECK_ARG(logits && token_ids && logprobs && entropies && (top_n == 0 || (top_tokens && top_logprobs)),
               "hl_token_logprobs: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_fp32) {
    token_logprobs_kernel<float><<<unsigned(rows), kLpThreads, 0, s>>>(
        static_cast<const float*>(logits), row_stride, vocab, token_ids, top_n, logprobs, entropies, top_tokens,
        top_logprobs);
  } else {
    token_logprobs_kernel<__nv_bfloat16><<<unsigned(rows), kLpThreads, 0, s>>>(
        static_cast<const __nv_bfloat16*>(logits), row_stride, vocab, token_ids, top_n, logprobs, entropies,
        top_tokens, top_logprobs);
  }
  HL_CHECK_LAUNCH("hl_token_logprobs");
  return HL_OK;
}
