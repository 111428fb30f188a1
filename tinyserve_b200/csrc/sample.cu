// Token sampling with temperature, top-k, top-p and min-p from given random
// numbers (tsb_sample).
//
// Tokens are ranked by the 64-bit key (order-preserving bits of the logit,
// ~index): larger is better, no two are equal.  Every filter keeps a prefix of
// the ranking, so a row's kept set is {key >= T}:
//   top-k  T = the largest C with #{key >= C} >= k,
//   top-p  T = the largest C with mass{key >= C} >= p * mass of the k kept,
//   min-p  w >= min_p, w = exp((x - max) / temperature), monotone in the key.
#include <cfloat>

#include "tsb_common.cuh"
#include "tsb_internal.h"

namespace tsb {
namespace {

constexpr int kThreads = 1024;

struct SampleArgs {
  const void* logits;
  const float* noise;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
  float* logprobs;
  int64_t row_stride, noise_stride;
  int vocab;
};

template <int DT>
__device__ __forceinline__ float logit(const void* base, int64_t i) {
  float x;
  if constexpr (DT == TSB_DT_F32)
    x = static_cast<const float*>(base)[i];
  else if constexpr (DT == TSB_DT_BF16)
    x = bf16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
  else
    x = half_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
  return x != x ? -INFINITY : x;
}

// Ascending unsigned order of the floats' order; -0 and +0 alike.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_key(float x, int i) {
  return ((uint64_t)order_bits(x) << 32) | (uint32_t)~i;
}

template <typename T, typename F>
__device__ T block_reduce(T v, F f, T* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One CTA per row; each bit of a threshold costs one pass over the row.
template <int DT>
__global__ void __launch_bounds__(kThreads) sample_rows(const SampleArgs a) {
  __shared__ uint64_t red64[32];
  __shared__ double redd[32];
  const int row = blockIdx.x, V = a.vocab;
  constexpr int64_t EB = DT == TSB_DT_F32 ? 4 : 2;
  const void* x = static_cast<const char*>(a.logits) + row * a.row_stride * EB;
  const float* noise = a.noise ? a.noise + row * a.noise_stride : nullptr;
  const float t = a.temperature ? a.temperature[row] : 1.f;
  const bool greedy = !(t > 0.f) || !noise;
  const float inv = greedy ? 1.f : fminf(1.f / t, FLT_MAX);
  const auto more = [](uint64_t p, uint64_t q) { return p > q ? p : q; };
  uint64_t best = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) best = more(best, rank_key(logit<DT>(x, i), i));
  best = block_reduce(best, more, red64);
  const int first = (int)~(uint32_t)best;
  const float top = logit<DT>(x, first);
  if (top == -INFINITY) {
    if (threadIdx.x == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  // (x - max) / temperature, without 0 * infinity at either end
  const auto scaled = [&](float v) {
    if (v == top) return 0.f;
    return top == INFINITY || v == -INFINITY ? -INFINITY : fmaxf(v - top, -FLT_MAX) * inv;
  };
  const auto add = [](double p, double q) { return p + q; };
  const auto mass = [&](uint64_t c) {
    double s = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float v = logit<DT>(x, i);
      if (rank_key(v, i) >= c) s += expf(scaled(v));
    }
    return block_reduce(s, add, redd);
  };
  const double total = mass(0);
  uint64_t threshold = 0;
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < V) {
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t c = threshold | (1ull << bit);
      uint64_t n = 0;
      for (int i = threadIdx.x; i < V; i += kThreads) n += rank_key(logit<DT>(x, i), i) >= c;
      n = block_reduce(n, [](uint64_t p, uint64_t q) { return p + q; }, red64);
      if (n >= (uint64_t)k) threshold = c;
    }
  }
  const float p = a.top_p ? a.top_p[row] : 1.f;
  if (p < 1.f) {
    const double want = (double)p * (threshold ? mass(threshold) : total);
    uint64_t lower = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t c = lower | (1ull << bit);
      if (mass(c) >= want && c <= best) lower = c;
    }
    threshold = more(threshold, lower);
  }
  const float least = a.min_p ? a.min_p[row] : 0.f;
  int token = first;
  if (!greedy) {
    uint64_t win = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float v = logit<DT>(x, i), d = scaled(v);
      if (i != first && (rank_key(v, i) < threshold || d == -INFINITY || !(expf(d) >= least))) continue;
      const float r = d - logf(noise[i]);
      win = more(win, rank_key(r == r ? r : -INFINITY, i));
    }
    token = (int)~(uint32_t)block_reduce(win, more, red64);
  }
  if (threadIdx.x == 0) {
    a.tokens[row] = token;
    if (a.logprobs) a.logprobs[row] = scaled(logit<DT>(x, token)) - (float)log(total);
  }
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb_sample(const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t row_stride,
                          const float* noise, int64_t noise_stride, const float* temperature, const int32_t* top_k,
                          const float* top_p, const float* min_p, int64_t* tokens, float* logprobs, void* stream) {
  if (dtype != TSB_DT_F32 && dtype != TSB_DT_BF16 && dtype != TSB_DT_F16)
    return set_error(TSB_ERR_UNSUPPORTED, "logits must be fp32, bf16 or f16");
  if (rows < 0 || vocab <= 0) return set_error(TSB_ERR_INVALID, "rows must not be negative, vocab must be positive");
  if (row_stride < vocab || (noise && noise_stride < vocab)) return set_error(TSB_ERR_INVALID, "rows must not overlap");
  if (rows == 0) return TSB_OK;
  if (!logits || !tokens) return set_error(TSB_ERR_INVALID, "null pointer");
  const SampleArgs a{logits, noise,  temperature, top_k,        top_p, min_p,
                     tokens, logprobs, row_stride,  noise_stride, vocab};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TSB_DT_F32)
    sample_rows<TSB_DT_F32><<<rows, kThreads, 0, st>>>(a);
  else if (dtype == TSB_DT_BF16)
    sample_rows<TSB_DT_BF16><<<rows, kThreads, 0, st>>>(a);
  else
    sample_rows<TSB_DT_F16><<<rows, kThreads, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TSB_OK : set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
}
