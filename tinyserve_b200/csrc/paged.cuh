// What the paged-cache kernels share: the arguments of a call, the map from
// a token to its sequence and position, and the one place that turns a cached
// position into an address (with its bounds checks).
#pragma once
#include <cuda_fp8.h>

#include <type_traits>

#include "tsb_common.cuh"
#include "tsb_internal.h"

namespace tsb {

struct PagedArgs {
  const uint8_t* kc;
  const uint8_t* vc;
  int64_t page_stride, head_stride, row_stride;  // elements
  const int32_t* table;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  int32_t* err;
  int num_pages, page_size, table_stride, max_pos;  // max_pos: table_width * page_size
  int n_seqs, n_tokens, max_q, nq, nkv, G;
};

// One sequence of the batch: its rows of q / out and its cached positions.
struct SeqSpan {
  int q0, q_len, kv_len;
};

// Lengths that contradict the call are reported and cut to what can be read.
__device__ __forceinline__ SeqSpan seq_span(const PagedArgs& a, int b) {
  SeqSpan s;
  s.q0 = a.cu_q[b];
  const int q1 = a.cu_q[b + 1];
  s.kv_len = a.kv_lens[b];
  if (s.q0 < 0 || q1 < s.q0 || q1 > a.n_tokens || q1 - s.q0 > a.max_q || s.kv_len < 0 || s.kv_len > a.max_pos) {
    atomicExch(a.err, kDevBadPlan);
    s.q0 = min(max(s.q0, 0), a.n_tokens);
    s.q_len = 0;
    s.kv_len = 0;
    return s;
  }
  s.q_len = q1 - s.q0;
  return s;
}

// Element offset of (sequence b, position j, KV head 0) in either pool; -1
// for a page outside the pool.
__device__ __forceinline__ int64_t cached_row(const PagedArgs& a, int b, int j) {
  const int pg = j / a.page_size;
  const int page = a.table[(int64_t)b * a.table_stride + pg];
  if (page < 0 || page >= a.num_pages) {
    atomicExch(a.err, kDevBadPlan);
    return -1;
  }
  return page * a.page_stride + (j - pg * a.page_size) * a.row_stride;
}

// The sequence that owns a token row: the last b with cu_q[b] <= token; -1
// when the row lies outside every sequence.
__device__ __forceinline__ int seq_of(const PagedArgs& a, int token) {
  int lo = 0, hi = a.n_seqs;  // cu_q[lo] <= token < cu_q[hi]
  if (a.n_seqs == 0 || token < a.cu_q[0] || token >= a.cu_q[a.n_seqs]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= token)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <int DT>  // TSB_DT_BF16 / TSB_DT_F16
__device__ __forceinline__ float to_f32(uint16_t b) {
  if constexpr (DT == TSB_DT_BF16)
    return __uint_as_float(static_cast<uint32_t>(b) << 16);
  else
    return __half2float(__ushort_as_half(b));
}
template <int DT>
__device__ __forceinline__ uint16_t from_f32(float x) {
  if constexpr (DT == TSB_DT_BF16)
    return f32_to_bf16_bits(x);
  else
    return __half_as_ushort(__float2half_rn(x));
}
__device__ __forceinline__ float e4m3_to_f32(uint8_t b) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(b, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

// One attention call.
struct AttnCall {
  PagedArgs p;
  const uint16_t* q;
  uint16_t* out;
  int64_t q_token_stride, q_head_stride;  // elements
  const float* sinks;
  unsigned* counters;  // zero between calls
  float* part;         // partial results of split key ranges
  float scale;
  int window, keep_first;  // keep_first is 0 without a window
  int short_rows;          // the long kernel leaves sequences with at most so many rows per KV head to the short one
};

// A sequence with at most this many rows (new tokens x query heads of a KV
// head) per KV head goes to the short kernel, one with more to the long one
// (which takes all where there is no launch of the short one).
constexpr int kShortRows = 16;

// Workspace: the error word, the counters, the partial results.
constexpr size_t kPagedHead = TSB_PAGED_ZEROED;  // of the first two; the last are written before they are read
size_t long_partial_bytes(int head_dim);
size_t short_partial_bytes(int head_dim);
int launch_paged_short(const TsbPagedCache& cache, const AttnCall& c, cudaStream_t st);
int launch_paged_long(const TsbPagedCache& cache, const AttnCall& c, cudaStream_t st);

// Calls f with the cache's type, head size and storage as constants.
template <class F>
void dispatch_paged(const TsbPagedCache& c, F f) {
  auto by_type = [&](auto dt, auto d) {
    if (c.cache_fp8)
      f(dt, d, std::true_type{});
    else
      f(dt, d, std::false_type{});
  };
  auto by_dim = [&](auto dt) {
    if (c.head_dim == 64)
      by_type(dt, std::integral_constant<int, 64>{});
    else
      by_type(dt, std::integral_constant<int, 128>{});
  };
  if (c.dtype == TSB_DT_BF16)
    by_dim(std::integral_constant<int, TSB_DT_BF16>{});
  else
    by_dim(std::integral_constant<int, TSB_DT_F16>{});
}

}  // namespace tsb
