// RoPE + store into a paged KV cache, and the entry points of the paged
// operators (tsb_paged_kv_store, tsb_paged_attention).
//
// The cache is a pool of pages shared by all requests
// (tinyserve/paged_kv_cache.py:20-122); a sliding window may keep the first
// tokens visible (tinyserve/static_kv_cache.py:282-389); GPT-OSS adds a sink
// logit per head to the softmax denominator.
//
//   out_t = sum_j e^(s_tj - m) v_j / (e^(sink - m) + sum_j e^(s_tj - m)),
//   s_tj = scale * q_t . k_j,  j visible to t,  m the largest of them.
//
// Sequences with few rows are bound by the cache's bytes, longer chunks by
// products and exponentials: one kernel each (paged_attn_short.cu,
// paged_attn_long.cu); a batch that may have both takes two launches.
#include "paged.cuh"

namespace tsb {
namespace {

// ------------------------------------------------------------------ store
// Bound by the bytes of the rows.  A thread takes 8 dims of a head's lower half
// with the 8 of its upper half (two 16-byte loads, two 16-byte stores), so
// rotation needs no exchange, for every 32nd (D = 64) or 16th head of its
// token: the table's values are read once for all of them, and up to three
// heads' loads are under way together, ahead of the look-ups of sequence and
// page that the stores wait for.  Products and sums are rounded one by one in
// fp32 (no contraction), then once to the 16-bit type.  Measured: 8192 tokens of
// 64 + 16 heads of 64 into a bf16 cache 28.8 us, 91% of the measured copy rate
// (one CTA per token, the table read for every head: 87 us).
constexpr int kStoreToken = 128;  // threads of a token
struct StoreArgs {
  PagedArgs p;
  const uint16_t* qkv;
  int64_t qkv_stride;
  const void* cos;
  const void* sin;
  uint16_t* q_out;
  int max_rope;
};

template <int TT>
__device__ __forceinline__ void load_table8(const void* t, int64_t at, float (&r)[8]) {
  if constexpr (TT == TSB_DT_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(t) + at);
    const float4 a = p[0], b = p[1];
    r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w;
    r[4] = b.x, r[5] = b.y, r[6] = b.z, r[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(t) + at);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[2 * i] = to_f32<TT>((uint16_t)w[i]);
      r[2 * i + 1] = to_f32<TT>((uint16_t)(w[i] >> 16));
    }
  }
}

template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == TSB_DT_F16)
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    else
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 8 values of the 16-bit type, rounded once more to e4m3.  The hardware's
// conversion saturates; a plain cast makes NaN (with the value's sign) of what
// rounds past 448, that is of what lies above 464.
template <int DT>
__device__ __forceinline__ uint2 pack8_e4m3(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = to_f32<DT>((uint16_t)w[i]), hi = to_f32<DT>((uint16_t)(w[i] >> 16));
    uint16_t b;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(hi), "f"(lo));
    uint32_t two = b;
    if (!(fabsf(lo) <= 464.f)) two |= 0x007Fu;
    if (!(fabsf(hi) <= 464.f)) two |= 0x7F00u;
    o[i / 2] |= two << (16 * (i & 1));
  }
  return make_uint2(o[0], o[1]);
}

template <int DT, int D, bool FP8, int TT>
__global__ void __launch_bounds__(256, 4) paged_store_kernel(const StoreArgs s) {
  const PagedArgs& a = s.p;
  constexpr int kC = D / 16;  // 8-dim chunks of a half
  constexpr int kSlots = kStoreToken / kC, kAhead = 3;
  const int token = blockIdx.x * (256 / kStoreToken) + threadIdx.x / kStoreToken;
  if (token >= a.n_tokens) return;
  const int c = threadIdx.x % kC, slot = threadIdx.x % kStoreToken / kC, heads = a.nq + 2 * a.nkv;
  const uint16_t* src = s.qkv + (int64_t)token * s.qkv_stride + c * 8;
  uint4 r1[kAhead], r2[kAhead];
  const auto load = [&](int first) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int head = first + u * kSlots;
      if (head < heads) {
        r1[u] = *reinterpret_cast<const uint4*>(src + head * D);
        r2[u] = *reinterpret_cast<const uint4*>(src + head * D + D / 2);
      }
    }
  };
  load(slot);
  const int b = seq_of(a, token);
  if (b < 0) return;
  const SeqSpan sp = seq_span(a, b);
  const int pos = sp.kv_len - sp.q_len + (token - sp.q0);
  if (token - sp.q0 >= sp.q_len) return;  // a span that was reported and cut
  if (pos < 0 || pos >= s.max_rope) {
    if (threadIdx.x % kStoreToken == 0) atomicExch(a.err, kDevBadPlan);
    return;
  }
  float cs[8], sn[8];
  load_table8<TT>(s.cos, (int64_t)pos * (D / 2) + c * 8, cs);
  load_table8<TT>(s.sin, (int64_t)pos * (D / 2) + c * 8, sn);
  const int64_t row = cached_row(a, b, pos);
  for (int first = slot; first < heads; first += kAhead * kSlots) {
    if (first > slot) load(first);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int head = first + u * kSlots;
      if (head >= heads) break;
      uint4 o1 = r1[u], o2 = r2[u];
      if (head < a.nq + a.nkv) {
        float y1[8], y2[8];
        const uint32_t w1[4] = {o1.x, o1.y, o1.z, o1.w}, w2[4] = {o2.x, o2.y, o2.z, o2.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x1 = to_f32<DT>((uint16_t)(w1[i / 2] >> (16 * (i & 1))));
          const float x2 = to_f32<DT>((uint16_t)(w2[i / 2] >> (16 * (i & 1))));
          y1[i] = __fsub_rn(__fmul_rn(x1, cs[i]), __fmul_rn(x2, sn[i]));
          y2[i] = __fadd_rn(__fmul_rn(x2, cs[i]), __fmul_rn(x1, sn[i]));
        }
        o1 = pack8<DT>(y1);
        o2 = pack8<DT>(y2);
      }
      if (head < a.nq) {
        uint16_t* q = s.q_out + ((int64_t)token * a.nq + head) * D + c * 8;
        *reinterpret_cast<uint4*>(q) = o1;
        *reinterpret_cast<uint4*>(q + D / 2) = o2;
      } else if (row >= 0) {
        const bool key = head < a.nq + a.nkv;
        const int64_t at = row + (int64_t)(head - a.nq - (key ? 0 : a.nkv)) * a.head_stride + c * 8;
        uint8_t* pool = const_cast<uint8_t*>(key ? a.kc : a.vc);
        if constexpr (FP8) {
          *reinterpret_cast<uint2*>(pool + at) = pack8_e4m3<DT>(o1);
          *reinterpret_cast<uint2*>(pool + at + D / 2) = pack8_e4m3<DT>(o2);
        } else {
          *reinterpret_cast<uint4*>(pool + 2 * at) = o1;
          *reinterpret_cast<uint4*>(pool + 2 * (at + D / 2)) = o2;
        }
      }
    }
  }
}

// ------------------------------------------------------------------ host
int fail(int code, const char* what) { return set_error(code, what); }

// Checks what both entry points share and fills the kernel's arguments.
int paged_args(const TsbPagedCache* c, const TsbPagedBatch* b, int n_q_heads, void* ws, size_t ws_bytes, PagedArgs& a) {
  if (!c || !b || !ws) return fail(TSB_ERR_INVALID, "null pointer");
  if (c->head_dim != 64 && c->head_dim != 128) return fail(TSB_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (c->dtype != TSB_DT_BF16 && c->dtype != TSB_DT_F16) return fail(TSB_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  if (c->cache_fp8 != 0 && c->cache_fp8 != 1) return fail(TSB_ERR_INVALID, "cache_fp8 must be 0 or 1");
  if (c->n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % c->n_kv_heads)
    return fail(TSB_ERR_INVALID, "n_q_heads must be a positive multiple of n_kv_heads");
  if (c->num_pages < 0 || c->page_size <= 0) return fail(TSB_ERR_INVALID, "page_size must be positive");
  if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_q < 0 || b->table_width < 0 || b->table_stride < b->table_width)
    return fail(TSB_ERR_INVALID, "bad batch sizes");
  if ((int64_t)b->table_width * c->page_size > INT32_MAX / 2) return fail(TSB_ERR_UNSUPPORTED, "page table too wide");
  if ((int64_t)b->n_tokens * n_q_heads > INT32_MAX / 2) return fail(TSB_ERR_UNSUPPORTED, "too many tokens in one call");
  const int64_t per16 = c->cache_fp8 ? 16 : 8;
  if (c->page_stride % per16 || c->head_stride % per16 || c->row_stride % per16 || c->page_stride < 0 ||
      c->head_stride < 0 || c->row_stride < 0)
    return fail(TSB_ERR_INVALID, "cache strides must be multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(c->k_cache) | reinterpret_cast<uintptr_t>(c->v_cache)) & 15)
    return fail(TSB_ERR_INVALID, "caches must be 16-byte aligned");
  if (b->n_tokens > 0 && b->n_seqs > 0 &&
      (!c->k_cache || !c->v_cache || !b->cu_q || !b->kv_lens || (b->table_width > 0 && !b->page_table)))
    return fail(TSB_ERR_INVALID, "null pointer");
  if ((reinterpret_cast<uintptr_t>(b->page_table) | reinterpret_cast<uintptr_t>(b->cu_q) |
       reinterpret_cast<uintptr_t>(b->kv_lens)) & 3)
    return fail(TSB_ERR_INVALID, "page_table, cu_q and kv_lens must be 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(ws) & 255) return fail(TSB_ERR_INVALID, "workspace must be 256-byte aligned");
  if (ws_bytes < tsb_paged_workspace(c->head_dim)) return fail(TSB_ERR_WORKSPACE, "workspace too small");
  a.kc = static_cast<const uint8_t*>(c->k_cache);
  a.vc = static_cast<const uint8_t*>(c->v_cache);
  a.page_stride = c->page_stride;
  a.head_stride = c->head_stride;
  a.row_stride = c->row_stride;
  a.table = b->page_table;
  a.cu_q = b->cu_q;
  a.kv_lens = b->kv_lens;
  a.err = static_cast<int32_t*>(ws);
  a.num_pages = c->num_pages;
  a.page_size = c->page_size;
  a.table_stride = b->table_stride;
  a.max_pos = b->table_width * c->page_size;
  a.n_seqs = b->n_seqs;
  a.n_tokens = b->n_tokens;
  a.max_q = b->max_q;
  a.nq = n_q_heads;
  a.nkv = c->n_kv_heads;
  a.G = n_q_heads / c->n_kv_heads;
  return TSB_OK;
}

int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TSB_OK : fail(TSB_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace

int sm_count() {
  static int count[64];  // by device
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  if (dev < 64 && count[dev]) return count[dev];
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
  if (dev < 64) count[dev] = n;
  return n;
}

}  // namespace tsb

using namespace tsb;

extern "C" {

size_t tsb_paged_workspace(int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return 0;
  const size_t a = long_partial_bytes(head_dim), b = short_partial_bytes(head_dim);
  return kPagedHead + (a > b ? a : b);
}

int tsb_paged_kv_store(const TsbPagedCache* cache, const TsbPagedBatch* batch, const void* qkv, int64_t qkv_stride,
                       int32_t n_q_heads, const void* cos, const void* sin, int32_t table_dtype, int32_t max_pos,
                       void* q_out, void* workspace, size_t workspace_bytes, void* stream) {
  StoreArgs s{};
  const int rc = paged_args(cache, batch, n_q_heads, workspace, workspace_bytes, s.p);
  if (rc) return rc;
  if (table_dtype != TSB_DT_F32 && table_dtype != TSB_DT_BF16 && table_dtype != TSB_DT_F16)
    return fail(TSB_ERR_UNSUPPORTED, "cos / sin must be fp32, bf16 or f16");
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return TSB_OK;
  if (!qkv || !cos || !sin || !q_out) return fail(TSB_ERR_INVALID, "null pointer");
  if (qkv_stride < (int64_t)(n_q_heads + 2 * cache->n_kv_heads) * cache->head_dim || qkv_stride % 8)
    return fail(TSB_ERR_INVALID, "qkv rows must not overlap and be a multiple of 8 elements apart");
  const auto overlaps = [&](int n, int64_t stride) { return n > 1 && stride < cache->head_dim; };
  if (overlaps(cache->n_kv_heads, cache->head_stride) || overlaps(cache->page_size, cache->row_stride) ||
      overlaps(cache->num_pages, cache->page_stride))
    return fail(TSB_ERR_INVALID, "rows of the caches must not overlap");
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin) |
       reinterpret_cast<uintptr_t>(q_out)) & 15)
    return fail(TSB_ERR_INVALID, "qkv, cos, sin and q_out must be 16-byte aligned");
  s.qkv = static_cast<const uint16_t*>(qkv);
  s.qkv_stride = qkv_stride;
  s.cos = cos;
  s.sin = sin;
  s.q_out = static_cast<uint16_t*>(q_out);
  s.max_rope = max_pos;
  const dim3 grid((batch->n_tokens + 256 / kStoreToken - 1) / (256 / kStoreToken));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto dt, auto d, auto fp8, auto tt) {
    paged_store_kernel<decltype(dt)::value, decltype(d)::value, decltype(fp8)::value, decltype(tt)::value>
        <<<grid, 256, 0, st>>>(s);
  };
  dispatch_paged(*cache, [&](auto dt, auto d, auto fp8) {
    if (table_dtype == TSB_DT_F32)
      go(dt, d, fp8, std::integral_constant<int, TSB_DT_F32>{});
    else if (table_dtype == TSB_DT_BF16)
      go(dt, d, fp8, std::integral_constant<int, TSB_DT_BF16>{});
    else
      go(dt, d, fp8, std::integral_constant<int, TSB_DT_F16>{});
  });
  return launched();
}

int tsb_paged_attention(const TsbPagedCache* cache, const TsbPagedBatch* batch, const void* q, int64_t q_token_stride,
                        int64_t q_head_stride, int32_t n_q_heads, int32_t window, int32_t keep_first,
                        const float* sinks, float scale, void* out, void* workspace, size_t workspace_bytes,
                        void* stream) {
  AttnCall c{};
  const int rc = paged_args(cache, batch, n_q_heads, workspace, workspace_bytes, c.p);
  if (rc) return rc;
  if (window < 0 || keep_first < 0) return fail(TSB_ERR_INVALID, "window and keep_first must not be negative");
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return TSB_OK;
  if (!q || !out) return fail(TSB_ERR_INVALID, "null pointer");
  if (q_token_stride % 8 || q_head_stride % 8 || q_token_stride < 0 || q_head_stride < 0)
    return fail(TSB_ERR_INVALID, "q strides must be multiples of 8 elements");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
    return fail(TSB_ERR_INVALID, "q and out must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(sinks) & 3) return fail(TSB_ERR_INVALID, "sinks must be 4-byte aligned");
  c.q = static_cast<const uint16_t*>(q);
  c.out = static_cast<uint16_t*>(out);
  c.q_token_stride = q_token_stride;
  c.q_head_stride = q_head_stride;
  c.sinks = sinks;
  c.scale = scale;
  // No position is beyond the table's: a window that covers them all is none, and
  // what is left of either number stays far from the integers' end.
  c.window = window < c.p.max_pos ? window : 0;
  c.keep_first = c.window > 0 ? min(keep_first, c.p.max_pos) : 0;
  c.counters = static_cast<unsigned*>(workspace) + 64;
  c.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kPagedHead);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((int64_t)batch->max_q * c.p.G > kShortRows) {
    // Lengths are on the device.  Where the rows are as many as n_seqs sequences
    // of max_q tokens have, all sequences are long as a rule, and the long kernel
    // takes short ones too (a buffer that is not full) instead of a launch for
    // them: a prompt of 4096 tokens 268 us, 272 with the launch, 64 full sequences
    // of 4 tokens over 4096 bf16 positions 205 us and 214.  One token each in such a
    // buffer: 203 us, 103 with the launch.
    const bool full = (int64_t)batch->max_q * batch->n_seqs == batch->n_tokens;
    c.short_rows = full ? 0 : kShortRows;
    const int rl = launch_paged_long(*cache, c, st);
    if (rl || full) return rl;
  }
  return launch_paged_short(*cache, c, st);
}

}  // extern "C"
