// Token sampling with temperature, top-k, top-p and min-p from given random
// numbers (tsb_sample).
//
// Tokens are ranked by a 64-bit key, (order-preserving bits of the logit,
// inverted index): larger is better, no two are equal.  Every filter keeps a
// prefix of the ranking, so a row's kept set is {key >= T}:
//   top-k  T = the k-th largest key,
//   top-p  T = the last key whose better ones weigh less than p * (mass of the k kept),
//   min-p  w >= min_p, w = exp((x - max) / temperature), monotone in the key.
// The kept token with the largest (x - max) / temperature - log(noise) wins.
//
// A cluster of CTAs shares a row: the logits come from memory once and from L2
// in the few passes after the first.
//   1. the best key;
//   2. sum of w, and (for top-k, top-p) a histogram over the distance from the
//      maximum: tokens per bin and their mass; without those filters the race;
//   3. the bin where the k-th token or the p-th part of the mass lies; a bin with
//      more than kList tokens is divided again by its keys, until its tokens fit
//      a list, where each counts the tokens and the mass before it;
//   4. the race among the keys from T on; noise is read for those alone.
// Masses are sums of integers, w in units of 2^-31, so neither the order of the
// atomic additions nor the number of CTAs changes a result.
#include <cfloat>

#include "tc05.cuh"
#include "tsb_common.cuh"
#include "tsb_internal.h"

namespace tsb {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 1024;     // two a thread
constexpr int kList = 1024;     // tokens that are ranked one by one
constexpr float kPerUnit = 32;  // bins of a unit of logit: 32 units, e^-32 of the best token's weight
constexpr int kMaxCluster = 8;

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
  int vocab, chunk;  // chunk: tokens of a CTA, a multiple of 8
  int index_bits;
};

struct Shared {
  uint64_t mass[kBins];  // combined over the cluster, for this CTA's share of the bins
  uint32_t count[kBins];
  uint32_t n[kBins], lo[kBins], hi[kBins];  // this CTA's tokens: count, mass (two words, carried by hand)
  uint64_t list[kList];                     // the first CTA's: keys of the chosen bin, and their masses
  uint32_t list_mass[kList];
  uint32_t listed;
  uint64_t red[kWarps], red2[kWarps];
  // read by the other CTAs
  uint64_t best, race, low, result_key, result_mass;
  double sum;
  // the bin that a scan found
  int bin;
  uint32_t bin_count, before_count;
  uint64_t before_mass;
};

template <int DT>
__device__ __forceinline__ float to_logit(uint32_t bits) {
  float x;
  if constexpr (DT == TSB_DT_F32)
    x = __uint_as_float(bits);
  else if constexpr (DT == TSB_DT_BF16)
    x = bf16_bits_to_f32((uint16_t)bits);
  else
    x = half_bits_to_f32((uint16_t)bits);
  return x != x ? -INFINITY : x;
}

// Ascending unsigned order of the floats' order; -0 and +0 alike.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// A value of another CTA's shared memory.
template <typename T>
__device__ __forceinline__ T remote(const T* mine, int rank) {
  const uint32_t at = mapa_shared(smem_u32(mine), rank);
  if constexpr (sizeof(T) == 8) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return *reinterpret_cast<T*>(&v);
  } else {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return *reinterpret_cast<T*>(&v);
  }
}

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, F f, T* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ uint64_t more(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ void sync_all() {
  __syncthreads();
  cluster_sync();
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_rows(const SampleArgs a) {
  __shared__ Shared sh;
  const int rank = (int)cluster_rank(), V = a.vocab;
  int ctas;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int row = blockIdx.x / ctas;
  constexpr int EB = DT == TSB_DT_F32 ? 4 : 2, PER = 16 / EB;  // tokens of a 16-byte load
  const char* x = static_cast<const char*>(a.logits) + row * a.row_stride * EB;
  const float* noise = a.noise ? a.noise + row * a.noise_stride : nullptr;
  const float t = a.temperature ? a.temperature[row] : 1.f;
  const bool greedy = !(t > 0.f) || !noise;
  const float inv = greedy ? 1.f : fminf(1.f / t, FLT_MAX);
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.f, least = a.min_p ? a.min_p[row] : 0.f;
  const bool by_k = !greedy && k > 0 && k < V, by_p = !greedy && p < 1.f;
  const uint64_t index_mask = (1ull << a.index_bits) - 1;
  const auto key_of = [&](float v, int i) { return ((uint64_t)order_bits(v) << a.index_bits) | (index_mask - i); };
  const auto index_of = [&](uint64_t key) { return (int)(index_mask - (key & index_mask)); };

  // f(index, logit) of this CTA's tokens.  Loads are 16 bytes wide on 16-byte
  // boundaries; a row that starts off them begins a few tokens early.
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / EB);
  const int v0 = rank * a.chunk, v1 = min(v0 + a.chunk, V + skew);  // places from the boundary on
  const auto each = [&](auto f) {
    const uint4* src = reinterpret_cast<const uint4*>(x - skew * EB);
    constexpr int kAhead = 4;
    for (int b = v0 / PER + threadIdx.x; b * PER < v1; b += kAhead * kThreads) {
      uint4 r[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int at = (b + u * kThreads) * PER;
        if (at >= skew && at + PER <= v1) r[u] = __ldg(src + b + u * kThreads);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int at = (b + u * kThreads) * PER;
        if (at >= v1) break;
        if (at >= skew && at + PER <= v1) {
          const uint32_t w[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
#pragma unroll
          for (int e = 0; e < PER; ++e)
            f(at + e - skew, to_logit<DT>(PER == 4 ? w[e] : w[e / 2] >> (16 * (e & 1))));
        } else {  // the row's ends
          for (int e = 0; e < PER; ++e) {
            const int i = at + e - skew;
            if (i < 0 || i >= V) continue;
            uint32_t bits;
            if constexpr (EB == 4)
              bits = reinterpret_cast<const uint32_t*>(x)[i];
            else
              bits = reinterpret_cast<const uint16_t*>(x)[i];
            f(i, to_logit<DT>(bits));
          }
        }
      }
    }
  };

  // ---- 1. the best key
  uint64_t best = 0;
  each([&](int i, float v) { best = more(best, key_of(v, i)); });
  best = block_reduce(best, more, sh.red);
  if (threadIdx.x == 0) {
    sh.best = best;
    sh.listed = 0;
  }
  sync_all();
  for (int c = 0; c < ctas; ++c) best = more(best, remote(&sh.best, c));
  const int first = index_of(best);
  float top;
  {
    const uint32_t o = (uint32_t)(best >> a.index_bits);
    top = __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
  }
  if (top == -INFINITY) {  // the same for the whole cluster
    if (threadIdx.x == 0 && rank == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    sync_all();
    return;
  }
  // (x - max) / temperature, without 0 * infinity at either end
  const auto scaled = [&](float v) {
    if (v == top) return 0.f;
    return top == INFINITY || v == -INFINITY ? -INFINITY : fmaxf(v - top, -FLT_MAX) * inv;
  };
  // weight in units of 2^-31
  const auto mass_of = [&](float v) { return __float2uint_rn(expf(scaled(v)) * 2147483648.f); };
  const auto bin_of = [&](float v) {  // distance from the maximum, monotone in the logit
    const float d = v == top ? 0.f : top - v;
    return min(kBins - 1, (int)fminf(d * kPerUnit, 2e9f));
  };
  const auto race_key = [&](int i, float v, float d) {
    const float r = d - logf(__ldg(noise + i));
    return key_of(r == r ? r : -INFINITY, i);
  };

  // ---- histograms: of the whole row by distance, or of one bin by keys
  uint64_t key_hi = 0;
  int level = 0, shift = 0, whole_bin = 0;
  uint64_t key_lo = 0;
  const auto clear = [&] {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.n[i] = sh.hi[i] = sh.lo[i] = 0;
    __syncthreads();
  };
  const auto put = [&](int bin, float v) {
    atomicAdd(&sh.n[bin], 1u);
    if (by_p) {
      const uint32_t m = mass_of(v);
      if (m && atomicAdd(&sh.lo[bin], m) > ~m) atomicAdd(&sh.hi[bin], 1u);
    }
  };
  const auto in_range = [&](int i, float v) {
    if (bin_of(v) != whole_bin) return false;
    const uint64_t key = key_of(v, i);
    return level == 0 || (key >= key_lo && key <= key_hi);
  };
  const int share = (kBins + ctas - 1) / ctas;  // bins that a CTA adds up
  const auto combine = [&] {
    sync_all();
    for (int b = rank * share + threadIdx.x; b < min(kBins, (rank + 1) * share); b += kThreads) {
      uint32_t n = 0;
      uint64_t m = 0;
      for (int c = 0; c < ctas; ++c) {
        n += remote(&sh.n[b], c);
        if (by_p) m += ((uint64_t)remote(&sh.hi[b], c) << 32) + remote(&sh.lo[b], c);
      }
      sh.count[b] = n;
      sh.mass[b] = m;
    }
    sync_all();
  };
  // The first bin at which `by count: base + counts reach k` or `base + masses
  // reach want` (for masses: the last kept token's bin).
  const auto scan = [&](bool count, uint32_t base_n, uint64_t base_m, double want) {
    uint32_t n[2];
    uint64_t m[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int b = 2 * threadIdx.x + e;
      n[e] = remote(&sh.count[b], b / share);
      m[e] = by_p ? remote(&sh.mass[b], b / share) : 0;
    }
    // exclusive sums over the threads, both in 64 bits
    uint64_t sn = n[0] + n[1], sm = m[0] + m[1];
    const uint64_t own_n = sn, own_m = sm;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t un = __shfl_up_sync(0xffffffffu, sn, o), um = __shfl_up_sync(0xffffffffu, sm, o);
      if ((threadIdx.x & 31) >= o) sn += un, sm += um;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) {
      sh.red[threadIdx.x >> 5] = sn;
      sh.red2[threadIdx.x >> 5] = sm;
    }
    if (threadIdx.x == 0) sh.bin = -1;
    __syncthreads();
    uint64_t bn = base_n + sn - own_n, bm = base_m + sm - own_m;
    for (int w = 0; w < (int)threadIdx.x >> 5; ++w) bn += sh.red[w], bm += sh.red2[w];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool here = n[e] && (count ? bn < (uint64_t)k && bn + n[e] >= (uint64_t)k
                                       : (double)bm < want && (double)(bm + m[e]) >= want);
      if (here) {  // one thread at most
        sh.bin = 2 * threadIdx.x + e;
        sh.bin_count = n[e];
        sh.before_count = (uint32_t)bn;
        sh.before_mass = bm;
      }
      bn += n[e];
      bm += m[e];
    }
    __syncthreads();
  };

  // ---- 2. the sum of all weights, with the histogram or the race
  const bool filtered = by_k || by_p;
  double sum = 0;
  uint64_t win = 0;
  if (filtered) clear();
  {
    double part = 0;  // so that a row's place in memory does not show in its last bit
    each([&](int i, float v) {
      const float d = scaled(v), w = expf(d);
      part += w;
      if (filtered)
        put(bin_of(v), v);
      else if (!greedy && (i == first || (d != -INFINITY && w >= least)))
        win = more(win, race_key(i, v, d));
    });
    sum = block_reduce(part, [](double q, double r) { return q + r; }, reinterpret_cast<double*>(sh.red));
  }
  if (threadIdx.x == 0) sh.sum = sum;

  // ---- 3. the threshold: top-k, then top-p of what it keeps
  uint64_t threshold = 0;
  if (filtered) {
    combine();
    bool whole = true;  // the histogram is the row's
    uint64_t kept_mass = 0;
    if (by_p) {  // of the whole row, until top-k says less
      uint64_t m = 0;
      for (int b = threadIdx.x; b < kBins; b += kThreads) m += remote(&sh.mass[b], b / share);
      kept_mass = block_reduce(m, [](uint64_t q, uint64_t r) { return q + r; }, sh.red);
    }
    for (int step = by_k ? 0 : 1; step < (by_p ? 2 : 1); ++step) {
      const bool count = step == 0;
      const double want = count ? 0. : (double)p * (double)kept_mass;
      if (!count && !(want > 0.)) {  // nothing but the first token
        threshold = best;
        break;
      }
      if (!whole) {
        clear();
        each([&](int i, float v) { put(bin_of(v), v); });
        combine();
      }
      whole = true;
      level = 0;
      scan(count, 0, 0, want);
      while (sh.bin >= 0 && sh.bin_count > kList) {
        // divide the bin by its keys: first the span of logits that it can hold
        const int bin = sh.bin;
        const uint32_t bn = sh.before_count;
        const uint64_t bm = sh.before_mass;
        if (level == 0) {
          whole_bin = bin;
          uint64_t low = ~0ull, high = 0;
          each([&](int i, float v) {
            if (bin_of(v) != whole_bin) return;
            const uint64_t key = key_of(v, i);
            low = key < low ? key : low;
            high = more(high, key);
          });
          low = block_reduce(low, [](uint64_t q, uint64_t r) { return q < r ? q : r; }, sh.red);
          high = block_reduce(high, more, sh.red);
          if (threadIdx.x == 0) {
            sh.low = low;
            sh.race = high;
          }
          sync_all();
          for (int c = 0; c < ctas; ++c) {
            const uint64_t l = remote(&sh.low, c);
            low = l < low ? l : low;
            high = more(high, remote(&sh.race, c));
          }
          key_lo = low;
          key_hi = high;
        } else {
          key_hi -= (uint64_t)bin << shift;
          const uint64_t span = (1ull << shift) - 1;
          key_lo = key_hi - key_lo > span ? key_hi - span : key_lo;
        }
        ++level;
        whole = false;
        shift = max(0, 64 - __clzll((long long)(key_hi - key_lo)) - 10);
        clear();
        each([&](int i, float v) {
          if (in_range(i, v)) put((int)((key_hi - key_of(v, i)) >> shift), v);
        });
        combine();
        scan(count, bn, bm, want);
      }
      // list the bin's tokens in the first CTA
      const int bin = sh.bin;
      const uint32_t bn = sh.before_count;
      const uint64_t bm = sh.before_mass;
      if (level == 0) whole_bin = bin;
      const uint32_t counter = mapa_shared(smem_u32(&sh.listed), 0), keys = mapa_shared(smem_u32(sh.list), 0),
                     masses = mapa_shared(smem_u32(sh.list_mass), 0);
      each([&](int i, float v) {
        if (!in_range(i, v)) return;
        const uint64_t key = key_of(v, i);
        if (level > 0 && (int)((key_hi - key) >> shift) != bin) return;
        uint32_t at;
        asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(counter) : "memory");
        if (at < kList) {
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(keys + 8 * at), "l"(key) : "memory");
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(masses + 4 * at), "r"(by_p ? mass_of(v) : 0u) : "memory");
        }
      });
      sync_all();
      if (rank == 0) {
        const int n = min((int)sh.listed, kList);
        uint64_t last = ~0ull;  // the smallest kept key
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const uint64_t key = sh.list[i];
          uint32_t better = 0;
          uint64_t m = bm;
          for (int j = 0; j < n; ++j)
            if (sh.list[j] > key) {
              ++better;
              m += sh.list_mass[j];
            }
          if (count) {
            if (bn + better == (uint32_t)k - 1) {
              sh.result_key = key;
              sh.result_mass = m + sh.list_mass[i];
            }
          } else if ((double)m < want && key < last) {
            last = key;
          }
        }
        if (!count) {
          last = block_reduce(last, [](uint64_t q, uint64_t r) { return q < r ? q : r; }, sh.red);
          if (threadIdx.x == 0) sh.result_key = last;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.listed = 0;
      }
      sync_all();
      threshold = more(threshold, remote(&sh.result_key, 0));
      if (count) kept_mass = remote(&sh.result_mass, 0);
    }

    // ---- 4. the race of the kept
    each([&](int i, float v) {
      if (i != first && key_of(v, i) < threshold) return;
      const float d = scaled(v);
      if (i != first && (d == -INFINITY || !(expf(d) >= least))) return;
      win = more(win, race_key(i, v, d));
    });
  }
  if (!greedy) win = block_reduce(win, more, sh.red);
  if (threadIdx.x == 0) sh.race = win;
  sync_all();
  if (rank == 0 && threadIdx.x == 0) {
    for (int c = 0; c < ctas; ++c) win = more(win, remote(&sh.race, c));
    sum = 0;
    for (int c = 0; c < ctas; ++c) sum += remote(&sh.sum, c);
    const int token = greedy ? first : index_of(win);
    a.tokens[row] = token;
    if (a.logprobs) {
      uint32_t bits;
      if constexpr (EB == 4)
        bits = reinterpret_cast<const uint32_t*>(x)[token];
      else
        bits = reinterpret_cast<const uint16_t*>(x)[token];
      a.logprobs[row] = scaled(to_logit<DT>(bits)) - (float)log(sum);
    }
  }
  sync_all();  // no CTA leaves while its memory may be read
}

template <int DT>
cudaError_t launch(const SampleArgs& a, int rows, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_rows<DT>, a);
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
  if (vocab > 1 << 28 || rows > 1 << 24) return set_error(TSB_ERR_UNSUPPORTED, "too many rows or tokens");
  if (row_stride < vocab || (noise && noise_stride < vocab)) return set_error(TSB_ERR_INVALID, "rows must not overlap");
  if (rows == 0) return TSB_OK;
  if (!logits || !tokens) return set_error(TSB_ERR_INVALID, "null pointer");
  SampleArgs a{logits, noise,  temperature, top_k,        top_p, min_p,
               tokens, logprobs, row_stride,  noise_stride, vocab, 0, 1};
  while ((1 << a.index_bits) < vocab) ++a.index_bits;
  // CTAs of a row: as many as still get 4096 tokens each, fewer once the rows
  // alone fill the GPU (a cluster's synchronisations cost about a pass over
  // 8192 tokens)
  int ctas = 1;
  while (ctas < kMaxCluster && vocab / (2 * ctas) >= 4096 && (int64_t)rows * ctas < 4 * sm_count()) ctas *= 2;
  a.chunk = ((vocab + 8 + ctas - 1) / ctas + 7) / 8 * 8;  // 8: a row may begin off a 16-byte boundary
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == TSB_DT_F32    ? launch<TSB_DT_F32>(a, rows, ctas, st)
                        : dtype == TSB_DT_BF16 ? launch<TSB_DT_BF16>(a, rows, ctas, st)
                                               : launch<TSB_DT_F16>(a, rows, ctas, st);
  return e == cudaSuccess ? TSB_OK : set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
}
