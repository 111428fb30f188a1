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
//   1. the best key, and every thread's largest logit;
//   2. a bound below which no token can be kept: min-p gives one, top-k the k-th
//      largest of the threads' maxima; then the sum of w and, where a bound is
//      known, a list of the tokens above it (each warp its own).  Top-p alone
//      takes a histogram of mass over the distance from the maximum in this
//      pass and has its bound and lists after it.  A row without filters runs
//      its race here;
//   3. T, from the lists (from the whole row where a list overflows): the
//      histogram's bin in which the limit lies, whose tokens are ranked one by
//      one in one CTA, each counting the tokens and the mass before it.  A bin
//      of more than kList tokens is divided again by its keys;
//   4. the race among the keys from T on; noise is read for those alone.
// Masses are sums of integers, w in units of 2^-31, so neither the order of the
// atomic additions nor the number of CTAs changes a result.
//
// One row is bound by the chain of its passes and synchronisations, many rows
// by instructions.  A pass over the row therefore spends a few instructions on
// a token, and what is done for few tokens is done from lists: in the pass, one
// such token in a warp holds up all 32 lanes (a third of the tokens' warps with
// one token in a hundred; 66 us for a row of 201088 with top-p).  A thread
// copies its 16-byte pieces ahead into shared memory with a ring of
// asynchronous copies; held in registers they were waited for when the ring
// moved on, and loops unrolled over several loads were bound by their own
// first fetch.  Measured (201088 tokens): one fp32 row with top-p 34 us; 32 fp32 rows
// without filters 28 us (1.8 TB/s of logits and noise); 64 bf16 rows 27 us greedy,
// 45 us without filters, 34 us with min-p, 41 us with top-k, with top-p of 0.9 69 us at
// temperature 0.7 and 118 us at 1, where rows keep more tokens than the lists
// hold and take two more passes.
#include <cfloat>

#include "tc05.cuh"
#include "tsb_common.cuh"
#include "tsb_internal.h"

namespace tsb {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kRing = 4;        // 16-byte pieces of a thread under way
constexpr int kOwn = 256;       // tokens of a warp's list
constexpr int kRingBytes = kRing * kThreads * 16;
constexpr int kBins = 1024;     // two a thread
constexpr int kList = 256;      // tokens that are ranked one by one; 800 of them took longer than two more divisions
constexpr int kMaxima = 1024;   // largest k that the threads' maxima are asked about
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
  uint32_t own_at[kWarps][kOwn];  // the warps' lists: index and logit
  float own[kWarps][kOwn];
  uint64_t red[kWarps], red2[kWarps];
  // read by the other CTAs
  uint64_t best, race, low, result_key, result_mass;
  uint64_t owned[2];  // taken in turn
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
__global__ void __launch_bounds__(kThreads, 2) sample_rows(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t ring[];
  Shared& sh = *reinterpret_cast<Shared*>(ring + kRingBytes);
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

  // f(index of the first, logits) of each 16 bytes of this CTA's part.  Copies
  // lie on 16-byte boundaries; a row that starts off them begins a few tokens
  // early, and its ends are put together token by token, -infinity outside.
  const int skew = (int)((reinterpret_cast<uintptr_t>(x) & 15) / EB);
  const int v0 = rank * a.chunk, v1 = min(v0 + a.chunk, V + skew);  // places from the boundary on
  const uint32_t mine = smem_u32(ring) + threadIdx.x * 16;
  const auto fetch = [&](int at, int place) {
    const uint32_t to = mine + place * (kThreads * 16);
    if (at >= skew && at + PER <= v1) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(x + (int64_t)(at - skew) * EB) : "memory");
    } else if (at < v1) {
#pragma unroll 1
      for (int e = 0; e < PER; ++e) {
        const int i = at + e - skew;
        const bool is = i >= 0 && i < V;
        if constexpr (EB == 4)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 4 * e), "r"(is ? reinterpret_cast<const uint32_t*>(x)[i] : 0xFF800000u)
                       : "memory");
        else
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(to + 2 * e),
                       "h"(is ? reinterpret_cast<const uint16_t*>(x)[i] : (uint16_t)(DT == TSB_DT_BF16 ? 0xFF80 : 0xFC00))
                       : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const auto each = [&](auto f) {  // whole warps stay in the loop: outside the row they see -infinity
    constexpr int kTurn = kThreads * PER;
    int at = v0 + threadIdx.x * PER, place = 0;
    const int ends = v1 + (threadIdx.x & 31) * PER;  // for the warp's first lane: v1
#pragma unroll 1
    for (int c = 0; c < kRing - 1; ++c) fetch(at + c * kTurn, c);
#pragma unroll 1
    for (; at < ends; at += kTurn) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "r"(mine + place * (kThreads * 16))
                   : "memory");
      fetch(at + (kRing - 1) * kTurn, place == 0 ? kRing - 1 : place - 1);
      place = place + 1 == kRing ? 0 : place + 1;
      float v[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e)
        v[e] = at < v1 ? to_logit<DT>(PER == 4 ? w[e] : w[e / 2] >> (16 * (e & 1))) : -INFINITY;
      f(at - skew, v);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  };
  // the best of the CTAs' values, read by the lanes side by side
  const auto of_cluster = [&](const uint64_t* mine, auto f) {
    const int lane = threadIdx.x & 31;
    uint64_t v = remote(mine, lane < ctas ? lane : 0);
#pragma unroll
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };

  // ---- 1. the best key
  float largest = -INFINITY;  // of this thread
  uint64_t best = 0;
  {
    int at = 0;
    each([&](int i, const float(&v)[PER]) {
      float m = v[0];
#pragma unroll
      for (int e = 1; e < PER; ++e) m = fmaxf(m, v[e]);
      if (m > largest) {
        largest = m;
#pragma unroll
        for (int e = PER - 1; e >= 0; --e)
          if (v[e] == m) at = i + e;
      }
    });
    if (largest > -INFINITY) best = key_of(largest, at);
  }
  best = block_reduce(best, more, sh.red);
  if (threadIdx.x == 0) {
    sh.best = best;
    sh.listed = 0;
  }
  sync_all();
  best = of_cluster(&sh.best, more);
  if (best == 0) {  // the same for the whole cluster
    if (threadIdx.x == 0 && rank == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    sync_all();
    return;
  }
  const int first = index_of(best);
  float top;
  {
    const uint32_t o = (uint32_t)(best >> a.index_bits);
    top = __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
  }
  // (x - max) / temperature, without 0 * infinity at either end
  const auto scaled = [&](float v) {
    if (v == top) return 0.f;
    return top == INFINITY || v == -INFINITY ? -INFINITY : fmaxf(v - top, -FLT_MAX) * inv;
  };
  const auto mass_of = [&](float w) { return __float2uint_rn(w * 2147483648.f); };  // in units of 2^-31
  const auto bin_of = [&](float v) {  // distance from the maximum, monotone in the logit
    const float d = v == top ? 0.f : top - v;
    return min(kBins - 1, (int)fminf(d * kPerUnit, 2e9f));
  };
  // A token's race; a fast logarithm (its error is far below 1e-3) tells which
  // are worth an exact one.
  const bool wide_noise = ((reinterpret_cast<uintptr_t>(noise) / 4 - skew) & 3) == 0;
  const auto noise_of = [&](int i, const float(&v)[PER], float(&z)[PER]) {
    if (wide_noise && i >= 0 && i + PER <= V) {
#pragma unroll
      for (int e = 0; e < PER; e += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(noise + i + e));
        z[e] = q.x, z[e + 1] = q.y, z[e + 2] = q.z, z[e + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) z[e] = v[e] > -INFINITY ? __ldg(noise + i + e) : 1.f;
    }
  };
  float ahead = -INFINITY;
  uint64_t win = 0;
  const auto race = [&](int i, float d, float z) {
    if (d - __logf(z) < ahead - 1e-3f) return;
    float r = d - logf(z);
    r = r == r ? r : -INFINITY;
    ahead = fmaxf(ahead, r);
    win = more(win, key_of(r, i));
  };

  // The warp's lanes learn of each other's best races, one distance a call.
  int apart = 1;
  const auto share_ahead = [&] {
    ahead = fmaxf(ahead, __shfl_xor_sync(0xffffffffu, ahead, apart));
    apart = apart == 16 ? 1 : 2 * apart;
  };

  // ---- histograms: of the whole row by distance, or of one bin by keys
  uint64_t key_hi = 0;
  int level = 0, shift = 0, whole_bin = 0;
  uint64_t key_lo = 0;
  const auto clear = [&] {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.n[i] = sh.hi[i] = sh.lo[i] = 0;
    __syncthreads();
  };
  const auto put = [&](int bin, float w) {
    atomicAdd(&sh.n[bin], 1u);
    if (by_p) {
      const uint32_t m = mass_of(w);
      if (m && atomicAdd(&sh.lo[bin], m) > ~m) atomicAdd(&sh.hi[bin], 1u);
    }
  };
  uint64_t floor_key = 0;  // top-p looks at what top-k keeps
  const auto counts = [&](int i, float v) { return v > -INFINITY && (floor_key == 0 || key_of(v, i) >= floor_key); };
  const auto in_range = [&](int i, float v) {  // of these, the ones in the bin that is divided
    if (!counts(i, v) || bin_of(v) != whole_bin) return false;
    const uint64_t key = key_of(v, i);
    return level == 0 || (key >= key_lo && key <= key_hi);
  };
  // ---- the warps' lists of tokens with logits from `cut` to `cap`
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int owned = 0;  // of this warp
  float cut = -INFINITY, cap = INFINITY;
  bool listed = false;  // the lists hold all of them, in every CTA
  const auto own = [&](int i, const float(&v)[PER]) {
    if (owned > kOwn) return;  // full: it does not matter by how much
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const bool is = v[e] >= cut && v[e] <= cap;
      const uint32_t all = __ballot_sync(0xffffffffu, is);
      if (!all) continue;
      const int at = owned + __popc(all & ((1u << lane) - 1));
      if (is && at < kOwn) {
        sh.own_at[warp][at] = i + e;
        sh.own[warp][at] = v[e];
      }
      owned += __popc(all);
    }
  };
  // Whether every list of the cluster holds its tokens.  Two calls may follow
  // each other with no barrier between one's reads and the other's write, so they
  // take two words in turn: a word is written again after the barrier of the call
  // in between, which nobody passes before everyone has read it.
  int turn = 0;
  const auto agree = [&] {
    const uint64_t most = block_reduce((uint64_t)owned, more, sh.red);
    if (threadIdx.x == 0) sh.owned[turn] = most;
    sync_all();
    listed = of_cluster(&sh.owned[turn], more) <= kOwn;
    turn ^= 1;
  };
  const auto visit = [&](auto f) {  // f(index, logit) of the lists, or of the row
    if (listed) {
      for (int j = lane; j < owned; j += 32) f((int)sh.own_at[warp][j], sh.own[warp][j]);
      __syncwarp();
    } else {
      each([&](int i, const float(&v)[PER]) {
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (v[e] > -INFINITY) f(i + e, v[e]);
      });
    }
  };

  const int share = (kBins + ctas - 1) / ctas;  // bins that a CTA adds up
  const auto combine = [&] {
    sync_all();
    for (int b = rank * share + threadIdx.x; b < min(kBins, (rank + 1) * share); b += kThreads) {
      uint32_t n = 0;
      uint64_t m = 0;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < ctas) {
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

  // ---- 2. what is known of the bound before the sum
  const bool filtered = by_k || by_p;
  const bool by_min = !greedy && least > 0.f;
  const float slack = fabsf(top) * 2.4e-7f;  // roundings of top - distance
  clear();
  if (by_k && k <= kMaxima) {
    if (largest > -INFINITY) atomicAdd(&sh.n[bin_of(largest)], 1u);
    combine();
    scan(true, 0, 0, 0.);
    // none: fewer threads than k have a token.  Half a bin more than the bin's edge, for its rounding
    if (sh.bin >= 0 && sh.bin < kBins - 1) cut = top - (sh.bin + 1.5f) / kPerUnit - slack;
    __syncthreads();
    clear();
  }
  if (by_min && !by_p) {
    // w >= min_p: a distance of log(min_p), a little more for its rounding
    const float d = logf(fminf(least, 1.f)) * 1.0001f - 1e-4f;
    cut = fmaxf(cut, top + fmaxf(d / inv, -FLT_MAX) - slack);
  }
  if (!(cut < top)) cut = -INFINITY;  // beyond what fp32 tells apart, or infinite
  const bool early = cut > -INFINITY;
  const bool mass_first = by_p && !by_k;
  // ---- the sum of all weights; without filters the race
  double sum;
  {
    // Two floats, so that a row's place in memory does not show in its last bit;
    // from 1 on, so that w is never the larger summand and the rounding of a sum
    // is what comes out of undoing it.
    float part = 1.f, rest = 0.f;
    const auto add = [&](float w) {
      const float s = part + w;
      rest += w - (s - part);
      part = s;
    };
    const bool free_race = !filtered && !by_min && !greedy;
    if (top < INFINITY && inv > 1e-30f && inv < 1e30f) {  // no 0 * infinity, no infinity - infinity
      const float c = inv * 1.4426950408889634f;
      each([&](int i, const float(&v)[PER]) {
        float d[PER], z[PER];
        if (free_race) noise_of(i, v, z);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          d[e] = fmaxf(v[e] - top, -FLT_MAX);
          float w;
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(d[e] * c));
          add(w);
          if (mass_first && v[e] > -INFINITY) put(bin_of(v[e]), w);
        }
        if (early) own(i, v);
        if (free_race) {
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (v[e] > -INFINITY) race(i + e, d[e] * inv, z[e]);
          share_ahead();
        }
      });
    } else {
      each([&](int i, const float(&v)[PER]) {
        float z[PER];
        if (free_race) noise_of(i, v, z);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const float d = scaled(v[e]), w = expf(d);
          add(w);
          if (mass_first && v[e] > -INFINITY) put(bin_of(v[e]), w);
          if (free_race && (i + e == first || d > -INFINITY)) race(i + e, d, z[e]);
        }
        if (early) own(i, v);
      });
    }
    sum = block_reduce(((double)part - 1.) + (double)rest, [](double q, double r) { return q + r; },
                       reinterpret_cast<double*>(sh.red));
  }
  if (threadIdx.x == 0) sh.sum = sum;
  if (early) agree();

  // ---- 3. the threshold: top-k, then top-p of what it keeps
  uint64_t threshold = 0;
  if (filtered) {
    sync_all();  // every CTA has to go by the same sums below
    const uint32_t counter = mapa_shared(smem_u32(&sh.listed), 0), keys = mapa_shared(smem_u32(sh.list), 0),
                   masses = mapa_shared(smem_u32(sh.list_mass), 0);
    const auto enlist = [&](uint64_t key, float v) {  // into the first CTA's list
      uint32_t at;
      asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(counter) : "memory");
      if (at < kList) {
        const uint32_t m = by_p ? mass_of(expf(scaled(v))) : 0u;
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(keys + 8 * at), "l"(key) : "memory");
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(masses + 4 * at), "r"(m) : "memory");
      }
    };
    const auto least_of = [](uint64_t q, uint64_t r) { return q < r ? q : r; };
    bool todo_k = by_k;
    double kept_mass = 0;  // of what top-k keeps, or of the row
    bool ready = mass_first, dirty = mass_first;  // the histogram: of the whole row already, used
    for (int step = by_k ? 0 : 1; step < (by_p ? 2 : 1); ++step) {
      const bool count = step == 0;
      if (!count && !todo_k) {  // top-p of the whole row
        double total = remote(&sh.sum, lane < ctas ? lane : 0);
        if (lane >= ctas) total = 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        kept_mass = total * 2147483648.;
      }
      const double want = count ? 0. : (double)p * kept_mass;
      if (!count && !(want > 0.)) {  // nothing but the first token
        threshold = best;
        break;
      }
      level = 0;
      floor_key = threshold;
      if (!ready) {
        if (dirty) clear();
        visit([&](int i, float v) {
          if (counts(i, v)) put(bin_of(v), by_p ? expf(scaled(v)) : 0.f);
        });
      }
      ready = false;
      dirty = true;
      combine();
      scan(count, 0, 0, want);
      if (!listed && sh.bin >= 0 && sh.bin < kBins - 1) {
        // lists of what may be kept; where that is too much, of the bin alone
        cut = top - (sh.bin + 1.5f) / kPerUnit - slack;
        const bool many = sh.before_count + sh.bin_count > (uint32_t)(kOwn * kWarps / 2 * ctas);
        for (int only = many; only < 2 && !listed && cut < top && cut > -INFINITY; ++only) {
          if (only) cap = fminf(top, top - (sh.bin - 0.5f) / kPerUnit + slack);
          owned = 0;
          each(own);
          agree();
        }
      }
      while (sh.bin >= 0 && sh.bin_count > kList) {
        // divide the bin by its keys: first the span of logits that it can hold
        const int bin = sh.bin;
        const uint32_t bn = sh.before_count;
        const uint64_t bm = sh.before_mass;
        if (level == 0) {
          whole_bin = bin;
          uint64_t low = ~0ull, high = 0;
          visit([&](int i, float v) {
            if (!in_range(i, v)) return;
            const uint64_t key = key_of(v, i);
            low = least_of(low, key);
            high = more(high, key);
          });
          low = block_reduce(low, least_of, sh.red);
          high = block_reduce(high, more, sh.red);
          if (threadIdx.x == 0) {
            sh.low = low;
            sh.race = high;
          }
          sync_all();
          key_lo = of_cluster(&sh.low, least_of);
          key_hi = of_cluster(&sh.race, more);
        } else {
          key_hi -= (uint64_t)bin << shift;
          const uint64_t span = (1ull << shift) - 1;
          key_lo = key_hi - key_lo > span ? key_hi - span : key_lo;
        }
        ++level;
        shift = max(0, 64 - __clzll((long long)(key_hi - key_lo)) - 10);
        clear();
        visit([&](int i, float v) {
          if (in_range(i, v)) put((int)((key_hi - key_of(v, i)) >> shift), by_p ? expf(scaled(v)) : 0.f);
        });
        combine();
        scan(count, bn, bm, want);
      }
      const int bin = sh.bin;
      if (bin < 0) {
        // Fewer tokens than k; or rounding leaves the limit past the last token: of
        // the row, or of the bin that was divided, whose masses come from another
        // exponential the second time.  That bin is kept to its end.
        if (count) todo_k = false;
        if (level > 0) threshold = more(threshold, key_lo);
        if (cap < INFINITY) listed = false;
        cap = INFINITY;
        continue;
      }
      const uint32_t bn = sh.before_count;
      const uint64_t bm = sh.before_mass;
      if (level == 0) whole_bin = bin;
      visit([&](int i, float v) {
        if (!in_range(i, v)) return;
        const uint64_t key = key_of(v, i);
        if (level == 0 || (int)((key_hi - key) >> shift) == bin) enlist(key, v);
      });
      sync_all();
      if (rank == 0) {
        const int n = min((int)sh.listed, kList);
        uint64_t last = ~0ull;  // the smallest kept key
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const uint64_t key = sh.list[i];
          uint32_t better = 0;
          uint64_t m = bm;
#pragma unroll 4
          for (int j = 0; j < n; ++j) {
            const bool is = sh.list[j] > key;
            better += is;
            m += is ? sh.list_mass[j] : 0u;
          }
          if (count) {
            if (bn + better == (uint32_t)k - 1) {
              sh.result_key = key;
              sh.result_mass = m + sh.list_mass[i];
            }
          } else if ((double)m < want) {
            last = least_of(last, key);
          }
        }
        if (!count) {
          last = block_reduce(last, least_of, sh.red);
          if (threadIdx.x == 0) sh.result_key = last;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.listed = 0;
      }
      sync_all();
      threshold = more(threshold, remote(&sh.result_key, 0));
      if (cap < INFINITY) listed = false;  // the lists are of no further use
      cap = INFINITY;
      if (count) kept_mass = (double)remote(&sh.result_mass, 0);
      sync_all();
    }

  }
  // ---- 4. the race of the kept
  if ((filtered || by_min) && listed) {
    visit([&](int i, float v) {
      if (i != first && key_of(v, i) < threshold) return;
      const float d = scaled(v);
      if (i == first || (d > -INFINITY && (least <= 0.f || expf(d) >= least))) race(i, d, __ldg(noise + i));
    });
  } else if (filtered || by_min) {
    // many are kept: a pass over the row with its noise
    const uint32_t edge = (uint32_t)(threshold >> a.index_bits);
    const float floor_x = edge == 0 ? -INFINITY : __uint_as_float(edge ^ ((edge >> 31) ? 0x80000000u : 0xFFFFFFFFu));
    each([&](int i, const float(&v)[PER]) {
      float z[PER];
      noise_of(i, v, z);
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const float d = scaled(v[e]);
        const bool kept = v[e] > floor_x || (v[e] == floor_x && key_of(v[e], i + e) >= threshold);
        if (i + e == first || (kept && d > -INFINITY && (least <= 0.f || expf(d) >= least))) race(i + e, d, z[e]);
      }
      share_ahead();
    });
  }
  if (!greedy) win = block_reduce(win, more, sh.red);
  if (threadIdx.x == 0) sh.race = win;
  sync_all();
  if (rank == 0 && threadIdx.x < 32) {
    win = of_cluster(&sh.race, more);
    sum = remote(&sh.sum, threadIdx.x < ctas ? threadIdx.x : 0);
    if (threadIdx.x >= ctas) sum = 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) {
      const int token = greedy ? first : index_of(win);
      a.tokens[row] = token;
      if (a.logprobs) {
        uint32_t bits;
        if constexpr (EB == 4)
          bits = reinterpret_cast<const uint32_t*>(x)[token];
        else
          bits = reinterpret_cast<const uint16_t*>(x)[token];
        a.logprobs[row] = scaled(to_logit<DT>(bits)) - logf((float)sum);
      }
    }
  }
  sync_all();  // no CTA leaves while its memory may be read
}

template <int DT>
cudaError_t launch(const SampleArgs& a, int rows, int ctas, cudaStream_t st) {
  static bool ready[64];  // by device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev]))
    e = cudaFuncSetAttribute(sample_rows<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kRingBytes + (int)sizeof(Shared));
  if (e != cudaSuccess) return e;
  if (dev < 64) ready[dev] = true;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kRingBytes + sizeof(Shared);
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
  const auto off = [](const void* p, uintptr_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
  if (off(logits, dtype == TSB_DT_F32 ? 4 : 2) || off(noise, 4) || off(temperature, 4) || off(top_k, 4) ||
      off(top_p, 4) || off(min_p, 4) || off(tokens, 8) || off(logprobs, 4))
    return set_error(TSB_ERR_INVALID, "pointers must be aligned to their type");
  SampleArgs a{logits, noise,  temperature, top_k,        top_p, min_p,
               tokens, logprobs, row_stride,  noise_stride, vocab, 0, 1};
  while ((1 << a.index_bits) < vocab) ++a.index_bits;
  // CTAs of a row: as many as still get 4096 tokens each, until the rows' CTAs
  // reach the SMs (64 rows of 201088, mixed: 2 CTAs 215 us, 8 CTAs 180 us; 200 rows
  // of 32001, top-k: 1 CTA 37 us, 2 CTAs 46 us)
  int ctas = 1;
  while (ctas < kMaxCluster && vocab / (2 * ctas) >= 4096 && (int64_t)rows * ctas < sm_count()) ctas *= 2;
  a.chunk = ((vocab + 8 + ctas - 1) / ctas + 7) / 8 * 8;  // 8: a row may begin off a 16-byte boundary
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == TSB_DT_F32    ? launch<TSB_DT_F32>(a, rows, ctas, st)
                        : dtype == TSB_DT_BF16 ? launch<TSB_DT_BF16>(a, rows, ctas, st)
                                               : launch<TSB_DT_F16>(a, rows, ctas, st);
  return e == cudaSuccess ? TSB_OK : set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
}
