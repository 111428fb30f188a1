// Attention of single decode tokens (and a few tokens of a sequence: up to
// kShortRows rows per KV head) over a paged KV cache (tsb_paged_attention).
//
// Bound by the cache's bytes.  The up to 16 (token, query head) rows of a KV
// head are one side of mma.sync m16n8k16 tiles, so each key and value is read
// once for all of them and costs a warp no arithmetic of its own beyond its
// share of the products.  Each warp keeps a ring of steps (K and V of kStep
// positions) on their way to shared memory with 16-byte asynchronous copies;
// loaded to registers right before their use, one step at a time, the copies
// in flight covered a third of the memory's latency (116 us for 64 tokens over
// up to 4096 e4m3 positions).  Both products allow any order of their inner
// dimension, and the sums any order of their columns, so a lane takes 16 (or
// 8) contiguous bytes of a row and the rows of Q, and the columns of the
// output, are permuted to match.
//
//   S = Q K^T, P = 2^(c S - c m), O = O + P V   (c = scale * log2(e))
//
// with a running maximum m per row that moves only when a row outgrows it by
// 2^6.  Types and the scaling of bf16 queries over e4m3 caches are those of the
// long kernel, and so is what the weights' rounding costs (one token over 500
// bf16 positions: 0.0022 against 64 bits, 0.0017 from the output's rounding).
//
// Work: steps of kStep positions of all (sequence, KV head) items form a
// line.  Where items are alike a CTA takes whole items; else the line is cut
// into equal pieces, and an item's last piece joins its parts in key order.
// The four warps of a CTA take a piece's steps in turn and are joined in
// shared memory.
//
// Measured: 64 tokens over up to 4096 positions, 8 KV heads of 64: 61 us from a
// bf16 cache (5.0 TB/s, 77% of the measured copy rate), 48 us from an e4m3 one (50%:
// half the bytes a step, the same chain of copy, widening, products and exponentials; neither
// memory, 38% of its cycles, nor the schedulers, 46%, are full);
// one token over 500 positions 9 us, launch and the chain of look-up, copy,
// products and joining.
#include "paged.cuh"

namespace tsb {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kMaxSeqs = 512;    // sequences of one launch
constexpr int kMaxCtas = 592;    // four on each SM of a B200
constexpr int kItemCost = 12;    // a part's fixed work in steps (look-ups, first copies, joining): three a warp
// Steps: four a warp; joining parts costs as much as five or six.  Where the rule for
// whole items ends, one token over 512 positions takes 8.9 us, over 513 12.0, over 1024 12.0.
constexpr int kMinPiece = 16;
constexpr int kMaxParts = 64;    // of an item
constexpr float kGrow = 6.f;
constexpr int kRows = kShortRows;
constexpr int kCounters = 1024;  // first of this kernel's counters

template <int D>
constexpr int step_of() {
  return D == 64 ? 32 : 16;
}

struct ShortArgs {
  AttnCall c;
};

// A warp's ring: steps in it, bytes of a step's K or V; CTAs of an SM.
template <int D, bool FP8>
struct Ring {
  static constexpr int kRowBytes = D * (FP8 ? 1 : 2);
  static constexpr int kHalf = step_of<D>() * kRowBytes;
  static constexpr int kSteps = 3;
  static constexpr int kBytes = kWarps * kSteps * 2 * kHalf;
  static constexpr int kPerSm = !FP8 ? 2 : D == 64 ? 4 : 3;
};
// Byte of 16-byte chunk c of row r: chunks of a row are exchanged so that the
// rows and chunks that lanes read together lie in different banks.
template <int RB>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return RB == 64 ? r * 64 + ((c ^ (r >> 1)) & 3) * 16 : r * RB + (c ^ ((r & 6) ^ ((r & 1) << 2))) * 16;
}

template <int D>
struct Sums {  // the four warps' results; lies over the rings
  float o[kWarps][kRows][D + 4];
  float m[kWarps][kRows], l[kWarps][kRows];
};

struct Shared {
  int q_len[kMaxSeqs], kv_len[kMaxSeqs];
  int pre[kMaxSeqs + 1];  // line length of the sequences before, per KV head
  int longest[kWarps], poison, last;
};

// Positions that some row of a sequence sees: [0, nfirst), then [first, kv_len).
struct Span {
  int nfirst, first, nf, n;  // nf: steps of the first part, n: of both
};
template <int STEP>
__device__ __forceinline__ Span visible(const AttnCall& c, int q_len, int kv_len) {
  Span s{0, 0, 0, 0};
  if (kv_len <= 0) return s;
  s.first = c.window > 0 ? max(0, kv_len - q_len - c.window + 1) : 0;
  s.nfirst = min(c.keep_first, s.first);
  s.nf = (s.nfirst + STEP - 1) / STEP;
  s.n = s.nf + (kv_len - s.first + STEP - 1) / STEP;
  return s;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t b) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)b));
  return r;
}
template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    mma_f16(d, a, b0, b1);
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One CTA's part of one item.
struct Segment {
  int b, head, q_len, kv_len, k0, k1;
  Span v;
  int part, parts, c_first;
};

template <int DT, int D, bool FP8>
__global__ void __launch_bounds__(kThreads, Ring<D, FP8>::kPerSm) paged_attn_short(const __grid_constant__ ShortArgs sa) {
  using Rg = Ring<D, FP8>;
  constexpr int STEP = step_of<D>(), NT = STEP / 8, RB = Rg::kRowBytes;
  constexpr int KW = FP8 ? D / 16 : D / 8;   // words of a lane's share of a key
  constexpr int VW = FP8 ? D / 32 : D / 16;  // words of a lane's share of a value
  constexpr bool kF16 = FP8 || DT == TSB_DT_F16;
  constexpr float kBias = kF16 ? 8.f : 0.f;
  constexpr int EB = FP8 ? 1 : 2;
  constexpr int KS = D / 16;  // inner steps of S
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared sh;
  Sums<D>& sums = *reinterpret_cast<Sums<D>*>(dyn);
  const AttnCall& c = sa.c;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int G = c.p.G;
  pdl_wait();
  pdl_launch_dependents();

  // ---- the line
  int longest = 0;
  for (int b = threadIdx.x; b < c.p.n_seqs; b += kThreads) {
    const SeqSpan sp = seq_span(c.p, b);
    const bool mine = sp.q_len > 0 && sp.q_len * G <= kRows;
    sh.q_len[b] = mine ? sp.q_len : 0;
    sh.kv_len[b] = sp.kv_len;
    const int u = mine ? visible<STEP>(c, sp.q_len, sp.kv_len).n + kItemCost : 0;
    sh.pre[b + 1] = u;
    longest = max(longest, u);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  if (lane == 0) sh.longest[warp] = longest;
  if (threadIdx.x == 0) sh.poison = 0;
  __syncthreads();
  longest = max(max(sh.longest[0], sh.longest[1]), max(sh.longest[2], sh.longest[3]));
  if (longest == 0) return;
  int64_t total = 0;
  int n = 1;
  bool whole = false;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    // running sums: of steps, and again of items where a CTA takes whole ones
    if (pass == 1 && !whole) break;
    if (warp == 0) {
      int run = 0;
      for (int b0 = 0; b0 < c.p.n_seqs; b0 += 32) {
        const int b = b0 + lane;
        int v = 0;
        if (b < c.p.n_seqs) v = pass == 0 ? sh.pre[b + 1] : sh.q_len[b] > 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        if (b < c.p.n_seqs) sh.pre[b + 1] = run + v;
        run += __shfl_sync(0xffffffffu, v, 31);
      }
      if (lane == 0) sh.pre[0] = 0;
    }
    __syncthreads();
    total = (int64_t)sh.pre[c.p.n_seqs] * c.p.nkv;
    if (pass == 0) {
      const int64_t share = (total + gridDim.x - 1) / gridDim.x;
      const int64_t items = total / max(1, longest);  // at least so many
      whole = longest <= kMinPiece + kItemCost || (items <= gridDim.x && 8 * (int64_t)longest <= 9 * share);
      const int64_t piece = max((int64_t)kMinPiece, (int64_t)(longest + kMaxParts - 1) / kMaxParts);
      n = (int)min((int64_t)gridDim.x, max((int64_t)1, total / piece));
    } else {
      n = (int)min((int64_t)gridDim.x, total);
    }
    __syncthreads();
  }
  if ((int)blockIdx.x >= n) return;
  const bool small = total <= INT32_MAX / kMaxCtas;  // 32-bit quotients do
  const auto ratio = [&](int64_t a, int64_t b, int64_t q) {
    return small ? (int64_t)((uint32_t)a * (uint32_t)b / (uint32_t)q) : a * b / q;
  };
  const auto cut = [&](int i) { return ratio(total, i, n); };
  const auto cta_of = [&](int64_t p) {
    int i = (int)ratio(p, n, total);
    while (i > 0 && cut(i) > p) --i;
    while (i + 1 < n && cut(i + 1) <= p) ++i;
    return i;
  };
  int64_t x = cut(blockIdx.x);
  const int64_t end = cut(blockIdx.x + 1);
  const float c0 = fmaxf(fabsf(c.scale) * 1.4426950408889634f, 1e-37f);
  const uint32_t flip = c.scale < 0.f ? 0x80008000u : 0u;

  while (x < end) {
    Segment s;
    {  // the item at x
      int lo = 0, hi = c.p.n_seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)sh.pre[mid] * c.p.nkv <= x)
          lo = mid;
        else
          hi = mid;
      }
      const int u = sh.pre[lo + 1] - sh.pre[lo];
      const int64_t first = (int64_t)sh.pre[lo] * c.p.nkv;
      s.b = lo;
      s.head = small ? (int)((uint32_t)(x - first) / (uint32_t)u) : (int)((x - first) / u);
      s.q_len = sh.q_len[lo];
      s.kv_len = sh.kv_len[lo];
      s.v = visible<STEP>(c, s.q_len, s.kv_len);
      const int64_t at = first + (int64_t)s.head * u;
      s.parts = 1;
      s.part = 0;
      s.c_first = 0;
      if (whole) {
        s.k0 = 0;
        s.k1 = s.v.n;
        x = at + 1;
      } else {
        const int64_t keys = at + kItemCost, stop = at + u, to = min(end, stop);
        s.k0 = (int)max((int64_t)0, x - keys);
        s.k1 = (int)max((int64_t)0, to - keys);
        const bool starts = x == at;
        x = to;
        if (s.k1 > s.k0 && (s.k0 > 0 || s.k1 < s.v.n)) {
          s.c_first = cta_of(keys);
          s.parts = cta_of(stop - 1) - s.c_first + 1;
          s.part = (int)blockIdx.x - s.c_first;
        }
        if (s.k1 == s.k0 && !(s.v.n == 0 && starts)) continue;
      }
    }
    const int R = s.q_len * G, base = s.kv_len - s.q_len, q0 = c.p.cu_q[s.b];
    const bool several = s.q_len > 1;
    const int row[2] = {g, g + 8};
    int pos[2];
    // ---- Q as the left operand: rows g and g + 8, the dims that this lane has of a key
    uint32_t q[KS][4];
    float cr[2] = {c0, c0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tok = row[h] < R ? row[h] / G : 0;
      pos[h] = row[h] < R ? base + tok : -1;
      uint2 w[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = FP8 ? 16 * (t + 4 * (k / 4)) + 4 * (k % 4) : 8 * (t + 4 * (k / 2)) + 4 * (k % 2);
        w[k] = make_uint2(0, 0);
        if (row[h] < R)
          w[k] = *reinterpret_cast<const uint2*>(c.q + (int64_t)(q0 + tok) * c.q_token_stride +
                                                 (int64_t)(s.head * G + row[h] - tok * G) * c.q_head_stride + d);
      }
      if constexpr (FP8 && DT == TSB_DT_BF16) {
        uint32_t big = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
          big = max(big, max(max(w[k].x & 0x7FFFu, (w[k].x >> 16) & 0x7FFFu), max(w[k].y & 0x7FFFu, (w[k].y >> 16) & 0x7FFFu)));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int e = (int)(big >> 7);
        const int shift = e == 255 || big == 0 ? 0 : min(127, 14 + 127 - max(e, 1));
        const float f1 = __int_as_float((127 + shift / 2) << 23), f2 = __int_as_float((127 + shift - shift / 2) << 23);
        cr[h] = fmaxf(ldexpf(c0, -shift), 1e-37f);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          w[k].x = pack2<true>(__uint_as_float(w[k].x << 16) * f1 * f2, __uint_as_float(w[k].x & 0xFFFF0000u) * f1 * f2);
          w[k].y = pack2<true>(__uint_as_float(w[k].y << 16) * f1 * f2, __uint_as_float(w[k].y & 0xFFFF0000u) * f1 * f2);
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        q[k][h] = w[k].x ^ flip;
        q[k][2 + h] = w[k].y ^ flip;
      }
    }
    // ---- this warp's steps
    float o[D / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const uint32_t ring = smem_u32(dyn) + warp * (Rg::kSteps * 2 * Rg::kHalf);
    const auto first_of = [&](int k) { return k < s.v.nf ? k * STEP : s.v.first + (k - s.v.nf) * STEP; };
    const auto end_of = [&](int k) { return k < s.v.nf ? s.v.nfirst : s.kv_len; };
    const auto find = [&](int k) {  // byte offset of this lane's position of step k
      int64_t off = -1;
      if (k < s.k1 && lane < STEP && first_of(k) + lane < end_of(k)) {
        off = cached_row(c.p, s.b, first_of(k) + lane);
        if (off >= 0) off = (off + s.head * c.p.head_stride) * EB;
      }
      return off;
    };
    const auto fetch = [&](int k, int place, int64_t off) {
      if (k < s.k1) {
        constexpr int CH = RB / 16, RPI = 32 / CH;  // chunks of a row, rows a copy instruction
        const uint32_t at = ring + place * 2 * Rg::kHalf;
#pragma unroll
        for (int i = 0; i < STEP / RPI; ++i) {
          const int row_i = i * RPI + lane / CH, ch = lane % CH;
          const int64_t a = __shfl_sync(0xffffffffu, off, row_i);
          const int64_t from = a < 0 ? 0 : a + ch * 16;
          const uint32_t to = at + chunk_at<RB>(row_i, ch);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(c.p.kc + from), "r"(a < 0 ? 0 : 16)
                       : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + Rg::kHalf), "l"(c.p.vc + from),
                       "r"(a < 0 ? 0 : 16)
                       : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int64_t ahead;
    {
      int64_t off[Rg::kSteps];  // looked up together
#pragma unroll
      for (int i = 0; i < Rg::kSteps; ++i) off[i] = find(s.k0 + warp + i * kWarps);
#pragma unroll
      for (int i = 0; i < Rg::kSteps - 1; ++i) fetch(s.k0 + warp + i * kWarps, i, off[i]);
      ahead = off[Rg::kSteps - 1];
    }
    int place = 0;
#pragma unroll 1
    for (int k = s.k0 + warp; k < s.k1; k += kWarps) {
      const int j0 = first_of(k), je = end_of(k);
      asm volatile("cp.async.wait_group %0;" ::"n"(Rg::kSteps - 2) : "memory");
      __syncwarp();  // everyone's copies of this step; and the step before has been read
      fetch(k + (Rg::kSteps - 1) * kWarps, place == 0 ? Rg::kSteps - 1 : place - 1, ahead);
      ahead = find(k + Rg::kSteps * kWarps);
      const uint32_t here = ring + place * 2 * Rg::kHalf;
      place = place + 1 == Rg::kSteps ? 0 : place + 1;
      // S = Q K^T: row g (and g + 8) against keys 8 i + 2 t, + 1
      float sc[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        uint32_t kf[KW];  // key 8 i + g, dims by chunks of 16 bytes: t, t + 4, ...
#pragma unroll
        for (int w = 0; w < KW; w += 4)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(kf[w]), "=r"(kf[w + 1]), "=r"(kf[w + 2]), "=r"(kf[w + 3])
                       : "r"(here + chunk_at<RB>(8 * i + g, t + w)));
        sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          if constexpr (FP8)
            mma<kF16>(sc[i], q[kk], e4m3x2_to_f16x2(kf[kk]), e4m3x2_to_f16x2(kf[kk] >> 16));
          else
            mma<kF16>(sc[i], q[kk], kf[2 * kk], kf[2 * kk + 1]);
        }
      }
      const bool open = j0 + STEP - 1 <= base && j0 + STEP <= je &&
                        (c.window == 0 || j0 > s.kv_len - 1 - c.window || j0 + STEP - 1 < c.keep_first);
      if (!open) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + 8 * i + 2 * t + (e & 1), p = pos[e / 2];
            if (!(j < je && j <= p && (c.window == 0 || j > p - c.window || j < c.keep_first))) sc[i][e] = -INFINITY;
          }
      }
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        top[0] = fmaxf(top[0], fmaxf(sc[i][0], sc[i][1]));
        top[1] = fmaxf(top[1], fmaxf(sc[i][2], sc[i][3]));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      }
      if (__any_sync(0xffffffffu, (top[0] - m[0]) * cr[0] > kGrow || (top[1] - m[1]) * cr[1] > kGrow)) {
        float keep[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          keep[h] = m[h] == -INFINITY ? 0.f : ex2((m[h] - top[h]) * cr[h]);
          m[h] = top[h];
          l[h] *= keep[h];
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= keep[0], o[i][1] *= keep[0];
          o[i][2] *= keep[1], o[i][3] *= keep[1];
        }
      }
      uint32_t p[NT][2];
      const float mc[2] = {(m[0] == -INFINITY ? 0.f : m[0] * cr[0]) - kBias, (m[1] == -INFINITY ? 0.f : m[1] * cr[1]) - kBias};
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float a = ex2(fmaf(sc[i][2 * h], cr[h], -mc[h])), b = ex2(fmaf(sc[i][2 * h + 1], cr[h], -mc[h]));
          l[h] += a + b;
          p[i][h] = pack2<kF16>(a, b);
        }
      // O += P V: column n of the product's tile j is dim of (n, j) below
#pragma unroll
      for (int kk = 0; kk < STEP / 16; ++kk) {
        const uint32_t a[4] = {p[2 * kk][0], p[2 * kk][1], p[2 * kk + 1][0], p[2 * kk + 1][1]};
        uint32_t vf[4][VW];  // values 16 kk + 2 t + {0, 1, 8, 9}, chunk g (and g + 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rv = 16 * kk + 2 * t + (i & 1) + 4 * (i & 2);
          if constexpr (VW == 2) {
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                         : "=r"(vf[i][0]), "=r"(vf[i][1])
                         : "r"(here + Rg::kHalf + chunk_at<RB>(rv, g / 2) + (g & 1) * 8));
          } else {
#pragma unroll
            for (int w = 0; w < VW; w += 4)
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(vf[i][w]), "=r"(vf[i][w + 1]), "=r"(vf[i][w + 2]), "=r"(vf[i][w + 3])
                           : "r"(here + Rg::kHalf + chunk_at<RB>(rv, g + 2 * w)));
          }
        }
        if (!open && several) {  // a value that one row sees and another does not has to be finite
          bool any = false;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              uint32_t bad;
              if constexpr (FP8) {
                bad = __vcmpeq4(vf[i][w] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
              } else {
                constexpr uint32_t ex = DT == TSB_DT_F16 ? 0x7C007C00u : 0x7F807F80u;
                bad = __vcmpeq2(vf[i][w] & ex, ex);
              }
              vf[i][w] &= ~bad;
              any |= bad != 0;
            }
          if (any) sh.poison = 1;
        }
        const auto& v0 = vf[0];
        const auto& v1 = vf[1];
        const auto& v2 = vf[2];
        const auto& v3 = vf[3];
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          if constexpr (FP8) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t sel = e ? 0x7362 : 0x5140;
              const uint32_t x01 = prmt(v0[w], v1[w], sel), x23 = prmt(v2[w], v3[w], sel);
              mma<kF16>(o[4 * w + 2 * e], a, e4m3x2_to_f16x2(x01), e4m3x2_to_f16x2(x23));
              mma<kF16>(o[4 * w + 2 * e + 1], a, e4m3x2_to_f16x2(x01 >> 16), e4m3x2_to_f16x2(x23 >> 16));
            }
          } else {
            mma<kF16>(o[2 * w], a, prmt(v0[w], v1[w], 0x5410), prmt(v2[w], v3[w], 0x5410));
            mma<kF16>(o[2 * w + 1], a, prmt(v0[w], v1[w], 0x7632), prmt(v2[w], v3[w], 0x7632));
          }
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the rings are read: the sums take their place
    // ---- the four warps joined
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t == 0) {
        sums.m[warp][row[h]] = m[h] == -INFINITY ? -INFINITY : m[h] * cr[h] - kBias;  // weights are 2^(c s - this)
        sums.l[warp][row[h]] = l[h];
      }
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int nn = 2 * t + (e & 1);
        const int d = D == 64 ? 8 * nn + j : FP8 ? 16 * nn + j : 64 * (j / 8) + 8 * nn + j % 8;
        sums.o[warp][row[e / 2]][d] = o[j][e];
      }
    __syncthreads();
    // thread: a row, and D / 8 of its dims
    const int r = threadIdx.x / 8, d0 = (threadIdx.x % 8) * (D / 8);
    const int tok = r < R ? r / G : 0, qh = s.head * G + (r - tok * G);
    const float sink = c.sinks && r < R ? c.sinks[qh] * 1.4426950408889634f : -INFINITY;
    float acc[D / 8] = {}, top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sums.m[w][r]);
    {
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(sums.m[w][r] - ref);
        sum += sums.l[w][r] * f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) acc[d] = fmaf(f, sums.o[w][r][d0 + d], acc[d]);
      }
    }
    const bool poisoned = sh.poison != 0;
    if (poisoned && r < R) {
      // values taken out of closed steps, for the rows that see them
      const int p = base + tok;
      for (int k = s.k0; k < s.k1; ++k) {
        const int j0 = k < s.v.nf ? k * STEP : s.v.first + (k - s.v.nf) * STEP;
        const int je = min(j0 + STEP, k < s.v.nf ? s.v.nfirst : s.kv_len);
        const bool open = j0 + STEP - 1 <= base && j0 + STEP <= je &&
                          (c.window == 0 || j0 > s.kv_len - 1 - c.window || j0 + STEP - 1 < c.keep_first);
        if (open) continue;
        for (int j = j0; j < je && j <= p; ++j) {
          if (c.window > 0 && j <= p - c.window && j >= c.keep_first) continue;
          const int64_t at = cached_row(c.p, s.b, j);
          if (at < 0) continue;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            const int64_t i = at + s.head * c.p.head_stride + d0 + d;
            float v;
            if constexpr (FP8)
              v = e4m3_to_f32(c.p.vc[i]);
            else
              v = to_f32<DT>(reinterpret_cast<const uint16_t*>(c.p.vc)[i]);
            if (!isfinite(v)) acc[d] += v;
          }
        }
      }
    }
    bool write = r < R;
    if (s.parts > 1) {
      constexpr int kPart = kRows * (D + 2);
      const auto slot = [&](int i) { return c.part + (int64_t)(2 * (s.c_first + i) + (i == 0 ? 1 : 0)) * kPart; };
      float* mine = slot(s.part);
#pragma unroll
      for (int d = 0; d < D / 8; d += 4)
        *reinterpret_cast<float4*>(mine + r * D + d0 + d) = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
      if (threadIdx.x % 8 == 0) {
        mine[kRows * D + r] = top;
        mine[kRows * D + kRows + r] = sum;
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        unsigned prev;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                     : "=r"(prev)
                     : "l"(c.counters + kCounters + s.c_first)
                     : "memory");
        sh.last = prev == (unsigned)(s.parts - 1);
        if (sh.last) c.counters[kCounters + s.c_first] = 0;
      }
      __syncthreads();
      write = write && sh.last;
      if (write) {
        __threadfence();
        top = -INFINITY;
        for (int i = 0; i < s.parts; ++i) top = fmaxf(top, __ldcg(slot(i) + kRows * D + r));
        const float ref = top == -INFINITY ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) acc[d] = 0.f;
#pragma unroll 4
        for (int i = 0; i < s.parts; ++i) {
          const float* sl = slot(i);
          const float f = ex2(__ldcg(sl + kRows * D + r) - ref);
          sum = fmaf(__ldcg(sl + kRows * D + kRows + r), f, sum);
#pragma unroll
          for (int d = 0; d < D / 8; d += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(sl + r * D + d0 + d));
            acc[d] = fmaf(f, v.x, acc[d]);
            acc[d + 1] = fmaf(f, v.y, acc[d + 1]);
            acc[d + 2] = fmaf(f, v.z, acc[d + 2]);
            acc[d + 3] = fmaf(f, v.w, acc[d + 3]);
          }
        }
      }
    }
    if (write) {
      if (sink != -INFINITY) {
        // sums are 2^(c s - top): the sink joins them, above or below
        const float ref = fmaxf(sink, top), f = ex2(top - ref);
        sum = sum * f + ex2(sink - ref);
#pragma unroll
        for (int d = 0; d < D / 8; ++d) acc[d] *= f;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      uint16_t* out = c.out + ((int64_t)(q0 + tok) * c.p.nq + qh) * D + d0;
#pragma unroll
      for (int d = 0; d < D / 8; d += 8) {
        uint4 w;
        w.x = pack2<DT == TSB_DT_F16>(acc[d] * inv, acc[d + 1] * inv);
        w.y = pack2<DT == TSB_DT_F16>(acc[d + 2] * inv, acc[d + 3] * inv);
        w.z = pack2<DT == TSB_DT_F16>(acc[d + 4] * inv, acc[d + 5] * inv);
        w.w = pack2<DT == TSB_DT_F16>(acc[d + 6] * inv, acc[d + 7] * inv);
        *reinterpret_cast<uint4*>(out + d) = w;
      }
    }
    __syncthreads();  // the shared sums are read
    if (threadIdx.x == 0) sh.poison = 0;
    __syncthreads();
  }
}

}  // namespace

size_t short_partial_bytes(int head_dim) { return sizeof(float) * 2 * kMaxCtas * kRows * (head_dim + 2); }

int launch_paged_short(const TsbPagedCache& cache, const AttnCall& call, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  dispatch_paged(cache, [&](auto dt, auto d, auto fp8) {
    constexpr int DT = decltype(dt)::value, D = decltype(d)::value;
    constexpr bool FP8 = decltype(fp8)::value;
    ShortArgs a{call};
    // a launch's sequences: their steps are summed in 32 bits
    const int steps = call.p.max_pos / step_of<D>() + 3 + kItemCost;
    const int seqs = min(kMaxSeqs, INT32_MAX / steps);
    for (int b0 = 0; b0 < call.p.n_seqs && e == cudaSuccess; b0 += seqs) {
      a.c.p.table = call.p.table + (int64_t)b0 * call.p.table_stride;
      a.c.p.cu_q = call.p.cu_q + b0;
      a.c.p.kv_lens = call.p.kv_lens + b0;
      a.c.p.n_seqs = min(seqs, call.p.n_seqs - b0);
      // no more CTAs than pieces of the least size in the longest tables
      const int64_t most = (int64_t)a.c.p.n_seqs * call.p.nkv * (steps / kMinPiece + 1);
      auto kern = paged_attn_short<DT, D, FP8>;
      using Rg = Ring<D, FP8>;
      constexpr int smem = Rg::kBytes > (int)sizeof(Sums<D>) ? Rg::kBytes : (int)sizeof(Sums<D>);
      static bool ready[64];  // by device
      int dev = 0;
      e = cudaGetDevice(&dev);
      if (e == cudaSuccess && (dev >= 64 || !ready[dev]))
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return;
      if (dev < 64) ready[dev] = true;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)min(most, (int64_t)min(kMaxCtas, Rg::kPerSm * sm_count())));
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = smem;
      cfg.stream = st;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, kern, a);
    }
  });
  return e == cudaSuccess ? TSB_OK : set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace tsb
