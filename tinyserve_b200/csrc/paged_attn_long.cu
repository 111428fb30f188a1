// Attention of prompt chunks over a paged KV cache on the tensor cores
// (sequences with more than kShortRows rows per KV head; tsb_paged_attention).
//
// Rows: the query heads of a KV head share its keys, so a sequence's rows for
// one KV head are (token, head of the group), token-major; 256 of them, two
// tiles of 128, make an item.  An item walks its visible key tiles (128
// positions; with a window the tiles of the first tokens, then those from the
// window of its first row on) with a running maximum m and sum l per row:
//
//   S = Q K^T             tcgen05, both operands in shared memory, S in TMEM
//   P = 2^(c S - c m)     one thread per row, c = scale * log2(e)
//   O = O + P V           tcgen05, P from TMEM, V by its K rows
//
// m moves (and O, l are rescaled) only when a row's maximum has grown by more
// than 2^6 in weight, so O is rarely touched; every weight then stays below
// 2^6.  P is rounded to 16 bits (the sums l are not).  f16 weights are kept
// 2^8 times larger so that small ones stay above f16's smallest step.
//
// Types: 16-bit caches multiply in their type.  e4m3 caches multiply in f16,
// which holds every e4m3 value; bf16 queries are scaled per row by a power of
// two into f16's upper range first (exact but for elements 2^-38 below the
// row's largest).
//
// Work: the key tiles of all items form one line that is cut into equal
// pieces, one per CTA, so long and short rows and few or many items balance;
// an item that is cut leaves partial (O, m, l) and its last piece joins them
// in key order.
//
// Warps: 0-3 and 4-7 hold the rows of the two tiles, 8 issues the products,
// 9-10 load.  While one tile's rows are in the exponential the tensor core
// runs the other tile's products.
//
// A weight of zero times a value that is not finite would be NaN: in tiles
// where the mask hides something from some row, values that are not finite
// are replaced by zeros as they are loaded, and rows that do see them get them
// added at the end.
#include "paged.cuh"
#include "tmem_io.cuh"

namespace tsb {
namespace {

constexpr int kTileQ = 128, kTileK = 128;
constexpr int kItemRows = 2 * kTileQ;
constexpr int kWarpMma = 8, kWarpLoad = 9, kLoadWarps = 2;
constexpr int kThreads = 32 * (kWarpLoad + kLoadWarps);
constexpr int kMaxSeqs = 1024;  // sequences of one launch
constexpr int kItemCost = 2;    // an item's fixed work in key tiles
constexpr int kMinPiece = 6;    // a CTA's least share
constexpr int kMaxCtas = 148;
constexpr float kGrow = 6.f;    // rescale when the maximum grows by more (log2)

template <int D>
constexpr int stages() {
  return D == 64 ? 6 : 4;
}
template <int D>
constexpr int tile_bytes() {
  return kTileK * D * 2;
}

struct Shared {
  uint64_t q_full, q_empty, s_full[2], p_ready[2], o_full[2], drained;
  uint64_t part_left, part_said;  // a part is written; whether it was the item's last
  uint64_t kv_full[6], kv_empty[6];
  uint32_t tmem;
  int abort;
  int poison[4];   // the segment (number + 1, by its low bits) that met values that are not finite
  int last;        // this CTA joins the parts of the current item
  int start_seq, start_tile;
  int64_t start_off;
  int8_t q_exp[2][kItemRows];
  int q_len[kMaxSeqs], kv_len[kMaxSeqs];
  int64_t pre[kMaxSeqs + 1];
};

struct LongArgs {
  AttnCall c;
  int part_stride;  // floats of one partial result
};

// ------------------------------------------------------------------ geometry
struct Range {
  int nf, lo, n;  // tiles [0, nf), then from tile lo on; n in all
};
// Key tiles that some row of tile t of a sequence sees.
__device__ __forceinline__ Range key_tiles(const AttnCall& c, int q_len, int kv_len, int t) {
  const int G = c.p.G, base = kv_len - q_len;
  const int p0 = base + t * kItemRows / G;
  const int p1 = base + min(q_len - 1, (t * kItemRows + kItemRows - 1) / G);
  Range r{0, 0, 0};
  if (p1 < 0) return r;
  const int hi = p1 / kTileK + 1;
  const int first = c.window > 0 ? max(0, p0 - c.window + 1) : 0;
  r.lo = first / kTileK;
  r.nf = min((c.keep_first + kTileK - 1) / kTileK, r.lo);
  r.n = r.nf + hi - r.lo;
  return r;
}
__device__ __forceinline__ int tiles_of(const AttnCall& c, int q_len) {
  const int rows = q_len * c.p.G;
  return rows > kShortRows ? (rows + kItemRows - 1) / kItemRows : 0;
}
// Every row with a position in [p0, p1] sees all keys of the tile at j0.
__device__ __forceinline__ bool open_tile(const AttnCall& c, int p0, int p1, int j0) {
  return j0 + kTileK - 1 <= p0 && (c.window == 0 || j0 > p1 - c.window || j0 + kTileK - 1 < c.keep_first);
}

// One CTA's part of one item.
struct Segment {
  int b, head, q_len, kv_len, row0, rows;  // row0: first row of the item, rows: rows of the sequence
  Range r;
  int k0, k1;          // of r's n tiles
  int part, parts, c_first;
  bool zero;           // an item that sees nothing: write zeros
  int tiles;           // 1 or 2 tiles of rows
};

// The walk of one CTA over its piece of the line; every role runs it.
struct Walk {
  int64_t x, end, at, total;  // at: where the current item begins
  int n, head, b, t;
  __device__ int64_t cut(int c) const { return total * c / n; }
  __device__ int cta_of(int64_t p) const {
    int c = (int)(p * n / total);
    while (c > 0 && cut(c) > p) --c;
    while (c + 1 < n && cut(c + 1) <= p) ++c;
    return c;
  }
  __device__ bool next(const AttnCall& c, const Shared& sh, Segment& s) {
    while (x < end) {
      s.b = b;
      s.head = head;
      s.q_len = sh.q_len[b];
      s.kv_len = sh.kv_len[b];
      s.row0 = t * kItemRows;
      s.rows = s.q_len * c.p.G;
      s.r = key_tiles(c, s.q_len, s.kv_len, t);
      s.tiles = s.rows - s.row0 > kTileQ ? 2 : 1;
      const int64_t keys = at + kItemCost, stop = keys + s.r.n;
      const int64_t to = min(end, stop);
      s.k0 = (int)max((int64_t)0, x - keys);
      s.k1 = (int)max((int64_t)0, to - keys);
      s.zero = s.r.n == 0 && x == at;
      s.parts = 1;
      s.part = 0;
      if (s.k1 > s.k0 && (s.k0 > 0 || s.k1 < s.r.n)) {
        s.c_first = cta_of(keys);
        s.parts = cta_of(stop - 1) - s.c_first + 1;
        s.part = (int)blockIdx.x - s.c_first;
      }
      x = to;
      if (to == stop) {
        at = stop;
        if (++t >= tiles_of(c, s.q_len)) {
          t = 0;
          for (;;) {
            if (++b >= c.p.n_seqs) {
              b = 0;
              ++head;
            }
            if (tiles_of(c, sh.q_len[b])) break;  // some sequence has tiles: total > 0
          }
        }
      }
      if (s.k1 > s.k0 || s.zero) return true;
    }
    return false;
  }
};

// Key tile number of index k of a segment's list.
__device__ __forceinline__ int tile_at(const Range& r, int k) { return k < r.nf ? k : r.lo + (k - r.nf); }

// ------------------------------------------------------------------ waits
// Bounded; when one gives up the CTA's other waits give up too, and every
// role falls through to the kernel's end.
__device__ __forceinline__ bool wait_for(Shared& sh, uint64_t* bar, uint32_t parity, int32_t* err) {
  for (uint32_t i = 0; i < kMaxPolls; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(&sh.abort)) return false;
  }
  *reinterpret_cast<volatile int*>(&sh.abort) = 1;
  atomicExch(err, kDevWaitTimeout);
  return false;
}

// The same for a whole warp, which goes on or gives up together.
__device__ __forceinline__ bool warp_wait_for(Shared& sh, uint64_t* bar, uint32_t parity, int32_t* err) {
  return __all_sync(0xffffffffu, wait_for(sh, bar, parity, err));
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
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t b) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(b));
  return r;
}
// Zeroes the 16-bit elements of a word that are not finite; true if any was.
template <bool F16>
__device__ __forceinline__ bool drop_nonfinite(uint32_t& w) {
  constexpr uint32_t e = F16 ? 0x7C007C00u : 0x7F807F80u;
  const uint32_t bad = __vcmpeq2(w & e, e);
  w &= ~bad;
  return bad != 0;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// ------------------------------------------------------------------ loaders
template <int DT, int D, bool FP8>
struct Loader {
  static constexpr bool kF16 = FP8 || DT == TSB_DT_F16;
  static constexpr int NS = stages<D>(), TB = tile_bytes<D>();
  static constexpr int kLag = NS / 2;  // copies in flight, in units of one K or V tile
  const AttnCall& c;
  Shared& sh;
  uint32_t q_smem, kv_smem;
  int warp, lane;
  uint32_t unit = 0, signalled = 0;  // tiles begun / announced
  uint32_t bound_units = 0;          // bit u % 32: unit u holds values of a tile that is not open
  int live = 0;
  bool ok = true;

  __device__ bool wait_slot() {
    const uint32_t round = unit / NS;
    if (round > 0) ok = ok && warp_wait_for(sh, &sh.kv_empty[unit % NS], (round - 1) & 1, c.p.err);
    return ok;
  }
  __device__ void announce(uint32_t u) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.kv_full[u % NS]);
  }
  __device__ void flag_poison() {
    *reinterpret_cast<volatile int*>(&sh.poison[live & 3]) = live + 1;
    __threadfence_block();
  }

  // Element offsets of this warp's 64 rows of the tile at j0: lane l holds
  // rows l and l + 32; -1 past the end of the sequence.
  __device__ void row_offsets(const Segment& s, int j0, int64_t (&off)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = j0 + warp * 64 + i * 32 + lane;
      off[i] = j < s.kv_len ? cached_row(c.p, s.b, j) : -1;
      if (off[i] >= 0) off[i] += s.head * c.p.head_stride;
    }
  }
  __device__ static int64_t pick(const int64_t (&off)[2], int r) {  // r: row of this warp's 64
    const int64_t a = __shfl_sync(0xffffffffu, off[0], r & 31), b = __shfl_sync(0xffffffffu, off[1], r & 31);
    return r < 32 ? a : b;
  }

  __device__ void load_q(const Segment& s) {
    constexpr int CH = D / 8, RPI = 32 / CH;  // 16-byte chunks of a row, rows per step
    const int G = c.p.G;
    const uint32_t flip = c.scale < 0.f ? 0x80008000u : 0u;
    for (int r0 = warp * RPI; r0 < s.tiles * kTileQ; r0 += 4 * kLoadWarps * RPI) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int R = s.row0 + r0 + u * kLoadWarps * RPI + lane / CH;
        v[u] = make_uint4(0, 0, 0, 0);
        if (R < s.rows) {
          const int i = R / G, g = R - i * G;
          v[u] = *reinterpret_cast<const uint4*>(c.q + (int64_t)(c.p.cu_q[s.b] + i) * c.q_token_stride +
                                                 (int64_t)(s.head * G + g) * c.q_head_stride + (lane % CH) * 8);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = r0 + u * kLoadWarps * RPI + lane / CH;
        uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        if constexpr (FP8 && DT == TSB_DT_BF16) {
          // the row's largest element to [2^14, 2^15): exponents only
          uint32_t big = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) big = max(big, max(w[k] & 0x7FFFu, (w[k] >> 16) & 0x7FFFu));
#pragma unroll
          for (int o = CH / 2; o; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
          const int e = (int)(big >> 7);
          const int shift = e == 255 || big == 0 ? 0 : min(127, 14 + 127 - max(e, 1));
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float lo = ldexpf(__uint_as_float(w[k] << 16), shift);
            const float hi = ldexpf(__uint_as_float(w[k] & 0xFFFF0000u), shift);
            w[k] = pack2<true>(lo, hi);
          }
          if (lane % CH == 0) sh.q_exp[live & 1][r] = (int8_t)shift;
        }
        const int ch = lane % CH;
        const uint32_t dst = q_smem + (r / kTileQ) * TB + (ch / 8) * (kTileQ * 128) + sw128_off(r % kTileQ, ch % 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0] ^ flip), "r"(w[1] ^ flip),
                     "r"(w[2] ^ flip), "r"(w[3] ^ flip)
                     : "memory");
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.q_full);
  }

  // ---- 16-bit caches: asynchronous copies, announced kLag units later
  __device__ void copy_unit(const uint8_t* pool, const int64_t (&off)[2], bool closed) {
    constexpr int CH = D / 8, RPI = 32 / CH;
    if (!wait_slot()) return;
    const uint32_t base = kv_smem + (unit % NS) * TB;
    const int ch = lane % CH;
#pragma unroll
    for (int i = 0; i < 64 / RPI; ++i) {
      const int r = i * RPI + lane / CH;
      const int64_t o = pick(off, r);
      const uint32_t dst = base + (ch / 8) * (kTileK * 128) + sw128_off(warp * 64 + r, ch % 8);
      cp_async16(dst, pool + 2 * ((o < 0 ? 0 : o) + ch * 8), o >= 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (closed)
      bound_units |= 1u << (unit % 32);
    else
      bound_units &= ~(1u << (unit % 32));
    ++unit;
  }
  __device__ void finish_unit() {  // the copies of unit `signalled` have landed
    constexpr int CH = D / 8, RPI = 32 / CH;
    if (bound_units >> (signalled % 32) & 1) {
      const uint32_t base = kv_smem + (signalled % NS) * TB;
      const int ch = lane % CH;
      bool any = false;
      for (int i = 0; i < 64 / RPI; ++i) {
        const uint32_t at = base + (ch / 8) * (kTileK * 128) + sw128_off(warp * 64 + i * RPI + lane / CH, ch % 8);
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(at)
                     : "memory");
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) bad |= drop_nonfinite<kF16>(w[k]);
        if (bad)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
        any |= bad;
      }
      if (any) flag_poison();
    }
    announce(signalled);
    ++signalled;
  }
  __device__ void drain() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    while (signalled < unit) finish_unit();
  }

  // ---- e4m3 caches: through registers, one unit ahead
  static constexpr int kRegs = FP8 ? 64 * D / 16 / 32 : 1;
  __device__ void fetch(const uint8_t* pool, const int64_t (&off)[2], uint4 (&v)[kRegs]) const {
    constexpr int CH = D / 16, RPI = 32 / CH;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int64_t o = pick(off, i * RPI + lane / CH);
      v[i] = make_uint4(0, 0, 0, 0);
      if (o >= 0) v[i] = *reinterpret_cast<const uint4*>(pool + o + (lane % CH) * 16);
    }
  }
  __device__ void put(uint4 (&v)[kRegs], bool closed) {
    constexpr int CH = D / 16, RPI = 32 / CH;
    if (!wait_slot()) return;
    const uint32_t base = kv_smem + (unit % NS) * TB;
    bool any = false;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      uint32_t b[4] = {v[i].x, v[i].y, v[i].z, v[i].w}, h[8];
      if (closed) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t bad = __vcmpeq4(b[k] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
          b[k] &= ~bad;
          any |= bad != 0;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[2 * k] = e4m3x2_to_f16x2((uint16_t)b[k]);
        h[2 * k + 1] = e4m3x2_to_f16x2((uint16_t)(b[k] >> 16));
      }
      const int r = warp * 64 + i * RPI + lane / CH, ch = 2 * (lane % CH);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t dst = base + ((ch + k) / 8) * (kTileK * 128) + sw128_off(r, (ch + k) % 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(h[4 * k]), "r"(h[4 * k + 1]),
                     "r"(h[4 * k + 2]), "r"(h[4 * k + 3])
                     : "memory");
      }
    }
    if (any) flag_poison();
    announce(unit);
    ++unit;
  }

  __device__ void run(Walk w) {
    Segment s;
    while (ok && w.next(c, sh, s)) {
      if (s.k1 == s.k0) continue;
      if (live > 0) ok = warp_wait_for(sh, &sh.q_empty, (live - 1) & 1, c.p.err);
      if (!ok) break;
      load_q(s);
      const int base = s.kv_len - s.q_len;
      const int p0 = base + s.row0 / c.p.G, p1 = base + min(s.q_len - 1, (s.row0 + kItemRows - 1) / c.p.G);
      int64_t off[2];
      int j0 = tile_at(s.r, s.k0) * kTileK;
      row_offsets(s, j0, off);
      if constexpr (FP8) {
        uint4 k[kRegs], v[kRegs];
        fetch(c.p.kc, off, k);
        for (int i = s.k0; i < s.k1 && ok; ++i) {
          const bool closed = !open_tile(c, p0, p1, j0);
          fetch(c.p.vc, off, v);
          put(k, false);
          if (i + 1 < s.k1) {
            j0 = tile_at(s.r, i + 1) * kTileK;
            row_offsets(s, j0, off);
            fetch(c.p.kc, off, k);
          }
          put(v, closed);
        }
      } else {
        for (int i = s.k0; i < s.k1 && ok; ++i) {
          const bool closed = !open_tile(c, p0, p1, j0);
          copy_unit(c.p.kc, off, false);
          if (unit - signalled > kLag) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
            finish_unit();
          }
          int64_t next[2] = {-1, -1};
          const int jn = i + 1 < s.k1 ? tile_at(s.r, i + 1) * kTileK : 0;
          if (i + 1 < s.k1) row_offsets(s, jn, next);
          if (ok) copy_unit(c.p.vc, off, closed);
          if (unit - signalled > kLag) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
            finish_unit();
          }
          off[0] = next[0];
          off[1] = next[1];
          j0 = jn;
        }
        drain();
      }
      ++live;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
};

// ------------------------------------------------------------------ products
template <int DT, int D, bool FP8>
__device__ void issue_products(const AttnCall& c, Shared& sh, Walk w, uint32_t q_smem, uint32_t kv_smem, uint32_t tmem) {
  constexpr bool kF16 = FP8 || DT == TSB_DT_F16;
  constexpr int NS = stages<D>(), TB = tile_bytes<D>();
  constexpr uint32_t kQk = idesc_f16(kTileQ, kTileK, kF16 ? 0 : 1);
  constexpr uint32_t kPv = idesc_f16(kTileQ, D, kF16 ? 0 : 1) | kIdescBTransposed;
  const auto s_at = [&](int x) { return tmem + x * kTileK; };
  const auto o_at = [&](int x) { return tmem + 2 * kTileK + x * D; };
  uint32_t used = 0;        // K and V tiles consumed
  uint32_t p_phase = 0;     // p_ready completions waited for (both tiles alike, tile 1 only if present)
  uint32_t p_phase1 = 0;
  int live = 0;
  bool ok = true;
  const auto tile_full = [&](uint32_t u) { return wait_for(sh, &sh.kv_full[u % NS], (u / NS) & 1, c.p.err); };
  const auto qk = [&](int x, uint32_t u) {
    const uint32_t a = q_smem + x * TB, b = kv_smem + (u % NS) * TB;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t o = (k / 4) * (128 * 128) + (k % 4) * 32;
      umma_f16(s_at(x), sw128_desc(a + o), sw128_desc(b + o), kQk, k > 0);
    }
    umma_commit(&sh.s_full[x]);
  };
  const auto pv = [&](int x, uint32_t u, bool first) {
    const uint32_t b = kv_smem + (u % NS) * TB;
#pragma unroll
    for (int k = 0; k < kTileK / 16; ++k)
      umma_f16_ta(o_at(x), s_at(x) + 8 * k, sw128_mn_desc(b + k * 16 * 128, D == 64 ? 1024 : kTileK * 128), kPv,
                  !(first && k == 0));
  };
  Segment s;
  while (ok && w.next(c, sh, s)) {
    const int n = s.k1 - s.k0;
    if (n == 0) continue;
    ok = wait_for(sh, &sh.q_full, live & 1, c.p.err) && tile_full(used);
    if (!ok) break;
    tc_fence_after();
    for (int x = 0; x < s.tiles; ++x) qk(x, used);
    umma_commit(&sh.kv_empty[used % NS]);
    if (n == 1) umma_commit(&sh.q_empty);
    for (int i = 0; i < n && ok; ++i) {
      const uint32_t v = used + 1, k = used + 2;
      ok = tile_full(v) && (i + 1 == n || tile_full(k));
      for (int x = 0; x < s.tiles && ok; ++x) {
        uint32_t& ph = x ? p_phase1 : p_phase;
        ok = wait_for(sh, &sh.p_ready[x], ph & 1, c.p.err);
        if (!ok) break;
        ++ph;
        tc_fence_after();
        pv(x, v, i == 0);
        if (i + 1 < n)
          qk(x, k);
        else
          umma_commit(&sh.o_full[x]);
      }
      if (!ok) break;
      umma_commit(&sh.kv_empty[v % NS]);
      if (i + 1 < n) umma_commit(&sh.kv_empty[k % NS]);
      if (i + 2 == n) umma_commit(&sh.q_empty);
      used += 2;
    }
    // used: one K and one V tile per index
    ++live;
  }
  // nothing may be in flight when tensor memory is given back
  umma_commit(&sh.drained);
  for (uint32_t i = 0; i < kMaxPolls && !mbar_try_wait(&sh.drained, 0); ++i) {
  }
}

// ------------------------------------------------------------------ rows
// One row of an item from its parts, in key order.
template <int DT, int D>
__device__ void join_parts(const LongArgs& la, const Segment& s, int row, float sink, uint16_t* out) {
  const auto slot = [&](int i) {
    return la.c.part + (int64_t)(2 * (s.c_first + i) + (i == 0 ? 1 : 0)) * la.part_stride + row;
  };
  constexpr int kM = D * kItemRows, kL = (D + 1) * kItemRows;
  float top = sink;
  for (int i = 0; i < s.parts; ++i) top = fmaxf(top, __ldcg(slot(i) + kM));
  const float ref = top == -INFINITY ? 0.f : top;
  float all = ex2(sink - ref);
  for (int i = 0; i < s.parts; ++i) all += __ldcg(slot(i) + kL) * ex2(__ldcg(slot(i) + kM) - ref);
  const float inv = all == 0.f ? 0.f : 1.f / all;
#pragma unroll 1
  for (int d = 0; d < D; d += 16) {
    float o[16] = {};
    for (int i = 0; i < s.parts; ++i) {
      const float* sl = slot(i);
      const float f = ex2(__ldcg(sl + kM) - ref);
#pragma unroll
      for (int k = 0; k < 16; ++k) o[k] = fmaf(f, __ldcg(sl + (d + k) * kItemRows), o[k]);
    }
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
      uint4 q;
      uint32_t* qw = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
      for (int e = 0; e < 4; ++e) qw[e] = pack2<DT == TSB_DT_F16>(o[k + 2 * e] * inv, o[k + 2 * e + 1] * inv);
      *reinterpret_cast<uint4*>(out + d + k) = q;
    }
  }
}

template <int DT, int D, bool FP8>
__device__ void softmax_rows(const LongArgs& la, Shared& sh, Walk w, uint32_t tmem) {
  const AttnCall& c = la.c;
  constexpr bool kF16 = FP8 || DT == TSB_DT_F16;
  constexpr float kBias = kF16 ? 8.f : 0.f;
  const int x = threadIdx.x / kTileQ, r = threadIdx.x % kTileQ;  // tile and row
  const uint32_t lanes = (uint32_t)((threadIdx.x / 32) % 4) << 21;  // warp's first lane << 16
  const uint32_t s_at = tmem + lanes + x * kTileK, o_at = tmem + lanes + 2 * kTileK + x * D;
  const int G = c.p.G;
  const float c0 = fmaxf(fabsf(c.scale) * 1.4426950408889634f, 1e-37f);  // positive: -infinity stays so
  uint32_t s_phase = 0, o_phase = 0, cut_parts = 0;
  int live = 0;
  bool ok = true;
  Segment s;
  while (ok && w.next(c, sh, s)) {
    const int n = s.k1 - s.k0, R = s.row0 + x * kTileQ + r;
    const int base = s.kv_len - s.q_len;
    const int token = R < s.rows ? R / G : 0, pos = R < s.rows ? base + token : -1;
    const int q0 = c.p.cu_q[s.b];
    const bool mine = x < s.tiles;
    float m = -INFINITY, l = 0.f, cr = c0;
    if (n > 0 && mine) {
      const int first = s.row0 + x * kTileQ;
      const int p0 = base + first / G, p1 = base + min(s.q_len - 1, (first + kTileQ - 1) / G);
      for (int i = 0; i < n; ++i) {
        const int j0 = tile_at(s.r, s.k0 + i) * kTileK;
        ok = warp_wait_for(sh, &sh.s_full[x], s_phase & 1, c.p.err);
        if (!ok) break;
        ++s_phase;
        tc_fence_after();
        if constexpr (FP8 && DT == TSB_DT_BF16) {
          if (i == 0) cr = fmaxf(ldexpf(c0, -(int)sh.q_exp[live & 1][x * kTileQ + r]), 1e-37f);
        }
        uint32_t v[kTileK];
        tmem_load_row128(s_at, v);
        if (!open_tile(c, p0, p1, j0)) {
          const int hi = pos - j0, lo = c.window > 0 ? pos - c.window - j0 : -1, f = c.keep_first - j0;
#pragma unroll
          for (int k = 0; k < kTileK; ++k)
            if (!(k <= hi && (k > lo || k < f))) v[k] = 0xFF800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < kTileK; ++k) mx[k % 4] = fmaxf(mx[k % 4], __uint_as_float(v[k]));
        const float top = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
        if (__any_sync(0xffffffffu, (top - m) * cr > kGrow)) {
          const float keep = m == -INFINITY ? 0.f : ex2((m - top) * cr);
          m = top;
          l *= keep;
          if (i > 0) {
#pragma unroll
            for (int d = 0; d < D; d += 32) {
              uint32_t o[32];
              tmem_load_row32(o_at + d, o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
              tmem_store_row32(o_at + d, o);
            }
          }
        }
        const float mc = (m == -INFINITY ? 0.f : m * cr) - kBias;
        float sum[4] = {};
        uint32_t p[kTileK / 2];
#pragma unroll
        for (int k = 0; k < kTileK / 2; ++k) {
          const float a = ex2(fmaf(__uint_as_float(v[2 * k]), cr, -mc));
          const float b = ex2(fmaf(__uint_as_float(v[2 * k + 1]), cr, -mc));
          sum[k % 4] += a + b;
          p[k] = pack2<kF16>(a, b);
        }
        tmem_store_row32(s_at, p);
        tmem_store_row32(s_at + 32, p + 32);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sh.p_ready[x]);
      }
      if (!ok) break;
      ok = warp_wait_for(sh, &sh.o_full[x], o_phase & 1, c.p.err);
      if (!ok) break;
      ++o_phase;
      tc_fence_after();
    }
    // the row's result: written, or left as one part
    const bool poisoned = n > 0 && *reinterpret_cast<volatile int*>(&sh.poison[live & 3]) == live + 1;
    const float sink = c.sinks && R < s.rows ? c.sinks[s.head * G + (R - token * G)] * 1.4426950408889634f : -INFINITY;
    const float mlog = m == -INFINITY ? -INFINITY : m * cr - kBias;  // weights are 2^(c s - mlog)
    float inv = 0.f;
    if (s.parts == 1) {
      const float all = l + (sink == -INFINITY ? 0.f : ex2(sink - (m == -INFINITY ? sink : mlog)));
      inv = all == 0.f ? 0.f : 1.f / all;
    }
    float* part = la.c.part + (int64_t)(2 * blockIdx.x + (s.part == 0 ? 1 : 0)) * la.part_stride;
    const int rr = x * kTileQ + r;
#pragma unroll
    for (int d = 0; d < D; d += 32) {
      uint32_t o[32];
      if (n > 0 && mine) {
        tmem_load_row32(o_at + d, o);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0;
      }
      if (poisoned && pos >= 0) {
        for (int i = s.k0; i < s.k1; ++i) {
          const int t0 = tile_at(s.r, i) * kTileK;
          const int pa = base + s.row0 / G, pb = base + min(s.q_len - 1, (s.row0 + kItemRows - 1) / G);
          if (open_tile(c, pa, pb, t0)) continue;
          for (int j = t0; j <= min(pos, t0 + kTileK - 1); ++j) {
            if (c.window > 0 && j <= pos - c.window && j >= c.keep_first) continue;
            const int64_t row = cached_row(c.p, s.b, j);
            if (row < 0) continue;
            const int64_t at = row + s.head * c.p.head_stride + d;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              float vv;
              if constexpr (FP8)
                vv = e4m3_to_f32(c.p.vc[at + k]);
              else
                vv = to_f32<DT>(reinterpret_cast<const uint16_t*>(c.p.vc)[at + k]);
              if (!isfinite(vv)) o[k] = __float_as_uint(__uint_as_float(o[k]) + vv);
            }
          }
        }
      }
      __syncwarp();
      if (s.parts > 1) {
#pragma unroll
        for (int k = 0; k < 32; ++k) part[(d + k) * kItemRows + rr] = __uint_as_float(o[k]);
      } else if (R < s.rows) {
        uint16_t* out = c.out + ((int64_t)(q0 + token) * c.p.nq + s.head * G + (R - token * G)) * D + d;
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          uint4 q;
          uint32_t* qw = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            qw[e] = pack2<DT == TSB_DT_F16>(__uint_as_float(o[k + 2 * e]) * inv, __uint_as_float(o[k + 2 * e + 1]) * inv);
          *reinterpret_cast<uint4*>(out + k) = q;
        }
      }
    }
    if (n > 0) ++live;
    tc_fence_before();
    if (s.parts == 1) continue;
    // parts are joined by whoever comes last
    part[D * kItemRows + rr] = mlog;
    part[(D + 1) * kItemRows + rr] = l;
    __threadfence();
    mbar_arrive(&sh.part_left);
    if (threadIdx.x == 0) {
      if (wait_for(sh, &sh.part_left, cut_parts & 1, c.p.err)) {
        unsigned prev;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                     : "=r"(prev)
                     : "l"(c.counters + s.c_first)
                     : "memory");
        sh.last = prev == (unsigned)(s.parts - 1);
        if (sh.last) c.counters[s.c_first] = 0;
        mbar_arrive(&sh.part_said);
      }
    }
    __syncwarp();
    ok = warp_wait_for(sh, &sh.part_said, cut_parts & 1, c.p.err);
    if (!ok) break;
    ++cut_parts;
    if (!*reinterpret_cast<volatile int*>(&sh.last)) continue;
    if (R < s.rows) {
      __threadfence();
      join_parts<DT, D>(la, s, rr, sink,
                        c.out + ((int64_t)(q0 + token) * c.p.nq + s.head * G + (R - token * G)) * D);
    }
    __syncwarp();
  }
}

// ------------------------------------------------------------------ kernel
template <int DT, int D, bool FP8>
__global__ void __launch_bounds__(kThreads, 1) paged_attn_long(const __grid_constant__ LongArgs la) {
  extern __shared__ uint8_t dyn[];
  __shared__ Shared sh;
  const AttnCall& c = la.c;
  constexpr int NS = stages<D>(), TB = tile_bytes<D>();
  const uint32_t kv_smem = (smem_u32(dyn) + 1023u) & ~1023u, q_smem = kv_smem + NS * TB;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, kLoadWarps);
    mbar_init(&sh.q_empty, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sh.s_full[x], 1);
      mbar_init(&sh.p_ready[x], kTileQ);
      mbar_init(&sh.o_full[x], 1);
      sh.poison[x] = sh.poison[2 + x] = 0;
    }
    mbar_init(&sh.drained, 1);
    mbar_init(&sh.part_left, 2 * kTileQ);
    mbar_init(&sh.part_said, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh.kv_full[i], kLoadWarps);
      mbar_init(&sh.kv_empty[i], 1);
    }
    sh.abort = 0;
    fence_barrier_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch_dependents();
  // lengths, and each sequence's key tiles per KV head
  for (int b = warp; b < c.p.n_seqs; b += kThreads / 32) {
    SeqSpan sp{0, 0, 0};
    if (lane == 0) sp = seq_span(c.p, b);
    const int q_len = __shfl_sync(0xffffffffu, sp.q_len, 0), kv_len = __shfl_sync(0xffffffffu, sp.kv_len, 0);
    int64_t sum = 0;
    for (int t = lane; t < tiles_of(c, q_len); t += 32) sum += key_tiles(c, q_len, kv_len, t).n + kItemCost;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      sh.q_len[b] = q_len;
      sh.kv_len[b] = kv_len;
      sh.pre[b + 1] = sum;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) {  // sums to running sums
    int64_t run = 0;
    for (int b0 = 0; b0 < c.p.n_seqs; b0 += 32) {
      int64_t v = b0 + lane < c.p.n_seqs ? sh.pre[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (b0 + lane < c.p.n_seqs) sh.pre[b0 + lane + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) sh.pre[0] = 0;
  }
  __syncthreads();
  const int64_t per_head = sh.pre[c.p.n_seqs];
  Walk w;
  w.total = per_head * c.p.nkv;
  w.n = (int)min((int64_t)gridDim.x, max((int64_t)1, w.total / kMinPiece));
  const bool works = w.total > 0 && (int)blockIdx.x < w.n;
  if (works) {
    w.x = w.cut(blockIdx.x);
    w.end = w.cut(blockIdx.x + 1);
    w.head = (int)(w.x / per_head);
    const int64_t off = w.x - w.head * per_head;
    if (warp == 0) {  // the sequence and tile the piece starts in
      int lo = 0, hi = c.p.n_seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sh.pre[mid] <= off)
          lo = mid;
        else
          hi = mid;
      }
      // of sequences that start at the same place only the last has tiles
      int64_t begin = sh.pre[lo];
      int t0 = 0;
      const int nt = tiles_of(c, sh.q_len[lo]);
      for (;; t0 += 32) {
        int v = t0 + lane < nt ? key_tiles(c, sh.q_len[lo], sh.kv_len[lo], t0 + lane).n + kItemCost : 0;
        const int own = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        const unsigned past = __ballot_sync(0xffffffffu, begin + v > off);
        if (past || t0 + 32 >= nt) {
          const int l0 = past ? __ffs(past) - 1 : 31;
          if (lane == l0) {
            sh.start_seq = lo;
            sh.start_tile = t0 + lane;
            sh.start_off = w.head * per_head + begin + v - own;
          }
          break;
        }
        begin += __shfl_sync(0xffffffffu, v, 31);
      }
    }
  }
  __syncthreads();
  if (works) {
    w.b = sh.start_seq;
    w.t = sh.start_tile;
    w.at = sh.start_off;
    const uint32_t tmem = sh.tmem;
    if (warp < kWarpMma) {
      softmax_rows<DT, D, FP8>(la, sh, w, tmem);
    } else if (warp == kWarpMma) {
      if (lane == 0) issue_products<DT, D, FP8>(c, sh, w, q_smem, kv_smem, tmem);
    } else {
      Loader<DT, D, FP8> ld{c, sh, q_smem, kv_smem, warp - kWarpLoad, lane};
      ld.run(w);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, 512);
  }
}

int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    return v;
  }();
  return n;
}

constexpr int part_floats(int d) { return (d + 2) * kItemRows; }

}  // namespace

size_t long_partial_bytes(int head_dim) { return sizeof(float) * 2 * kMaxCtas * part_floats(head_dim); }

int launch_paged_long(const TsbPagedCache& cache, const AttnCall& call, cudaStream_t st) {
  int rc = TSB_OK;
  dispatch_paged(cache, [&](auto dt, auto d, auto fp8) {
    constexpr int D = decltype(d)::value;
    auto kern = paged_attn_long<decltype(dt)::value, D, decltype(fp8)::value>;
    constexpr int smem = (stages<D>() + 2) * tile_bytes<D>() + 1024;
    static bool ready[64];  // by device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !ready[dev]))
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
      rc = set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
      return;
    }
    if (dev < 64) ready[dev] = true;
    LongArgs la{call, part_floats(D)};
    for (int b0 = 0; b0 < call.p.n_seqs && rc == TSB_OK; b0 += kMaxSeqs) {
      la.c.p.table = call.p.table + (int64_t)b0 * call.p.table_stride;
      la.c.p.cu_q = call.p.cu_q + b0;
      la.c.p.kv_lens = call.p.kv_lens + b0;
      la.c.p.n_seqs = min(kMaxSeqs, call.p.n_seqs - b0);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(min(kMaxCtas, sm_count()));
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = smem;
      cfg.stream = st;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, kern, la);
      if (e != cudaSuccess) rc = set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
    }
  });
  return rc;
}

}  // namespace tsb
