// Attention of prompt chunks over a paged KV cache on the tensor cores
// (sequences with more than short_rows rows per KV head; tsb_paged_attention).
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
// 2^6.  P is rounded to 16 bits for the product (the sums l are not).  f16 weights are kept
// 2^8 times larger so that small ones stay above f16's smallest step.
//
// Types: 16-bit caches multiply in their type.  e4m3 caches multiply in f16,
// which holds every e4m3 value; bf16 queries are scaled per row by a power of
// two into f16's upper range first: elements down to 2^-31 of the row's largest
// stay exact, smaller ones are off by up to 2^-39 of it.
//
// Error: scores and sums are fp32, each weight is rounded once to P's type, l is
// summed from the unrounded ones.  Outputs against 64 bits, relative L2: prompt of
// 4096 tokens in bf16 0.0021, where the output's own rounding alone gives 0.0017; over
// e4m3 caches (f16 weights) 0.0017; f16 0.00025, where its rounding alone gives 0.00021.
//
// Work: the key tiles of all items form one line that is cut into equal
// pieces, one per CTA, so long and short rows and few or many items balance;
// an item that is cut leaves partial (O, m, l) and its last piece joins them
// in key order.
//
// Warps: 0-3 and 4-7 hold the rows of the two tiles, 8 issues the products, 9
// the tensor copies, 10-11 load Q, 12-15 load or finish K and V.  While one
// tile's rows are in the exponential the tensor core runs the other tile's
// products.
//
// K and V reach shared memory in one of three ways: 16-bit pools whose pages
// hold whole groups of 8 rows by tensor copies (boxes of the largest power of
// two that divides the page size), other 16-bit pools by 16-byte asynchronous
// copies, e4m3 pools through registers, widened on the way.
//
// What bounds it: exponentials first (16 a cycle and SM: 122 us for a prompt of
// 4096 tokens with 64 heads; its products would take 83 us at the measured bf16
// rate), then what a step costs around them.  Measured there: 267 us, 0.51
// PFLOP/s, the two tiles' rows 2200 of a step's 3700 cycles in their exponentials,
// 600 waiting for scores, the rest finding the maximum, masking and handing
// over.  What decided the time otherwise: 128 keys a step (S, P and O fill
// tensor memory), code that stays in the instruction caches (loops unrolled to
// 275 KB took 516 us, rolled 364), S read twice in 32-column pieces (held whole, its 128
// registers left none to keep exponentials in flight), scores of the next step
// issued as soon as a row is read.  Exponentials on the multiply-add units for a
// quarter of the weights made it slower: instructions, not the exponential
// unit alone, fill a step.
//
// A weight of zero times a value that is not finite would be NaN: in tiles
// where the mask hides something from some row, values that are not finite
// are replaced by zeros as they are loaded, and rows that do see them get them
// added at the end.
#include <cuda.h>

#include "paged.cuh"
#include "tmem_io.cuh"

namespace tsb {
namespace {

constexpr int kTileQ = 128, kTileK = 128;
constexpr int kItemRows = 2 * kTileQ;
constexpr int kWarpMma = 8, kWarpTma = 9, kWarpQ = 10, kQWarps = 2, kWarpKv = 12, kKvWarps = 4;
constexpr int kThreads = 32 * (kWarpKv + kKvWarps);
enum Feed { kFeedTma, kFeedCopy, kFeedWiden };  // how K and V reach shared memory
constexpr int kMaxSeqs = 512;   // sequences of one launch
constexpr int kItemCost = 4;    // an item's fixed work (Q, output) in key tiles; below kMinPiece
constexpr int kMinPiece = 6;    // a CTA's least share
constexpr int kMaxCtas = 148;
constexpr float kGrow = 6.f;    // rescale when the maximum grows by more (log2)

template <int D>
constexpr int stages() {
  return D == 64 ? 6 : 4;
}
template <int D>
constexpr int q_buffers() {  // two where they fit: the next segment's rows arrive during this one
  return D == 64 ? 2 : 1;
}
// Tensor memory (all 512 columns are the CTA's, so columns are plain
// numbers): S of both tiles, then P where there is room for it beside S
// (else in S's place), then O.
template <int D>
constexpr bool p_beside_s() {
  return D == 64;
}
template <int D>
constexpr int p_column(int x) {
  return p_beside_s<D>() ? 2 * kTileK + x * (kTileK / 2) : x * kTileK;
}
template <int D>
constexpr int o_column(int x) {
  return 512 - (2 - x) * D;
}
constexpr int kOutStage = 2048;  // bytes a row warp stages of its output: 32 rows of 32 elements
template <int D>
constexpr int tile_bytes() {
  return kTileK * D * 2;
}

struct Shared {
  uint64_t q_full[2], q_empty[2], s_full[2], s_read[2], p_ready[2], o_done[2], drained;
  uint64_t part_left, part_said;  // a part is written; whether it was the item's last
  uint64_t seg_done;              // the row threads are done with a segment
  uint64_t kv_full[6], kv_empty[6];
  uint64_t v_ok[6];             // tensor copies: the V tile is fit for the product
  uint32_t tmem;
  int abort;
  int poison[8];   // the segment (number + 1, by its low bits) that met values that are not finite
  int last;        // this CTA joins the parts of the current item
  int start_seq, start_tile;
  int64_t start_off;
  int8_t q_exp[4][kItemRows];
  int q_len[kMaxSeqs], kv_len[kMaxSeqs];
  int64_t pre[kMaxSeqs + 1];
};

struct LongArgs {
  CUtensorMap k_map, v_map;  // tensor copies only
  AttnCall c;
  int part_stride;  // floats of one partial result
  int box_rows;     // rows of one tensor copy
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
  return rows > c.short_rows ? (rows + kItemRows - 1) / kItemRows : 0;
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
// Bounded (some seconds); when one gives up the CTA's other waits give up too,
// and every role falls through to the kernel's end.
constexpr uint32_t kPollNs = 10000, kPolls = 1u << 18;
__device__ __forceinline__ bool phase_done(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(kPollNs)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_for(Shared& sh, uint64_t* bar, uint32_t parity, int32_t* err) {
  uint32_t polls = 0;
#pragma unroll 1
  while (!phase_done(bar, parity)) {
    volatile int* abort = &sh.abort;
    if (*abort) return false;
    if (++polls == kPolls) {
      *abort = 1;
      atomicExch(err, kDevWaitTimeout);
      return false;
    }
  }
  return true;
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Pairs of floats in one register pair: half the instructions of the scalar forms.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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
// Q rows of each segment, 16 bytes a lane.
template <int DT, int D, bool FP8>
__device__ void load_queries(const AttnCall& c, Shared& sh, Walk w, uint32_t q_smem, int warp, int lane) {
  constexpr int TB = tile_bytes<D>();
  constexpr int CH = D / 8, RPI = 32 / CH;  // 16-byte chunks of a row, rows per step
  constexpr int kBatch = 8;
  const int G = c.p.G;
  const uint32_t flip = c.scale < 0.f ? 0x80008000u : 0u;
  Segment s;
  for (int live = 0; w.next(c, sh, s);) {
    if (s.k1 == s.k0) continue;
    const uint16_t* q0 = c.q + (int64_t)c.p.cu_q[s.b] * c.q_token_stride;
    constexpr int NQ = q_buffers<D>();
    const int buf = live % NQ;
    if (live >= NQ && !warp_wait_for(sh, &sh.q_empty[buf], (live / NQ - 1) & 1, c.p.err)) return;
    for (int r0 = warp * RPI; r0 < s.tiles * kTileQ; r0 += kBatch * kQWarps * RPI) {
      uint4 v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int R = s.row0 + r0 + u * kQWarps * RPI + lane / CH;
        v[u] = make_uint4(0, 0, 0, 0);
        if (R < s.rows) {
          const int i = R / G, g = R - i * G;
          v[u] = *reinterpret_cast<const uint4*>(q0 + i * c.q_token_stride +
                                                 (int64_t)(s.head * G + g) * c.q_head_stride + (lane % CH) * 8);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int r = r0 + u * kQWarps * RPI + lane / CH;
        uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        if constexpr (FP8 && DT == TSB_DT_BF16) {
          // the row's largest element to [2^14, 2^15): exponents only
          uint32_t big = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) big = max(big, max(x[k] & 0x7FFFu, (x[k] >> 16) & 0x7FFFu));
#pragma unroll
          for (int o = CH / 2; o; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
          const int e = (int)(big >> 7);
          const int shift = e == 255 || big == 0 ? 0 : min(127, 14 + 127 - max(e, 1));
          // 2^shift in two factors, both in range
          const float f1 = __int_as_float((127 + shift / 2) << 23), f2 = __int_as_float((127 + shift - shift / 2) << 23);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            x[k] = pack2<true>(__uint_as_float(x[k] << 16) * f1 * f2, __uint_as_float(x[k] & 0xFFFF0000u) * f1 * f2);
          if (lane % CH == 0) sh.q_exp[live & 3][r] = (int8_t)shift;
        }
        const int ch = lane % CH;
        const uint32_t dst = q_smem + (2 * buf + r / kTileQ) * TB + (ch / 8) * (kTileQ * 128) + sw128_off(r % kTileQ, ch % 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x[0] ^ flip), "r"(x[1] ^ flip),
                     "r"(x[2] ^ flip), "r"(x[3] ^ flip)
                     : "memory");
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.q_full[buf]);
    ++live;
  }
}

// Tensor copies: lane i moves box i of each K and V tile.
template <int D>
__device__ void copy_tiles(const LongArgs& la, Shared& sh, Walk w, uint32_t kv_smem, int lane) {
  constexpr int NS = stages<D>(), TB = tile_bytes<D>();
  const AttnCall& c = la.c;
  const int rows = la.box_rows, boxes = kTileK / rows;
  uint32_t unit = 0;
  Segment s;
  while (w.next(c, sh, s)) {
    const auto find = [&](int k, int& page, int& row) {  // box `lane` of tile k of the list
      const int j = tile_at(s.r, k) * kTileK + lane * rows;
      page = -1;
      if (k < s.k1 && lane < boxes && j < s.kv_len) {
        const int pg = j / c.p.page_size;
        row = j - pg * c.p.page_size;
        page = c.p.table[(int64_t)s.b * c.p.table_stride + pg];
        if (page < 0 || page >= c.p.num_pages) {
          atomicExch(c.p.err, kDevBadPlan);
          page = -1;
        }
      }
    };
    int page, row = 0;
    find(s.k0, page, row);
#pragma unroll 1
    for (int i = s.k0; i < s.k1; ++i) {
      int next, next_row = 0;
      find(i + 1, next, next_row);
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * rows * (D * 2);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv, ++unit) {
        const uint32_t st = unit % NS;
        if (unit >= NS && !warp_wait_for(sh, &sh.kv_empty[st], (unit / NS - 1) & 1, c.p.err)) return;
        if (lane == 0) mbar_arrive_expect_tx(&sh.kv_full[st], bytes);
        __syncwarp();
        if (page >= 0) {
          const CUtensorMap* map = kv ? &la.v_map : &la.k_map;
#pragma unroll
          for (int d = 0; d < D; d += 64)
            asm volatile(
                "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
                "%5}], [%6];" ::"r"(kv_smem + st * TB + (d / 64) * (kTileK * 128) + lane * rows * 128),
                "l"(map), "r"(d), "r"(row), "r"(s.head), "r"(page), "r"(smem_u32(&sh.kv_full[st]))
                : "memory");
        }
      }
      page = next;
      row = next_row;
    }
  }
}

// The four K / V warps; warp w has rows [32 w, 32 w + 32) of each tile, lane l
// looks up row l.
template <int DT, int D, int FEED>
struct Loader {
  static constexpr int NS = stages<D>(), TB = tile_bytes<D>();
  static constexpr int kRows = kTileK / kKvWarps;
  const AttnCall& c;
  Shared& sh;
  uint32_t kv_smem;
  int warp, lane;
  uint32_t unit = 0, signalled = 0;  // tiles begun / announced
  uint32_t closed_units = 0;         // bit u % 32: unit u is the V of a tile that is not open
  int live = 0;
  bool ok = true;

  __device__ bool wait_slot() {
    if (unit >= NS) ok = ok && warp_wait_for(sh, &sh.kv_empty[unit % NS], (unit / NS - 1) & 1, c.p.err);
    return ok;
  }
  __device__ void announce(uint64_t* bar) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  }
  __device__ void flag_poison() {
    *reinterpret_cast<volatile int*>(&sh.poison[live & 7]) = live + 1;
    __threadfence_block();
  }
  // Element offset of this lane's row of the tile at j0; -1 past the end.
  __device__ int64_t row_offset(const Segment& s, int j0) const {
    const int j = j0 + warp * kRows + lane;
    const int64_t o = j < s.kv_len ? cached_row(c.p, s.b, j) : -1;
    return o < 0 ? -1 : o + s.head * c.p.head_stride;
  }
  // Replaces what is not finite in this warp's rows of a V tile by zeros; rows
  // from `held` on hold no position (page tails, or what was there before).
  __device__ void clean(uint32_t base, int held) {
    constexpr int CH = D / 8, RPI = 32 / CH;
    const int ch = lane % CH;
    bool any = false;
    for (int i = 0; i < kRows / RPI; ++i) {
      const int row = warp * kRows + i * RPI + lane / CH;
      const uint32_t at = base + (ch / 8) * (kTileK * 128) + sw128_off(row, ch % 8);
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "r"(at)
                   : "memory");
      bool bad = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= drop_nonfinite<DT == TSB_DT_F16>(w[k]);
      if (bad)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
      any |= bad && row < held;
    }
    if (any) flag_poison();
    __syncwarp();
  }

  // ---- asynchronous copies, announced kLag units later
  __device__ void copy_unit(const uint8_t* pool, int64_t off, bool closed) {
    constexpr int CH = D / 8, RPI = 32 / CH;
    if (!wait_slot()) return;
    const uint32_t base = kv_smem + (unit % NS) * TB;
    const int ch = lane % CH;
#pragma unroll
    for (int i = 0; i < kRows / RPI; ++i) {
      const int r = i * RPI + lane / CH;
      const int64_t o = __shfl_sync(0xffffffffu, off, r);
      const uint32_t dst = base + (ch / 8) * (kTileK * 128) + sw128_off(warp * kRows + r, ch % 8);
      cp_async16(dst, pool + 2 * ((o < 0 ? 0 : o) + ch * 8), o >= 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    const uint32_t bit = 1u << (unit % 32);
    closed_units = closed ? closed_units | bit : closed_units & ~bit;
    // Copies in flight, in units of one K or V tile.  Not more: the products of
    // index i wait for K of i + 1 before they let go of V of i - 1, so that K
    // must be announced without waiting for V's place.
    constexpr int kLag = 2;
    if (++unit - signalled > kLag) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
      finish_unit();
    }
  }
  __device__ void finish_unit() {  // the copies of unit `signalled` have landed
    if (closed_units >> (signalled % 32) & 1) clean(kv_smem + (signalled % NS) * TB, kTileK);  // zeros past the end
    announce(&sh.kv_full[signalled % NS]);
    ++signalled;
  }

  // ---- e4m3: through registers, one unit ahead
  static constexpr int kRegs = FEED == kFeedWiden ? kRows * D / 16 / 32 : 1;
  __device__ void fetch(const uint8_t* pool, int64_t off, uint4 (&v)[kRegs]) const {
    constexpr int CH = D / 16, RPI = 32 / CH;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int64_t o = __shfl_sync(0xffffffffu, off, i * RPI + lane / CH);
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
      const int r = warp * kRows + i * RPI + lane / CH, ch = 2 * (lane % CH);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t dst = base + ((ch + k) / 8) * (kTileK * 128) + sw128_off(r, (ch + k) % 8);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(h[4 * k]), "r"(h[4 * k + 1]),
                     "r"(h[4 * k + 2]), "r"(h[4 * k + 3])
                     : "memory");
      }
    }
    if (any) flag_poison();
    announce(&sh.kv_full[unit % NS]);
    ++unit;
  }

  __device__ void run(Walk w) {
    Segment s;
    while (ok && w.next(c, sh, s)) {
      if (s.k1 == s.k0) continue;
      const int base = s.kv_len - s.q_len;
      const int p0 = base + s.row0 / c.p.G, p1 = base + min(s.q_len - 1, (s.row0 + kItemRows - 1) / c.p.G);
      int j0 = tile_at(s.r, s.k0) * kTileK;
      if constexpr (FEED == kFeedWiden) {
        uint4 k[kRegs], v[kRegs];
        int64_t off = row_offset(s, j0);
        fetch(c.p.kc, off, k);
#pragma unroll 1
        for (int i = s.k0; i < s.k1 && ok; ++i) {
          const bool closed = !open_tile(c, p0, p1, j0);
          fetch(c.p.vc, off, v);
          put(k, false);
          if (i + 1 < s.k1) {
            j0 = tile_at(s.r, i + 1) * kTileK;
            off = row_offset(s, j0);
            fetch(c.p.kc, off, k);
          }
          put(v, closed);
        }
      } else if constexpr (FEED == kFeedCopy) {
        int64_t off = row_offset(s, j0);
#pragma unroll 1
        for (int i = s.k0; i < s.k1 && ok; ++i) {
          const bool closed = !open_tile(c, p0, p1, j0);
          copy_unit(c.p.kc, off, false);
          int64_t next = -1;
          j0 = tile_at(s.r, i + 1) * kTileK;
          if (i + 1 < s.k1) next = row_offset(s, j0);
          if (ok) copy_unit(c.p.vc, off, closed);
          off = next;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        while (signalled < unit) finish_unit();
      } else {
#pragma unroll 1
        for (int i = s.k0; i < s.k1 && ok; ++i) {
          const uint32_t u = unit + 1, st = u % NS;  // the V tile of this index
          ok = warp_wait_for(sh, &sh.kv_full[st], (u / NS) & 1, c.p.err);
          if (!ok) break;
          const int at = tile_at(s.r, i) * kTileK;
          if (!open_tile(c, p0, p1, at)) clean(kv_smem + st * TB, s.kv_len - at);
          announce(&sh.v_ok[st]);
          unit += 2;
        }
      }
      ++live;
    }
    if constexpr (FEED == kFeedCopy) asm volatile("cp.async.wait_all;" ::: "memory");
  }
};

// ------------------------------------------------------------------ products
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

// One warp walks and waits, one thread of it issues: its chain of waits and
// issues is what both tiles' rows wait for, so each K and V is waited for once
// and a product is in one place of the code.  Where P lies beside S the next
// scores go first (S is free once its row has been read, and the row needs them
// before it needs the sums), else PV_x(i), QK_x(i+1), which the tensor core
// runs in this order.  Row warps that wait for a commit release the K and V
// tiles and Q that it covers.
template <int DT, int D, int FEED>
__device__ void issue_products(const AttnCall& c, Shared& sh, Walk w, uint32_t q_smem, uint32_t kv_smem) {
  constexpr bool kF16 = FEED == kFeedWiden || DT == TSB_DT_F16;
  constexpr int NP = stages<D>() / 2, TB = tile_bytes<D>(), NQ = q_buffers<D>();
  constexpr uint32_t kQk = idesc_f16(kTileQ, kTileK, kF16 ? 0 : 1);
  constexpr uint32_t kPv = idesc_f16(kTileQ, D, kF16 ? 0 : 1) | kIdescBTransposed;
  const bool leader = elect_one();
  const uint64_t q_desc = sw128_desc(q_smem), k_desc = sw128_desc(kv_smem);
  const uint64_t v_desc = sw128_mn_desc(kv_smem + TB, D == 64 ? 1024 : kTileK * 128);
  int place = 0;                // of the pair of index i, and the parity of its round
  uint32_t round = 0;
  uint32_t p_phase[2] = {0, 0}, r_phase[2] = {0, 0};
  int live = 0;
  bool ok = true;
  const auto k_wait = [&](int pl, uint32_t rd) { ok = ok && warp_wait_for(sh, &sh.kv_full[2 * pl], rd & 1, c.p.err); };
  const auto v_wait = [&](int pl, uint32_t rd) {
    ok = ok && warp_wait_for(sh, FEED == kFeedTma ? &sh.v_ok[2 * pl + 1] : &sh.kv_full[2 * pl + 1], rd & 1, c.p.err);
  };
  const auto read_wait = [&](int x) {  // the rows have read the scores issued last
    ok = ok && warp_wait_for(sh, &sh.s_read[x], (r_phase[x] - 1) & 1, c.p.err);
  };
  const auto qk = [&](auto X, int pl) {
    if (!ok) return;
    tc_fence_after();
    if (leader) {
      constexpr int x = decltype(X)::value;
      const uint64_t a = q_desc + (uint32_t)((live % NQ) * (2 * TB >> 4)), b = k_desc + (uint32_t)(pl * (2 * TB >> 4));
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t o = ((k / 4) * (128 * 128) + (k % 4) * 32) >> 4;
        umma_f16(x * kTileK, a + x * (TB >> 4) + o, b + o, kQk, k > 0);
      }
      umma_commit(&sh.s_full[x]);
    }
    __syncwarp();
    ++r_phase[decltype(X)::value];
  };
  const auto pv = [&](auto X, int pl, bool first) {
    constexpr int x = decltype(X)::value;
    ok = ok && warp_wait_for(sh, &sh.p_ready[x], p_phase[x] & 1, c.p.err);
    if (!ok) return;
    ++p_phase[x];
    tc_fence_after();
    if (leader) {
      const uint64_t b = v_desc + (uint32_t)(pl * (2 * TB >> 4));
#pragma unroll
      for (int k = 0; k < kTileK / 16; ++k)
        umma_f16_ta(o_column<D>(x), p_column<D>(x) + 8 * k, b + (k * 16 * 128 >> 4), kPv, k > 0 || !first);
      umma_commit(&sh.o_done[x]);
    }
    __syncwarp();
  };
  const std::integral_constant<int, 0> t0{};
  const std::integral_constant<int, 1> t1{};
  Segment s;
  while (ok && w.next(c, sh, s)) {
    const int n = s.k1 - s.k0;
    if (n == 0) continue;
    const bool two = s.tiles == 2;
    ok = warp_wait_for(sh, &sh.q_full[live % NQ], (live / NQ) & 1, c.p.err);
    // step i issues the scores of index i + 1 and the sums of index i
#pragma unroll 1
    for (int i = -1; i < n && ok; ++i) {
      const int next = i < 0 ? place : place + 1 == NP ? 0 : place + 1;
      const uint32_t next_round = round + (i >= 0 && next == 0);
      const bool more = i + 1 < n;
      if (more) k_wait(next, next_round);
      if (i >= 0) v_wait(place, round);
      const auto tile = [&](auto X) {
        if constexpr (p_beside_s<D>()) {
          if (more) {
            if (r_phase[decltype(X)::value] > 0) read_wait(decltype(X)::value);
            qk(X, next);
          }
          if (i >= 0) pv(X, place, i == 0);
        } else {
          if (i >= 0) pv(X, place, i == 0);
          if (more) qk(X, next);
        }
      };
      tile(t0);
      if (two) tile(t1);
      place = next;
      round = next_round;
    }
    ++live;
  }
  // nothing may be in flight when tensor memory is given back
  if (leader) {
    umma_commit(&sh.drained);
    for (uint32_t i = 0; i < kPolls && !phase_done(&sh.drained, 0); ++i) {
    }
  }
  __syncwarp();
}

// ------------------------------------------------------------------ rows
// Adds to a row's sums (a part's column, or the output) the values that were
// taken out of its V tiles because they are not finite, where it sees them.
template <int DT, int D, bool FP8>
__device__ __noinline__ void add_nonfinite(const AttnCall& c, const Segment& s, int pos, float* part, uint16_t* out) {
  const int base = s.kv_len - s.q_len;
  const int p0 = base + s.row0 / c.p.G, p1 = base + min(s.q_len - 1, (s.row0 + kItemRows - 1) / c.p.G);
  for (int i = s.k0; i < s.k1; ++i) {
    const int j0 = tile_at(s.r, i) * kTileK;
    if (open_tile(c, p0, p1, j0)) continue;
#pragma unroll 1
    for (int j = j0; j <= min(pos, j0 + kTileK - 1); ++j) {
      if (c.window > 0 && j <= pos - c.window && j >= c.keep_first) continue;
      const int64_t row = cached_row(c.p, s.b, j);
      if (row < 0) continue;
      const int64_t at = row + s.head * c.p.head_stride;
#pragma unroll 1
      for (int d = 0; d < D; ++d) {
        float v;
        if constexpr (FP8)
          v = e4m3_to_f32(c.p.vc[at + d]);
        else
          v = to_f32<DT>(reinterpret_cast<const uint16_t*>(c.p.vc)[at + d]);
        if (isfinite(v)) continue;
        if (part)
          part[d * kItemRows] += v;
        else
          out[d] = from_f32<DT>(to_f32<DT>(out[d]) + v);
      }
    }
  }
}

// Both tiles' rows release what they share; a lone tile speaks for both.
__device__ __forceinline__ void release(Shared& sh, int tiles, uint64_t* bar) {
  mbar_arrive(bar);
  if (tiles == 1) mbar_arrive(bar);
}

// One row of an item from its parts, in key order.
template <int DT, int D>
__device__ __noinline__ void join_parts(const LongArgs& la, const Segment& s, int row, float sink, uint16_t* out) {
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
  for (int d = 0; d < D; d += 32) {
    float o[32] = {};
    for (int i = 0; i < s.parts; ++i) {
      const float* sl = slot(i);
      const float f = ex2(__ldcg(sl + kM) - ref);
#pragma unroll
      for (int k = 0; k < 32; ++k) o[k] = fmaf(f, __ldcg(sl + (d + k) * kItemRows), o[k]);
    }
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
      uint4 q;
      uint32_t* qw = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
      for (int e = 0; e < 4; ++e) qw[e] = pack2<DT == TSB_DT_F16>(o[k + 2 * e] * inv, o[k + 2 * e + 1] * inv);
      *reinterpret_cast<uint4*>(out + d + k) = q;
    }
  }
}

template <int DT, int D, int FEED>
__device__ void softmax_rows(const LongArgs& la, Shared& sh, Walk w, uint32_t out_smem) {
  const AttnCall& c = la.c;
  constexpr bool FP8 = FEED == kFeedWiden;
  constexpr bool kF16 = FP8 || DT == TSB_DT_F16;
  constexpr int NS = stages<D>();
  constexpr float kBias = kF16 ? 8.f : 0.f;
  const int x = threadIdx.x / kTileQ, r = threadIdx.x % kTileQ;  // tile and row
  const uint32_t lanes = (uint32_t)((threadIdx.x / 32) % 4) << 21;  // warp's first lane << 16
  const uint32_t s_at = lanes + x * kTileK, p_at = lanes + (x ? p_column<D>(1) : p_column<D>(0));
  const uint32_t o_at = lanes + (x ? o_column<D>(1) : o_column<D>(0));
  const int G = c.p.G;
  const float c0 = fmaxf(fabsf(c.scale) * 1.4426950408889634f, 1e-37f);  // positive: -infinity stays so
  uint32_t s_phase = 0, o_phase = 0,  // scores waited for, weights handed over (one product each)
       cut_parts = 0, used = 0;
  int live = 0;
  bool ok = true;
  Segment s;
  while (ok && w.next(c, sh, s)) {
    const int n = s.k1 - s.k0, R = s.row0 + x * kTileQ + r;
    const int base = s.kv_len - s.q_len;
    const int token = R < s.rows ? R / G : 0, pos = R < s.rows ? base + token : -1;
    const int q0 = c.p.cu_q[s.b];
    const bool mine = x < s.tiles;
    const float sink = c.sinks && R < s.rows ? c.sinks[s.head * G + (R - token * G)] * 1.4426950408889634f : -INFINITY;
    float m = -INFINITY, l = 0.f, cr = c0;
    if (n > 0 && mine) {
      const int first = s.row0 + x * kTileQ;
      const int p0 = base + first / G, p1 = base + min(s.q_len - 1, (first + kTileQ - 1) / G);
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int j0 = tile_at(s.r, s.k0 + i) * kTileK;
        ok = warp_wait_for(sh, &sh.s_full[x], s_phase & 1, c.p.err);
        if (!ok) break;
        ++s_phase;
        tc_fence_after();
        // S is there, so this tile is done with its K, the V before it and, last, Q
        if (r == 32) release(sh, s.tiles, &sh.kv_empty[(used + 2 * i) % NS]);
        if (r == 96 && i + 1 == n) release(sh, s.tiles, &sh.q_empty[live % q_buffers<D>()]);
        if constexpr (FP8 && DT == TSB_DT_BF16) {
          if (i == 0) cr = fmaxf(ldexpf(c0, -(int)sh.q_exp[live & 3][x * kTileQ + r]), 1e-37f);
        }
        if (!open_tile(c, p0, p1, j0)) {
          // masked in place, so that the registers below have one source
          const int hi = pos - j0, lo = c.window > 0 ? pos - c.window - j0 : -1, f = c.keep_first - j0;
#pragma unroll 1
          for (int k0 = 0; k0 < kTileK; k0 += 32) {
            uint32_t u[32];
            tmem_load_row32(s_at + k0, u);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!(k0 + k <= hi && (k0 + k > lo || k0 + k < f))) u[k] = 0xFF800000u;
            tmem_store_row32(s_at + k0, u);
          }
          tmem_st_wait();
        }
        // The row is read twice, 32 columns at a time with the next ones on their
        // way: held whole, its 128 registers leave too few to keep the
        // exponentials in flight.
        float mx[4] = {m, -INFINITY, -INFINITY, -INFINITY};
        uint32_t v[2][32];
        tmem_start_row32(s_at, v[0]);
#pragma unroll 1
        for (int h = 0; h < kTileK; h += 64) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            tmem_finish_row32(v[g]);
            if (g == 0 || h == 0) tmem_start_row32(s_at + h + 32 * (g + 1), v[1 - g]);
#pragma unroll
            for (int k = 0; k < 32; k += 2)
              mx[k / 2 % 4] = max3(mx[k / 2 % 4], __uint_as_float(v[g][k]), __uint_as_float(v[g][k + 1]));
          }
        }
        const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
        if (__any_sync(0xffffffffu, (top - m) * cr > kGrow)) {
          const float keep = m == -INFINITY ? 0.f : ex2((m - top) * cr);
          m = top;
          l *= keep;
          if (i > 0) {
            // the product before has to be in O
            ok = warp_wait_for(sh, &sh.o_done[x], (o_phase - 1) & 1, c.p.err);
            if (!ok) break;
            tc_fence_after();
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
        const uint64_t cr2 = pair(cr, cr), mc2 = pair(-mc, -mc);
        uint64_t sum[2] = {0, 0};
        // O and P of the product before: done, and its V with it
        if (i > 0) {
          ok = warp_wait_for(sh, &sh.o_done[x], (o_phase - 1) & 1, c.p.err);
          if (!ok) break;
          if (r == 64) release(sh, s.tiles, &sh.kv_empty[(used + 2 * i - 1) % NS]);
        }
        tmem_start_row32(s_at, v[0]);
#pragma unroll 1
        for (int h = 0; h < kTileK; h += 64) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t p[16];
            tmem_finish_row32(v[g]);
            if (g == 0 || h == 0) tmem_start_row32(s_at + h + 32 * (g + 1), v[1 - g]);
            if (p_beside_s<D>() && g == 1 && h > 0) {  // the scores have been read
              tc_fence_before();
              __syncwarp();
              if (r % 32 == 0) mbar_arrive(&sh.s_read[x]);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const uint64_t e = fma2(pair(__uint_as_float(v[g][2 * k]), __uint_as_float(v[g][2 * k + 1])), cr2, mc2);
              float2 w = unpair(e);
              w.x = ex2(w.x);
              w.y = ex2(w.y);
              sum[k % 2] = add2(sum[k % 2], pair(w.x, w.y));
              p[k] = pack2<kF16>(w.x, w.y);
            }
            // where P lies in S: the columns from 32 on in S have been read
            tmem_store_row16(p_at + h / 2 + 16 * g, p);
          }
        }
        ++o_phase;
        const float2 sums = unpair(add2(sum[0], sum[1]));
        l += sums.x + sums.y;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (threadIdx.x % 32 == 0) mbar_arrive(&sh.p_ready[x]);
      }
      if (!ok) break;
      ok = warp_wait_for(sh, &sh.o_done[x], (o_phase - 1) & 1, c.p.err);
      if (!ok) break;
      tc_fence_after();
      if (r == 64) release(sh, s.tiles, &sh.kv_empty[(used + 2 * n - 1) % NS]);
    }
    used += 2 * n;
    // the row's result: written, or left as one part
    const bool poisoned = n > 0 && *reinterpret_cast<volatile int*>(&sh.poison[live & 7]) == live + 1;
    const float mlog = m == -INFINITY ? -INFINITY : m * cr - kBias;  // weights are 2^(c s - mlog)
    float inv = 0.f;
    if (s.parts == 1) {
      const float all = l + (sink == -INFINITY ? 0.f : ex2(sink - (m == -INFINITY ? sink : mlog)));
      inv = all == 0.f ? 0.f : 1.f / all;
    }
    const int out_row = R < s.rows ? (q0 + token) * c.p.nq + s.head * G + (R - token * G) : -1;
    float* part = la.c.part + (int64_t)(2 * blockIdx.x + (s.part == 0 ? 1 : 0)) * la.part_stride;
    const int rr = x * kTileQ + r;
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
      uint32_t o[32];
      if (n > 0 && mine) {
        tmem_load_row32(o_at + d, o);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0;
      }
      if (s.parts > 1) {
#pragma unroll
        for (int k = 0; k < 32; ++k) part[(d + k) * kItemRows + rr] = __uint_as_float(o[k]);
      } else {
        // through shared memory, so that rows are written in whole 64-byte pieces
        const uint32_t mine_at = out_smem + (threadIdx.x / 32) * kOutStage, ln = r % 32;
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            q[e] = pack2<DT == TSB_DT_F16>(__uint_as_float(o[8 * k + 2 * e]) * inv, __uint_as_float(o[8 * k + 2 * e + 1]) * inv);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine_at + ln * 64 + ((k ^ (ln >> 1)) & 3) * 16),
                       "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                       : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = k * 8 + ln / 4, ch = ln % 4;
          const int to = __shfl_sync(0xffffffffu, out_row, row);
          uint4 q;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                       : "r"(mine_at + row * 64 + ((ch ^ (row >> 1)) & 3) * 16)
                       : "memory");
          if (to >= 0) *reinterpret_cast<uint4*>(c.out + (int64_t)to * D + d + ch * 8) = q;
        }
      }
    }
    tc_fence_before();
    __syncwarp();
    if (poisoned && pos >= 0) {
      if (s.parts > 1)
        add_nonfinite<DT, D, FP8>(c, s, pos, part + rr, nullptr);
      else
        add_nonfinite<DT, D, FP8>(c, s, pos, nullptr, c.out + (int64_t)out_row * D);
    }
    __syncwarp();
    if (n > 0) {
      // no row thread runs more than one segment ahead of another
      if (live > 0) ok = warp_wait_for(sh, &sh.seg_done, (live - 1) & 1, c.p.err);
      if (!ok) break;
      if (r % 32 == 0) mbar_arrive(&sh.seg_done);
      ++live;
    }
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
      join_parts<DT, D>(la, s, rr, sink, c.out + (int64_t)out_row * D);
    }
    __syncwarp();
  }
}

// ------------------------------------------------------------------ kernel
template <int DT, int D, int FEED>
__global__ void __launch_bounds__(kThreads, 1) paged_attn_long(const __grid_constant__ LongArgs la) {
  extern __shared__ uint8_t dyn[];
  __shared__ Shared sh;
  const AttnCall& c = la.c;
  constexpr int NS = stages<D>(), TB = tile_bytes<D>();
  const uint32_t kv_smem = (smem_u32(dyn) + 1023u) & ~1023u, q_smem = kv_smem + NS * TB;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) sh.poison[i] = 0;
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sh.q_full[x], kQWarps);
      mbar_init(&sh.q_empty[x], 2);
      mbar_init(&sh.s_full[x], 1);
      mbar_init(&sh.p_ready[x], kTileQ / 32);
      mbar_init(&sh.s_read[x], kTileQ / 32);
      mbar_init(&sh.o_done[x], 1);
    }
    mbar_init(&sh.drained, 1);
    mbar_init(&sh.part_left, 2 * kTileQ);
    mbar_init(&sh.part_said, 1);
    mbar_init(&sh.seg_done, 2 * kTileQ / 32);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh.kv_full[i], FEED == kFeedTma ? 1 : kKvWarps);
      mbar_init(&sh.kv_empty[i], 2);
      mbar_init(&sh.v_ok[i], kKvWarps);
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
  }
  if (works) {  // the same for the whole CTA
    if (warp < kWarpMma) {
      softmax_rows<DT, D, FEED>(la, sh, w, q_smem + 2 * q_buffers<D>() * TB);
    } else {
      if (warp == kWarpMma) {
        issue_products<DT, D, FEED>(c, sh, w, q_smem, kv_smem);
      } else if (warp == kWarpTma) {
        if constexpr (FEED == kFeedTma) copy_tiles<D>(la, sh, w, kv_smem, lane);
      } else if (warp < kWarpKv) {
        load_queries<DT, D, FEED == kFeedWiden>(c, sh, w, q_smem, warp - kWarpQ, lane);
      } else {
        Loader<DT, D, FEED> ld{c, sh, kv_smem, warp - kWarpKv, lane};
        ld.run(w);
      }
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

constexpr int part_floats(int d) { return (d + 2) * kItemRows; }

}  // namespace

size_t long_partial_bytes(int head_dim) { return sizeof(float) * 2 * kMaxCtas * part_floats(head_dim); }

// A map of one pool for boxes of `rows` rows of one head of one page, 64
// elements wide, in the 128-byte swizzle; false where the driver has no such
// map for these strides.
static bool pool_map(CUtensorMap* map, const TsbPagedCache& cache, void* pool, int rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  if (!encode) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)cache.head_dim, (cuuint64_t)cache.page_size, (cuuint64_t)cache.n_kv_heads,
                              (cuuint64_t)cache.num_pages};
  // a dimension of one entry may have any stride: give it a valid one
  const cuuint64_t row = 2 * (cuuint64_t)cache.head_dim;
  const cuuint64_t strides[3] = {cache.page_size > 1 ? 2 * (cuuint64_t)cache.row_stride : row,
                                 cache.n_kv_heads > 1 ? 2 * (cuuint64_t)cache.head_stride : row,
                                 cache.num_pages > 1 ? 2 * (cuuint64_t)cache.page_stride : row};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
  for (int i = 0; i < 3; ++i)
    if (strides[i] < row || strides[i] >= (1ull << 40)) return false;
  return encode(map, cache.dtype == TSB_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                pool, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int D, int FEED>
static int launch_long(LongArgs& la, const AttnCall& call, cudaStream_t st) {
  auto kern = paged_attn_long<DT, D, FEED>;
  constexpr int smem = (stages<D>() + 2 * q_buffers<D>()) * tile_bytes<D>() + 8 * kOutStage + 1024;
  static bool ready[64];  // by device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev])) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (e != cudaSuccess) return set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
  la.part_stride = part_floats(D);
  for (int b0 = 0; b0 < call.p.n_seqs; b0 += kMaxSeqs) {
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
    if (e != cudaSuccess) return set_error(TSB_ERR_CUDA, cudaGetErrorString(e));
  }
  return TSB_OK;
}

int launch_paged_long(const TsbPagedCache& cache, const AttnCall& call, cudaStream_t st) {
  LongArgs la{};
  la.c = call;
  int rc = TSB_OK;
  dispatch_paged(cache, [&](auto dt, auto d, auto fp8) {
    constexpr int DT = decltype(dt)::value, D = decltype(d)::value;
    if constexpr (decltype(fp8)::value) {
      rc = launch_long<DT, D, kFeedWiden>(la, call, st);
    } else {
      // boxes of whole groups of 8 rows: the swizzle's period
      la.box_rows = 1;
      while (la.box_rows < kTileK && cache.page_size % (2 * la.box_rows) == 0) la.box_rows *= 2;
      if (la.box_rows >= 8 && pool_map(&la.k_map, cache, cache.k_cache, la.box_rows) &&
          pool_map(&la.v_map, cache, cache.v_cache, la.box_rows))
        rc = launch_long<DT, D, kFeedTma>(la, call, st);
      else
        rc = launch_long<DT, D, kFeedCopy>(la, call, st);
    }
  });
  return rc;
}

}  // namespace tsb
