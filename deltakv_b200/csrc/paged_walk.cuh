// What the attention kernels over a paged cache share (paged_attn.cu: 16- and 32-bit pages, paged_attn8.cuh: 8-bit
// pages): the line of tokens cut into ranges, a warp's walk over its range, its stream of tiles into shared memory, and
// the joins of parts, within a CTA and by a second launch.
#pragma once

#include "dkv_common.cuh"

namespace dkv {
namespace pattn {

constexpr int kTile = 16;  // borders fall on multiples of it; a pipeline stage has 16 or 8 tokens
// Virtual tokens per sequence: what starting and finishing one costs a warp (Params::seq_cost).  16-bit walk of 256
// sequences of 1..600 tokens at 16 / 32 / 48 / 64 / 96: 38 / 34 / 31 / 34 / 39 us; of 64 of 1..8192:
// 73 / 61 / 59 / 60 / 61 us; long sequences do not notice.
constexpr int kSeqCost = 48;
// Up to so many tiles a warp, a batch runs as one launch, a CTA for each sequence and unit, of as many warps
// as let all CTAs run at once (an SM holds the warps of one CTA of the walk).  Split and joined / one launch, us,
// bf16, 8 KV heads x 128: 4 sequences of 100 / 200 / 300 tokens (1 / 2 / 2 tiles) 9.7 / 5.0, 10.2 / 6.6, 10.6 / 7.0;
// 60 of 100 / 200 / 300 (3 / 5 / 7 tiles of 3 warps) 11.8 / 8.7, 14.7 / 11.8, 16.8 / 14.7, and of 1..100 / 200 /
// 300 10.4 / 6.6, 10.6 / 9.1, 11.1 / 11.7.  The border is at 5 to 7 tiles for other head sizes and fp32 as well.
constexpr int kLocalTiles = 5;
// Tokens below which a range is not cut further (at least two tiles: the join counts on it).  Sixteen mixed
// shapes at 32 / 64 / 96: geometric mean 14.2 / 14.9 / 15.6 us.
constexpr int kMinRange = 32;
static_assert(kMinRange >= 2 * kTile, "a range inside a sequence has at least one tile");

struct Params {
  const char *q;
  int64_t q_seq, q_head;  // bytes
  char *out;
  int64_t out_seq, out_head;  // bytes
  float *lse;
  const int32_t *cu, *tables, *table_lens;
  int64_t table_stride;
  const char *k, *v;
  int64_t k_block, k_slot, k_head, v_block, v_slot, v_head;  // bytes
  int num_blocks;
  // parts: [range][unit][starts before / in the range][head of the unit][head_dim], and m, l of each
  float *part_o, *part_ml;
  int32_t *status;
  float bias;        // l and O of the parts carry 2^bias
  float scale_log2;  // scale * log2(e): scores are kept in base 2
  int n_seqs, n_kv, heads, group, chunks, units, ranges;
  int seq_cost;
  int alone;  // parts that a warp joins by itself, at most 64
  int hd, block_size;
  uint32_t div_mul, div_shift;  // i / block_size = i div_mul >> div_shift
  int local;  // not 0: a CTA of so many warps per (sequence, unit), no ranges, no parts
  int copy;   // kPlain, kRows or kPages
  int piece;  // kPlain: bytes of an asynchronous piece, 8 or 4, or 0 (element by element)
  int pairs;  // rows of q and out in whole pairs of 16-bit elements
  // 8-bit pages: the scale of a block's head
  const float *k_scale, *v_scale;
  int64_t ks_block, ks_head, vs_block, vs_head;  // elements
};

// ---------------------------------------------------------------------------------------
// the line of tokens and its ranges (at most 2^31 tokens and 2^16 sequences: 32 bits hold it)
// ---------------------------------------------------------------------------------------
struct Line {
  uint32_t total;  // virtual tokens
  uint32_t ranges; // in use
  uint32_t each, more;  // range r has each tokens, the first `more` ranges one more
  __device__ __forceinline__ uint32_t start(uint32_t r) const { return r * each + min(r, more); }
  __device__ __forceinline__ uint32_t owner(uint32_t x) const {  // the range of token x < total
    const uint32_t big = more * (each + 1);
    return x < big ? x / (each + 1) : more + (x - big) / each;
  }
};
__device__ __forceinline__ Line line_of(const Params &p, uint32_t tokens) {
  Line ln;
  ln.total = tokens + static_cast<uint32_t>(p.seq_cost) * p.n_seqs;
  ln.ranges = min(max(ln.total / kMinRange, 1u), static_cast<uint32_t>(p.ranges));
  ln.each = ln.total / ln.ranges;
  ln.more = ln.total - ln.each * ln.ranges;
  return ln;
}
// the token of sequence [at, at + len) that a range border at x falls on: a multiple of the tile
__device__ __forceinline__ int border(const Params &p, uint32_t x, uint32_t at, int len) {
  if (x <= at) return 0;
  if (x - at >= static_cast<uint32_t>(len) + p.seq_cost) return len;
  return static_cast<int>(min((x - at) & ~static_cast<uint32_t>(kTile - 1), static_cast<uint32_t>(len)));
}

// cu_seqlens and table lengths of 32 consecutive sequences in a warp's registers, so that
// walking from one sequence to the next waits for memory once in 31 sequences
//
// kEarly: for a kernel that has not waited for the one before it yet, see join_kernel; lengths only.
template <bool kEarly>
struct WindowOf {
  int base;  // lane i holds cu[base + i] and the table length of sequence base + i
  int cu, tlen;
  static __device__ __forceinline__ int cu_at(const Params &p, int b) {
    if (!kEarly) return p.cu[b];
    int v;
    asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.cu + b) : "memory");
    return v;
  }
  __device__ __forceinline__ void load(const Params &p, int b, int lane) {
    base = b;
    const int at = b + lane;
    cu = cu_at(p, min(at, p.n_seqs));
    tlen = !kEarly && p.table_lens ? p.table_lens[min(at, p.n_seqs - 1)] : 0;
  }
  __device__ __forceinline__ void need(const Params &p, int b, int lane) {
    if (b - base > 30) load(p, b, lane);
  }
  __device__ __forceinline__ int at(int b) const { return __shfl_sync(0xffffffffu, cu, b - base); }
  __device__ __forceinline__ int table_len(int b) const { return __shfl_sync(0xffffffffu, tlen, b - base); }
  // the first look of find, which does not depend on x: issued while the line's length is loaded
  __device__ __forceinline__ void look(const Params &p, int lane) {
    if (p.n_seqs > 31)
      cu = cu_at(p, min(lane * ((p.n_seqs + 31) / 32), p.n_seqs));
    else
      load(p, 0, lane);
  }
  // the largest b with cu[b] + seq_cost b <= x, and a window that starts at or before it
  __device__ __forceinline__ int find(const Params &p, uint32_t x, int lane) {
    int lo = 0, hi = p.n_seqs;
    while (hi - lo > 31) {
      const int step = (hi - lo + 31) / 32;
      const int b = lo + lane * step;
      if (lo > 0 || hi < p.n_seqs) cu = cu_at(p, min(b, p.n_seqs));
      const bool in = b < hi && static_cast<uint32_t>(cu) + static_cast<uint32_t>(p.seq_cost) * b <= x;
      const int k = __popc(__ballot_sync(0xffffffffu, in));
      if (k > 1) lo += (k - 1) * step;
      hi = min(hi, lo + step);
    }
    if (p.n_seqs > 31) load(p, lo, lane);
    const bool in = lo + lane < hi && static_cast<uint32_t>(cu) + static_cast<uint32_t>(p.seq_cost) * (lo + lane) <= x;
    return lo + max(__popc(__ballot_sync(0xffffffffu, in)) - 1, 0);
  }
};
using Window = WindowOf<false>;

// ---------------------------------------------------------------------------------------
// a warp's walk over its range: one tile of tokens after the other
// ---------------------------------------------------------------------------------------
enum { kFirst = 1, kLast = 2, kFromStart = 4, kToEnd = 8 };

struct Walk {
  Window win;
  uint32_t x0, x1;  // the range
  int b;            // sequence
  int i, end;       // tile start and end of the piece within the sequence
  int step;         // tokens from one tile to the next (more than a tile: the other warps' tiles between)
  int64_t tlen;     // valid entries of its table row
  uint32_t flags;
  bool live;
};

// zero output of a sequence without tokens
template <typename T>
__device__ __forceinline__ void write_empty(const Params &p, int b, int h0, int n_h, int lane) {
  for (int h = h0; h < h0 + n_h; ++h) {
    T *o = reinterpret_cast<T *>(p.out + b * p.out_seq + h * p.out_head);
    for (int d = lane; d < p.hd; d += 32) o[d] = T(0.f);
    if (p.lse && lane == 0) p.lse[static_cast<int64_t>(b) * p.heads + h] = __int_as_float(0xff800000);
  }
}

// moves w to the next piece of the range that has tokens, starting with sequence w.b
template <typename T>
__device__ __forceinline__ void walk_seq(const Params &p, Walk &w, int h0, int n_h, int lane) {
  w.live = false;
  for (; w.b < p.n_seqs; ++w.b) {
    w.win.need(p, w.b, lane);
    const int first = w.win.at(w.b);
    const uint32_t at = static_cast<uint32_t>(first) + static_cast<uint32_t>(p.seq_cost) * w.b;
    if (at >= w.x1) return;
    const int len = max(w.win.at(w.b + 1) - first, 0);
    const int i0 = border(p, w.x0, at, len), i1 = border(p, w.x1, at, len);
    if (i1 > i0) {
      w.i = i0, w.end = i1;
      w.flags = kFirst | (i0 == 0 ? kFromStart : 0) | (i1 == len ? kToEnd : 0);
      w.tlen = p.table_lens ? w.win.table_len(w.b) : p.table_stride;
      w.live = true;
      return;
    }
    if (len == 0 && at >= w.x0) write_empty<T>(p, w.b, h0, n_h, lane);
  }
}
template <typename T>
__device__ __forceinline__ void walk_next(const Params &p, Walk &w, int h0, int n_h, int lane) {
  w.flags &= ~kFirst;
  if (w.end - w.i > w.step) {
    w.i += w.step;
    return;
  }
  if (p.local) {
    w.live = false;
    return;
  }
  ++w.b;
  walk_seq<T>(p, w, h0, n_h, lane);
}
// the walk of range r
__device__ __forceinline__ Walk range_walk(const Params &p, const Window &win, const Line &ln, uint32_t r, int tokens,
                                           int lane) {
  Walk w;
  w.win = win;
  w.x0 = ln.start(r), w.x1 = ln.start(r + 1);
  w.b = w.win.find(p, w.x0, lane);
  w.step = tokens;
  return w;
}
// every n_warps-th tile of sequence b
__device__ __forceinline__ Walk local_walk(const Params &p, int b, int tokens, int warp, int n_warps) {
  Walk w;
  w.b = b;
  w.i = warp * tokens, w.step = n_warps * tokens;
  w.end = max(p.cu[b + 1] - p.cu[b], 0);
  w.tlen = p.table_lens ? p.table_lens[b] : p.table_stride;
  w.flags = kFirst;
  w.live = w.i < w.end;
  return w;
}

// One warp's stream of tiles into its ring of kStages shared-memory stages.  A stage holds kTok
// rows of K, then as many of V, kRow bytes apart (16 more than a row: consecutive rows start 4
// banks apart, so neither the fragment loads nor 16-byte reads of 8 rows conflict).  Three ways to
// copy:
//   kPages  block_size a multiple of the tile: a tile lies in one block, its rows a fixed stride
//           apart, and a lane's addresses are one base and an immediate or a running sum.  Each
//           lane holds the block id of another tile to come, so the table is waited for once in
//           32 tiles;
//   kRows   any block_size: the first kTok lanes look up the K rows, the next the V rows, a tile
//           ahead, and pass them on;
//   kPlain  rows that do not start or end on 16 bytes: in asynchronous pieces of 8 or 4 bytes, or
//           (16-bit rows that start on odd elements) element by element.
// A bulk copy per row (one instruction instead of 8 to 32) is slower for rows of 128 and 256 bytes:
// such copies start at about one in 14 clocks on an SM, 18 B/clock (681 us against 545 for the
// 3.5 GB of 32 long sequences).
enum { kPlain = 0, kRows = 1, kPages = 2 };

template <typename T, int HD, int kStages, int kTok>
struct Stream {
  static constexpr int kSize = static_cast<int>(sizeof(T));
  static constexpr int kRow = HD * kSize + 16;
  static constexpr int kStage = 2 * kTok * kRow;
  static constexpr int kBytes = kStages * (kStage + 16);  // the stages' descriptions behind them
  static constexpr int kPieces = HD * kSize / 16;         // 16-byte pieces of a row
  static constexpr int kRowLanes = kPieces < 32 ? kPieces : 32;
  static constexpr int kAtOnce = 32 / kRowLanes;          // rows a copy instruction covers

  const Params &p;
  Walk w;
  char *ring;
  uint4 *meta;  // per stage: sequence, flags, bit per token that takes part, end of the stream
  const char *k, *v;  // kPages: this lane's first piece of slot 0 of block 0; else its side's base
  int h0, n_h, lane;
  int id, slot;  // block and slot of this lane's row of the next tile; kPages: block of the tile
  int tile;      // kPages: of the 32 tiles that the lanes hold ids of, the next
  static constexpr int kNoRow = -1, kShort = INT32_MIN;  // negative ids in a table read as kNoRow

  __device__ __forceinline__ Stream(const Params &p_, char *mine, int u, int h0_, int n_h_, int lane_)
      : p(p_), ring(mine), meta(reinterpret_cast<uint4 *>(mine + kStages * kStage)), h0(h0_), n_h(n_h_), lane(lane_),
        id(kNoRow), slot(0), tile(0) {
    const int row = lane / kRowLanes, piece = lane % kRowLanes;
    k = p.k + u * p.k_head, v = p.v + u * p.v_head;
    if (p.copy == kPages) {
      k += row * p.k_slot + piece * 16;
      v += row * p.v_slot + piece * 16;
    }
    if (p.hd < HD) {  // columns past head_dim stay zero in every stage: nothing writes them again
      for (int i = lane; i < kStages * kStage / 16; i += 32)
        reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
  }
  __device__ __forceinline__ int block_of(int i) const {  // i / block_size for any i < 2^31
    return static_cast<int>((static_cast<uint64_t>(i) * p.div_mul) >> p.div_shift);
  }
  // (not through the read-only path: the plan before this launch may have written the table while this grid
  // was already in place)
  __device__ __forceinline__ int id_at(int blk) const {
    return blk < w.tlen ? max(p.tables[w.b * p.table_stride + blk], kNoRow) : kShort;
  }
  __device__ __forceinline__ void look_up() {
    if (!w.live) return;
    if (p.copy == kPages) {
      if (++tile < 32 && !(w.flags & kFirst)) return;
      tile = 0;
      const int ahead = lane * w.step;
      id = ahead < w.end - w.i ? id_at(block_of(w.i + ahead)) : kNoRow;
    } else {
      id = kNoRow;
      if (lane >= 2 * kTok || lane % kTok >= w.end - w.i) return;
      const int i = w.i + lane % kTok, blk = block_of(i);
      slot = i - blk * p.block_size;
      id = id_at(blk);
    }
  }
  __device__ __forceinline__ void start(const Walk &from) {
    w = from;
    if (!p.local) walk_seq<T>(p, w, h0, n_h, lane);
    look_up();
  }
  // the rows of one side of a tile in one block, `rows` of them (the others zero)
  __device__ __forceinline__ void copy_side(uint32_t dst, const char *src, int64_t slot_bytes, int rows) {
    const int64_t step = slot_bytes * kAtOnce;
#pragma unroll
    for (int r = 0; r < kTok; r += kAtOnce) {
#pragma unroll
      for (int c = 0; c < kPieces; c += 32) {
        if ((c + lane % kRowLanes) * 16 < p.hd * kSize)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + r * kRow + c * 16), "l"(src + c * 16),
                       "r"(r + lane / kRowLanes < rows ? 16 : 0)
                       : "memory");
      }
      src += step;
    }
  }
  __device__ __forceinline__ void copy_side(uint32_t dst, const char *src, int64_t slot_bytes) {  // all of them
    const int64_t step = slot_bytes * kAtOnce;
#pragma unroll
    for (int r = 0; r < kTok; r += kAtOnce) {
#pragma unroll
      for (int c = 0; c < kPieces; c += 32)
        if ((c + lane % kRowLanes) * 16 < p.hd * kSize) cp_async_16(dst + r * kRow + c * 16, src + c * 16);
      src += step;
    }
  }
  // rows whose addresses the lanes hold (0: zeros), in pieces smaller than 16 bytes
  __device__ __forceinline__ void copy_plain(char *stage, uint64_t addr) {
    const int row_bytes = p.hd * kSize;
    if (p.piece >= 4) {
      for (int row = 0; row < 2 * kTok; ++row) {
        const uint64_t a = __shfl_sync(0xffffffffu, addr, row);
        const char *src = a ? reinterpret_cast<const char *>(a) : p.k;
        for (int at = lane * p.piece; at < row_bytes; at += 32 * p.piece) {
          if (p.piece == 8)
            cp_async8(stage + row * kRow + at, src + at, a ? 8 : 0);
          else
            cp_async4(stage + row * kRow + at, src + at, a ? 4 : 0);
        }
      }
      return;
    }
    for (int d = lane; d < (p.hd + 31) / 32 * 32; d += 32) {
      for (int row = 0; row < 2 * kTok; row += 8) {  // eight rows' loads in flight
        T x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint64_t a = __shfl_sync(0xffffffffu, addr, row + r);
          x[r] = a && d < p.hd ? reinterpret_cast<const T *>(a)[d] : T(0.f);
        }
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (d < p.hd) reinterpret_cast<T *>(stage + (row + r) * kRow)[d] = x[r];
      }
    }
  }
  // issues the next tile's copies into stage s (one cp.async group, empty past the end)
  __device__ __forceinline__ void fill(int s) {
    if (w.live) {
      char *stage = ring + s * kStage;
      uint32_t there;
      if (p.copy == kPages) {
        int rows = min(w.end - w.i, kTok);
        const int block = __shfl_sync(0xffffffffu, id, tile);
        if (block < 0 || block >= p.num_blocks) {
          if (lane == 0) record_error(p.status, block == kShort ? DKV_ERR_BLOCK_TABLE_SHORT : DKV_ERR_PAGE_RANGE);
          rows = 0;
        }
        there = (1u << rows) - 1;
        const uint32_t dst = smem_u32(stage) + lane / kRowLanes * kRow + lane % kRowLanes * 16;
        const int64_t at = rows ? block : 0, in = w.i - block_of(w.i) * p.block_size;
        const char *ks = k + at * p.k_block + in * p.k_slot, *vs = v + at * p.v_block + in * p.v_slot;
        if (rows == kTok) {
          copy_side(dst, ks, p.k_slot);
          copy_side(dst + kTok * kRow, vs, p.v_slot);
        } else {
          copy_side(dst, ks, p.k_slot, rows);
          copy_side(dst + kTok * kRow, vs, p.v_slot, rows);
        }
      } else {
        const bool wanted = lane < 2 * kTok && lane % kTok < w.end - w.i;
        const bool good = wanted && id >= 0 && id < p.num_blocks;
        if (wanted && !good) record_error(p.status, id == kShort ? DKV_ERR_BLOCK_TABLE_SHORT : DKV_ERR_PAGE_RANGE);
        there = __ballot_sync(0xffffffffu, good) & ((1u << kTok) - 1);
        const char *src = lane < kTok ? k + id * p.k_block + slot * p.k_slot : v + id * p.v_block + slot * p.v_slot;
        const uint64_t addr = good ? reinterpret_cast<uint64_t>(src) : 0;
        if (p.copy == kRows) {
#pragma unroll
          for (int c = lane; c < 2 * kTok * kPieces; c += 32) {
            const int row = c / kPieces, piece = c % kPieces;
            const uint64_t a = __shfl_sync(0xffffffffu, addr, row);
            if (piece * 16 < p.hd * kSize)
              cp_async16(stage + row * kRow + piece * 16, a ? reinterpret_cast<const char *>(a) + piece * 16 : p.k,
                         a ? 16 : 0);
          }
        } else {
          copy_plain(stage, addr);
        }
      }
      const bool last = !p.local && w.end - w.i <= kTok;
      if (lane == 0) meta[s] = make_uint4(w.b, w.flags | (last ? kLast : 0), there, 0);
      walk_next<T>(p, w, h0, n_h, lane);
      look_up();
    } else if (lane == 0) {
      meta[s] = make_uint4(0, 0, 0, 1);  // the end
    }
    cp_async_commit();
  }
};

__device__ __forceinline__ float ex2(float x) {  // 2^x to 2 ulp, subnormal results 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The join within a CTA: each warp's (m, l) and O (rows of HD + 4: no bank conflicts) lie at the
// front of its ring.  Sixteen lanes a head (there are at most 16 warps) turn every warp's m into that warp's
// weight, then the threads sum the weighted O, four columns at a time.
template <int HD, int kRows>
struct LocalState {
  float o[kRows][HD + 4];
  float m[kRows], l[kRows];
};
template <int DT, int HD, int kRows>
__device__ __forceinline__ void local_join(const Params &p, char *smem, int warp_bytes, int n_warps, int b, int h0,
                                           int n_h) {
  using T = typename Elem<DT>::T;
  using State = LocalState<HD, kRows>;
  const float kNegInf = __int_as_float(0xff800000);
  auto state = [&](int w) { return reinterpret_cast<State *>(smem + w * warp_bytes); };
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int i0 = threadIdx.x - lane; i0 < n_h * 16; i0 += n_warps * 32) {  // 16 lanes a head, one a warp's part
    const int g = min((i0 + lane) / 16, n_h - 1), w = lane & 15;
    const bool mine = w < n_warps && i0 + lane < n_h * 16;
    const float m = w < n_warps ? state(w)->m[g] : kNegInf;
    float top = m;
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    const float e = ex2(m - (top == kNegInf ? 0.f : top));
    float total = w < n_warps ? state(w)->l[g] * e : 0.f;
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) total += __shfl_xor_sync(0xffffffffu, total, k);
    if (mine) state(w)->m[g] = total == 0.f ? 0.f : e / total;
    if (mine && w == 0 && p.lse)
      p.lse[static_cast<int64_t>(b) * p.heads + h0 + g] = (top + (log2f(total) - p.bias)) * 0.6931471805599453f;
  }
  __syncthreads();
  constexpr int kCols = HD / 4;
  for (int i = threadIdx.x; i < n_h * kCols; i += n_warps * 32) {
    const int g = i / kCols, d = i % kCols * 4;
    if (d >= p.hd) continue;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < n_warps; ++w) {
      const float e = state(w)->m[g];
      const float4 y = *reinterpret_cast<const float4 *>(&state(w)->o[g][d]);
      x[0] = fmaf(y.x, e, x[0]), x[1] = fmaf(y.y, e, x[1]), x[2] = fmaf(y.z, e, x[2]), x[3] = fmaf(y.w, e, x[3]);
    }
    T *dst = reinterpret_cast<T *>(p.out + b * p.out_seq + (h0 + g) * p.out_head) + d;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (d + k < p.hd) dst[k] = Elem<DT>::from_f(x[k]);
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
struct Shape {
  int hd_pad, g, warps, tokens;  // kernel variant
  int chunks, units;     // chunks of a group, KV heads x chunks
  int local;             // warps of a CTA per (sequence, unit), or 0: ranges
  int ranges;            // upper bound of the ranges in use
  int64_t parts;         // part slots
  int seq_cost;
  int sms;
  int64_t o_bytes, bytes;
};

// Warps of a CTA (one CTA an SM), stages of a warp's ring and tokens of a stage.
struct Variant {
  int warps, stages, tokens;
};

inline bool float_dtype(int dt) { return dt == DKV_F32 || dt == DKV_F16 || dt == DKV_BF16; }

inline int check_args(const dkv_paged_decode_args &a) {
  const dkv_paged_cache &k = a.k_pages, &v = a.v_pages;
  if (k.dtype != v.dtype || k.block_size != v.block_size || k.n_heads != v.n_heads || k.head_dim != v.head_dim ||
      k.block_size <= 0 || k.n_heads <= 0 || k.head_dim <= 0 || k.num_blocks < 0 || v.num_blocks < 0)
    return DKV_ERR_LAYOUT;
  if (k.head_dim > 256) return DKV_ERR_UNSUPPORTED;
  if (a.n_q_heads <= 0 || a.n_q_heads % k.n_heads || a.n_q_heads > 65535) return DKV_ERR_UNSUPPORTED;
  if (a.seqs.n_seqs < 0 || a.seqs.max_seq_len < 0) return DKV_ERR_INVALID_ARGUMENT;
  if (a.seqs.n_seqs > 65535) return DKV_ERR_UNSUPPORTED;
  return DKV_OK;
}

constexpr int kMaxRanges = 2048;

// how a batch is cut, given the kernel variant: s->hd_pad and s->g are set; least_local: fewest warps of a CTA of the one-launch form
inline int cut_up(const dkv_paged_decode_args &a, const Variant &v, int seq_cost, int least_local, Shape *s) {
  const int rc = sm_count(&s->sms);
  if (rc != DKV_OK) return rc;
  const int64_t sms = s->sms;
  const int hd = a.k_pages.head_dim, group = a.n_q_heads / a.k_pages.n_heads;
  s->warps = v.warps, s->tokens = v.tokens;
  s->chunks = (group + s->g - 1) / s->g;
  s->units = a.k_pages.n_heads * s->chunks;
  const int64_t pairs = static_cast<int64_t>(a.seqs.n_seqs) * s->units;
  s->local = s->warps;
  while (s->local > 0 && pairs > sms * (s->warps / s->local)) --s->local;
  if (s->local < least_local) s->local = 0;
  if (a.seqs.max_seq_len > static_cast<int64_t>(kLocalTiles) * s->tokens * s->local) s->local = 0;
  const int64_t most = sms * s->warps / s->units;
  const int64_t line = static_cast<int64_t>(a.seqs.n_seqs) * (static_cast<int64_t>(a.seqs.max_seq_len) + seq_cost);
  const int64_t want = line / kMinRange;
  s->ranges = static_cast<int>(s->local || most < 1 || want < 1 ? 1 : (want < most ? want : most));
  if (s->ranges > kMaxRanges) s->ranges = kMaxRanges;
  s->parts = s->ranges > 1 ? static_cast<int64_t>(s->ranges) * s->units * 2 * s->g : 0;
  s->o_bytes = (s->parts * hd * 4 + 15) / 16 * 16;
  s->bytes = s->o_bytes + s->parts * 8;
  s->seq_cost = seq_cost;
  return DKV_OK;
}

// everything but the workspace's parts and bias; sizes: bytes of an element of the pages, and of q and out
inline void fill_params(const dkv_paged_decode_args &a, const Shape &s, int64_t sz, int64_t q_sz, Params *to) {
  Params &p = *to;
  const dkv_paged_cache &k = a.k_pages, &v = a.v_pages;
  p.q = static_cast<const char *>(a.q), p.q_seq = a.q_stride_seq * q_sz, p.q_head = a.q_stride_head * q_sz;
  p.out = static_cast<char *>(a.out), p.out_seq = a.out_stride_seq * q_sz, p.out_head = a.out_stride_head * q_sz;
  p.lse = a.lse;
  p.cu = a.seqs.cu_seqlens, p.tables = a.seqs.block_tables, p.table_lens = a.seqs.table_lens;
  p.table_stride = a.seqs.table_stride;
  if (p.tables == nullptr) p.table_lens = nullptr, p.table_stride = 0;  // tables without columns
  p.k = static_cast<const char *>(k.base), p.v = static_cast<const char *>(v.base);
  p.k_block = k.stride_block * sz, p.k_slot = k.stride_slot * sz, p.k_head = k.stride_head * sz;
  p.v_block = v.stride_block * sz, p.v_slot = v.stride_slot * sz, p.v_head = v.stride_head * sz;
  const int64_t blocks = k.num_blocks < v.num_blocks ? k.num_blocks : v.num_blocks;
  p.num_blocks = static_cast<int>(blocks < INT32_MAX ? blocks : INT32_MAX);  // ids are 32-bit
  p.part_o = static_cast<float *>(a.workspace);
  p.part_ml = s.parts ? p.part_o + s.o_bytes / 4 : nullptr;
  p.status = a.status;
  p.bias = 0.f;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.n_seqs = a.seqs.n_seqs, p.n_kv = k.n_heads, p.heads = a.n_q_heads, p.group = a.n_q_heads / k.n_heads;
  p.chunks = s.chunks, p.units = s.units, p.ranges = s.ranges;
  p.seq_cost = s.seq_cost;
  p.alone = 64;
  p.local = s.local;
  p.hd = k.head_dim, p.block_size = k.block_size;
  // for i < 2^31 and 2^(s - 1) < block_size <= 2^s: mul = floor(2^(31 + s) / block_size) + 1 is off by at
  // most one part in 2^31 and fits 32 bits (division by invariant integers, Granlund and Montgomery)
  p.div_shift = 31;
  while ((1u << (p.div_shift - 31)) < static_cast<uint32_t>(k.block_size)) ++p.div_shift;
  p.div_mul = static_cast<uint32_t>((1ull << p.div_shift) / static_cast<uint32_t>(k.block_size) + 1);
  // 16-byte copies where every row of K and V starts on 16 bytes and is a multiple of 16 long
  const int64_t all = p.k_block | p.k_slot | p.k_head | p.v_block | p.v_slot | p.v_head | (p.hd * sz) |
                      static_cast<int64_t>(reinterpret_cast<uintptr_t>(k.base) | reinterpret_cast<uintptr_t>(v.base));
  // (without blocks there is no address to give to a copy of nothing)
  p.piece = blocks == 0 ? 0 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 0;
  p.copy = all % 16 || blocks == 0 ? kPlain : k.block_size % s.tokens ? kRows : kPages;
  const int64_t two = p.q_seq | p.q_head | p.out_seq | p.out_head | (p.hd * q_sz) |
                      static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out));
  p.pairs = two % 4 == 0;
  p.k_scale = p.v_scale = nullptr;
  p.ks_block = p.ks_head = p.vs_block = p.vs_head = 0;
}

// raises a kernel's shared-memory limit once per device
template <auto kKernel>
int allow_smem(int bytes) {
  static unsigned long long done = 0;  // a bit per device; a race only sets the same value twice
  int dev = 0;
  DKV_CUDA_CHECK(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (__atomic_load_n(&done, __ATOMIC_RELAXED) & bit)) return DKV_OK;
  DKV_CUDA_CHECK(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  __atomic_fetch_or(&done, bit, __ATOMIC_RELAXED);
  return DKV_OK;
}

// The second launch: joins the parts of the sequences that were cut into an output of type dt (paged_attn.cu).
int launch_join(int dt, const Params &p, const Shape &s, cudaStream_t st);

}  // namespace pattn
}  // namespace dkv
