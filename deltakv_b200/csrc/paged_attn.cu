// Attention of one new token per sequence over a paged KV cache.
//
// For sequence b, query head h of KV head u, with s_i = scale q.K_i over its tokens i:
//   m = max_i s_i,  l = sum_i exp(s_i - m),  O = sum_i exp(s_i - m) V_i,  out = O / l,  lse = m + ln l.
// (m, l, O) of two disjoint parts of the tokens join exactly: with M = max(m1, m2) each part's l
// and O are multiplied by exp(m - M) and added.  So the cache's length can be cut anywhere.
//
// Every K and V element is used for the query heads of its group, 2 to 16 of them mostly: 2 to 16
// flops a byte, far below the ridge, so the kernel is built as a stream of the pages.  Work is
// cut without regard to sequences: the tokens of all sequences are laid end to end (cu_seqlens
// is that layout), with kSeqCost virtual tokens of overhead behind those of each sequence, and the
// line is cut into equal ranges.  One warp walks one range of one KV head, so a batch of any
// raggedness keeps all warps equally busy and the host needs no lengths.  A sequence inside
// one range is finished by its warp; a sequence cut by a range border leaves (m, l, O) of its
// parts in the workspace, and a second launch joins them in the order of the ranges (the
// result does not depend on scheduling).  A batch of short sequences takes one launch instead: a CTA for
// each sequence and KV head, its warps' parts joined in shared memory.
//
// Measured on a B200 (calls back to back; HBM floor at the measured 6535 GB/s): 32 sequences of
// 20000..32768, 8 KV heads x 128, bf16: 551-591 us by the box's power (floor 529); one of 131071: 98-103 us
// (82); 64 of 1..8192: 63-65 us (46); 256 of 1..600, f16: 29.4 us (17); fp32, 16 of 4096: 98 us (82).  About
// 12 us of each are the launch, the dependent loads before the first copy, the last warps and the join; the
// rest streams at 0.93-0.97 of the peak.
#include "dkv_common.cuh"

namespace dkv {
namespace pattn {

constexpr int kTile = 16;  // borders fall on multiples of it; a pipeline stage has 16 or 8 tokens
// Virtual tokens per sequence: what starting and finishing one costs a warp.  Walk of 256 sequences
// of 1..600 tokens at 16 / 32 / 48 / 64 / 96: 38 / 34 / 31 / 34 / 39 us; of 64 of 1..8192:
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
  int hd, block_size;
  uint32_t div_mul, div_shift;  // i / block_size = i div_mul >> div_shift
  int local;  // not 0: a CTA of so many warps per (sequence, unit), no ranges, no parts
  int copy;   // kPlain, kRows or kPages
  int piece;  // kPlain: bytes of an asynchronous piece, 8 or 4, or 0 (element by element)
  int pairs;  // rows of q and out in whole pairs of 16-bit elements
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
__device__ __forceinline__ Line line_of(uint32_t tokens, int n_seqs, int most) {
  Line ln;
  ln.total = tokens + static_cast<uint32_t>(kSeqCost) * n_seqs;
  ln.ranges = min(max(ln.total / kMinRange, 1u), static_cast<uint32_t>(most));
  ln.each = ln.total / ln.ranges;
  ln.more = ln.total - ln.each * ln.ranges;
  return ln;
}
// the token of sequence [at, at + len) that a range border at x falls on: a multiple of the tile
__device__ __forceinline__ int border(uint32_t x, uint32_t at, int len) {
  if (x <= at) return 0;
  if (x - at >= static_cast<uint32_t>(len) + kSeqCost) return len;
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
  // the largest b with cu[b] + kSeqCost b <= x, and a window that starts at or before it
  __device__ __forceinline__ int find(const Params &p, uint32_t x, int lane) {
    int lo = 0, hi = p.n_seqs;
    while (hi - lo > 31) {
      const int step = (hi - lo + 31) / 32;
      const int b = lo + lane * step;
      if (lo > 0 || hi < p.n_seqs) cu = cu_at(p, min(b, p.n_seqs));
      const bool in = b < hi && static_cast<uint32_t>(cu) + static_cast<uint32_t>(kSeqCost) * b <= x;
      const int k = __popc(__ballot_sync(0xffffffffu, in));
      if (k > 1) lo += (k - 1) * step;
      hi = min(hi, lo + step);
    }
    if (p.n_seqs > 31) load(p, lo, lane);
    const bool in = lo + lane < hi && static_cast<uint32_t>(cu) + static_cast<uint32_t>(kSeqCost) * (lo + lane) <= x;
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
    const uint32_t at = static_cast<uint32_t>(first) + static_cast<uint32_t>(kSeqCost) * w.b;
    if (at >= w.x1) return;
    const int len = max(w.win.at(w.b + 1) - first, 0);
    const int i0 = border(w.x0, at, len), i1 = border(w.x1, at, len);
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
// the walk with fp32 arithmetic on the ordinary pipes
// ---------------------------------------------------------------------------------------
// fp32 pages (the tensor cores round fp32 operands).  HD: head_dim rounded up (columns past
// head_dim are zero), G: query heads of the unit (rounded up), W: warps per CTA.  Scores: lane =
// (token, half or quarter of the head); output: lane = 4 columns, the tokens dealt to 128 / HD
// groups of lanes where the head is shorter than 128.
template <int HD, int G, int W, int kStages_, int kTok>
struct Simt {
  static constexpr int kStages = kStages_;
  using S = Stream<float, HD, kStages, kTok>;
  static constexpr int kParts = 32 / kTok;              // lanes that share a token's score
  static constexpr int kQRow = (HD + 4 * kParts) * 4;  // the parts of a head 16 B apart in banks
  static constexpr int kWarpBytes = S::kBytes + G * kQRow + kTok * G * 8;
  static constexpr int kWarp = kWarpBytes;
};

template <int HD, int G, int W, int kStages, int kTok>
__global__ void __launch_bounds__(W * 32, 1) simt_kernel(const __grid_constant__ Params p) {
  using C = Simt<HD, G, W, kStages, kTok>;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  begin_overlapped();
  const int gw = p.local ? blockIdx.x : blockIdx.x * W + warp;
  const int r = gw / p.units, unit = gw - r * p.units;  // r: the range, or the sequence where local
  Line ln;
  Window win;
  if (!p.local) {
    win.look(p, lane);
    ln = line_of(p.cu[p.n_seqs], p.n_seqs, p.ranges);
    if (r >= static_cast<int>(ln.ranges)) return;
  }
  const int u = unit / p.chunks, chunk = unit - u * p.chunks;
  const int n_h = min(G, p.group - chunk * G), h0 = u * p.group + chunk * G;

  char *mine = smem + warp * C::kWarpBytes;
  float *qs = reinterpret_cast<float *>(mine + C::S::kBytes);
  uint64_t *ps = reinterpret_cast<uint64_t *>(qs + C::kQRow / 4 * G);  // [token][head]: the weight, twice
  typename C::S stream(p, mine, u, h0, n_h, lane);
  stream.start(p.local ? local_walk(p, r, kTok, warp, p.local) : range_walk(p, win, ln, r, kTok, lane));

  constexpr int kVec = HD >= 128 ? HD / 128 : 1;         // float4 columns per lane
  constexpr int kLanes = HD >= 128 ? 32 : HD / 4;        // lanes per token in the output product
  constexpr int kSplit = 32 / kLanes;                    // tokens handled at once there
  float m[G], l[G];
  uint64_t o[G][kVec][2];  // pairs of columns, for the packed fma
  const int key = lane % kTok, part = lane / kTok;
  const int oc = lane % kLanes, ok = lane / kLanes;
  auto clear = [&]() {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      m[g] = __int_as_float(0xff800000), l[g] = 0.f;
#pragma unroll
      for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[g][j][e] = 0;
    }
  };
  // sums over the lanes that share a head (l) or a column (o)
  auto reduce = [&](int g) {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], k);
#pragma unroll
    for (int j = 0; j < kVec; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = kLanes; k < 32; k <<= 1) o[g][j][i] = add2(o[g][j][i], __shfl_xor_sync(0xffffffffu, o[g][j][i], k));
  };
  auto column = [&](int g, int j, int e) {
    float x, y;
    f2unpack(o[g][j][e / 2], x, y);
    return e & 1 ? y : x;
  };
  clear();

  for (int s = 0; s < C::kStages; ++s) stream.fill(s);
  for (int s = 0;; s = s + 1 == C::kStages ? 0 : s + 1) {
    __syncwarp();
    const uint4 mt = stream.meta[s];
    if (mt.w) break;
    const int b = mt.x;
    if (mt.y & kFirst) {
      // loads in flight together (8 heads x 32 with more of them spill)
      constexpr int kLoads = G * HD / 32, kAtOnce = HD == 32 ? 4 : kLoads < 16 ? kLoads : 16;
#pragma unroll 1
      for (int k0 = 0; k0 < kLoads; k0 += kAtOnce) {
        float x[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int g = (k0 + k) * 32 / HD, d = (k0 + k) * 32 % HD + lane;
          x[k] = g < n_h && d < p.hd ? reinterpret_cast<const float *>(p.q + b * p.q_seq + (h0 + g) * p.q_head)[d] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
          const int g = (k0 + k) * 32 / HD, d = (k0 + k) * 32 % HD + lane;
          qs[g * (C::kQRow / 4) + d + d / (HD / C::kParts) * 4] = x[k];
        }
      }
      clear();
    }
    cp_async_wait<C::kStages - 1>();  // after a first tile's q is on its way
    __syncwarp();
    const float *kr = reinterpret_cast<const float *>(mine + s * C::S::kStage + key * C::S::kRow) + part * (HD / C::kParts);
    uint64_t acc[G];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g] = 0;
#pragma unroll 4
    for (int d = 0; d < HD / C::kParts; d += 4) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(kr + d);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const ulonglong2 y =
            *reinterpret_cast<const ulonglong2 *>(qs + g * (C::kQRow / 4) + part * (HD / C::kParts + 4) + d);
        acc[g] = fma2(x.y, y.y, fma2(x.x, y.x, acc[g]));
      }
    }
    const bool there = (mt.z >> key) & 1;
    float x[G];
    bool past = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float lo, hi;
      f2unpack(acc[g], lo, hi);
      lo += hi;
#pragma unroll
      for (int k = kTok; k < 32; k <<= 1) lo += __shfl_xor_sync(0xffffffffu, lo, k);
      x[g] = there ? lo * p.scale_log2 : __int_as_float(0xff800000);
      past |= x[g] > m[g];
    }
    if (__any_sync(0xffffffffu, past)) {  // as in the tensor-core walk: m moves only when it must
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float top = x[g];
#pragma unroll
        for (int k = kTok / 2; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        top = fmaxf(m[g], top);
        const float keep = ex2(m[g] - (top == __int_as_float(0xff800000) ? 0.f : top));
        m[g] = top;
        l[g] *= keep;
        const uint64_t two = f2pack(keep, keep);
#pragma unroll
        for (int j = 0; j < kVec; ++j) o[g][j][0] = mul2(o[g][j][0], two), o[g][j][1] = mul2(o[g][j][1], two);
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float e = ex2(x[g] - (m[g] == __int_as_float(0xff800000) ? 0.f : m[g]));
      if (part == 0) {
        l[g] += e;
        ps[key * G + g] = f2pack(e, e);
      }
    }
    __syncwarp();
#pragma unroll 4
    for (int t = ok; t < kTok; t += kSplit) {
      const float *vr = reinterpret_cast<const float *>(mine + s * C::S::kStage + (kTok + t) * C::S::kRow);
      uint64_t e[G];
#pragma unroll
      for (int g = 0; g < G; g += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(ps + t * G + g);
        e[g] = two.x, e[g + 1] = two.y;
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(vr + j * 128 + oc * 4);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          o[g][j][0] = fma2(e[g], y.x, o[g][j][0]);
          o[g][j][1] = fma2(e[g], y.y, o[g][j][1]);
        }
      }
    }
    if (mt.y & kLast) {
      const bool whole = (mt.y & kFromStart) && (mt.y & kToEnd);
      const int64_t slot = (static_cast<int64_t>(r) * p.units + unit) * 2 + (mt.y & kFromStart ? 1 : 0);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        reduce(g);
        const float sum = l[g];
        if (g < n_h && lane < kLanes) {
          const int h = h0 + g;
          if (whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            float *dst = reinterpret_cast<float *>(p.out + b * p.out_seq + h * p.out_head);
#pragma unroll
            for (int j = 0; j < kVec; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (j * 128 + oc * 4 + i < p.hd) dst[j * 128 + oc * 4 + i] = column(g, j, i) * inv;
            if (p.lse && lane == 0)
              p.lse[static_cast<int64_t>(b) * p.heads + h] = (m[g] + log2f(sum)) * 0.6931471805599453f;
          } else {
            float *dst = p.part_o + (slot * G + g) * p.hd;
#pragma unroll
            for (int j = 0; j < kVec; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (j * 128 + oc * 4 + i < p.hd) dst[j * 128 + oc * 4 + i] = column(g, j, i);
            if (lane == 0) {
              p.part_ml[(slot * G + g) * 2] = m[g];
              p.part_ml[(slot * G + g) * 2 + 1] = sum;
            }
          }
        }
      }
    }
    __syncwarp();
    stream.fill(s);
  }
  cp_async_wait<0>();
  if (p.local) {
    __syncwarp();
    LocalState<HD, G> *mine_out = reinterpret_cast<LocalState<HD, G> *>(mine);
    static_assert(sizeof(LocalState<HD, G>) <= C::kStages * C::S::kStage, "the state fits the ring");
#pragma unroll
    for (int g = 0; g < G; ++g) {
      reduce(g);
      if (lane < kLanes) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) mine_out->o[g][j * 128 + oc * 4 + e] = column(g, j, e);
      }
      if (lane == 0) mine_out->m[g] = m[g], mine_out->l[g] = l[g];
    }
    local_join<DKV_F32, HD, G>(p, smem, C::kWarpBytes, p.local, r, h0, n_h);
  }
}

// ---------------------------------------------------------------------------------------
// the walk with 16-bit pages on the tensor cores
// ---------------------------------------------------------------------------------------
// Transposed products, so that the query heads (few) are the narrow side n = 8 of
// mma.m16n8k16 and nothing is wasted on padding a group of 1..8 heads to 16:
//   S^T [16 tokens x 8 heads] = K [16 x 16 per step] . Q^T,  K fragments by ldmatrix,
//   O^T [16 columns x 8 heads] += V^T . P^T [16 tokens x 8 heads], V^T by ldmatrix.trans.
// P^T needs the tokens along the operand's k side where S^T has them along m: movmatrix
// transposes each 8 x 8 block in registers.  A K or V element meets 8 multiply-adds a head
// block: at the HBM rate of 12 elements a clock and SM that is 100 of the ~1000 a clock that
// mma.sync can do, so the tensor cores are far from the bound and tcgen05's 128-row tiles
// (16 times the padding, operands through tensor memory) would buy nothing.
// Weights enter the product as two 16-bit terms (value and rest: 2^-17 relative for bf16) -
// one term would add an error as large as the output's own rounding.  In f16 they are scaled by
// 2^14, which l shares, so that weights down to 2^-28 of the largest keep all their bits.
// The rest of a weight may be 0 or negative, so an infinite V element gives NaN where its weight as one
// number gives infinity: columns that end as NaN are looked through, see infinite_columns.
template <int DT>
struct Half;
template <>
struct Half<DKV_BF16> {
  static constexpr float kBias = 0.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float lo(uint32_t w) { return bf16lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return bf16hi(w); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma16816_bf16(c, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <>
struct Half<DKV_F16> {
  static constexpr float kBias = 14.f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_f16x2(a, b); }
  static __device__ __forceinline__ float lo(uint32_t w) { return f16lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return f16hi(w); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma16816(c, a[0], a[1], a[2], a[3], b0, b1);
  }
};
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <int DT, int HD, int W, int kStages_>
struct Mma {
  static constexpr int kStages = kStages_;
  using T = typename Elem<DT>::T;
  using S = Stream<T, HD, kStages, kTile>;
  static constexpr int kWarp = S::kBytes;
};

// After a piece of sequence b (tokens i0 to i1, its tiles `step` apart) left something in O that is not finite: the
// columns that are NaN though no weight is, as their V elements have them, infinite where these are infinite with
// one sign.  (Whatever the weights: they are positive.)  A lane has columns 16 k + g and 16 k + 8 + g and looks
// at every fourth token.  Rare, so it reads V again, and is given what the walk holds anyway: with values of its own
// kept for it, the walk was 1 % slower, now 0.5 %.
template <int DT, int kSteps>
__device__ __forceinline__ void infinite_columns(const Params &p, float (&o)[kSteps][4], const float (&sum)[2], int u, int b,
                                                 int i0, int i1, int step, int g, int t) {
  constexpr uint32_t kExp = DT == DKV_BF16 ? 0x7f80 : 0x7c00;
  auto of_row = [](uint32_t x) {  // over the four lanes that share columns
    x |= __shfl_xor_sync(0xffffffffu, x, 1);
    return x | __shfl_xor_sync(0xffffffffu, x, 2);
  };
  uint32_t asked = 0, up = 0, down = 0, nan = 0;  // a bit per column of the lane
#pragma unroll
  for (int c = 0; c < 2 * kSteps; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float x = o[c / 2][c % 2 * 2 + h];
      asked |= static_cast<uint32_t>(x != x && sum[h] == sum[h]) << c;
    }
  asked = of_row(asked);
  const int64_t tlen = p.table_lens ? p.table_lens[b] : p.table_stride;
  // until every column asked for is known to be NaN (i + kTile and i + step are not formed where they could pass 2^31)
  for (int i = i0; i < i1 && __any_sync(0xffffffffu, (asked & ~(nan | (up & down))) != 0); i += step) {
    const int n = min(i1 - i, kTile);
    for (int j = t; j < n; j += 4) {
      const int blk = (i + j) / p.block_size;
      const int id = blk < tlen ? p.tables[b * p.table_stride + blk] : -1;
      if (id < 0 || id >= p.num_blocks) continue;
      const unsigned short *row = reinterpret_cast<const unsigned short *>(
          p.v + u * p.v_head + id * p.v_block + (i + j - blk * p.block_size) * p.v_slot);
#pragma unroll
      for (int c = 0; c < 2 * kSteps; ++c) {
        const int d = c * 8 + g;
        const uint32_t x = d < p.hd ? row[d] : 0, size = x & 0x7fff;
        nan |= static_cast<uint32_t>(size > kExp) << c;
        up |= static_cast<uint32_t>(x == kExp) << c;
        down |= static_cast<uint32_t>(x == (kExp | 0x8000)) << c;
      }
    }
    nan = of_row(nan), up = of_row(up), down = of_row(down);
    if (i1 - i <= step) break;
  }
  up &= ~nan, down &= ~nan;
#pragma unroll
  for (int c = 0; c < 2 * kSteps; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float &x = o[c / 2][c % 2 * 2 + h];
      if (x != x && sum[h] == sum[h] && ((up ^ down) >> c & 1)) x = __int_as_float((up >> c & 1) ? 0x7f800000 : 0xff800000);
    }
}

template <int DT, int HD, int W, int kStages>
__global__ void __launch_bounds__(W * 32, 1) mma_kernel(const __grid_constant__ Params p) {
  using C = Mma<DT, HD, W, kStages>;
  using T = typename C::T;
  using E = Half<DT>;
  constexpr int kSteps = HD / 16;
  const float kNegInf = __int_as_float(0xff800000);
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  begin_overlapped();
  const int gw = p.local ? blockIdx.x : blockIdx.x * W + warp;
  const int r = gw / p.units, unit = gw - r * p.units;  // r: the range, or the sequence where local
  Line ln;
  Window win;
  if (!p.local) {
    win.look(p, lane);
    ln = line_of(p.cu[p.n_seqs], p.n_seqs, p.ranges);
    if (r >= static_cast<int>(ln.ranges)) return;
  }
  const int u = unit / p.chunks, chunk = unit - u * p.chunks;
  const int n_h = min(8, p.group - chunk * 8), h0 = u * p.group + chunk * 8;

  char *mine = smem + warp * C::S::kBytes;
  typename C::S stream(p, mine, u, h0, n_h, lane);
  stream.start(p.local ? local_walk(p, r, kTile, warp, p.local) : range_walk(p, win, ln, r, kTile, lane));

  const int g = lane >> 2, t = lane & 3;
  // ldmatrix rows: K as (token, k half), V as (token half, column half) of a 16 x 16 block
  const uint32_t k_at = smem_u32(mine) + (lane & 15) * C::S::kRow + (lane >> 4) * 16;
  const uint32_t v_at =
      smem_u32(mine) + (kTile + (lane & 7) + (lane >> 4) * 8) * C::S::kRow + ((lane >> 3) & 1) * 16;
  uint32_t qf[kSteps][2];
  float o[kSteps][4], m[2], l[2];
  auto clear = [&]() {
    m[0] = m[1] = kNegInf;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[k][e] = 0.f;
  };
  auto sum_of = [&](int c) {  // l over the lanes that share a head
    float x = l[c];
    x += __shfl_xor_sync(0xffffffffu, x, 4);
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    return x + __shfl_xor_sync(0xffffffffu, x, 16);
  };
  auto all_finite = [&]() {  // of O: 0 times anything else is NaN
    float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = fmaf(o[k][e], 0.f, z[e]);
    return __all_sync(0xffffffffu, (z[0] + z[1]) + (z[2] + z[3]) == 0.f);
  };
  clear();

  for (int s = 0; s < kStages; ++s) stream.fill(s);
  for (int s = 0;; s = s + 1 == kStages ? 0 : s + 1) {
    __syncwarp();
    const uint4 mt = stream.meta[s];
    if (mt.w) break;
    const int b = mt.x;
    if (mt.y & kFirst) {
      // (lanes past the unit's heads repeat the last one; their results are not stored)
      const unsigned short *qr =
          reinterpret_cast<const unsigned short *>(p.q + b * p.q_seq + (h0 + min(g, n_h - 1)) * p.q_head) + t * 2;
      if (p.pairs) {  // outside the loop: a branch between the loads would have each waited for
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = k * 16 + e * 8;
            qf[k][e] = d + t * 2 < p.hd ? *reinterpret_cast<const uint32_t *>(qr + d) : 0;
          }
      } else {
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = k * 16 + e * 8;
            const uint32_t lo = d + t * 2 < p.hd ? qr[d] : 0, hi = d + t * 2 + 1 < p.hd ? qr[d + 1] : 0;
            qf[k][e] = lo | hi << 16;
          }
      }
      clear();
    }
    cp_async_wait<kStages - 1>();  // after a first tile's q is on its way
    __syncwarp();
    float sc[2][4];  // two chains over the head: even and odd steps
#pragma unroll
    for (int e = 0; e < 4; ++e) sc[0][e] = sc[1][e] = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      uint32_t a[4];
      ldmatrix_x4(a[0], a[1], a[2], a[3], k_at + s * C::S::kStage + k * 32);
      E::mma(sc[k & 1], a, qf[k][0], qf[k][1]);
    }
    uint32_t ph[2], pl[2];
    // x: {token g, token g + 8} x {head 2t, head 2t + 1}
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (sc[0][e] + sc[1][e]) * p.scale_log2;
    if (mt.z != 0xffffu) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!((mt.z >> (g + (e & 2) * 4)) & 1)) x[e] = kNegInf;
    }
    // m is any value not far below the scores so far: it moves (and O with it) only when a
    // score passes it, which after the first tiles is rare
    const float top0 = fmaxf(x[0], x[2]), top1 = fmaxf(x[1], x[3]);
    if (__any_sync(0xffffffffu, top0 > m[0] || top1 > m[1])) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = c ? top1 : top0;
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        top = fmaxf(top, m[c]);
        const float keep = ex2(m[c] - (top == kNegInf ? 0.f : top));
        m[c] = top;
        l[c] *= keep;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) o[k][c] *= keep, o[k][2 + c] *= keep;
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float base = (m[c] == kNegInf ? 0.f : m[c]) - E::kBias;  // nothing seen yet: any finite base
      x[c] = ex2(x[c] - base);
      x[c + 2] = ex2(x[c + 2] - base);
      l[c] += x[c] + x[c + 2];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t w = E::pack(x[2 * c], x[2 * c + 1]);
      ph[c] = transpose8x8(w);
      pl[c] = transpose8x8(E::pack(x[2 * c] - E::lo(w), x[2 * c + 1] - E::hi(w)));
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      uint32_t a[4];
      ldmatrix_x4_trans(a[0], a[1], a[2], a[3], v_at + s * C::S::kStage + k * 32);
      E::mma(o[k], a, ph[0], ph[1]);
      E::mma(o[k], a, pl[0], pl[1]);
    }
    if (mt.y & kLast) {
      const bool whole = (mt.y & kFromStart) && (mt.y & kToEnd);
      const int64_t part = (static_cast<int64_t>(r) * p.units + unit) * 2 + (mt.y & kFromStart ? 1 : 0);
      const float sum[2] = {sum_of(0), sum_of(1)};
      if (!all_finite()) {
        const int first = p.cu[b], len = max(p.cu[b + 1] - first, 0);
        const uint32_t at = static_cast<uint32_t>(first) + static_cast<uint32_t>(kSeqCost) * b;
        infinite_columns<DT>(p, o, sum, h0 / p.group, b, border(stream.w.x0, at, len), border(stream.w.x1, at, len), kTile,
                             g, t);
      }
      if (whole) {
        // heads to rows, so that a lane stores two neighbouring columns of one head
        const float inv0 = sum[0] == 0.f ? 0.f : 1.f / sum[0], inv1 = sum[1] == 0.f ? 0.f : 1.f / sum[1];
        T *dst = reinterpret_cast<T *>(p.out + b * p.out_seq + (h0 + g) * p.out_head);
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t w = transpose8x8(E::pack(o[k][e * 2] * inv0, o[k][e * 2 + 1] * inv1));
            const int d = k * 16 + e * 8 + t * 2;
            if (g < n_h) {
              if (p.pairs) {
                if (d < p.hd) *reinterpret_cast<uint32_t *>(dst + d) = w;
              } else {
                unsigned short *two = reinterpret_cast<unsigned short *>(dst + d);
                if (d < p.hd) two[0] = static_cast<unsigned short>(w);
                if (d + 1 < p.hd) two[1] = static_cast<unsigned short>(w >> 16);
              }
            }
          }
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (p.lse && g == 0 && t * 2 + c < n_h)
            p.lse[static_cast<int64_t>(b) * p.heads + h0 + t * 2 + c] =
                (m[c] + (log2f(sum[c]) - E::kBias)) * 0.6931471805599453f;
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int in = t * 2 + c;
          if (in >= n_h) continue;
          float *dst = p.part_o + (part * 8 + in) * p.hd;
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (k * 16 + e * 8 + g < p.hd) dst[k * 16 + e * 8 + g] = o[k][e * 2 + c];
          if (g == 0) {
            p.part_ml[(part * 8 + in) * 2] = m[c];
            p.part_ml[(part * 8 + in) * 2 + 1] = sum[c];
          }
        }
      }
    }
    __syncwarp();
    stream.fill(s);
  }
  cp_async_wait<0>();
  if (p.local) {
    __syncwarp();
    LocalState<HD, 8> *mine_out = reinterpret_cast<LocalState<HD, 8> *>(mine);
    static_assert(sizeof(LocalState<HD, 8>) <= kStages * C::S::kStage, "the state fits the ring");
    const float sum[2] = {sum_of(0), sum_of(1)};
    if (!all_finite())
      infinite_columns<DT>(p, o, sum, h0 / p.group, r, warp * kTile, max(p.cu[r + 1] - p.cu[r], 0), p.local * kTile, g, t);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int in = t * 2 + c;
      if (g == 0) mine_out->m[in] = m[c], mine_out->l[in] = sum[c];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        mine_out->o[in][k * 16 + g] = o[k][c];
        mine_out->o[in][k * 16 + 8 + g] = o[k][2 + c];
      }
    }
    local_join<DT, HD, 8>(p, smem, C::S::kBytes, p.local, r, h0, n_h);
  }
}

// ---------------------------------------------------------------------------------------
// join of the parts
// ---------------------------------------------------------------------------------------
constexpr int kMaxRanges = 2048;

// A CTA has `hpc` query heads (1 or a warp each) of a cut sequence.  blockIdx.x is a sequence
// where by_seq, else a range border (at most ranges - 1 sequences are cut); gridDim.z CTAs share a
// head's columns.  Which parts there are follows from the lengths alone and is worked out before
// the walk's end is waited for.  Up to 32 parts a warp joins alone, a lane per part's weight; more are
// joined by the CTA: a thread per part's weight, then VW columns a thread, a group of threads for
// every so many-th part.  The parts' addresses are an arithmetic sequence, so that several parts'
// loads are in flight: with a test in front of each load, the 222 parts of one long sequence took
// 12 us.  (At head_dim 128 and 16 bits the walk's CTA leaves no registers, so a CTA starts where one of the
// walk has ended.)
constexpr int kJoinThreads = 128;
constexpr int kJoinWide = 256;

// acc += sum of w(i) part(i) over i = i0, i0 + by, ... < n, eight loads at a time (past the end the last
// part is loaded again and left out: a loop for the remainder would wait for each)
template <int VW, typename W>
__device__ __forceinline__ void add_parts(float (&acc)[VW], const float *src, int64_t stride, int first, int i0, int by,
                                          int n, W weight) {
  for (int i = i0; i < n; i += 8 * by) {
    float x[8][VW];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int j = min(i + k * by, n - 1);
      const float *at = src + j * stride + (j ? 0 : first);
      if constexpr (VW == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(at);
        x[k][0] = v.x, x[k][1] = v.y, x[k][2] = v.z, x[k][3] = v.w;
      } else {
        x[k][0] = *at;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float w = weight(min(i + k * by, n - 1));
      if (i + k * by < n) {
#pragma unroll
        for (int e = 0; e < VW; ++e) acc[e] = fmaf(x[k][e], w, acc[e]);
      }
    }
  }
}

template <int DT, int VW, int kThreads>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ Params p, int g_unit, int by_seq,
                                                           int hpc) {
  using T = typename Elem<DT>::T;
  extern __shared__ __align__(16) char smem[];
  float *weight = reinterpret_cast<float *>(smem), *part_l = weight + p.ranges;
  __shared__ float red[kThreads * VW];
  __shared__ float red_m[kThreads / 32], red_l[kThreads / 32];
  const float kNegInf = __int_as_float(0xff800000);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Which parts there are follows from the lengths, and these are read before the walk is waited for: this grid is
  // put in place once every CTA of the walk has said let_next_start, that is when whatever wrote the lengths
  // has ended and its results are in global memory (the walk waited for that).  What this SM's L1 holds of them
  // may be older, so they are read past it (ld.relaxed.gpu).  The parts may be read after the wait only.
  // The kernel after this one may start when this grid has ended, and many of its CTAs end early, without a
  // wait: one waits for the walk whatever it has to do, so that the grid cannot end before the walk.
  // One warp reads the lengths for its CTA.  256 sequences of 1..600: 29.4 us; each warp for itself, queued at a
  // few lines of L2, 32.7; every CTA waiting before it reads them, 32.9 (and 84 of 1..3200 17.1 against 15.7).
  using Early = WindowOf<true>;
  let_next_start();
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) wait_for_earlier();
  __shared__ int seen[4];  // cu_seqlens at n_seqs, the sequence (-1: no such border), its start and end
  if (warp == 0) {
    const int tokens = Early::cu_at(p, p.n_seqs);
    const Line ln = line_of(tokens, p.n_seqs, p.ranges);
    const uint32_t rb = blockIdx.x + 1;
    int b = blockIdx.x, first = 0, next = 0;
    if (by_seq) {
      first = Early::cu_at(p, b), next = Early::cu_at(p, b + 1);
    } else if (rb >= ln.ranges) {
      b = -1;
    } else {
      Early win;
      win.look(p, lane);
      b = win.find(p, ln.start(rb), lane);
      win.need(p, b, lane);
      first = win.at(b), next = win.at(b + 1);
      const uint32_t at = static_cast<uint32_t>(first) + static_cast<uint32_t>(kSeqCost) * b;
      if (rb > 1 && ln.start(rb - 1) >= at) b = -1;  // an earlier border has this sequence
    }
    if (lane == 0) seen[0] = tokens, seen[1] = b, seen[2] = first, seen[3] = next;
  }
  __syncthreads();
  const Line ln = line_of(seen[0], p.n_seqs, p.ranges);
  const int b = seen[1], first = seen[2], next = seen[3];
  if (b < 0) return;
  const int len = max(next - first, 0);
  if (len == 0) return;
  const uint32_t at = static_cast<uint32_t>(first) + static_cast<uint32_t>(kSeqCost) * b;
  // the ranges with a part: a range is at least two tiles wide, so only those at the ends of the
  // sequence and of its virtual tokens can have none
  // (the bound changes nothing for lengths that are prefix sums; it keeps any others within the parts)
  const uint32_t last = ln.ranges - 1;
  uint32_t r0 = min(ln.owner(at), last), r1 = min(ln.owner(at + len + kSeqCost - 1), last);
  while (r0 < r1 && border(ln.start(r0 + 1), at, len) == 0) ++r0;
  while (r0 < r1 && border(ln.start(r1), at, len) == len) --r1;
  if (r1 == r0) return;  // not cut: written by its warp
  const int n = r1 - r0 + 1;
  // part i of head h: slots as the walk numbers them, [range][unit][0, or 1 for the first part][head]
  auto part_at = [&](int h) {
    const int u = h / p.group, in = h - u * p.group;
    return ((static_cast<int64_t>(r0) * p.units + u * p.chunks + in / g_unit) * 2) * g_unit + in % g_unit;
  };
  const int64_t stride = static_cast<int64_t>(p.units) * 2 * g_unit;
  auto store = [&](int h, int c, const float (&x)[VW], float inv) {
    T *dst = reinterpret_cast<T *>(p.out + b * p.out_seq + h * p.out_head) + c * VW;
#pragma unroll
    for (int e = 0; e < VW; ++e) dst[e] = Elem<DT>::from_f(x[e] * inv);
  };
  const int share = (p.hd / VW + gridDim.z - 1) / gridDim.z, col0 = blockIdx.z * share;
  const int cols = min(p.hd / VW, col0 + share);
  const int h0 = blockIdx.y * hpc, h1 = min(h0 + hpc, p.heads);

  if (n <= 32) {
    const int h = h0 + warp;
    if (h >= h1) return;
    const int64_t part0 = part_at(h);
    wait_for_earlier();
    float m = kNegInf, l = 0.f;
    if (lane < n) {
      const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + 2 * (part0 + lane * stride + (lane ? 0 : g_unit)));
      m = ml.x, l = ml.y;
    }
    float top = m;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    const float w = exp2f(m - (top == kNegInf ? 0.f : top));
    float total = l * w;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) total += __shfl_xor_sync(0xffffffffu, total, k);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    for (int c0 = col0; c0 < cols; c0 += 32) {
      const int c = min(c0 + lane, cols - 1);  // lanes past the end repeat the last column
      float acc[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) acc[e] = 0.f;
      add_parts<VW>(acc, p.part_o + part0 * p.hd + c * VW, stride * p.hd, g_unit * p.hd, 0, 1, n,
                    [&](int i) { return __shfl_sync(0xffffffffu, w, i); });
      if (c0 + lane < cols) store(h, c, acc, inv);
    }
    if (p.lse && lane == 0 && blockIdx.z == 0)
      p.lse[static_cast<int64_t>(b) * p.heads + h] = (top + (log2f(total) - p.bias)) * 0.6931471805599453f;
    return;
  }

  wait_for_earlier();
  for (int h = h0; h < h1; ++h) {
    const int64_t part0 = part_at(h);
    float top = kNegInf;
    for (int i = tid; i < n; i += kThreads) {
      const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + 2 * (part0 + i * stride + (i ? 0 : g_unit)));
      weight[i] = ml.x, part_l[i] = ml.y;
      top = fmaxf(top, ml.x);
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    if (lane == 0) red_m[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) top = fmaxf(top, red_m[i]);
    const float base = top == kNegInf ? 0.f : top;
    float sum = 0.f;
    for (int i = tid; i < n; i += kThreads) {
      const float e = exp2f(weight[i] - base);
      weight[i] = e;
      sum = fmaf(part_l[i], e, sum);
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (lane == 0) red_l[warp] = sum;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) total += red_l[i];
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int wide = min(share, kThreads), groups = kThreads / wide;
    for (int c0 = col0; c0 < cols; c0 += wide) {  // one pass unless head_dim is odd and above 128
      const int c = min(c0 + tid % wide, cols - 1), pg = tid / wide;
      float acc[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) acc[e] = 0.f;
      if (pg < groups) {
        add_parts<VW>(acc, p.part_o + part0 * p.hd + c * VW, stride * p.hd, g_unit * p.hd, pg, groups, n,
                      [&](int i) { return weight[i]; });
      }
#pragma unroll
      for (int e = 0; e < VW; ++e) red[tid * VW + e] = acc[e];
      __syncthreads();
      // the groups' sums: every eighth of them, then the eight
      if (pg < min(groups, 8))
        for (int i = pg + 8; i < groups; i += 8)
#pragma unroll
          for (int e = 0; e < VW; ++e) acc[e] += red[(i * wide + tid % wide) * VW + e];
      if (groups > 8) {
        __syncthreads();
        if (pg < 8)
#pragma unroll
          for (int e = 0; e < VW; ++e) red[tid * VW + e] = acc[e];
        __syncthreads();
      }
      if (pg == 0 && c0 + tid < cols) {
        for (int i = 1; i < min(groups, 8); ++i)
#pragma unroll
          for (int e = 0; e < VW; ++e) acc[e] += red[(i * wide + tid) * VW + e];
        store(h, c, acc, inv);
      }
      __syncthreads();
    }
    if (p.lse && tid == 0 && blockIdx.z == 0)
      p.lse[static_cast<int64_t>(b) * p.heads + h] = (top + (log2f(total) - p.bias)) * 0.6931471805599453f;
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
  int sms;
  int64_t o_bytes, bytes;
};

// Warps of a CTA (one CTA an SM) and stages of a warp's ring: as many warps as registers and 220 KB
// allow.  More warps hide each other's latency better than more stages: at head_dim 128 and 16 bits,
// 4 x 6 / 6 x 4 / 8 x 3 / 12 x 2 (warps x stages) walk 32 long sequences in 653 / 596 / 564 / 549 us.
// fp32 walks, which do more arithmetic a byte, want whole sets of four warps (one a scheduler), and tiles
// of 8 tokens to have them at 128 columns: at 8 KV heads x 128, 64 sequences of 1..8192, 4 / 8 heads a KV
// head take 115 / 170 us with 6 / 5 warps of 16 tokens, 119 / 154 with 11 / 10 of 8, 110 / 145 with 8 of 8.
// Groups of more than 8 heads are several units, whose warps read the pages one after the other out of L2; a warp
// of 16 heads takes more registers than 12 warps leave (8 of them an SM at head_dim 128) and a kernel of its own.
// 16 sequences, 8 KV heads of 16 query heads, bf16, us, two units / 16 heads a warp (floor): 2048
// tokens x 256 77 / 98 (41), 4096 x 128 65 / 63 (41), 8192 x 64 77 / 66 (41), 8192 x 32 60 / 48 (20.5): one form, which is
// the better one at the largest heads.
struct Variant {
  int warps, stages, tokens;
};
constexpr Variant variant(bool f32, int hd, int g) {
  if (f32 && hd == 256) return {4, 2, 8};
  if (f32 && hd == 128) return {8, 2, 8};
  if (f32 && hd == 64) return g == 4 ? Variant{8, 3, 16} : Variant{10, 2, 16};
  if (f32) return {12, 3, 16};
  if (hd == 256) return {6, 2, 16};
  return hd == 128 ? Variant{12, 2, 16} : hd == 64 ? Variant{12, 4, 16} : Variant{16, 4, 16};
}

bool float_dtype(int dt) { return dt == DKV_F32 || dt == DKV_F16 || dt == DKV_BF16; }

int check(const dkv_paged_decode_args *a) {
  if (a == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  const dkv_paged_cache &k = a->k_pages, &v = a->v_pages;
  if (!float_dtype(k.dtype)) return DKV_ERR_UNSUPPORTED;
  if (k.dtype != v.dtype || k.block_size != v.block_size || k.n_heads != v.n_heads || k.head_dim != v.head_dim ||
      k.block_size <= 0 || k.n_heads <= 0 || k.head_dim <= 0 || k.num_blocks < 0 || v.num_blocks < 0)
    return DKV_ERR_LAYOUT;
  if (k.head_dim > 256) return DKV_ERR_UNSUPPORTED;
  if (a->n_q_heads <= 0 || a->n_q_heads % k.n_heads || a->n_q_heads > 65535) return DKV_ERR_UNSUPPORTED;
  if (a->seqs.n_seqs < 0 || a->seqs.max_seq_len < 0) return DKV_ERR_INVALID_ARGUMENT;
  if (a->seqs.n_seqs > 65535) return DKV_ERR_UNSUPPORTED;
  return DKV_OK;
}

int shape_of(const dkv_paged_decode_args *a, Shape *s) {
  const int rc = sm_count(&s->sms);
  if (rc != DKV_OK) return rc;
  const int64_t sms = s->sms;
  const int hd = a->k_pages.head_dim, group = a->n_q_heads / a->k_pages.n_heads;
  s->hd_pad = hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
  const bool f32 = a->k_pages.dtype == DKV_F32;
  s->g = f32 && group <= 4 ? 4 : 8;
  const Variant v = variant(f32, s->hd_pad, s->g);
  s->warps = v.warps, s->tokens = v.tokens;
  s->chunks = (group + s->g - 1) / s->g;
  s->units = a->k_pages.n_heads * s->chunks;
  const int64_t pairs = static_cast<int64_t>(a->seqs.n_seqs) * s->units;
  s->local = s->warps;
  while (s->local > 0 && pairs > sms * (s->warps / s->local)) --s->local;
  if (a->seqs.max_seq_len > static_cast<int64_t>(kLocalTiles) * s->tokens * s->local) s->local = 0;
  const int64_t most = sms * s->warps / s->units;
  const int64_t line = static_cast<int64_t>(a->seqs.n_seqs) * (static_cast<int64_t>(a->seqs.max_seq_len) + kSeqCost);
  const int64_t want = line / kMinRange;
  s->ranges = static_cast<int>(s->local || most < 1 || want < 1 ? 1 : (want < most ? want : most));
  if (s->ranges > kMaxRanges) s->ranges = kMaxRanges;
  s->parts = s->ranges > 1 ? static_cast<int64_t>(s->ranges) * s->units * 2 * s->g : 0;
  s->o_bytes = (s->parts * hd * 4 + 15) / 16 * 16;
  s->bytes = s->o_bytes + s->parts * 8;
  return DKV_OK;
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

template <int HD, int G, int W, int kStages, int kTok>
int launch_simt(const Params &p, int grid, cudaStream_t st) {
  using C = Simt<HD, G, W, kStages, kTok>;
  static_assert(W * C::kWarp <= 227 * 1024, "shared memory of the walk");
  const int rc = allow_smem<simt_kernel<HD, G, W, kStages, kTok>>(W * C::kWarp);
  if (rc != DKV_OK) return rc;
  const int warps = p.local ? p.local : W;
  DKV_CUDA_CHECK(launch_overlapped(simt_kernel<HD, G, W, kStages, kTok>, dim3(grid), warps * 32, warps * C::kWarp, st, p));
  return DKV_OK;
}

template <int DT, int HD, int W, int kStages>
int launch_mma(const Params &p, int grid, cudaStream_t st) {
  using C = Mma<DT, HD, W, kStages>;
  static_assert(W * C::kWarp <= 227 * 1024, "shared memory of the walk");
  const int rc = allow_smem<mma_kernel<DT, HD, W, kStages>>(W * C::kWarp);
  if (rc != DKV_OK) return rc;
  const int warps = p.local ? p.local : W;
  DKV_CUDA_CHECK(launch_overlapped(mma_kernel<DT, HD, W, kStages>, dim3(grid), warps * 32, warps * C::kWarp, st, p));
  return DKV_OK;
}

#define DKV_WALK_CASE(HD, G)        \
  if (s.hd_pad == HD && s.g == G) { \
    constexpr Variant v = variant(kF32, HD, G); \
    DKV_WALK_LAUNCH(HD, G, v)       \
  }
template <int DT>
int launch_walk(const Params &p, const Shape &s, int grid, cudaStream_t st) {
  constexpr bool kF32 = DT == DKV_F32;
  if constexpr (kF32) {
#define DKV_WALK_LAUNCH(HD, G, v) return launch_simt<HD, G, v.warps, v.stages, v.tokens>(p, grid, st);
    DKV_WALK_CASE(32, 4)
    DKV_WALK_CASE(32, 8)
    DKV_WALK_CASE(64, 4)
    DKV_WALK_CASE(64, 8)
    DKV_WALK_CASE(128, 4)
    DKV_WALK_CASE(128, 8)
    DKV_WALK_CASE(256, 4)
    DKV_WALK_CASE(256, 8)
#undef DKV_WALK_LAUNCH
  } else {
#define DKV_WALK_LAUNCH(HD, G, v) return launch_mma<DT, HD, v.warps, v.stages>(p, grid, st);
    DKV_WALK_CASE(32, 8)
    DKV_WALK_CASE(64, 8)
    DKV_WALK_CASE(128, 8)
    DKV_WALK_CASE(256, 8)
#undef DKV_WALK_LAUNCH
  }
#undef DKV_WALK_CASE
  return DKV_ERR_UNSUPPORTED;
}

template <int DT>
int launch(const Params &p, const Shape &s, cudaStream_t st) {
  const int64_t warps = static_cast<int64_t>(s.ranges) * s.units;
  const int64_t ctas = s.local ? static_cast<int64_t>(p.n_seqs) * s.units : (warps + s.warps - 1) / s.warps;
  const int rc = launch_walk<DT>(p, s, static_cast<int>(ctas), st);
  if (rc != DKV_OK || s.ranges == 1) return rc;
  const int by_seq = p.n_seqs <= s.ranges - 1;
  const int cut = by_seq ? p.n_seqs : s.ranges - 1;
  // A CTA for each head, or a warp where more CTAs than run at once would come of it (CTA / warp, us, bf16: 9
  // sequences of 30000 x 16 heads x 64 38.2 / 42.5, 20 of 3000 x 32 heads x 128 51.5 / 52.4; at the border, 36 of
  // 2000 x 32 heads 61.3 / 60.6, 74 of 1..6000 x 16 heads 111.7 / 113.1; 74 of 1000 x 32 heads 65.1 / 62.1)
  const int64_t heads = static_cast<int64_t>(cut) * p.heads;  // to join at most
  const int hpc = heads <= s.sms * 8 ? 1 : kJoinThreads / 32;
  // Few heads: several CTAs for each, as long as an SM has one of them (1 / 2 / 4 CTAs a head, us, bf16: one sequence
  // of 4000 x 32 heads x 128 15.8 / 14.0 / 13.0, of 30000 x 8 heads x 32 14.6 / 12.8 / 12.5, 6 of 6000 x 8 x 256 24.9 /
  // 23.6 / 22.6; 12 of 8000 x 8 x 64 18.1 / 18.0 / 21.4, 4 of 8000 x 32 x 128 33.0 / 33.0 / 36.5; 5 of them 38.5 / 41.6
  // / 45.0)
  const int split = p.hd < 32 ? 1 : heads <= s.sms / 2 ? 4 : heads <= s.sms ? 2 : 1;
  const dim3 grid(cut, (p.heads + hpc - 1) / hpc, split);
  // heads of which some may have more parts than a CTA has threads: more threads (one sequence of 131071, 8 KV heads:
  // 99.5 -> 97.5 us; three of up to 13687, 2 KV heads: 17.4 -> 14.8; 5 of 15930, 40 heads: 54 -> 52), which cost time
  // where there are fewer parts (one of 47238, 16 KV heads of 7 query heads each, 111 ranges: 72.9 -> 75.5) and
  // where not all CTAs run at once (62 of 6119, 6 heads: 72.8 -> 74.3; 84 of 1..3200, 12 heads: 11.6 -> 15.5)
  const bool wide = heads <= s.sms * 2 && s.ranges > kJoinThreads;
  const auto kernel = wide ? (p.hd % 4 == 0 ? join_kernel<DT, 4, kJoinWide> : join_kernel<DT, 1, kJoinWide>)
                           : (p.hd % 4 == 0 ? join_kernel<DT, 4, kJoinThreads> : join_kernel<DT, 1, kJoinThreads>);
  DKV_CUDA_CHECK(launch_overlapped(kernel, grid, wide ? kJoinWide : kJoinThreads, s.ranges * 8, st, p, s.g, by_seq, hpc));
  return DKV_OK;
}

}  // namespace pattn
}  // namespace dkv

using namespace dkv;

extern "C" int dkv_paged_decode_workspace_bytes(const dkv_paged_decode_args *args, int64_t *bytes) {
  if (bytes == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  const int rc = pattn::check(args);
  if (rc != DKV_OK) return rc;
  pattn::Shape s;
  const int rs = pattn::shape_of(args, &s);
  if (rs != DKV_OK) return rs;
  *bytes = s.bytes;
  return DKV_OK;
}

extern "C" int dkv_paged_decode_attention(const dkv_paged_decode_args *args, dkv_stream_t stream) {
  const int rc = pattn::check(args);
  if (rc != DKV_OK) return rc;
  const dkv_paged_decode_args &a = *args;
  const dkv_paged_cache &k = a.k_pages, &v = a.v_pages;
  if (a.seqs.n_seqs == 0) return DKV_OK;
  if (a.q == nullptr || a.out == nullptr || a.seqs.cu_seqlens == nullptr)
    return DKV_ERR_INVALID_ARGUMENT;
  if ((k.base == nullptr && k.num_blocks > 0) || (v.base == nullptr && v.num_blocks > 0)) return DKV_ERR_INVALID_ARGUMENT;
  pattn::Shape s;
  const int rs = pattn::shape_of(args, &s);
  if (rs != DKV_OK) return rs;
  if (s.bytes > 0 && (a.workspace == nullptr || a.workspace_bytes < s.bytes)) return DKV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16) return DKV_ERR_ALIGNMENT;
  const int64_t sz = k.dtype == DKV_F32 ? 4 : 2;
  pattn::Params p;
  p.q = static_cast<const char *>(a.q), p.q_seq = a.q_stride_seq * sz, p.q_head = a.q_stride_head * sz;
  p.out = static_cast<char *>(a.out), p.out_seq = a.out_stride_seq * sz, p.out_head = a.out_stride_head * sz;
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
  p.bias = k.dtype == DKV_F16 ? pattn::Half<DKV_F16>::kBias : 0.f;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.n_seqs = a.seqs.n_seqs, p.n_kv = k.n_heads, p.heads = a.n_q_heads, p.group = a.n_q_heads / k.n_heads;
  p.chunks = s.chunks, p.units = s.units, p.ranges = s.ranges;
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
  p.copy = all % 16 || blocks == 0 ? pattn::kPlain : k.block_size % s.tokens ? pattn::kRows : pattn::kPages;
  const int64_t two = p.q_seq | p.q_head | p.out_seq | p.out_head | (p.hd * sz) |
                      static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out));
  p.pairs = two % 4 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (k.dtype) {
    case DKV_F32: return pattn::launch<DKV_F32>(p, s, st);
    case DKV_F16: return pattn::launch<DKV_F16>(p, s, st);
    default: return pattn::launch<DKV_BF16>(p, s, st);
  }
}
