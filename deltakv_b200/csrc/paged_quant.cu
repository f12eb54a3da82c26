// The 8-bit paged cache: K and V quantised as they are stored, read back, and patched in place.
//   dkv_append_paged_quant   RoPE of the new q and k rows, K and V quantised into their slots
//   dkv_scatter_paged_quant  value + delta for the rows of every sequence, quantised again
//   dkv_gather_paged_quant   the values of every sequence's rows
//   dkv_append_paged_quant_check, dkv_scatter_paged_quant_check   whether a call would write a block in two places
// The layouts and the page arithmetic are those of the paged scatter / gather (src/deltakv/paged.py:8-70).
#include "code8.cuh"
#include "paged_rows.cuh"

namespace dkv {
namespace quant {

using code8::Code;
using step::Append;
using step::Columns;
using step::Raw;
using step::Rotary;

// What a store writes of K or V.  Strides in bytes (pages), elements (source, scales).
struct Side {
  const void *src;
  int64_t src_row, src_head;
  uint8_t *pages;
  int64_t block, slot, head;
  float *scale;
  int64_t scale_block, scale_head;
};

// Rows of one call.  A run is the rows that follow one another in one block.  A CTA looks through a window of rows for
// the runs that begin there; each of its warps takes the K or V of a run's head, and with it alone the head's scale in that
// block.  (grid: the chunks of heads and sides of a window are neighbours.)
struct Store {
  Side side[2];
  int64_t n_rows, n_blocks, n_slots;
  const int64_t *slots;  // append
  const int32_t *positions;
  const float *cos_t, *sin_t;
  int rope_max_pos;
  dkv_seq_batch seqs;  // patch
  int32_t *status;
  int heads, hd, block_size;
  Rotary rot;
  int window;   // rows that a CTA looks through for the first ones of runs
  int narrow;   // the cache's slots fit 32 bits
  int pairs;    // heads times sides
  int chunks;   // CTAs of a window, with `each` pairs
  int each;
  int64_t ctas; // of the store
  uint32_t spread;  // every so many-th CTA is one of them, the others are q's
  int watchers;     // the launch's first CTAs, which look for blocks of two runs
  int places;       // of a watcher's table, a power of two
  int64_t segment, segments;  // the rows that a watcher takes at once, and how many of them there are
};

constexpr int kThreads = 128;
constexpr int kStaged = 4;  // pieces of two times VEC columns of a lane that wait in shared memory
// Pieces that a lane reads at once, and CTAs of an SM (which leave a thread 96 or 128 registers).  us: 16384 rows of 32 + 8 + 8
// heads x 128, bf16, appended: 1 piece, 5 CTAs 92.5; 1, 6 103 (spilled); 2, 5 95; 2, 4 96; 4, 4 100.  8192 such rows of fp32: 2, 4 68;
// 1, 5 75; 2, 5 83.  73000 rows of 8 x 128 patched, bf16: 4, 4 75; 2, 5 79; fp32: 2, 5 94; 4, 4 99 to 107.
constexpr int items_of(bool patch, int sdt) { return patch ? (sdt == DKV_F32 ? 2 : 4) : (sdt == DKV_F32 ? 2 : 1); }
constexpr int resident_of(bool patch, int sdt) { return patch == (sdt == DKV_F32) ? 5 : 4; }

// The largest magnitude of several values, and whether all are finite (0 times anything else is NaN).
struct Largest {
  float top = 0.f;
  uint64_t zero = 0;
  __device__ __forceinline__ void add(uint64_t pair) {
    float x, y;
    f2unpack(pair, x, y);
    top = fmaxf(fmaxf(top, fabsf(x)), fabsf(y));
    zero = fma2(pair, 0ull, zero);
  }
  __device__ __forceinline__ uint32_t bits() const {  // of the magnitude; not finite: above all finite ones
    float x, y;
    f2unpack(zero, x, y);
    return x + y == 0.f ? __float_as_uint(top) : 0x7fffffffu;
  }
};
// pieces of 8 columns are always two
template <int VEC>
__device__ __forceinline__ bool paired(const Columns &at) {
  return VEC > 1 || at.pair;
}
// strides that pieces of 8 columns take are below 2^31 (the host checks)
template <int VEC>
__device__ __forceinline__ int64_t times(int n, int64_t stride) {
  return VEC > 1 ? static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * static_cast<uint32_t>(stride))
                 : n * stride;
}

// block of a row's slot, -1 for none
__device__ __forceinline__ int64_t row_block(const Store &s, int64_t row) {
  const int64_t slot = s.slots[row];
  if (slot < 0 || slot >= s.n_slots) return -1;
  return s.narrow ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(s.block_size) : slot / s.block_size;
}
__device__ __forceinline__ int slot_in(const Store &s, int64_t row, int64_t block) {
  return static_cast<int>(s.slots[row] - block * s.block_size);
}

// whether the tables have a row's position
__device__ __forceinline__ bool turns(const Store &s, int pos) { return pos >= 0 && pos < s.rope_max_pos; }

// ---------------------------------------------------------------------------------------
// blocks of two runs
// ---------------------------------------------------------------------------------------
// Two runs of one block in a call would be two warps that choose its scale and round its codes again at the same time: what
// the block holds then is anything.  (Every run would have to know all others before it stores, so a launch before this
// one: 2 us of a decode step's 5.5.)  So the launch's first CTAs watch, beside the store's.  The rows are cut into segments; a watcher
// has two of them (or one, with itself), puts the blocks of the first one's runs into a table in shared memory and looks up the
// second one's: every pair of runs is some watcher's.  us without / with them: 16384 rows of 32 + 8 + 8 heads x 128 92.4 / 93.1, of one
// KV head x 64 11.4 / 11.9 (32 with four watchers, each for a quarter of the blocks and all rows), 4096 single rows 28.5 / 29.2, 73000 rows
// of 8 x 128 patched 75.2 / 75.5; 100000 rows of 4 + 1 + 1 x 128, 25 segments, 103 / 113.  16 segments instead of eight cost another 1 us.
constexpr int kMostPlaces = 8192;
constexpr int kQueue = 64;  // blocks of a warp that wait to be looked up, 32 at once
struct Watch {
  uint32_t *table;  // block + 1, 0: free
  uint32_t *queue;  // of the warp
  uint32_t places, seen = 0, queued = 0;
  int lane;
  bool adds = true, twice = false;
  // all threads of the CTA
  __device__ __forceinline__ Watch(uint32_t *memory, int places_)
      : table(memory), queue(memory + places_ + (threadIdx.x >> 5) * kQueue), places(places_), lane(threadIdx.x & 31) {
    for (uint32_t i = threadIdx.x; i < places; i += kThreads) table[i] = 0;
    __syncthreads();
  }
  // (multiplicative hashing, Knuth: the top bits of the product with an odd number near 2^32 / phi)
  __device__ __forceinline__ void look_up(uint32_t block) {
    uint32_t at = __umulhi(block * 0x9e3779b1u, places);
    for (uint32_t i = 0; i < places; ++i, at = (at + 1) & (places - 1)) {
      const uint32_t was = adds ? atomicCAS(table + at, 0u, block + 1) : table[at];
      twice |= was == block + 1;
      if (was == 0 || was == block + 1) return;
    }
  }
  // a warp's blocks, where `there`
  __device__ __forceinline__ void see(uint32_t block, bool there) {
    const uint32_t who = __ballot_sync(0xffffffffu, there);
    if (there) queue[(queued + __popc(who & ((1u << lane) - 1))) % kQueue] = block;
    queued += __popc(who);
    __syncwarp();
    if (queued - seen < 32) return;
    look_up(queue[(seen + lane) % kQueue]);
    seen += 32;
    __syncwarp();
  }
  __device__ __forceinline__ void rest() {
    if (lane < queued - seen) look_up(queue[(seen + lane) % kQueue]);
    seen = queued;
    __syncwarp();
  }
};

// Rows [from, to) of an append: a run begins where a row's block is not the one of the row before.
__device__ __forceinline__ void watch_rows(const Store &s, Watch &w, int64_t from, int64_t to) {
  constexpr int kAtOnce = 4;
  constexpr uint32_t kNone = 0xffffffffu;
  const int64_t *slots = s.slots;
  const uint64_t n_slots = s.n_slots;
  const uint32_t size = s.block_size, inverse = 0xffffffffu / size;
  const bool narrow = s.narrow;
  const auto block_of = [&](int64_t slot) -> uint32_t {
    if (static_cast<uint64_t>(slot) >= n_slots) return kNone;
    if (!narrow) return static_cast<uint32_t>(slot / size);
    const uint32_t x = static_cast<uint32_t>(slot), q = __umulhi(x, inverse);  // x / size, or one less: inverse is 2^32 / size less at most 1
    return q + (x - q * size >= size);
  };
  for (int64_t row0 = from + (threadIdx.x & ~31u) * kAtOnce; row0 < to; row0 += kThreads * kAtOnce) {
    int64_t slot[kAtOnce];  // all loads first
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) slot[k] = slots[min(row0 + k * 32 + w.lane, to - 1)];
    const int64_t before = slots[max(row0 - 1, static_cast<int64_t>(0))];
    uint32_t last = row0 > 0 ? block_of(before) : kNone;  // of the row before a warp's 32
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const uint32_t block = row0 + k * 32 + w.lane < to ? block_of(slot[k]) : kNone;
      const uint32_t up = __shfl_up_sync(0xffffffffu, block, 1);
      w.see(block, block != kNone && block != (w.lane == 0 ? last : up));
      last = __shfl_sync(0xffffffffu, block, 31);
    }
  }
}

// The blocks of a patch that begin in rows [from, to): a warp takes 32 sequences and their blocks one after the other, 128 at once.
__device__ __forceinline__ void watch_blocks(const Store &s, Watch &w, int64_t from, int64_t to) {
  constexpr int kAtOnce = 4;
  const dkv_seq_batch &q = s.seqs;
  const int32_t *cu = q.cu_seqlens, *tables = q.block_tables;
  const int64_t n_blocks = s.n_blocks, stride = q.table_stride, size = s.block_size, zero = 0;
  int first = 0, end = q.n_seqs;  // the last sequence that begins at `from` or before it is in [first, end)
  while (end - first > 1) {
    const int step = (end - first + 31) / 32, b = first + w.lane * step;
    const int k = __popc(__ballot_sync(0xffffffffu, b < end && cu[min(b, end - 1)] <= from));
    first += max(k - 1, 0) * step;
    end = min(end, first + step);
  }
  for (int b0 = first + static_cast<int>(threadIdx.x & ~31u); b0 < q.n_seqs; b0 += kThreads) {
    const int b = b0 + w.lane;
    int begin = 0, mine = 0;  // this lane's sequence's first block here, and how many of them the table has
    bool beyond = false;
    if (b < q.n_seqs) {
      const int64_t start = cu[b], stop = min(static_cast<int64_t>(cu[b + 1]), to);
      const int64_t tlen = q.table_lens ? q.table_lens[b] : stride;
      beyond = start >= to;
      if (start >= 0 && stop > start) {
        const int64_t one = max(from - start + size - 1, zero) / size, n = min((stop - start + size - 1) / size, tlen) - one;
        begin = static_cast<int>(one);
        mine = static_cast<int>(max(min(n, static_cast<int64_t>(1 << 25)), zero));  // (32 of them fit an int)
      }
    }
    int upto = mine;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, k);
      if (w.lane >= k) upto += y;
    }
    const int all = __shfl_sync(0xffffffffu, upto, 31);
    for (int i0 = 0; i0 < all; i0 += 32 * kAtOnce) {
      int32_t id[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int i = min(i0 + j * 32 + w.lane, all - 1);
        int l = 0;  // the sequence of block i: as many lanes have no more than i blocks up to theirs
#pragma unroll
        for (int k = 16; k > 0; k >>= 1)
          if (__shfl_sync(0xffffffffu, upto, l + k - 1) <= i) l += k;
        const int blk = i + __shfl_sync(0xffffffffu, begin - (upto - mine), l);
        id[j] = tables[static_cast<int64_t>(b0 + l) * stride + blk];
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        w.see(id[j], i0 + j * 32 + w.lane < all && id[j] >= 0 && id[j] < n_blocks);
    }
    if (__any_sync(0xffffffffu, beyond)) break;
  }
}

// one watcher (not part of the kernels' own code, whose registers it would cost)
template <bool kPatch>
__device__ __noinline__ void watch_runs(const Store &s, uint32_t *memory) {
  int64_t one = 0, two = blockIdx.x;  // its segments: the pairs one <= two in order
  for (int64_t more = s.segments; two >= more; --more) two -= more, ++one;
  two += one;
  Watch w(memory, s.places);
  const auto go = [&](int64_t i) {
    const int64_t from = i * s.segment, to = min(from + s.segment, s.n_rows);
    if (kPatch) watch_blocks(s, w, from, to); else watch_rows(s, w, from, to);
    w.rest();
  };
  go(one);
  if (two != one) {
    __syncthreads();
    w.adds = false;
    go(two);
  }
  if (w.twice) record_error(s.status, DKV_ERR_BLOCK_TWICE);
}
// the watchers alone
template <bool kPatch>
__global__ void __launch_bounds__(kThreads) watch_kernel(const __grid_constant__ Store s) {
  __shared__ uint32_t memory[kMostPlaces + kThreads / 32 * kQueue];
  begin_overlapped();
  watch_runs<kPatch>(s, memory);
}

// VEC values in pairs, as the packed fp32 operations of sm_100 take them; one value has a zero beside it.  (Where a product
// and a sum are rounded one after the other the single operations are used: packed ones are merged into one.)
template <int VEC>
struct Values {
  static constexpr int kPairs = VEC == 1 ? 1 : VEC / 2;
  uint64_t pair[kPairs];
};

// codes of VEC consecutive columns
template <int VEC>
struct Codes {
  uint32_t w[VEC / 4];
  __device__ __forceinline__ void load(const uint8_t *src) {
    const uint2 x = *reinterpret_cast<const uint2 *>(src);
    w[0] = x.x, w[1] = x.y;
  }
  __device__ __forceinline__ void store(uint8_t *dst) const { *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]); }
  template <int PT>
  __device__ __forceinline__ Values<VEC> get() const {
    Values<VEC> v;
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      float y[4];
      Code<PT>::unpack(w[i], y);
      v.pair[2 * i] = f2pack(y[0], y[1]), v.pair[2 * i + 1] = f2pack(y[2], y[3]);
    }
    return v;
  }
  template <int PT>
  __device__ __forceinline__ void set(const Values<VEC> &v, float by) {
    const uint64_t two = f2pack(by, by);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      float y[4];
      f2unpack(mul2(v.pair[2 * i], two), y[0], y[1]);
      f2unpack(mul2(v.pair[2 * i + 1], two), y[2], y[3]);
      w[i] = Code<PT>::pack(y[0], y[1], y[2], y[3]);
    }
  }
};
template <>
struct Codes<1> {
  uint32_t w;
  __device__ __forceinline__ void load(const uint8_t *src) { w = *src; }
  __device__ __forceinline__ void store(uint8_t *dst) const { *dst = static_cast<uint8_t>(w); }
  template <int PT>
  __device__ __forceinline__ Values<1> get() const {
    float y[4];
    Code<PT>::unpack(w, y);
    return {{f2pack(y[0], 0.f)}};
  }
  template <int PT>
  __device__ __forceinline__ void set(const Values<1> &v, float by) {
    float x, y;
    f2unpack(v.pair[0], x, y);
    w = Code<PT>::pack(__fmul_rn(x, by), 0.f, 0.f, 0.f);
  }
};
static_assert(sizeof(Codes<8>) == 8, "eight columns are one load");

// What stays of a block whose head's scale moves from held to scale, by the lanes of a warp.  mine: bit i of lane l says
// that slot 32 l + i is being stored.
template <int PDT, int VEC>
__device__ __forceinline__ void scale_again(const Store &s, const Side &side, uint8_t *pages, float held, float by, uint32_t mine,
                                            int lane) {
  constexpr int kAtOnce = 4;
  const int units = (s.hd + VEC - 1) / VEC, all = s.block_size * units;
  for (int i0 = 0; i0 < all; i0 += 32 * kAtOnce) {
    Codes<VEC> c[kAtOnce];
    int o[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = i0 + k * 32 + lane;
      const int u = min(i, all - 1) / units;
      const bool stored = __shfl_sync(0xffffffffu, mine, u >> 5) >> (u & 31) & 1;
      o[k] = i < all && !stored ? u : -1;
      if (o[k] >= 0) c[k].load(pages + times<VEC>(u, side.slot) + (i - u * units) * VEC);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (o[k] < 0) continue;
      Values<VEC> v = c[k].template get<PDT>();
#pragma unroll
      for (int e = 0; e < Values<VEC>::kPairs; ++e) v.pair[e] = mul2(v.pair[e], f2pack(held, held));
      c[k].template set<PDT>(v, by);
      c[k].store(pages + times<VEC>(o[k], side.slot) + (i0 + k * 32 + lane - o[k] * units) * VEC);
    }
  }
}

// a pair of columns turned; the columns of two pairs that lie in lo and hi
__device__ __forceinline__ uint64_t turned(uint64_t pair, float c, float s) {
  float x, y;
  f2unpack(pair, x, y);
  step::turn_pair(x, y, c, s);
  return f2pack(x, y);
}
__device__ __forceinline__ void turn_two(uint64_t &lo, uint64_t &hi, float c0, float c1, float s0, float s1) {
  float x0, x1, y0, y1;
  f2unpack(lo, x0, x1), f2unpack(hi, y0, y1);
  step::turn_pair(x0, y0, c0, s0), step::turn_pair(x1, y1, c1, s1);
  lo = f2pack(x0, x1), hi = f2pack(y0, y1);
}

// The runs that begin in a CTA's window, as its first warp finds them: a bit for each row where one begins, and for these
// how many rows they have and their block.  An append's rows: their slots in their blocks (-1: nothing to store) and
// positions, so that no run of a head waits for them again before it reads the tables.
struct Runs {
  uint32_t first;
  int n[32];
  int64_t block[32];
  int slot[32], pos[32];
};

// A lane's piece of a row: as read, and its values.
template <int SDT, int PDT, int VEC>
struct Piece {
  Raw<SDT, VEC> raw[2];
  Codes<VEC> old[2];
  int slot, pos;  // slot in the block; -1: nothing to store
  // src: the row's head; held: its slot, the block's r-th (kPatch); else it is the r-th row from the window's first on
  template <bool kPatch>
  __device__ __forceinline__ void load(const Store &s, const typename Elem<SDT>::T *src, const uint8_t *held, const Columns &at,
                                       int64_t row, int r, int64_t block, const Runs &runs) {
    raw[0].load(src + at.one);
    if (paired<VEC>(at)) raw[1].load(src + at.two);
    pos = 0;
    if (kPatch) {
      slot = r;
      old[0].load(held + at.one);
      if (paired<VEC>(at)) old[1].load(held + at.two);
    } else {
      if (r < 32) {
        slot = runs.slot[r], pos = runs.pos[r];
      } else {
        slot = slot_in(s, row, block);
        if (s.cos_t) pos = s.positions[row];
        if (s.cos_t && !turns(s, pos)) slot = -1;
      }
    }
  }
  template <bool kPatch>
  __device__ __forceinline__ void values(const Store &s, const Rotary &rot, const Columns &at, float held, Values<VEC> &lo,
                                         Values<VEC> &hi) const {
    constexpr int kPairs = Values<VEC>::kPairs;
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      lo.pair[e] = VEC == 1 ? f2pack(raw[0].get(0), 0.f) : f2pack(raw[0].get(2 * e), raw[0].get((2 * e + 1) % VEC));
      hi.pair[e] = !paired<VEC>(at) ? 0
                   : VEC == 1 ? f2pack(raw[1].get(0), 0.f)
                              : f2pack(raw[1].get(2 * e), raw[1].get((2 * e + 1) % VEC));
    }
    if (kPatch) {
      const auto add = [&](uint64_t code, uint64_t x) {  // code times held, plus x
        float a, b, c, d;
        f2unpack(code, a, b), f2unpack(x, c, d);
        return f2pack(__fadd_rn(__fmul_rn(a, held), c), __fadd_rn(__fmul_rn(b, held), d));
      };
      Values<VEC> y = old[0].template get<PDT>();
#pragma unroll
      for (int e = 0; e < kPairs; ++e) lo.pair[e] = add(y.pair[e], lo.pair[e]);
      if (paired<VEC>(at)) {
        y = old[1].template get<PDT>();
#pragma unroll
        for (int e = 0; e < kPairs; ++e) hi.pair[e] = add(y.pair[e], hi.pair[e]);
      }
    } else if (at.turn) {
      const int64_t angle = static_cast<int64_t>(pos) * (rot.dim / 2) + at.angle;
      if constexpr (VEC == 1) {
        float x, y, none;
        f2unpack(lo.pair[0], x, none), f2unpack(hi.pair[0], y, none);
        step::turn_pair(x, y, s.cos_t[angle], s.sin_t[angle]);
        lo.pair[0] = f2pack(x, 0.f), hi.pair[0] = f2pack(y, 0.f);
      } else {
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {  // four angles at a time: eight registers less
          const float4 c = reinterpret_cast<const float4 *>(s.cos_t + angle)[i], sn = reinterpret_cast<const float4 *>(s.sin_t + angle)[i];
          if (rot.interleaved) {
            Values<VEC> &v = i == 0 ? lo : hi;
            v.pair[0] = turned(v.pair[0], c.x, sn.x), v.pair[1] = turned(v.pair[1], c.y, sn.y);
            v.pair[2] = turned(v.pair[2], c.z, sn.z), v.pair[3] = turned(v.pair[3], c.w, sn.w);
          } else {
            turn_two(lo.pair[2 * i], hi.pair[2 * i], c.x, c.y, sn.x, sn.y);
            turn_two(lo.pair[2 * i + 1], hi.pair[2 * i + 1], c.z, c.w, sn.z, sn.w);
          }
        }
      }
    }
  }
};

template <int PDT, int VEC>
__device__ __forceinline__ void store_piece(uint8_t *dst, const Columns &at, const Values<VEC> &lo, const Values<VEC> &hi,
                                            float by) {
  Codes<VEC> c;
  c.template set<PDT>(lo, by), c.store(dst + at.one);
  if (paired<VEC>(at)) c.template set<PDT>(hi, by), c.store(dst + at.two);
}

// How a warp's lanes share rows: `wide` lanes a row (the pieces of a head, at most 32), several rows at once.
struct Lanes {
  int pieces, wide, rows, my_row, my_piece;
  __device__ __forceinline__ Lanes(int pieces_, int lane) : pieces(pieces_), wide(min(pieces_, 32)) {
    rows = 32 / wide;
    my_row = lane / wide, my_piece = lane - my_row * wide;
  }
};

// Values of a warp between the two passes over a run: pieces of the lanes, in 16-byte parts of which neighbouring lanes have
// neighbouring ones, and their slots.
template <int VEC>
struct Stage {
  static constexpr int kParts = VEC == 1 ? 1 : VEC / 4;  // of each of a piece's two halves
  ulonglong2 part[kStaged][2][kParts][32];
  int slot[kStaged][32];  // -1: nothing to store
  __device__ __forceinline__ void put(int k, int half, int lane, const Values<VEC> &v) {
#pragma unroll
    for (int i = 0; i < kParts; ++i)
      part[k][half][i][lane] = make_ulonglong2(v.pair[2 * i], v.pair[(2 * i + 1) % Values<VEC>::kPairs]);
  }
  __device__ __forceinline__ void get(int k, int half, int lane, Values<VEC> &v) const {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const ulonglong2 x = part[k][half][i][lane];
      v.pair[2 * i] = x.x;
      if (VEC > 1) v.pair[(2 * i + 1) % Values<VEC>::kPairs] = x.y;
    }
  }
};

// A run of n rows from the window's row i0 on, in `block`; kPatch: the block's first n slots, whose values the rows are added to.
// A lane has one piece of two times VEC columns of every so many-th row.  A run that fits the warp's kStaged pieces a lane (16
// rows of 128 columns) is read once, its values wait in shared memory for the scale; longer runs are read again, out of L1
// or L2, and worked out twice.
template <int SDT, int PDT, int VEC, bool kPatch>
__device__ __forceinline__ void store_run(const Store &s, const Side &side, int h, const Rotary &rot, const Lanes &lanes,
                                          const Runs &runs, int64_t r0, int i0, int n, int64_t block, Stage<VEC> &stage, int lane) {
  const int64_t row = r0 + i0;
  using ST = typename Elem<SDT>::T;
  uint8_t *pages = side.pages + block * side.block + h * side.head;
  float *scale_at = side.scale + block * side.scale_block + h * side.scale_head;
  const ST *src = static_cast<const ST *>(side.src) + row * side.src_row + h * side.src_head;
  const int64_t src_step = times<VEC>(lanes.rows, side.src_row), slot_step = times<VEC>(lanes.rows, side.slot);
  constexpr int kItems = items_of(kPatch, SDT);
  const bool once = (VEC > 1 || lanes.pieces <= 32) && n <= lanes.rows * kStaged;
  const float held = *scale_at;

  Largest largest;
  float by = 0.f, scale = 0.f;
  bool begun = false;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {  // the largest value; then the codes
    int at_stage = 0;
#pragma unroll 1
    for (int p0 = 0; p0 < (VEC > 1 ? 1 : lanes.pieces); p0 += 32) {  // (pieces of 8 columns are 32 at most: the host checks)
      const bool inside = lanes.my_row < lanes.rows && p0 + lanes.my_piece < lanes.pieces;
      const Columns at = step::columns_of<VEC>(rot, s.hd, min(p0 + lanes.my_piece, lanes.pieces - 1));
      int r = lanes.my_row;
      const ST *from = src + times<VEC>(r, side.src_row);
      const uint8_t *was = kPatch ? pages + times<VEC>(r, side.slot) : nullptr;
#pragma unroll 1
      for (int r0 = 0; r0 < n; r0 += lanes.rows * kItems) {
        if (pass == 0 || !once) {
          Piece<SDT, PDT, VEC> piece[kItems];
#pragma unroll
          for (int k = 0; k < kItems; ++k) {
            piece[k].slot = -1;
            if (inside && r < n)
              piece[k].template load<kPatch>(s, kPatch ? from : src + times<VEC>(r, side.src_row), was, at, row + r,
                                             kPatch ? r : i0 + r, block, runs);
            r += lanes.rows;
            if (kPatch) from += src_step, was += slot_step;
          }
#pragma unroll
          for (int k = 0; k < kItems; ++k) {
            stage.slot[at_stage + k][lane] = piece[k].slot;
            if (piece[k].slot < 0) continue;
            begun |= piece[k].slot == 0;
            Values<VEC> lo, hi;
            piece[k].template values<kPatch>(s, rot, at, held, lo, hi);
            stage.put(at_stage + k, 0, lane, lo), stage.put(at_stage + k, 1, lane, hi);
#pragma unroll
            for (int e = 0; e < Values<VEC>::kPairs; ++e) largest.add(lo.pair[e]), largest.add(hi.pair[e]);
          }
        }
        if (pass == 1) {
#pragma unroll
          for (int k = 0; k < kItems; ++k) {
            const int slot = stage.slot[at_stage + k][lane];
            if (slot < 0) continue;
            Values<VEC> lo, hi;
            stage.get(at_stage + k, 0, lane, lo), stage.get(at_stage + k, 1, lane, hi);
            store_piece<PDT, VEC>(pages + times<VEC>(slot, side.slot), at, lo, hi, by);
          }
        }
        if (once) at_stage += kItems;
      }
    }
    if (pass == 1) break;
    const uint32_t top_bits = __reduce_max_sync(0xffffffffu, largest.bits());  // (magnitudes compare as their bits do)
    // nothing is kept: a block that a token begins, or one that is patched whole
    begun = kPatch ? n == s.block_size : __any_sync(0xffffffffu, begun) != 0;
    scale = code8::scale_for<PDT>(top_bits, begun ? 0.f : held);
    by = code8::inverse_of(scale);
    if (!begun && !(scale == held)) {
      uint32_t mine = 0;
      if (kPatch) {
        const int past = n - lane * 32;
        mine = past >= 32 ? 0xffffffffu : past > 0 ? (1u << past) - 1 : 0u;
      } else {
        for (int i = 0; i < n; ++i) {
          const int o = slot_in(s, row + i, block);
          if (o >> 5 == lane && (!s.cos_t || turns(s, s.positions[row + i]))) mine |= 1u << (o & 31);
        }
      }
      scale_again<PDT, VEC>(s, side, pages, held, by, mine, lane);
    }
  }
  if (lane == 0) *scale_at = scale;
}

// The runs of a CTA's window and its pairs of head and side, dealt to its warps: f(i, n, block, pair) for the run that begins
// at the window's row i.
template <typename F>
__device__ __forceinline__ void each_run(const Store &s, int chunk, const Runs &runs, F f) {
  uint32_t first = runs.first;
  const int pair0 = chunk * s.each, pairs = min(s.each, s.pairs - pair0);
  int left = static_cast<int>(threadIdx.x >> 5);  // this warp's next pair, counted from the current run's first
  while (first) {
    const int i = __ffs(first) - 1;
    first &= first - 1;
    for (; left < pairs; left += kThreads / 32) f(i, runs.n[i], runs.block[i], pair0 + left);
    left -= pairs;
  }
}

// The runs of a window that all have one row (a decode step's): a few lanes have each, so that a warp has several at once.
template <int SDT, int PDT, int VEC>
__device__ __forceinline__ void store_single_rows(const Store &s, int chunk, const Runs &runs, uint32_t first, int64_t block, int64_t r0,
                                                   int lane) {
  using ST = typename Elem<SDT>::T;
  const int pair0 = chunk * s.each, pairs = min(s.each, s.pairs - pair0);
  const int all = __popc(first) * pairs;
  const int pieces = step::pieces_of(s.rot, s.hd, VEC);
  const int wide = pieces <= 1 ? 1 : 1 << (32 - __clz(pieces - 1));  // lanes of a row
  const int groups = 32 / wide, mine_in = lane & (wide - 1);
  const int nth = __fns(first, 0, lane + 1);  // the window's row with the lane-th run
  for (int base = static_cast<int>(threadIdx.x >> 5) * groups; base < all; base += kThreads / 32 * groups) {
    const int item = min(base + lane / wide, all - 1);
    const int run = item / pairs, pair = pair0 + item - run * pairs;
    const int i = __shfl_sync(0xffffffffu, nth, run);
    const int64_t at_block = __shfl_sync(0xffffffffu, block, i);
    const int which = pair >= s.heads, h = which ? pair - s.heads : pair;
    const Side &side = s.side[which];
    const Rotary rot = which == 0 ? s.rot : Rotary{0, 0};
    const Columns at = step::columns_of<VEC>(rot, s.hd, min(mine_in, pieces - 1));
    uint8_t *pages = side.pages + at_block * side.block + h * side.head;
    float *scale_at = side.scale + at_block * side.scale_block + h * side.scale_head;
    const float held = *scale_at;
    Piece<SDT, PDT, VEC> piece;
    piece.template load<false>(s, static_cast<const ST *>(side.src) + (r0 + i) * side.src_row + h * side.src_head, nullptr, at,
                               r0 + i, i, at_block, runs);
    const bool there = base + lane / wide < all && piece.slot >= 0;
    Values<VEC> lo, hi;
    Largest largest;
    if (there) {
      piece.template values<false>(s, rot, at, held, lo, hi);
#pragma unroll
      for (int e = 0; e < Values<VEC>::kPairs; ++e) largest.add(lo.pair[e]), largest.add(hi.pair[e]);
    }
    uint32_t top_bits = largest.bits();
    for (int k = wide / 2; k > 0; k >>= 1) top_bits = max(top_bits, __shfl_xor_sync(0xffffffffu, top_bits, k));
    const bool begun = piece.slot == 0;
    const float scale = code8::scale_for<PDT>(top_bits, begun ? 0.f : held);
    const float by = code8::inverse_of(scale);
    uint32_t moved = __ballot_sync(0xffffffffu, there && mine_in == 0 && !begun && !(scale == held));
    while (moved) {  // the warp scales again what the block of one row holds, after the other
      const int from = __ffs(moved) - 1;
      moved &= moved - 1;
      const int its_pair = __shfl_sync(0xffffffffu, pair, from), its_slot = __shfl_sync(0xffffffffu, piece.slot, from);
      const int64_t its_block = __shfl_sync(0xffffffffu, at_block, from);
      const Side &its = s.side[its_pair >= s.heads];
      scale_again<PDT, VEC>(s, its, its.pages + its_block * its.block + (its_pair >= s.heads ? its_pair - s.heads : its_pair) * its.head,
                            __shfl_sync(0xffffffffu, held, from), __shfl_sync(0xffffffffu, by, from),
                            its_slot >> 5 == lane ? 1u << (its_slot & 31) : 0u, lane);
    }
    if (there && mine_in < pieces) {
      store_piece<PDT, VEC>(pages + times<VEC>(piece.slot, side.slot), at, lo, hi, by);
      if (mine_in == 0) *scale_at = scale;
    }
  }
}

// k, v and q are read once, codes and q written once, so memory would bound it (57.8 us for 16384 rows of 32 + 8 + 8 heads x 128,
// bf16 to e4m3); it takes 93 us (without q about 50, floor 17), half of the issue slots used by 18 warps an SM: a run of 16 rows of a head takes some 1100
// instructions (the rotation, the largest, two conversions), and registers leave no room for more warps.  The store's CTAs,
// which wait for memory several times, lie evenly among those of q, which only stream.  4096 single rows of the same heads 29 us
// (a run a warp: 103), 64 of them 6 us of device time from cold caches.  Left out, for the 16384 rows: values kept in registers
// 140 us (spilled), a run for the whole CTA 123, rows kept as read and rotated twice 106, L2 asked for a CTA's rows before their
// runs are found 98.
template <int SDT, int PDT, int VEC>
__global__ void __launch_bounds__(kThreads, resident_of(false, SDT)) append_kernel(const __grid_constant__ Store s,
                                                                     const __grid_constant__ Append q) {
  __shared__ Stage<VEC> stage[kThreads / 32];
  __shared__ Runs runs;
  begin_overlapped();
  if (blockIdx.x < s.watchers) {
    watch_runs<false>(s, reinterpret_cast<uint32_t *>(stage));
    return;
  }
  const uint32_t block_id = blockIdx.x - s.watchers;
  const uint32_t turn = block_id / s.spread;
  const bool stores = turn < s.ctas && block_id == turn * s.spread;
  if (!stores) {
    const int64_t cta = static_cast<int64_t>(block_id) - min(static_cast<int64_t>(turn) + 1, s.ctas);
    step::append_rows<SDT, SDT, VEC, true>(q, cta * kThreads + threadIdx.x);
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t r0 = static_cast<int64_t>(turn / s.chunks) * s.window;
  const int chunk = static_cast<int>(turn % s.chunks);
  if (threadIdx.x < 32) {
    const int64_t row = r0 + lane;
    const int rows = static_cast<int>(min(static_cast<int64_t>(s.window), s.n_rows - r0));
    int64_t block = -1;
    runs.slot[lane] = -1;
    if (row < s.n_rows) {
      const int pos = s.cos_t ? s.positions[row] : 0;
      const int64_t at = row_block(s, row);
      const bool turned = s.cos_t == nullptr || turns(s, pos);
      if (at >= 0 && turned) runs.slot[lane] = slot_in(s, row, at);
      runs.pos[lane] = pos;
      if (lane < rows) {
        block = at;
        if (chunk == 0 && at < 0 && s.slots[row] >= 0) record_error(s.status, DKV_ERR_PAGE_RANGE);
        if (chunk == 0 && at >= 0 && !turned) record_error(s.status, DKV_ERR_ROPE_RANGE);
      }
    }
    int64_t before = __shfl_up_sync(0xffffffffu, block, 1);
    if (lane == 0) before = r0 > 0 ? row_block(s, r0 - 1) : -1;
    const uint32_t first = __ballot_sync(0xffffffffu, block >= 0 && block != before);
    const uint32_t more = __ballot_sync(0xffffffffu, block >= 0 && block == before);  // rows that go on with a run
    int n = __ffs(~(lane == 31 ? 0u : more >> (lane + 1)));
    const int last = first ? 31 - __clz(first) : 0;  // the run that may go on behind the window
    if (first && last + __shfl_sync(0xffffffffu, n, last) == rows) {
      const int64_t mine = __shfl_sync(0xffffffffu, block, last);
      int64_t end = r0 + rows;
      while (end - (r0 + last) < s.block_size) {
        const int64_t at = end + lane;
        const uint32_t same = __ballot_sync(0xffffffffu, at < s.n_rows && row_block(s, at) == mine);
        end += same == 0xffffffffu ? 32 : __ffs(~same) - 1;
        if (same != 0xffffffffu) break;
      }
      if (lane == last) n = static_cast<int>(end - (r0 + last));
    }
    runs.n[lane] = min(n, s.block_size);  // more: a slot came twice
    runs.block[lane] = block;
    if (lane == 0) runs.first = first;
  }
  __syncthreads();
  const uint32_t first = runs.first;
  if (first == 0) return;
  if (__all_sync(0xffffffffu, runs.n[lane] == 1 || !(first >> lane & 1)) && step::pieces_of(s.rot, s.hd, VEC) <= 32) {
    store_single_rows<SDT, PDT, VEC>(s, chunk, runs, first, runs.block[lane], r0, lane);
    return;
  }
  const Lanes lanes(step::pieces_of(s.rot, s.hd, VEC), lane);  // (the same for V: dim is even)
  each_run(s, chunk, runs, [&](int i, int rows_of, int64_t at, int pair) {
    const int which = pair >= s.heads;
    store_run<SDT, PDT, VEC, false>(s, s.side[which], which ? pair - s.heads : pair, which ? Rotary{0, 0} : s.rot, lanes, runs, r0, i,
                                    rows_of, at, stage[threadIdx.x >> 5], lane);
  });
}

// the sequence of row r (its last one where empty ones begin there too), or n_seqs for a row behind the last
__device__ __forceinline__ int sequence_of(const dkv_seq_batch &q, int64_t r) {
  int lo = 0, hi = q.n_seqs;  // cu[lo] <= r, and cu[hi] > r or hi = n_seqs
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (q.cu_seqlens[mid] <= r) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// the block of token i of sequence b, or -1
__device__ __forceinline__ int64_t page_of(const dkv_seq_batch &q, int64_t n_blocks, int b, int blk, int32_t *status) {
  const int64_t tlen = q.table_lens ? q.table_lens[b] : q.table_stride;
  if (blk >= tlen) {
    record_error(status, DKV_ERR_BLOCK_TABLE_SHORT);
    return -1;
  }
  const int32_t id = q.block_tables[static_cast<int64_t>(b) * q.table_stride + blk];
  if (id < 0 || id >= n_blocks) {
    record_error(status, DKV_ERR_PAGE_RANGE);
    return -1;
  }
  return id;
}

// The rows and the codes are read once, codes written once: memory would bound it (46 us for 73200 rows of 8 x 128, bf16 on
// e4m3); it takes 76 us, 50 % of the issue slots used by 15 warps an SM, 1105 instructions a run of 16 rows of a head.
template <int SDT, int PDT, int VEC>
__global__ void __launch_bounds__(kThreads, resident_of(true, SDT)) patch_kernel(const __grid_constant__ Store s) {
  __shared__ Stage<VEC> stage[kThreads / 32];
  __shared__ Runs runs;
  begin_overlapped();
  if (blockIdx.x < s.watchers) {
    watch_runs<true>(s, reinterpret_cast<uint32_t *>(stage));
    return;
  }
  const uint32_t block_id = blockIdx.x - s.watchers;
  const int lane = threadIdx.x & 31;
  const int64_t r0 = static_cast<int64_t>(block_id / s.chunks) * s.window;
  const int chunk = static_cast<int>(block_id % s.chunks);
  if (threadIdx.x < 32) {
    const int64_t row = r0 + lane;
    int64_t block = -1;
    int n = 0;
    if (lane < s.window && row < s.n_rows) {
      const int b = sequence_of(s.seqs, row);
      if (b < s.seqs.n_seqs) {
        const int start = s.seqs.cu_seqlens[b], i = static_cast<int>(row - start);
        const int left = s.seqs.cu_seqlens[b + 1] - static_cast<int>(row);
        if (i >= 0 && left > 0 && i % s.block_size == 0) {  // (always so, where cu_seqlens are prefix sums)
          n = min(min(left, s.block_size), static_cast<int>(min(s.n_rows - row, static_cast<int64_t>(INT32_MAX))));
          block = page_of(s.seqs, s.n_blocks, b, i / s.block_size, s.status);
        }
      }
      if (row == s.n_rows - 1 && chunk == 0 && s.seqs.cu_seqlens[s.seqs.n_seqs] > s.n_rows)
        record_error(s.status, DKV_ERR_INVALID_ARGUMENT);
    }
    const uint32_t first = __ballot_sync(0xffffffffu, block >= 0);
    runs.n[lane] = n, runs.block[lane] = block;
    if (lane == 0) runs.first = first;
  }
  __syncthreads();
  const Lanes lanes(step::pieces_of(Rotary{0, 0}, s.hd, VEC), lane);
  each_run(s, chunk, runs, [&](int i, int rows_of, int64_t at, int head) {
    store_run<SDT, PDT, VEC, true>(s, s.side[0], head, Rotary{0, 0}, lanes, runs, r0, i, rows_of, at, stage[threadIdx.x >> 5], lane);
  });
}

// ---------------------------------------------------------------------------------------
// reading back
// ---------------------------------------------------------------------------------------
struct Read {
  const uint8_t *pages;
  int64_t block, slot, head;  // bytes
  const float *scale;
  int64_t scale_block, scale_head;
  dkv_seq_batch seqs;
  void *out;
  int64_t out_row, out_head;
  int64_t n_rows, n_blocks;
  int32_t *status;
  int heads, hd, block_size;
  int rows;       // of a CTA
  int zero_rest;  // rows behind the last sequence become zero (else they are left)
};

constexpr int kReadThreads = 256;
constexpr int kReadRows = 32;

// VEC codes to values; the value's rows are written in whole 16 (8, 1) elements' worth of bytes
template <int PDT, int ODT, int VEC>
__device__ __forceinline__ void read_piece(const uint8_t *src, float scale, bool there, typename Elem<ODT>::T *dst) {
  if constexpr (VEC == 1) {
    float y[4];
    Code<PDT>::unpack(there ? *src : 0, y);
    *dst = Elem<ODT>::from_f(there ? __fmul_rn(y[0], scale) : 0.f);
  } else {
    uint32_t c[VEC / 4] = {};
    if (there) {
      if constexpr (VEC == 16) {
        const uint4 w = *reinterpret_cast<const uint4 *>(src);
        c[0] = w.x, c[1] = w.y, c[2] = w.z, c[3] = w.w;
      } else if constexpr (VEC == 8) {
        const uint2 w = *reinterpret_cast<const uint2 *>(src);
        c[0] = w.x, c[1] = w.y;
      } else {
        c[0] = *reinterpret_cast<const uint32_t *>(src);
      }
    }
    float x[VEC];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      float y[4];
      Code<PDT>::unpack(c[i], y);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[4 * i + k] = there ? __fmul_rn(y[k], scale) : 0.f;
    }
    if constexpr (VEC * sizeof(typename Elem<ODT>::T) == 8) {
      uint2 w;
      if (ODT == DKV_BF16)
        w = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
      else
        w = make_uint2(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]));
      *reinterpret_cast<uint2 *>(dst) = w;
    } else {
      Raw<ODT, VEC> y;
      y.set(x), y.store(dst);
    }
  }
}

// Bound by memory: each code read once, each value written once.  A CTA first finds its rows' places (one lane each),
// then a thread has the same columns of every so many-th row.  73200 rows of 8 x 128: to bf16 43-44 us (floor 34.5; 16 bytes of
// values a thread instead of 32: 53), to fp32 75 (57.4; 64 bytes: 98).
template <int PDT, int ODT, int VEC>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const __grid_constant__ Read a) {
  using OT = typename Elem<ODT>::T;
  begin_overlapped();
  __shared__ int64_t row_at[kReadRows], scale_at[kReadRows];  // scale_at -1: zeros, -2: left alone
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.rows;
  const int n = static_cast<int>(min(static_cast<int64_t>(a.rows), a.n_rows - r0));
  const int tid = threadIdx.x;
  if (tid < n) {
    const int64_t row = r0 + tid;
    const int b = sequence_of(a.seqs, row);
    int64_t block = a.zero_rest ? -1 : -2;
    int slot = 0;
    if (b < a.seqs.n_seqs) {
      const int i = static_cast<int>(row - a.seqs.cu_seqlens[b]), blk = i / a.block_size;
      slot = i - blk * a.block_size;
      // (never negative, where cu_seqlens are prefix sums)
      block = i >= 0 ? page_of(a.seqs, a.n_blocks, b, blk, a.status) : -1;
    }
    if (row == a.n_rows - 1 && a.seqs.cu_seqlens[a.seqs.n_seqs] > a.n_rows) record_error(a.status, DKV_ERR_INVALID_ARGUMENT);
    row_at[tid] = block < 0 ? 0 : block * a.block + slot * a.slot;
    scale_at[tid] = block < 0 ? block : block * a.scale_block;
  }
  __syncthreads();
  const int pieces = a.hd / VEC, per_row = a.heads * pieces;
  const int wide = min(per_row, kReadThreads), rows_at_once = kReadThreads / wide;
  const int my_row = tid / wide;
  if (my_row >= rows_at_once) return;
  for (int in = tid - my_row * wide; in < per_row; in += wide) {
    const int h = in / pieces, d = (in - h * pieces) * VEC;
    const uint8_t *src = a.pages + h * a.head + d;
    const float *scales = a.scale + h * a.scale_head;
    OT *dst = static_cast<OT *>(a.out) + (r0 + my_row) * a.out_row + h * a.out_head + d;
    const int64_t step = rows_at_once * a.out_row;
#pragma unroll 4
    for (int r = my_row; r < n; r += rows_at_once, dst += step) {
      const int64_t at = scale_at[r];
      if (at == -2) continue;
      read_piece<PDT, ODT, VEC>(src + row_at[r], at >= 0 ? scales[at] : 0.f, at >= 0, dst);
    }
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
bool float_dtype(int dt) { return dt == DKV_F32 || dt == DKV_F16 || dt == DKV_BF16; }
bool code_dtype(int dt) { return dt == DKV_E4M3 || dt == DKV_I8; }
constexpr int kMaxBlock = 1024;  // a bit of a warp's 32-bit registers for each slot

int check_pages(const dkv_paged_cache &c, const dkv_page_scales &s) {
  if (!code_dtype(c.dtype)) return DKV_ERR_UNSUPPORTED;
  if (c.block_size <= 0 || c.n_heads <= 0 || c.head_dim <= 0 || c.num_blocks < 0) return DKV_ERR_LAYOUT;
  if (c.block_size > kMaxBlock) return DKV_ERR_UNSUPPORTED;
  if (c.num_blocks > 0 && (c.base == nullptr || s.base == nullptr)) return DKV_ERR_INVALID_ARGUMENT;
  if (s.stride_block < 0 || s.stride_head < 0) return DKV_ERR_LAYOUT;
  return DKV_OK;
}
int check_seqs(const dkv_seq_batch &q) {
  if (q.n_seqs < 0) return DKV_ERR_INVALID_ARGUMENT;
  if (q.n_seqs > 65535) return DKV_ERR_UNSUPPORTED;
  if (q.n_seqs > 0 && q.cu_seqlens == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  return DKV_OK;
}
// tables without columns have no address to read from
dkv_seq_batch readable(const dkv_seq_batch &q) {
  dkv_seq_batch r = q;
  if (r.block_tables == nullptr) r.table_lens = nullptr, r.table_stride = 0;
  return r;
}

Side side_of(const dkv_paged_cache &c, const dkv_page_scales &s, const void *src, int64_t row, int64_t head) {
  Side x;
  x.src = src, x.src_row = row, x.src_head = head;
  x.pages = static_cast<uint8_t *>(c.base);
  x.block = c.stride_block, x.slot = c.stride_slot, x.head = c.stride_head;
  x.scale = s.base, x.scale_block = s.stride_block, x.scale_head = s.stride_head;
  return x;
}
int64_t source_bits(const Side &x, int64_t size) {
  return reinterpret_cast<intptr_t>(x.src) | x.src_row * size | x.src_head * size;
}
bool short_strides(const Side &x) { return x.src_row >= 0 && x.src_row <= INT32_MAX && x.slot >= 0 && x.slot <= INT32_MAX; }
int64_t page_bits(const Side &x) { return reinterpret_cast<intptr_t>(x.pages) | x.block | x.slot | x.head; }

// How rows and pairs of head and side are dealt: as many rows a CTA (up to 16: one in a block's worth begins a run of a
// prefill) and as few CTAs a window as still give 8 CTAs an SM.
void deal(int64_t rows, int pairs, int sms, Store *s) {
  constexpr int kWarps = kThreads / 32;
  const int64_t want = static_cast<int64_t>(sms) * 8;
  s->pairs = pairs;
  s->window = 1;
  while (s->window < 16 && rows / (2 * s->window) * ((pairs + kWarps - 1) / kWarps) >= want) s->window *= 2;
  const int64_t windows = (rows + s->window - 1) / s->window;
  const int64_t most = (pairs + kWarps - 1) / kWarps, chunks = (want + windows - 1) / windows;
  s->each = static_cast<int>((pairs + (chunks < most ? chunks : most) - 1) / (chunks < most ? chunks : most));
  s->chunks = (pairs + s->each - 1) / s->each;
  s->ctas = windows * s->chunks;
}

// How the rows are cut for the watchers: into 8 segments, not below 512 rows (an append's: a load of four rows a thread) or 1024, and
// not above what a table half full holds, given that rows have a run each or (a patch) one in each block and sequence.
void watch(bool patch, int64_t most, Store *s) {
  const int64_t least = patch ? 1024 : 512;
  const auto runs = [&](int64_t rows) {
    const int64_t n = patch ? rows / s->block_size + s->seqs.n_seqs + 1 : rows;
    return n < rows ? n : rows;
  };
  s->segment = (s->n_rows + 7) / 8 > least ? (s->n_rows + 7) / 8 : least;
  while (2 * runs(s->segment) > most) s->segment = s->segment / 2 > most / 2 ? s->segment / 2 : most / 2;
  s->segments = (s->n_rows + s->segment - 1) / s->segment;
  s->places = 64;
  while (s->places < 2 * runs(s->segment) && s->places < 2 * s->n_rows) s->places *= 2;
  // ids are 32-bit in block tables, and so are a table's entries; more rows than any call has (2 million in an append) are not watched
  constexpr int64_t kMostSegments = 512;
  s->watchers = s->n_blocks >= UINT32_MAX || s->segments > kMostSegments ? 0 : static_cast<int>(s->segments * (s->segments + 1) / 2);
}
// the bytes of a launch's stages, as places
constexpr int64_t stage_places(bool wide) { return wide ? 8192 : 4096; }
static_assert(sizeof(Stage<8>) >= 4 * (stage_places(true) / (kThreads / 32) + kQueue) && stage_places(true) <= kMostPlaces, "a watcher's memory");
static_assert(sizeof(Stage<1>) >= 4 * (stage_places(false) / (kThreads / 32) + kQueue), "a watcher's memory");

// What the rows of an append say of themselves, without their values.
int check_append(const dkv_append_args &g) {
  const dkv_paged_cache &kp = g.k_pages, &vp = g.v_pages;
  if (!code_dtype(kp.dtype)) return DKV_ERR_UNSUPPORTED;
  if (kp.block_size <= 0 || kp.num_blocks < 0 || vp.num_blocks < 0) return DKV_ERR_LAYOUT;
  if (g.n_rows < 0 || (g.n_rows > 0 && g.slots == nullptr)) return DKV_ERR_INVALID_ARGUMENT;
  return DKV_OK;
}
void slots_of(const dkv_append_args &g, Store *s) {
  const dkv_paged_cache &kp = g.k_pages, &vp = g.v_pages;
  s->n_rows = g.n_rows;
  s->n_blocks = kp.num_blocks < vp.num_blocks ? kp.num_blocks : vp.num_blocks;
  s->n_slots = s->n_blocks * kp.block_size, s->narrow = s->n_slots <= UINT32_MAX;
  s->slots = g.slots, s->status = g.status, s->block_size = kp.block_size;
}
int launch_watch(Store *s, cudaStream_t st) {
  watch(s->slots == nullptr, kMostPlaces, s);
  const auto kernel = s->slots ? watch_kernel<false> : watch_kernel<true>;
  if (s->watchers > 0) DKV_CUDA_CHECK(launch_overlapped(kernel, dim3(s->watchers), kThreads, 0, st, *s));
  return DKV_OK;
}

}  // namespace quant
}  // namespace dkv

using namespace dkv;

extern "C" int dkv_append_paged_quant(const dkv_append_args *args, const dkv_rotary *rotary, const dkv_page_scales *k_scales,
                                      const dkv_page_scales *v_scales, dkv_stream_t stream) {
  if (args == nullptr || k_scales == nullptr || v_scales == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  const dkv_append_args &g = *args;
  const dkv_paged_cache &kp = g.k_pages, &vp = g.v_pages;
  if (!quant::code_dtype(kp.dtype) || !quant::float_dtype(g.in_dtype)) return DKV_ERR_UNSUPPORTED;
  if (kp.dtype != vp.dtype || kp.block_size != vp.block_size || kp.n_heads != vp.n_heads || kp.head_dim != vp.head_dim)
    return DKV_ERR_LAYOUT;
  int rc = quant::check_pages(kp, *k_scales);
  if (rc == DKV_OK) rc = quant::check_pages(vp, *v_scales);
  if (rc != DKV_OK) return rc;
  if (g.n_rows < 0 || (g.q != nullptr && g.n_q_heads <= 0)) return DKV_ERR_INVALID_ARGUMENT;
  if ((g.rope_cos == nullptr) != (g.rope_sin == nullptr)) return DKV_ERR_INVALID_ARGUMENT;
  step::Rotary rot;
  if (step::rotary_of(g.rope_cos != nullptr, rotary, kp.head_dim, &rot) < 0) return DKV_ERR_UNSUPPORTED;
  if (g.n_rows == 0) return DKV_OK;
  if (g.k == nullptr || g.v == nullptr || g.slots == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (g.rope_cos != nullptr && g.positions == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (g.q != nullptr && g.q_out == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc != DKV_OK) return rc;
  quant::Store s = {};
  s.side[0] = quant::side_of(kp, *k_scales, g.k, g.k_stride_row, g.k_stride_head);
  s.side[1] = quant::side_of(vp, *v_scales, g.v, g.v_stride_row, g.v_stride_head);
  quant::slots_of(g, &s);
  s.positions = g.positions, s.cos_t = g.rope_cos, s.sin_t = g.rope_sin;
  s.rope_max_pos = g.rope_max_pos;
  s.heads = kp.n_heads, s.hd = kp.head_dim;
  s.rot = rot;
  step::Append q;
  step::describe(g, rot, &q);
  const int64_t size = g.in_dtype == DKV_F32 ? 4 : 2;
  int64_t bits = quant::source_bits(s.side[0], size) | quant::source_bits(s.side[1], size);
  bits |= reinterpret_cast<intptr_t>(g.rope_cos) | reinterpret_cast<intptr_t>(g.rope_sin);
  if (g.q != nullptr)
    bits |= reinterpret_cast<intptr_t>(g.q) | reinterpret_cast<intptr_t>(g.q_out) |
            (q.src_row[0] | q.src_head[0] | q.dst_row[0] | q.dst_head[0]) * size;
  const bool wide = step::whole_pieces(rot, kp.head_dim, 8) && kp.head_dim % 16 == 0 && kp.head_dim <= 512 && bits % 16 == 0 &&
                    (quant::page_bits(s.side[0]) | quant::page_bits(s.side[1])) % 8 == 0 && quant::short_strides(s.side[0]) &&
                    quant::short_strides(s.side[1]);
  quant::deal(g.n_rows, 2 * kp.n_heads, sms, &s);
  const int64_t threads = q.heads[0] == 0 ? 0 : g.n_rows * ((q.heads[0] + step::kHeads - 1) / step::kHeads) *
                                                    step::pieces_of(rot, kp.head_dim, wide ? 8 : 1);
  q.wide = threads > UINT32_MAX;
  const int64_t work = s.ctas + (threads + quant::kThreads - 1) / quant::kThreads;
  s.spread = static_cast<uint32_t>(work / s.ctas);
  quant::watch(false, quant::stage_places(wide), &s);
  const int64_t ctas = work + s.watchers;
  if (ctas > INT32_MAX) return DKV_ERR_UNSUPPORTED;
  static_assert(quant::kThreads == step::kAppThreads, "one launch for both");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define DKV_QUANT_CASE(S, P)                                                                                  \
  if (g.in_dtype == S && kp.dtype == P) {                                                                     \
    const auto kernel = wide ? quant::append_kernel<S, P, 8> : quant::append_kernel<S, P, 1>;                 \
    DKV_CUDA_CHECK(launch_overlapped(kernel, dim3(static_cast<unsigned>(ctas)), quant::kThreads, 0, st, s, q)); \
    return DKV_OK;                                                                                            \
  }
  DKV_QUANT_CASE(DKV_BF16, DKV_E4M3)
  DKV_QUANT_CASE(DKV_F16, DKV_E4M3)
  DKV_QUANT_CASE(DKV_F32, DKV_E4M3)
  DKV_QUANT_CASE(DKV_BF16, DKV_I8)
  DKV_QUANT_CASE(DKV_F16, DKV_I8)
  DKV_QUANT_CASE(DKV_F32, DKV_I8)
#undef DKV_QUANT_CASE
  return DKV_ERR_UNSUPPORTED;
}

extern "C" int dkv_scatter_paged_quant(const void *delta, int32_t delta_dtype, int64_t n_rows, int64_t delta_stride_row,
                                       int64_t delta_stride_head, const dkv_paged_cache *cache,
                                       const dkv_page_scales *scales, const dkv_seq_batch *seqs, int32_t *status,
                                       dkv_stream_t stream) {
  if (cache == nullptr || scales == nullptr || seqs == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  int rc = quant::check_pages(*cache, *scales);
  if (rc == DKV_OK) rc = quant::check_seqs(*seqs);
  if (rc != DKV_OK) return rc;
  if (!quant::float_dtype(delta_dtype)) return DKV_ERR_UNSUPPORTED;
  if (n_rows < 0) return DKV_ERR_INVALID_ARGUMENT;
  if (n_rows == 0 || seqs->n_seqs == 0) return DKV_OK;
  if (delta == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc != DKV_OK) return rc;
  quant::Store s = {};
  s.side[0] = quant::side_of(*cache, *scales, delta, delta_stride_row, delta_stride_head);
  s.n_rows = n_rows, s.n_blocks = cache->num_blocks;
  s.seqs = quant::readable(*seqs);
  s.status = status;
  s.heads = cache->n_heads, s.hd = cache->head_dim, s.block_size = cache->block_size;
  const int64_t size = delta_dtype == DKV_F32 ? 4 : 2;
  const bool wide = cache->head_dim % 16 == 0 && cache->head_dim <= 512 && quant::source_bits(s.side[0], size) % 16 == 0 &&
                    quant::page_bits(s.side[0]) % 8 == 0 && quant::short_strides(s.side[0]);
  quant::deal(n_rows, cache->n_heads, sms, &s);
  quant::watch(true, quant::stage_places(wide), &s);
  const int64_t ctas = s.ctas + s.watchers;
  if (ctas > INT32_MAX) return DKV_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define DKV_QUANT_CASE(S, P)                                                                               \
  if (delta_dtype == S && cache->dtype == P) {                                                             \
    const auto kernel = wide ? quant::patch_kernel<S, P, 8> : quant::patch_kernel<S, P, 1>;                \
    DKV_CUDA_CHECK(launch_overlapped(kernel, dim3(static_cast<unsigned>(ctas)), quant::kThreads, 0, st, s)); \
    return DKV_OK;                                                                                         \
  }
  DKV_QUANT_CASE(DKV_BF16, DKV_E4M3)
  DKV_QUANT_CASE(DKV_F16, DKV_E4M3)
  DKV_QUANT_CASE(DKV_F32, DKV_E4M3)
  DKV_QUANT_CASE(DKV_BF16, DKV_I8)
  DKV_QUANT_CASE(DKV_F16, DKV_I8)
  DKV_QUANT_CASE(DKV_F32, DKV_I8)
#undef DKV_QUANT_CASE
  return DKV_ERR_UNSUPPORTED;
}

extern "C" int dkv_append_paged_quant_check(const dkv_append_args *args, dkv_stream_t stream) {
  if (args == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  const int rc = quant::check_append(*args);
  if (rc != DKV_OK || args->n_rows == 0) return rc;
  quant::Store s = {};
  quant::slots_of(*args, &s);
  return quant::launch_watch(&s, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int dkv_scatter_paged_quant_check(int64_t n_rows, const dkv_paged_cache *cache, const dkv_seq_batch *seqs, int32_t *status,
                                             dkv_stream_t stream) {
  if (cache == nullptr || seqs == nullptr || n_rows < 0) return DKV_ERR_INVALID_ARGUMENT;
  if (!quant::code_dtype(cache->dtype)) return DKV_ERR_UNSUPPORTED;
  if (cache->block_size <= 0 || cache->num_blocks < 0) return DKV_ERR_LAYOUT;
  const int rc = quant::check_seqs(*seqs);
  if (rc != DKV_OK || n_rows == 0 || seqs->n_seqs == 0) return rc;
  quant::Store s = {};
  s.n_rows = n_rows, s.n_blocks = cache->num_blocks, s.block_size = cache->block_size;
  s.seqs = quant::readable(*seqs), s.status = status;
  return quant::launch_watch(&s, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int dkv_gather_paged_quant(const dkv_paged_cache *cache, const dkv_page_scales *scales, const dkv_seq_batch *seqs,
                                      void *out, int32_t out_dtype, int64_t n_rows, int64_t out_stride_row,
                                      int64_t out_stride_head, int32_t zero_rest, int32_t *status, dkv_stream_t stream) {
  if (cache == nullptr || scales == nullptr || seqs == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  int rc = quant::check_pages(*cache, *scales);
  if (rc == DKV_OK) rc = quant::check_seqs(*seqs);
  if (rc != DKV_OK) return rc;
  if (!quant::float_dtype(out_dtype)) return DKV_ERR_UNSUPPORTED;
  if (n_rows < 0) return DKV_ERR_INVALID_ARGUMENT;
  if (n_rows == 0) return DKV_OK;
  if (out == nullptr || seqs->cu_seqlens == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc != DKV_OK) return rc;
  quant::Read a;
  a.pages = static_cast<const uint8_t *>(cache->base);
  a.block = cache->stride_block, a.slot = cache->stride_slot, a.head = cache->stride_head;
  a.scale = scales->base, a.scale_block = scales->stride_block, a.scale_head = scales->stride_head;
  a.seqs = quant::readable(*seqs);
  a.out = out, a.out_row = out_stride_row, a.out_head = out_stride_head;
  a.n_rows = n_rows, a.n_blocks = cache->num_blocks;
  a.status = status;
  a.heads = cache->n_heads, a.hd = cache->head_dim, a.block_size = cache->block_size;
  a.rows = n_rows >= static_cast<int64_t>(sms) * quant::kReadRows * 2 ? quant::kReadRows : 8;
  a.zero_rest = zero_rest != 0;
  const int64_t size = out_dtype == DKV_F32 ? 4 : 2;
  // codes of a thread: 32 bytes of values, or 4 codes, or one
  const int full = static_cast<int>(32 / size);
  const int64_t code_bits = reinterpret_cast<intptr_t>(a.pages) | a.block | a.slot | a.head | a.hd;
  const int64_t out_bits = reinterpret_cast<intptr_t>(out) | out_stride_row * size | out_stride_head * size;
  const int vec = code_bits % full == 0 && out_bits % 16 == 0 ? full : code_bits % 4 == 0 && out_bits % (4 * size) == 0 ? 4 : 1;
  const int64_t ctas = (n_rows + a.rows - 1) / a.rows;
  if (ctas > INT32_MAX || static_cast<int64_t>(a.heads) * a.hd > INT32_MAX / quant::kReadRows - quant::kReadThreads)
    return DKV_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define DKV_QUANT_CASE(P, O)                                                                                  \
  if (cache->dtype == P && out_dtype == O) {                                                                  \
    constexpr int kFull = O == DKV_F32 ? 8 : 16;                                                              \
    const auto kernel = vec == kFull ? quant::read_kernel<P, O, kFull>                                        \
                                     : (vec == 4 ? quant::read_kernel<P, O, 4> : quant::read_kernel<P, O, 1>); \
    DKV_CUDA_CHECK(launch_overlapped(kernel, dim3(static_cast<unsigned>(ctas)), quant::kReadThreads, 0, st, a)); \
    return DKV_OK;                                                                                            \
  }
  DKV_QUANT_CASE(DKV_E4M3, DKV_BF16)
  DKV_QUANT_CASE(DKV_E4M3, DKV_F16)
  DKV_QUANT_CASE(DKV_E4M3, DKV_F32)
  DKV_QUANT_CASE(DKV_I8, DKV_BF16)
  DKV_QUANT_CASE(DKV_I8, DKV_F16)
  DKV_QUANT_CASE(DKV_I8, DKV_F32)
#undef DKV_QUANT_CASE
  return DKV_ERR_UNSUPPORTED;
}
