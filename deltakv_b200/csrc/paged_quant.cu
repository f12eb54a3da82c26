// The 8-bit paged cache: K and V quantised as they are stored, read back, and patched in place.
//   dkv_append_paged_quant   RoPE of the new q and k rows, K and V quantised into their slots
//   dkv_scatter_paged_quant  value + delta for the rows of every sequence, quantised again
//   dkv_gather_paged_quant   the values of every sequence's rows
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

// Rows of one call.  A run is the rows that follow one another in one block; a warp has a run's K or V of one
// head, and with it alone the head's scale in that block.
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
  int window;   // rows that a warp looks through for the first ones of runs
  int narrow;   // the cache's slots fit 32 bits
  int64_t ctas; // of the store; behind them q's
};

constexpr int kThreads = 128;
constexpr int kItems = 4;  // pieces of two times VEC columns that a lane holds at once

// block of a row's slot, -1 for none
__device__ __forceinline__ int64_t row_block(const Store &s, int64_t row) {
  const int64_t slot = s.slots[row];
  if (slot < 0 || slot >= s.n_slots) return -1;
  return s.narrow ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(s.block_size) : slot / s.block_size;
}
__device__ __forceinline__ int slot_in(const Store &s, int64_t row, int64_t block) {
  return static_cast<int>(s.slots[row] - block * s.block_size);
}

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
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      float y[4];
      Code<PT>::unpack(w[i], y);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[4 * i + k] = y[k];
    }
  }
  template <int PT>
  __device__ __forceinline__ void set(const float (&x)[VEC], float by) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      w[i] = Code<PT>::pack(__fmul_rn(x[4 * i], by), __fmul_rn(x[4 * i + 1], by), __fmul_rn(x[4 * i + 2], by),
                            __fmul_rn(x[4 * i + 3], by));
  }
};
template <>
struct Codes<1> {
  uint32_t w;
  __device__ __forceinline__ void load(const uint8_t *src) { w = *src; }
  __device__ __forceinline__ void store(uint8_t *dst) const { *dst = static_cast<uint8_t>(w); }
  template <int PT>
  __device__ __forceinline__ void get(float (&x)[1]) const {
    float y[4];
    Code<PT>::unpack(w, y);
    x[0] = y[0];
  }
  template <int PT>
  __device__ __forceinline__ void set(const float (&x)[1], float by) { w = Code<PT>::pack(__fmul_rn(x[0], by), 0.f, 0.f, 0.f); }
};
static_assert(sizeof(Codes<8>) == 8, "eight columns are one load");

// A run of n rows from `row` on, in `block`; kPatch: the block's first n slots, whose values the rows are added to.
template <int SDT, int PDT, int VEC, bool kPatch>
__device__ __forceinline__ void store_run(const Store &s, const Side &side, int h, bool turns, int64_t row, int n,
                                          int64_t block, int lane) {
  using ST = typename Elem<SDT>::T;
  uint8_t *pages = side.pages + block * side.block + h * side.head;
  float *scale_at = side.scale + block * side.scale_block + h * side.scale_head;
  const ST *src = static_cast<const ST *>(side.src) + row * side.src_row + h * side.src_head;
  const Rotary rot = turns ? s.rot : Rotary{0, 0};
  const int pieces = step::pieces_of(rot, s.hd, VEC);
  const int items = n * pieces;
  const float held = *scale_at;

  float x[kItems][2][VEC];
  int at_slot[kItems];  // -1: nothing to store
  Columns at[kItems];
  // the values of items i0 + lane, i0 + 32 + lane, ...
  auto load = [&](int i0) {
    Raw<SDT, VEC> raw[kItems][2];
    Codes<VEC> old[kItems][2];
    int r[kItems], pos[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = i0 + k * 32 + lane;
      at_slot[k] = -1, pos[k] = 0, r[k] = i / pieces;
      if (i >= items) continue;
      at[k] = step::columns_of<VEC>(rot, s.hd, i - r[k] * pieces);
      const ST *p = src + r[k] * side.src_row;
      raw[k][0].load(p + at[k].one);
      if (at[k].pair) raw[k][1].load(p + at[k].two);
      if (kPatch) {
        at_slot[k] = r[k];
        old[k][0].load(pages + r[k] * side.slot + at[k].one);
        if (at[k].pair) old[k][1].load(pages + r[k] * side.slot + at[k].two);
      } else {
        at_slot[k] = slot_in(s, row + r[k], block);
        if (s.cos_t) pos[k] = s.positions[row + r[k]];
      }
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (at_slot[k] >= 0) {
        if (!kPatch && s.cos_t && (pos[k] < 0 || pos[k] >= s.rope_max_pos)) {
          record_error(s.status, DKV_ERR_ROPE_RANGE);
          at_slot[k] = -1;
        }
      }
      if (at_slot[k] < 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[k][0][e] = x[k][1][e] = 0.f;
        continue;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[k][0][e] = raw[k][0].get(e), x[k][1][e] = at[k].pair ? raw[k][1].get(e) : 0.f;
      if (kPatch) {
        float y[VEC];
        old[k][0].template get<PDT>(y);
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[k][0][e] = __fadd_rn(__fmul_rn(y[e], held), x[k][0][e]);
        if (at[k].pair) {
          old[k][1].template get<PDT>(y);
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[k][1][e] = __fadd_rn(__fmul_rn(y[e], held), x[k][1][e]);
        }
      } else if (at[k].turn) {
        Raw<DKV_F32, VEC> c, sn;
        const int64_t angle = static_cast<int64_t>(pos[k]) * (rot.dim / 2) + at[k].angle;
        c.load(s.cos_t + angle), sn.load(s.sin_t + angle);
        step::turn<VEC>(x[k][0], x[k][1], c, sn, rot.interleaved);
      }
    }
  };
  uint32_t top = 0;
  bool begun = false;
  for (int i0 = 0; i0 < items; i0 += 32 * kItems) {
    load(i0);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      begun |= at_slot[k] == 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        top = max(top, max(__float_as_uint(x[k][0][e]) & 0x7fffffffu, __float_as_uint(x[k][1][e]) & 0x7fffffffu));
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  // nothing is kept: a block that a token begins, or one that is patched whole
  begun = kPatch ? n == s.block_size : __any_sync(0xffffffffu, begun);
  const float scale = code8::scale_for<PDT>(top, begun ? 0.f : held);
  const float by = code8::inverse_of(scale);

  if (!begun && !(scale == held)) {  // what stays of the block, in the new scale
    uint32_t mine = 0;  // bit i of lane l: slot 32 l + i is stored by this run
    if (kPatch) {
      const int past = n - lane * 32;
      mine = past >= 32 ? 0xffffffffu : past > 0 ? (1u << past) - 1 : 0u;
    } else {
      for (int i = 0; i < n; ++i) {
        const int o = slot_in(s, row + i, block);
        if (o >> 5 == lane) mine |= 1u << (o & 31);
      }
    }
    const int units = (s.hd + VEC - 1) / VEC, all = s.block_size * units;
    for (int i0 = 0; i0 < all; i0 += 32 * 8) {
      Codes<VEC> c[8];
      int o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * 32 + lane;
        const int u = min(i, all - 1) / units;
        const bool stored = __shfl_sync(0xffffffffu, mine, u >> 5) >> (u & 31) & 1;
        o[k] = i < all && !stored ? u : -1;
        if (o[k] >= 0) c[k].load(pages + u * side.slot + (i - u * units) * VEC);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (o[k] < 0) continue;
        float y[VEC];
        c[k].template get<PDT>(y);
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[e] = __fmul_rn(y[e], held);
        c[k].template set<PDT>(y, by);
        c[k].store(pages + o[k] * side.slot + (i0 + k * 32 + lane - o[k] * units) * VEC);
      }
    }
  }
  for (int i0 = 0; i0 < items; i0 += 32 * kItems) {
    if (items > 32 * kItems) load(i0);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (at_slot[k] < 0) continue;
      uint8_t *dst = pages + at_slot[k] * side.slot;
      Codes<VEC> c;
      c.template set<PDT>(x[k][0], by), c.store(dst + at[k].one);
      if (at[k].pair) c.template set<PDT>(x[k][1], by), c.store(dst + at[k].two);
    }
  }
  if (lane == 0) *scale_at = scale;
}

// Bound by memory: k, v and q are read once, codes and q written once.
template <int SDT, int PDT, int VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ Store s, const __grid_constant__ Append q) {
  begin_overlapped();
  if (blockIdx.x >= s.ctas) {
    step::append_rows<SDT, SDT, VEC, true>(q, (static_cast<int64_t>(blockIdx.x) - s.ctas) * kThreads + threadIdx.x);
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int per = 2 * s.heads;
  const int64_t r0 = item / per * s.window;
  if (r0 >= s.n_rows) return;
  const int in = static_cast<int>(item % per), which = in >= s.heads, h = which ? in - s.heads : in;
  const int64_t row = r0 + lane;
  int64_t block = -1;
  if (lane < s.window && row < s.n_rows) {
    block = row_block(s, row);
    if (block < 0 && in == 0 && s.slots[row] >= 0) record_error(s.status, DKV_ERR_PAGE_RANGE);
  }
  int64_t before = __shfl_up_sync(0xffffffffu, block, 1);
  if (lane == 0) before = r0 > 0 ? row_block(s, r0 - 1) : -1;
  uint32_t first = __ballot_sync(0xffffffffu, block >= 0 && block != before);
  while (first) {
    const int i = __ffs(first) - 1;
    first &= first - 1;
    const int64_t mine = __shfl_sync(0xffffffffu, block, i);
    int64_t end = r0 + i + 1;  // the rows after it in the same block
    while (true) {
      const int64_t at = end + lane;
      const uint32_t same = __ballot_sync(0xffffffffu, at < s.n_rows && row_block(s, at) == mine);
      if (same != 0xffffffffu) {
        end += __ffs(~same) - 1;
        break;
      }
      end += 32;
    }
    const int64_t n = min(end - (r0 + i), static_cast<int64_t>(s.block_size));  // more: a slot came twice
    store_run<SDT, PDT, VEC, false>(s, s.side[which], h, which == 0 && s.cos_t != nullptr, r0 + i, static_cast<int>(n), mine,
                                    lane);
  }
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

template <int SDT, int PDT, int VEC>
__global__ void __launch_bounds__(kThreads) patch_kernel(const __grid_constant__ Store s) {
  begin_overlapped();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t r0 = item / s.heads * s.window;
  if (r0 >= s.n_rows) return;
  const int h = static_cast<int>(item % s.heads);
  const int64_t row = r0 + lane;
  int64_t block = -1;
  int n = 0;
  if (lane < s.window && row < s.n_rows) {
    const int b = sequence_of(s.seqs, row);
    if (b < s.seqs.n_seqs) {
      const int first = s.seqs.cu_seqlens[b], i = static_cast<int>(row - first);
      const int left = s.seqs.cu_seqlens[b + 1] - static_cast<int>(row);
      if (i >= 0 && left > 0 && i % s.block_size == 0) {  // (always so, where cu_seqlens are prefix sums)
        n = min(min(left, s.block_size), static_cast<int>(min(s.n_rows - row, static_cast<int64_t>(INT32_MAX))));
        block = page_of(s.seqs, s.n_blocks, b, i / s.block_size, s.status);
      }
    }
    if (row == s.n_rows - 1 && h == 0 && s.seqs.cu_seqlens[s.seqs.n_seqs] > s.n_rows)
      record_error(s.status, DKV_ERR_INVALID_ARGUMENT);
  }
  uint32_t first = __ballot_sync(0xffffffffu, block >= 0);
  while (first) {
    const int i = __ffs(first) - 1;
    first &= first - 1;
    store_run<SDT, PDT, VEC, true>(s, s.side[0], h, false, r0 + i, __shfl_sync(0xffffffffu, n, i),
                                   __shfl_sync(0xffffffffu, block, i), lane);
  }
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

template <int PDT, int ODT, int VEC>
__device__ __forceinline__ void read_piece(const uint8_t *src, float scale, bool there, typename Elem<ODT>::T *dst) {
  if constexpr (VEC == 16) {
    const uint4 w = there ? *reinterpret_cast<const uint4 *>(src) : make_uint4(0, 0, 0, 0);
    const uint32_t c[4] = {w.x, w.y, w.z, w.w};
    float x[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[4];
      Code<PDT>::unpack(c[i], y);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[4 * i + k] = there ? __fmul_rn(y[k], scale) : 0.f;
    }
    Raw<ODT, 16> y;
    y.set(x), y.store(dst);
  } else {
    float y[4];
    Code<PDT>::unpack(there ? *src : 0, y);
    *dst = Elem<ODT>::from_f(there ? __fmul_rn(y[0], scale) : 0.f);
  }
}

// Bound by memory: each code read once, each value written once.  A CTA first finds its rows' places (one lane each),
// then a thread has 16 columns of a head.
template <int PDT, int ODT, int VEC>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const __grid_constant__ Read a) {
  using OT = typename Elem<ODT>::T;
  begin_overlapped();
  __shared__ int64_t block_at[kReadRows];  // -1: zeros, -2: left alone
  __shared__ int slot_at[kReadRows];
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
    block_at[tid] = block, slot_at[tid] = slot;
  }
  __syncthreads();
  const int pieces = a.hd / VEC, per_row = a.heads * pieces, all = n * per_row;
#pragma unroll 4
  for (int i = tid; i < all; i += kReadThreads) {
    const int r = i / per_row, in = i - r * per_row, h = in / pieces, d = (in - h * pieces) * VEC;
    const int64_t block = block_at[r];
    if (block == -2) continue;
    const bool there = block >= 0;
    const int64_t at = there ? block : 0;
    const uint8_t *src = a.pages + at * a.block + slot_at[r] * a.slot + h * a.head + d;
    const float scale = there ? a.scale[at * a.scale_block + h * a.scale_head] : 0.f;
    read_piece<PDT, ODT, VEC>(src, scale, there, static_cast<OT *>(a.out) + (r0 + r) * a.out_row + h * a.out_head + d);
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
int64_t page_bits(const Side &x) { return reinterpret_cast<intptr_t>(x.pages) | x.block | x.slot | x.head; }

// Rows that a warp looks through: a row each as long as all warps that come of it run about at once (64 an SM), else up to
// 16, so that prefill rows, of which one in a block's worth begins a run, do not launch a warp each.
int window_of(int64_t rows, int64_t warps_a_row, int sms) {
  int w = 1;
  while (w < 16 && rows * warps_a_row > static_cast<int64_t>(sms) * 64 * w) w *= 2;
  return w;
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
  s.n_rows = g.n_rows;
  s.n_blocks = kp.num_blocks < vp.num_blocks ? kp.num_blocks : vp.num_blocks;
  s.n_slots = s.n_blocks * kp.block_size, s.narrow = s.n_slots <= UINT32_MAX;
  s.slots = g.slots, s.positions = g.positions, s.cos_t = g.rope_cos, s.sin_t = g.rope_sin;
  s.rope_max_pos = g.rope_max_pos;
  s.status = g.status;
  s.heads = kp.n_heads, s.hd = kp.head_dim, s.block_size = kp.block_size;
  s.rot = rot;
  step::Append q;
  step::describe(g, rot, &q);
  const int64_t size = g.in_dtype == DKV_F32 ? 4 : 2;
  int64_t bits = quant::source_bits(s.side[0], size) | quant::source_bits(s.side[1], size);
  bits |= reinterpret_cast<intptr_t>(g.rope_cos) | reinterpret_cast<intptr_t>(g.rope_sin);
  if (g.q != nullptr)
    bits |= reinterpret_cast<intptr_t>(g.q) | reinterpret_cast<intptr_t>(g.q_out) |
            (q.src_row[0] | q.src_head[0] | q.dst_row[0] | q.dst_head[0]) * size;
  const bool wide = step::whole_pieces(rot, kp.head_dim, 8) && kp.head_dim % 16 == 0 && bits % 16 == 0 &&
                    (quant::page_bits(s.side[0]) | quant::page_bits(s.side[1])) % 8 == 0;
  s.window = quant::window_of(g.n_rows, 2 * kp.n_heads, sms);
  const int64_t warps = (g.n_rows + s.window - 1) / s.window * 2 * kp.n_heads;
  s.ctas = (warps * 32 + quant::kThreads - 1) / quant::kThreads;
  const int64_t threads = q.heads[0] == 0 ? 0 : g.n_rows * ((q.heads[0] + step::kHeads - 1) / step::kHeads) *
                                                    step::pieces_of(rot, kp.head_dim, wide ? 8 : 1);
  q.wide = threads > UINT32_MAX;
  const int64_t ctas = s.ctas + (threads + quant::kThreads - 1) / quant::kThreads;
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
  const bool wide = cache->head_dim % 16 == 0 && quant::source_bits(s.side[0], size) % 16 == 0 &&
                    quant::page_bits(s.side[0]) % 8 == 0;
  s.window = quant::window_of(n_rows, cache->n_heads, sms);
  const int64_t warps = (n_rows + s.window - 1) / s.window * cache->n_heads;
  const int64_t ctas = (warps * 32 + quant::kThreads - 1) / quant::kThreads;
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
  const bool wide = cache->head_dim % 16 == 0 &&
                    (reinterpret_cast<intptr_t>(a.pages) | a.block | a.slot | a.head) % 16 == 0 &&
                    (reinterpret_cast<intptr_t>(out) | out_stride_row * size | out_stride_head * size) % 16 == 0;
  const int64_t ctas = (n_rows + a.rows - 1) / a.rows;
  if (ctas > INT32_MAX || static_cast<int64_t>(a.heads) * a.hd > INT32_MAX / quant::kReadRows - quant::kReadThreads)
    return DKV_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define DKV_QUANT_CASE(P, O)                                                                                  \
  if (cache->dtype == P && out_dtype == O) {                                                                  \
    const auto kernel = wide ? quant::read_kernel<P, O, 16> : quant::read_kernel<P, O, 1>;                    \
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
