// The rows that a step writes, for the stores into 16- and 32-bit pages (paged_step.cu) and 8-bit ones (paged_quant.cu):
// pieces of a head's columns, their rotation, and the append of rows that keep their type.
#pragma once

#include "dkv_common.cuh"

namespace dkv {
namespace step {

// A rotary form: the first dim columns of a head turn in pairs (i, i + dim / 2), or (2 i, 2 i + 1) where
// interleaved, by the angle i of the row's position; the other columns stay.  dim 0: none turn.
struct Rotary {
  int dim, interleaved;
};

// A thread's two pieces of VEC columns: of a pair's first and second columns, or (interleaved) one behind the other;
// of the columns that stay, a piece of each half.
struct Columns {
  int one, two, angle;
  bool pair, turn;  // pair: false where an odd number of columns stays and this one has no partner
};
__host__ __device__ __forceinline__ int pieces_of(const Rotary &r, int hd, int vec) {
  return r.dim / 2 / vec + ((hd - r.dim + 1) / 2 + vec - 1) / vec;
}
template <int VEC>
__device__ __forceinline__ Columns columns_of(const Rotary &r, int hd, int piece) {
  Columns c;
  const int turning = r.dim / 2 / VEC;
  c.turn = piece < turning;
  if (c.turn) {
    c.angle = piece * VEC;
    c.one = r.interleaved ? 2 * c.angle : c.angle;
    c.two = r.interleaved ? c.one + VEC : c.one + r.dim / 2;
    c.pair = true;
  } else {
    c.angle = 0;
    c.one = r.dim + (piece - turning) * VEC;
    c.two = c.one + (hd - r.dim + 1) / 2;
    c.pair = c.two < hd;
  }
  return c;
}
// whether pieces of vec columns cover the head: then they and the angles' start on whole pieces
__host__ __forceinline__ bool whole_pieces(const Rotary &r, int hd, int vec) {
  return r.dim % (2 * vec) == 0 && (hd - r.dim) % (2 * vec) == 0;
}

// VEC consecutive elements of a type as they lie in memory, in 16-byte pieces (one: as it is)
template <int DT, int VEC>
struct Raw {
  static constexpr int kPieces = VEC * static_cast<int>(sizeof(typename Elem<DT>::T)) / 16;
  uint4 v[kPieces];
  __device__ __forceinline__ void load(const typename Elem<DT>::T *src) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) v[i] = reinterpret_cast<const uint4 *>(src)[i];
  }
  __device__ __forceinline__ void store(typename Elem<DT>::T *dst) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4 *>(dst)[i] = v[i];
  }
  __device__ __forceinline__ float get(int i) const {
    const int per = VEC / kPieces;
    const uint4 u = v[i / per];
    const int e = i % per;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (DT == DKV_F32) return __uint_as_float(w[e & 3]);
    const uint32_t x = w[(e / 2) & 3];
    return DT == DKV_BF16 ? (e & 1 ? bf16hi(x) : bf16lo(x)) : (e & 1 ? f16hi(x) : f16lo(x));
  }
  __device__ __forceinline__ void set(const float (&x)[VEC]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const float *y = x + i * (VEC / kPieces);
      if constexpr (DT == DKV_F32)
        v[i] = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
      else if constexpr (DT == DKV_BF16)
        v[i] = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                          pack_bf16x2(y[6], y[7]));
      else
        v[i] = make_uint4(pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]), pack_f16x2(y[4], y[5]),
                          pack_f16x2(y[6], y[7]));
    }
  }
};
template <int DT>
struct Raw<DT, 1> {
  typename Elem<DT>::T v;
  __device__ __forceinline__ void load(const typename Elem<DT>::T *src) { v = src[0]; }
  __device__ __forceinline__ void store(typename Elem<DT>::T *dst) const { dst[0] = v; }
  __device__ __forceinline__ float get(int) const { return Elem<DT>::to_f(v); }
  __device__ __forceinline__ void set(const float (&x)[1]) { v = Elem<DT>::from_f(x[0]); }
};

// turns a thread's columns; products and sum are each rounded, as the reference's tensor operations do
__device__ __forceinline__ void turn_pair(float &u, float &v, float c, float s) {
  const float x = u, y = v;
  u = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
  v = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
}
template <int VEC>
__device__ __forceinline__ void turn(float (&lo)[VEC], float (&hi)[VEC], const Raw<DKV_F32, VEC> &c,
                                     const Raw<DKV_F32, VEC> &s, bool interleaved) {
  if (VEC > 1 && interleaved) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      turn_pair(lo[2 * i], lo[2 * i + 1], c.get(i), s.get(i));
      turn_pair(hi[2 * i], hi[2 * i + 1], c.get(VEC / 2 + i), s.get(VEC / 2 + i));
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) turn_pair(lo[i], hi[i], c.get(i), s.get(i));
  }
}

constexpr int kAppThreads = 128;

struct Append {
  const void *src[3];  // q, k, v
  void *dst[3];        // q_out, K pages, V pages
  int64_t src_row[3], src_head[3];
  int64_t dst_row[3], dst_head[3];  // dst_row: q_out's row stride, the pages' slot stride
  int64_t dst_block[3];
  const int64_t *slots;
  const int32_t *positions;
  const float *cos_t, *sin_t;
  int64_t n_rows, n_slots;
  int32_t *status;
  int heads[3];
  int hd, half, block_size, rope_max_pos;  // half: of the head
  Rotary rot;  // the forms' kernels only
  int wide;  // more than 2^32 threads
};

constexpr int kHeads = 4;  // of a thread, see append_kernel

// Thread e of an append: its piece of up to kHeads heads of its row.  kForms: any rotary form, else rotate-half over the
// whole head (or none), whose columns need no division.
template <int SDT, int PDT, int VEC, bool kForms>
__device__ __forceinline__ void append_rows(const Append &a, int64_t e) {
  using ST = typename Elem<SDT>::T;
  using PT = typename Elem<PDT>::T;
  const int all = a.heads[0] + a.heads[1] + a.heads[2];
  const int cols = kForms ? pieces_of(a.rot, a.hd, VEC) : a.half / VEC;
  const int groups = (all + kHeads - 1) / kHeads, per_row = cols * groups;
  const int64_t row = a.wide ? e / per_row : static_cast<uint32_t>(e) / static_cast<uint32_t>(per_row);
  if (row >= a.n_rows) return;
  const int in = static_cast<int>(e - row * per_row);
  const int hg = in / cols;
  Columns at;
  if (kForms) {
    at = columns_of<VEC>(a.rot, a.hd, in - hg * cols);
  } else {
    at.one = at.angle = (in - hg * cols) * VEC, at.two = at.one + a.half;
    at.pair = at.two < a.hd;  // false only for the middle of an odd head without RoPE
    at.turn = a.cos_t != nullptr;
  }

  const int64_t slot = a.slots[row];
  const int pos = a.cos_t ? a.positions[row] : 0;
  Raw<SDT, VEC> x[kHeads][2];
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    int h = hg + k * groups;
    if (h >= all) break;
    const int w = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
    h -= w == 0 ? 0 : w == 1 ? a.heads[0] : a.heads[0] + a.heads[1];
    const ST *src = static_cast<const ST *>(a.src[w]) + row * a.src_row[w] + h * a.src_head[w];
    x[k][0].load(src + at.one);
    if (at.pair) x[k][1].load(src + at.two);
  }
  if (a.cos_t && (pos < 0 || pos >= a.rope_max_pos)) {
    record_error(a.status, DKV_ERR_ROPE_RANGE);
    return;
  }
  if (slot >= a.n_slots) record_error(a.status, DKV_ERR_PAGE_RANGE);
  const bool kept = slot >= 0 && slot < a.n_slots;
  Raw<DKV_F32, VEC> c, s;
  if (at.turn) {
    const int64_t row_at = static_cast<int64_t>(pos) * (kForms ? a.rot.dim / 2 : a.half) + at.angle;
    c.load(a.cos_t + row_at);
    s.load(a.sin_t + row_at);
  }
  const int64_t block = kept ? slot / a.block_size : 0;
  const int64_t off = kept ? slot - block * a.block_size : 0;
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    int h = hg + k * groups;
    if (h >= all) break;
    const int w = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
    h -= w == 0 ? 0 : w == 1 ? a.heads[0] : a.heads[0] + a.heads[1];
    if (w && !kept) continue;
    float lo[VEC], hi[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) lo[i] = x[k][0].get(i), hi[i] = at.pair ? x[k][1].get(i) : 0.f;
    if (at.turn && w < 2) turn<VEC>(lo, hi, c, s, kForms && a.rot.interleaved);
    if (w == 0) {
      ST *dst = static_cast<ST *>(a.dst[0]) + row * a.dst_row[0] + h * a.dst_head[0];
      Raw<SDT, VEC> y;
      y.set(lo), y.store(dst + at.one);
      if (at.pair) y.set(hi), y.store(dst + at.two);
    } else {
      PT *dst = static_cast<PT *>(a.dst[w]) + block * a.dst_block[w] + off * a.dst_row[w] + h * a.dst_head[w];
      Raw<PDT, VEC> y;
      y.set(lo), y.store(dst + at.one);
      if (at.pair) y.set(hi), y.store(dst + at.two);
    }
  }
}

// ---- host side ----
// The form that an entry was given, into *to: 0 rotate-half over the whole head or none, 1 another, negative: none of
// the kernels'.
inline int rotary_of(bool turns, const dkv_rotary *asked, int hd, Rotary *to) {
  to->dim = turns ? (asked != nullptr ? asked->dim : hd) : 0;
  to->interleaved = turns && asked != nullptr && asked->interleaved != 0;
  if (!turns) return 0;
  if (to->dim <= 0 || to->dim > hd || (to->dim & 1)) return -1;
  return to->dim != hd || to->interleaved;
}

// everything but the numbers of K and V heads
inline void describe(const dkv_append_args &g, const Rotary &rot, Append *to) {
  Append &a = *to;
  const dkv_paged_cache &kp = g.k_pages, &vp = g.v_pages;
  a.src[0] = g.q, a.src[1] = g.k, a.src[2] = g.v;
  a.dst[0] = g.q_out, a.dst[1] = kp.base, a.dst[2] = vp.base;
  a.src_row[0] = g.q_stride_row, a.src_row[1] = g.k_stride_row, a.src_row[2] = g.v_stride_row;
  a.src_head[0] = g.q_stride_head, a.src_head[1] = g.k_stride_head, a.src_head[2] = g.v_stride_head;
  a.dst_row[0] = g.q_out_stride_row, a.dst_row[1] = kp.stride_slot, a.dst_row[2] = vp.stride_slot;
  a.dst_head[0] = g.q_out_stride_head, a.dst_head[1] = kp.stride_head, a.dst_head[2] = vp.stride_head;
  a.dst_block[0] = 0, a.dst_block[1] = kp.stride_block, a.dst_block[2] = vp.stride_block;
  a.slots = g.slots, a.positions = g.positions, a.cos_t = g.rope_cos, a.sin_t = g.rope_sin;
  a.n_rows = g.n_rows;
  a.n_slots = (kp.num_blocks < vp.num_blocks ? kp.num_blocks : vp.num_blocks) * kp.block_size;
  a.status = g.status;
  a.heads[0] = g.q != nullptr ? g.n_q_heads : 0, a.heads[1] = a.heads[2] = 0;
  a.hd = kp.head_dim, a.half = (kp.head_dim + 1) / 2, a.block_size = kp.block_size, a.rope_max_pos = g.rope_max_pos;
  a.rot = rot;
  a.wide = 0;
}

}  // namespace step
}  // namespace dkv
