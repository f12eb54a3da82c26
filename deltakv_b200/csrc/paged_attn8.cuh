// The walk of the paged decode attention over 8-bit pages (e4m3 or int8 codes, an fp32 scale for each block and KV head).
//
// For sequence b, query head h of KV head u, with codes c, d and scales k, v of the blocks:
//   s_i = scale k_i q.c_i,  m = max_i s_i,  l = sum_i exp(s_i - m),  out = sum_i exp(s_i - m) v_i d_i / l.
// A scale is one factor for a token's whole row, so it multiplies the row's score, or its weight, and the products run
// over the codes themselves: every e4m3 and int8 code is an f16 number, and
//   S^T [16 tokens x 8 heads] = C . Q^T,   O^T [16 columns x 8 heads] += D^T . W^T,   W_i = exp(s_i - m) v_i
// are mma.m16n8k16 in f16 with the tokens (columns) on the wide side, as in the 16-bit walk.  The weights W take V's
// scales, which differ from block to block, so they have a factor 2^up of their own that keeps the largest of them not far
// below 2^8 and all below 2^15 (f16 ends at 2^16): it moves, and O with it, when a scale could lift a weight past that, as m
// does when a score passes it.  m is set 4 above the largest score (a factor of 16), and 2^up so that scales of four times those
// of the heaviest tokens fit: otherwise half of the tiles of a range of a few hundred tokens had one to move.  What an
// f16 weight loses at least is then 2^-25 of 2^8, 2^-33 of the largest weight.
//
// Bytes to fragments: a lane's ldmatrix register holds four codes of one token's row, which become the k-indices
// (2t, 2t + 1) and (2t + 8, 2t + 9) of one product (any order of the head's columns gives the same score, as long as
// q's fragment has it too).  For V, ldmatrix.trans gives a lane the codes of two columns of two tokens; the columns are
// dealt so that a lane's rows g and g + 8 of O^T are neighbours, 16 k + 2 g and + 1, and outputs are stored in pairs.
//
// Measured on a B200 (calls back to back; HBM floor at the measured 6535 GB/s): 32 sequences of 20000..32768, 8 KV heads x 128,
// e4m3: 300-330 us by the box's power (floor 265); 16 of 8192: 56-66 us (41); one of 131071: 57 (41); 64 of 1..8192, int8, f16 q
// of 64 heads: 42-43 (23); 256 of 1..600: 25-26 (7.5).  12 to 15 us of each are fixed (the launch, the first tiles of all SMs at
// once, SMs that get less of the HBM than others, the join); the rest streams at 0.90-0.96 of the peak.
//
// A K or V byte meets twice the arithmetic that it meets in a 16-bit page, so the issue of instructions counts here:
// q is one f16 term where it has 16 bits (exact: scaled by a power of two, 11 bits hold it) and two where it is fp32; W is two
// (2^-22 of itself).  One term of W would do for a bf16 out's own rounding, but not where values cancel; it saves 0-6 %: us,
// bf16 q, one / two: 32 sequences of 26000..30200 303-311 / 316-325, 16 of 8192 62.5 / 64, with 16 heads a KV head 65.5 / 69.5,
// 16 of 16384 of head_dim 64 57.4 / 60.3, of 32768 of 32 85.9 / 89.3, 64 of 1..8192 34.9 / 35.2.
#pragma once

#include "code8.cuh"
#include "paged_walk.cuh"

namespace dkv {
namespace pattn {

__device__ __forceinline__ uint32_t shuffle_bytes(uint32_t a, uint32_t b, uint32_t how) { return __byte_perm(a, b, how); }
__device__ __forceinline__ uint32_t minus_1152(uint32_t x) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t *>(&r);
}

// codes to pairs of f16
template <int PT>
struct Pairs;
template <>
struct Pairs<DKV_E4M3> {
  // bytes 0, 1 and bytes 2, 3
  static __device__ __forceinline__ void in_order(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
  // bytes 0, 2 and bytes 1, 3
  static __device__ __forceinline__ void crossed(uint32_t w, uint32_t &even, uint32_t &odd) {
    in_order(shuffle_bytes(w, 0, 0x3120), even, odd);
  }
};
template <>
struct Pairs<DKV_I8> {  // a byte b behind 0x64 is the f16 number 1024 + b; with b + 128 for b, less 1152 is b
  static __device__ __forceinline__ void in_order(uint32_t w, uint32_t &lo, uint32_t &hi) {
    w ^= 0x80808080u;
    lo = minus_1152(shuffle_bytes(w, 0x64646464u, 0x4140)), hi = minus_1152(shuffle_bytes(w, 0x64646464u, 0x4342));
  }
  static __device__ __forceinline__ void crossed(uint32_t w, uint32_t &even, uint32_t &odd) {
    w ^= 0x80808080u;
    even = minus_1152(shuffle_bytes(w, 0x64646464u, 0x4240)), odd = minus_1152(shuffle_bytes(w, 0x64646464u, 0x4341));
  }
};

// (no side effects: left to the compiler's scheduler, not volatile)
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 16 bytes into shared memory; L2 takes 256 with them, for a row of the next head lies behind most rows and is read by a
// neighbouring warp (32 long sequences, 8 heads x 128: 320 us without, 310 with)
__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// One warp's stream of tiles of 32 tokens into its ring: a stage holds 32 rows of K, as many of V (16 bytes more than a row
// apart: no bank conflicts), their scales and its description.  Two ways to copy:
//   kPages  block_size a multiple of 16: each half of a tile lies in one block (borders fall on multiples of 16), its rows a
//           fixed stride apart.  A lane holds the addresses of one of the next 32 halves, so that the table is waited
//           for, and addresses are worked out, once in 16 tiles;
//   kRows, kPlain  a lane for each token's block and slot, a tile ahead; rows in pieces of 16 bytes, or smaller ones.
// Places in pages and rows are kept in units of 16 bytes, 32 bits for 64 GB (caches beyond that go the kPlain way).
template <int HD, int kStages, typename O>
struct Stream8 {
  static constexpr int kTok = 32;
  static constexpr int kRow = HD + 16;
  static constexpr int kSide = kTok * kRow;
  static constexpr int kStage = 2 * kSide + 2 * kTok * 4;  // K, V, K's scales, V's
  static constexpr int kBytes = kStages * (kStage + 16);   // the stages' descriptions behind them
  static constexpr int kPieces = HD / 16;                  // 16-byte pieces of a row
  static constexpr int kAtOnce = 32 / kPieces;             // rows a copy instruction covers

  const Params &p;
  Walk w;
  char *ring;
  uint4 *meta;  // per stage: sequence, flags, bit per token that takes part, end of the stream
  const char *k, *v;    // of slot 0 of block 0; kPages: this lane's row and piece behind it, kRows: its piece
  const float *ks, *vs;
  uint32_t to;          // where this lane's first piece goes in stage 0
  bool inside;          // this lane's piece is not past head_dim
  int h0, n_h, lane;
  uint64_t k_at, v_at;  // kPlain: the row of this lane's token (0: none); else the row (kPages: half) it looked up, from k, v
  int id, slot;         // its block and slot in it, negative: none
  int tile;             // kPages: of the 16 tiles that the lanes hold, the next
  static constexpr int kNoRow = -1, kShort = INT32_MIN;

  __device__ __forceinline__ Stream8(const Params &p_, char *mine, int u, int h0_, int n_h_, int lane_)
      : p(p_), ring(mine), meta(reinterpret_cast<uint4 *>(mine + kStages * kStage)), k(p_.k + u * p_.k_head),
        v(p_.v + u * p_.v_head), ks(p_.k_scale + u * p_.ks_head), vs(p_.v_scale + u * p_.vs_head), h0(h0_), n_h(n_h_),
        lane(lane_), k_at(0), v_at(0), id(kNoRow), slot(-1), tile(0) {
    const int row = lane / kPieces, piece = lane % kPieces;
    to = smem_u32(ring) + row * kRow + piece * 16;
    inside = piece * 16 < p.hd;
    if (p.copy == kPages) k += row * p.k_slot, v += row * p.v_slot;
    if (p.copy != kPlain) k += piece * 16, v += piece * 16;
    if (p.hd < HD) {  // columns past head_dim stay zero in every stage: only zeros are written there again
      for (int i = lane; i < kStages * kStage / 16; i += 32) reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
  }
  __device__ __forceinline__ float *scales(int s) const { return reinterpret_cast<float *>(ring + s * kStage + 2 * kSide); }
  // Loads a table entry for this lane; what follows from it is worked out (resolve) when the next tile is filled, so that
  // nothing waits for the load here.
  __device__ __forceinline__ void look_up() {
    if (!w.live) return;
    int ahead = lane;
    if (p.copy == kPages) {
      if (++tile < 16 && !(w.flags & kFirst)) return;
      tile = 0;
      ahead = (lane >> 1) * w.step + (lane & 1) * 16;
    }
    id = kNoRow, slot = -1;
    if (ahead >= w.end - w.i) return;
    const int i = w.i + ahead;
    const int blk = static_cast<int>((static_cast<uint64_t>(i) * p.div_mul) >> p.div_shift);
    slot = i - blk * p.block_size;
    id = blk < w.tlen ? max(p.tables[w.b * p.table_stride + blk], kNoRow) : kShort;
  }
  __device__ __forceinline__ void resolve() {
    if (p.copy == kPages && tile != 0) return;
    k_at = v_at = 0;
    if (slot < 0) return;
    if (id < 0 || id >= p.num_blocks) {
      record_error(p.status, id == kShort ? DKV_ERR_BLOCK_TABLE_SHORT : DKV_ERR_PAGE_RANGE);
      id = kNoRow;
      return;
    }
    const int64_t k_off = id * p.k_block + slot * p.k_slot, v_off = id * p.v_block + slot * p.v_slot;
    if (p.copy != kPlain)
      k_at = static_cast<uint32_t>(k_off >> 4), v_at = static_cast<uint32_t>(v_off >> 4);
    else
      k_at = reinterpret_cast<uint64_t>(k + k_off), v_at = reinterpret_cast<uint64_t>(v + v_off);
  }
  __device__ __forceinline__ void start(const Walk &from) {
    w = from;
    if (!p.local) walk_seq<O>(p, w, h0, n_h, lane);
    look_up();
  }
  // 16 rows from `off` on; kAll: else `rows` of them (the others zero)
  template <bool kAll>
  __device__ __forceinline__ void copy_half(uint32_t dst, const char *base, uint32_t off, uint32_t slot_bytes, int rows) {
    const char *src = base + static_cast<uint64_t>(off) * 16;
#pragma unroll
    for (int r = 0; r < 16; r += kAtOnce) {
      const char *from = src + static_cast<uint64_t>(slot_bytes) * static_cast<uint32_t>(r);
      if (kAll) {  // (a register for the size costs several instructions)
        if (inside) copy16(dst + r * kRow, from);
      } else {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + r * kRow), "l"(from),
                     "r"(inside && r + lane / kPieces < rows ? 16 : 0)
                     : "memory");
      }
    }
  }
  // the rows that the lanes looked up; those not in `there` zero
  __device__ __forceinline__ void copy_rows(char *to_rows, uint64_t addr, const char *base, uint32_t there) {
    if (p.copy == kRows) {
      const uint32_t dst = smem_u32(to_rows) + lane / kPieces * kRow + lane % kPieces * 16;
#pragma unroll
      for (int r = 0; r < kTok; r += kAtOnce) {
        const int row = r + lane / kPieces;
        const char *from = base + static_cast<uint64_t>(__shfl_sync(0xffffffffu, static_cast<uint32_t>(addr), row)) * 16;
        if (there == 0xffffffffu) {
          if (inside) copy16(dst + r * kRow, from);
        } else {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + r * kRow), "l"(from),
                       "r"(inside && (there >> row & 1) ? 16 : 0)
                       : "memory");
        }
      }
    } else if (p.piece >= 4) {
      for (int row = 0; row < kTok; ++row) {
        const uint64_t a = __shfl_sync(0xffffffffu, addr, row);
        const char *src = a ? reinterpret_cast<const char *>(a) : base;
        for (int at = lane * p.piece; at < p.hd; at += 32 * p.piece) {
          if (p.piece == 8)
            cp_async8(to_rows + row * kRow + at, src + at, a ? 8 : 0);
          else
            cp_async4(to_rows + row * kRow + at, src + at, a ? 4 : 0);
        }
      }
    } else {
      for (int d = lane; d < (p.hd + 31) / 32 * 32; d += 32) {
        for (int row = 0; row < kTok; row += 8) {  // eight rows' loads in flight
          uint8_t x[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const uint64_t a = __shfl_sync(0xffffffffu, addr, row + r);
            x[r] = a && d < p.hd ? reinterpret_cast<const uint8_t *>(a)[d] : 0;
          }
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (d < p.hd) to_rows[(row + r) * kRow + d] = static_cast<char>(x[r]);
        }
      }
    }
  }
  // issues the next tile's copies into stage s (one cp.async group, empty past the end)
  __device__ __forceinline__ void fill(int s) {
    if (w.live) {
      const int left = w.end - w.i;
      resolve();
      uint32_t there;
      int block;  // of this lane's token, negative: none
      if (p.copy == kPages) {
        block = __shfl_sync(0xffffffffu, id, 2 * tile + lane / 16);
        if (lane >= left) block = kNoRow;
        there = __ballot_sync(0xffffffffu, block >= 0);
        const uint32_t k_step = static_cast<uint32_t>(p.k_slot), v_step = static_cast<uint32_t>(p.v_slot);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t k_off = __shfl_sync(0xffffffffu, static_cast<uint32_t>(k_at), 2 * tile + h);
          const uint32_t v_off = __shfl_sync(0xffffffffu, static_cast<uint32_t>(v_at), 2 * tile + h);
          const uint32_t dst = to + s * kStage + 16 * h * kRow;
          if (there == 0xffffffffu) {
            copy_half<true>(dst, k, k_off, k_step, 16);
            copy_half<true>(dst + kSide, v, v_off, v_step, 16);
          } else {  // (where nothing is there the offsets are 0, and nothing is read)
            const int rows = __popc(there >> (16 * h) & 0xffffu);
            copy_half<false>(dst, k, k_off, k_step, rows);
            copy_half<false>(dst + kSide, v, v_off, v_step, rows);
          }
        }
      } else {
        block = id;
        there = __ballot_sync(0xffffffffu, block >= 0);
        copy_rows(ring + s * kStage, k_at, k, there);
        copy_rows(ring + s * kStage + kSide, v_at, v, there);
      }
      if (p.num_blocks > 0) {
        const uint32_t n = block < 0 ? 0 : 4, at = max(block, 0);
        cp_async4(scales(s) + lane, ks + static_cast<uint64_t>(at) * static_cast<uint32_t>(p.ks_block), n);
        cp_async4(scales(s) + kTok + lane, vs + static_cast<uint64_t>(at) * static_cast<uint32_t>(p.vs_block), n);
      } else {
        scales(s)[lane] = scales(s)[kTok + lane] = 0.f;
      }
      const bool last = !p.local && left <= kTok;
      if (lane == 0) meta[s] = make_uint4(w.b, w.flags | (last ? kLast : 0), there, 0);
      walk_next<O>(p, w, h0, n_h, lane);
      look_up();
    } else if (lane == 0) {
      meta[s] = make_uint4(0, 0, 0, 1);  // the end
    }
    cp_async_commit();
  }
};

constexpr float kSlack = 4.f;  // m above the largest score when it is set, in base 2

// PT: the codes, DT: q and out, NB: blocks of 8 query heads of a unit (a K or V byte becomes an f16 once for all of them).
template <int PT, int DT, int HD, int NB, int W, int kStages>
__global__ void __launch_bounds__(W * 32, 1) walk8_kernel(const __grid_constant__ Params p) {
  using T = typename Elem<DT>::T;
  using S = Stream8<HD, kStages, T>;
  constexpr int kTok = S::kTok;
  constexpr int kTerms = DT == DKV_F32 ? 2 : 1;  // of q
  constexpr int kGroups = HD / 32;  // of 32 columns: one ldmatrix
  constexpr int kBatch = kGroups < 4 ? kGroups : 4;
  constexpr int kSteps = HD / 16;
  constexpr int kHeadsOf = 8 * NB;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  begin_overlapped();
  const int gw = p.local ? blockIdx.x : blockIdx.x * W + warp;
  const int r = gw / p.units, unit = gw - r * p.units;  // r: the range, or the sequence where local
  Line ln;
  Window win;
  if (!p.local) {
    win.look(p, lane);
    ln = line_of(p, p.cu[p.n_seqs]);
    if (r >= static_cast<int>(ln.ranges)) return;
  }
  const int u = unit / p.chunks, chunk = unit - u * p.chunks;
  const int n_h = min(kHeadsOf, p.group - chunk * kHeadsOf), h0 = u * p.group + chunk * kHeadsOf;

  char *mine = smem + warp * S::kBytes;
  S stream(p, mine, u, h0, n_h, lane);
  stream.start(p.local ? local_walk(p, r, kTok, warp, p.local) : range_walk(p, win, ln, r, kTok, lane));

  const int g = lane >> 2, t = lane & 3;
  // ldmatrix rows: K as (token, half of 32 columns), V as (token half, 16 columns) of a 16 x 32 block
  const uint32_t k_at = smem_u32(mine) + (lane & 15) * S::kRow + (lane >> 4) * 16;
  uint32_t qf[NB][kTerms][kGroups][2][2];
  float unit_q[NB][2];  // what a score of heads 2t, 2t + 1 is in base 2, but for the token's scale
  float o[NB][kSteps][4], m[NB][2], l[NB][2], top_z[NB][2];
  int up[NB][2];  // O is in units of 2^-up
  float v_cap;    // V's scales up to which no weight passes 2^15; 0 while a head has no weight that `up` could be set by
  auto clear = [&]() {
    v_cap = 32768.f;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[n][c] = -3e38f;  // below any score, and finite: no case of its own
        l[n][c] = top_z[n][c] = 0.f, up[n][c] = 0;
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][k][e] = 0.f;
    }
  };
  auto over_tokens = [&](float x, auto f) {  // over the lanes that share a head
    x = f(x, __shfl_xor_sync(0xffffffffu, x, 4));
    x = f(x, __shfl_xor_sync(0xffffffffu, x, 8));
    return f(x, __shfl_xor_sync(0xffffffffu, x, 16));
  };
  const auto larger = [](float a, float b) { return fmaxf(a, b); };
  auto sum_of = [&](int n, int c) { return over_tokens(l[n][c], [](float a, float b) { return a + b; }); };
  auto load_q = [&](int b, int nb) {  // (lanes past the unit's heads repeat the last one; their results are not stored)
    const T *qr = reinterpret_cast<const T *>(p.q + b * p.q_seq + (h0 + min(8 * nb + g, n_h - 1)) * p.q_head);
    float x[kGroups][2][4];
    float top = 0.f;
    if (DT != DKV_F32 && p.pairs) {  // outside the loops: a branch between the loads would have each waited for
      uint32_t w[kGroups][2][2];
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int d = k * 32 + e * 16 + t * 4 + i * 2;
            w[k][e][i] = d < p.hd ? *reinterpret_cast<const uint32_t *>(qr + d) : 0;
          }
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[k][e][2 * i] = DT == DKV_BF16 ? bf16lo(w[k][e][i]) : f16lo(w[k][e][i]);
            x[k][e][2 * i + 1] = DT == DKV_BF16 ? bf16hi(w[k][e][i]) : f16hi(w[k][e][i]);
          }
    } else {
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = k * 32 + e * 16 + t * 4 + i;
            x[k][e][i] = d < p.hd ? Elem<DT>::to_f(qr[d]) : 0.f;
          }
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[k][e][i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the head's largest element to [2^13, 2^14) (an f16 q stays as it is): 27 binary places below it before an f16
    // subnormal loses any of 11 bits, and 448 x 2^14 x 256 columns far within fp32
    const int by_two = DT == DKV_F16 ? 0 : min(140 - static_cast<int>(__float_as_uint(top) >> 23), 126);
    const float by = exp2i(by_two);
#pragma unroll
    for (int k = 0; k < kGroups; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a = x[k][e][2 * i] * by, c = x[k][e][2 * i + 1] * by;
          const uint32_t w = pack_f16x2(a, c);
          qf[nb][0][k][e][i] = w;
          if (kTerms == 2) qf[nb][kTerms - 1][k][e][i] = pack_f16x2(a - f16lo(w), c - f16hi(w));
        }
    const float back = exp2i(-by_two) * p.scale_log2;
    unit_q[nb][0] = __shfl_sync(0xffffffffu, back, t * 8), unit_q[nb][1] = __shfl_sync(0xffffffffu, back, t * 8 + 4);
  };
  clear();

  for (int s = 0; s < kStages; ++s) stream.fill(s);
  for (int s = 0;; s = s + 1 == kStages ? 0 : s + 1) {
    __syncwarp();
    const uint4 mt = stream.meta[s];
    if (mt.w) break;
    const int b = mt.x;
    if (mt.y & kFirst) {
#pragma unroll
      for (int n = 0; n < NB; ++n) load_q(b, n);
      clear();
    }
    cp_async_wait<kStages - 1>();  // after a first tile's q is on its way
    __syncwarp();
    const uint32_t at = k_at + s * S::kStage;
    const float *scales = stream.scales(s);
    // {tokens 16 i + g, 16 i + g + 8} x {heads 2t, 2t + 1}: the codes' products
    float sc[NB][2][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][i][e] = 0.f;
#pragma unroll
    for (int k0 = 0; k0 < kGroups; k0 += kBatch) {
      uint32_t c[2][kBatch][4];  // all loads first: none waits for a product before it
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          ldmatrix_x4(c[i][k][0], c[i][k][1], c[i][k][2], c[i][k][3], at + 16 * i * S::kRow + (k0 + k) * 32);
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {  // tokens g and g + 8 of 16 columns
            uint32_t a[4];
            Pairs<PT>::in_order(c[i][k][2 * e], a[0], a[2]);
            Pairs<PT>::in_order(c[i][k][2 * e + 1], a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
              for (int x = 0; x < kTerms; ++x) mma_f16(sc[n][i], a, qf[n][x][k0 + k][e]);
          }
    }
    float k_scale[2][2], v_scale[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        k_scale[i][e] = scales[16 * i + g + 8 * e], v_scale[i][e] = scales[kTok + 16 * i + g + 8 * e];
    const float kNegInf = __int_as_float(0xff800000);
    auto absent = [&](int i, int e) { return !((mt.z >> (16 * i + g + (e & 2) * 4)) & 1); };
    const float most = fmaxf(fmaxf(fabsf(v_scale[0][0]), fabsf(v_scale[0][1])), fmaxf(fabsf(v_scale[1][0]), fabsf(v_scale[1][1])));
    float wt[NB][2][4];  // how far a score is above m, then its weight
    bool moves = most > v_cap;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) wt[n][i][e] = fmaf(sc[n][i][e], k_scale[i][e >> 1] * unit_q[n][e & 1], -m[n][e & 1]);
      if (mt.z != 0xffffffffu) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (absent(i, e)) wt[n][i][e] = kNegInf;
      }
      const float(&x)[2][4] = wt[n];
      moves |= fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                     fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3]))) > 0.f;
    }
    // m is any value not far from the largest score so far, 2^up any factor that keeps the weights of V's codes below
    // 2^15 and the largest of them not far below 2^8: they move (and l, O with them) only when a score passes m or a scale
    // of V's could lift a weight too high, which after the first tile is rare; and with every V scale that is not 0 until
    // there is a weight to set 2^up by (a range may begin with tokens whose values are all zero)
    if (__any_sync(0xffffffffu, moves)) {
      int highest = -126;
      bool unset = false;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            wt[n][i][e] = absent(i, e) ? kNegInf : sc[n][i][e] * (k_scale[i][e >> 1] * unit_q[n][e & 1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float(&x)[2][4] = wt[n];
          const float best = over_tokens(fmaxf(fmaxf(x[0][c], x[0][c + 2]), fmaxf(x[1][c], x[1][c + 2])), larger);
          const float next_m = best > m[n][c] ? best + kSlack : m[n][c];
          float z = 0.f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              x[i][c + 2 * e] -= next_m;
              z = fmaxf(z, fabsf(ex2(x[i][c + 2 * e]) * v_scale[i][e]));
            }
          const float keep = ex2(m[n][c] - next_m);
          top_z[n][c] = fmaxf(top_z[n][c] * keep, over_tokens(z, larger));
          // the largest weight to [2^8, 2^9)
          const int next = top_z[n][c] > 0.f
                               ? max(min(135 - static_cast<int>(__float_as_uint(top_z[n][c]) >> 23), 126), -111)
                               : up[n][c];
          // (O is 0 wherever the exponent could pass 126: it has no weight yet, or m has moved by more than 126)
          const float keep_o = ex2(fminf(m[n][c] - next_m + static_cast<float>(next - up[n][c]), 126.f));
          l[n][c] *= keep;
          m[n][c] = next_m, up[n][c] = next;
          highest = max(highest, next), unset |= top_z[n][c] == 0.f;
#pragma unroll
          for (int k = 0; k < kSteps; ++k) o[n][k][c] *= keep_o, o[n][k][2 + c] *= keep_o;
        }
      }
      v_cap = unset ? 0.f : exp2i(15 - highest);
    }
    uint32_t w[NB][2][2][2];  // two terms
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float lift[2] = {exp2i(up[n][0]), exp2i(up[n][1])};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = ex2(wt[n][i][e]);
          l[n][e & 1] += y;
          wt[n][i][e] = y * lift[e & 1] * v_scale[i][e >> 1];  // (the other product could be infinite where y is 0)
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float *y = wt[n][i] + 2 * c;
          const uint32_t v = pack_f16x2(y[0], y[1]);
          w[n][i][0][c] = transpose_8x8(v);
          w[n][i][1][c] = transpose_8x8(pack_f16x2(y[0] - f16lo(v), y[1] - f16hi(v)));
        }
      }
    }
#pragma unroll
    for (int k0 = 0; k0 < kGroups; k0 += kBatch) {
      uint32_t c[2][kBatch][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          ldmatrix_x4_trans(c[i][k][0], c[i][k][1], c[i][k][2], c[i][k][3],
                            at + S::kSide + 16 * i * S::kRow + (k0 + k) * 32);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // columns 32 k + 16 e + 2 g and + 1, tokens 2t, 2t + 1 and 2t + 8, 2t + 9
            uint32_t a[4];
            Pairs<PT>::crossed(c[i][k][2 * e], a[0], a[1]);
            Pairs<PT>::crossed(c[i][k][2 * e + 1], a[2], a[3]);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
              for (int x = 0; x < 2; ++x) mma_f16(o[n][2 * (k0 + k) + e], a, w[n][i][x]);
          }
    }
    if (mt.y & kLast) {
      const bool whole = (mt.y & kFromStart) && (mt.y & kToEnd);
      const int64_t part = (static_cast<int64_t>(r) * p.units + unit) * 2 + (mt.y & kFromStart ? 1 : 0);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int in = 8 * n + t * 2 + c;
          const float sum = sum_of(n, c), by = exp2i(-up[n][c]);
          if (in >= n_h) continue;
          if (whole) {
            const float inv = sum == 0.f ? 0.f : by / sum;
            T *dst = reinterpret_cast<T *>(p.out + b * p.out_seq + (h0 + in) * p.out_head);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              const int d = k * 16 + 2 * g;
              const float lo = o[n][k][c] * inv, hi = o[n][k][2 + c] * inv;
              if (DT != DKV_F32 && p.pairs) {
                if (d < p.hd)
                  *reinterpret_cast<uint32_t *>(dst + d) = DT == DKV_BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
              } else {
                if (d < p.hd) dst[d] = Elem<DT>::from_f(lo);
                if (d + 1 < p.hd) dst[d + 1] = Elem<DT>::from_f(hi);
              }
            }
            if (p.lse && g == 0)
              p.lse[static_cast<int64_t>(b) * p.heads + h0 + in] = (m[n][c] + log2f(sum)) * 0.6931471805599453f;
          } else {
            float *dst = p.part_o + (part * kHeadsOf + in) * p.hd;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              const int d = k * 16 + 2 * g;
              if (d < p.hd) dst[d] = o[n][k][c] * by;
              if (d + 1 < p.hd) dst[d + 1] = o[n][k][2 + c] * by;
            }
            if (g == 0) {
              p.part_ml[(part * kHeadsOf + in) * 2] = m[n][c];
              p.part_ml[(part * kHeadsOf + in) * 2 + 1] = sum;
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
    using State = LocalState<HD, kHeadsOf>;
    State *mine_out = reinterpret_cast<State *>(mine);
    static_assert(sizeof(State) <= kStages * S::kStage, "the state fits the ring");
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int in = 8 * n + t * 2 + c;
        const float sum = sum_of(n, c), by = exp2i(-up[n][c]);
        if (g == 0) mine_out->m[in] = m[n][c], mine_out->l[in] = sum;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          mine_out->o[in][k * 16 + 2 * g] = o[n][k][c] * by;
          mine_out->o[in][k * 16 + 2 * g + 1] = o[n][k][2 + c] * by;
        }
      }
    local_join<DT, HD, kHeadsOf>(p, smem, S::kBytes, p.local, r, h0, n_h);
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
// Warps of a CTA (one an SM) and stages of a warp's ring, as registers and 227 KB allow.  Three stages of eight warps stream
// better than two of twelve (one range's eight heads on one SM, whose rows are neighbours in memory); where arithmetic or
// many short sequences bound it, twelve are a little better.  us, 8 KV heads: head_dim 128, 8 x 3 / 12 x 2: 32 sequences of
// 26000..30200 303 / 323, 16 of 8192 61 / 61, 64 of 1..8192 35.6 / 36.5, 256 of 1..600 25.7 / 24.3, block_size 24 (rows looked up one
// by one) 74 / 63.  head_dim 64, 16 x 2 / 14 x 3 / 8 x 5: 16 of 16384 60.7 / 64.6 / 75.2.  32, 16 x 4 / 12 x 5 / 8 x 8: 16 of
// 32768 89.5 / 98.7 / 121.5.  256, 6 x 2 / 4 x 3: 16 of 4096 60.1 / 62.6.
constexpr Variant variant8(bool f32, int hd, int heads) {
  if (hd == 256) return {6, 2, 32};
  if (hd == 128) return {8, 3, 32};
  if (heads == 16) return hd == 64 ? Variant{12, 3, 32} : Variant{12, 4, 32};
  return hd == 64 ? (f32 ? Variant{12, 3, 32} : Variant{16, 2, 32}) : Variant{16, 4, 32};
}
// Query heads of a unit: 16 where a KV head has more than eight and registers allow it (16 sequences of 8192, 16 heads for each
// of 8 KV heads x 128: 70 us, as two units of eight 92, with twelve warps 105).
constexpr int heads8(bool f32, int hd, int group) { return !f32 && hd <= 128 && group > 8 ? 16 : 8; }
// A sequence costs more tokens than in the 16-bit walk, whose tokens take longer.  At 48 / 80 / 160, us: 64 sequences of
// 1..8192 41.0 / 35.6 / 36.7, 256 of 1..600 25.3 / 25.7 / 30.8.
constexpr int kSeqCost8 = 80;
// CTAs of one warp lose to ranges (148 sequences of 64 / 150 tokens: 13.7 / 20.1 us in one launch, 11.8 / 16.4 split); of two,
// they win (60 of 300: 12.8 against 17.0), as do more (37 of 500: 11.3 against 17.8; 18 of 1000: 11.6 against 16.3, of
// 1..1000 11.3 against 10.7).
constexpr int kLeastLocal8 = 2;

template <int PT, int DT, int HD, int NB>
int launch_walk8(const Params &p, const Shape &s, cudaStream_t st) {
  constexpr Variant v = variant8(DT == DKV_F32, HD, 8 * NB);
  constexpr int kWarp = Stream8<HD, v.stages, typename Elem<DT>::T>::kBytes;
  static_assert(v.warps * kWarp <= 227 * 1024, "shared memory of the walk");
  const auto kernel = walk8_kernel<PT, DT, HD, NB, v.warps, v.stages>;
  const int rc = allow_smem<walk8_kernel<PT, DT, HD, NB, v.warps, v.stages>>(v.warps * kWarp);
  if (rc != DKV_OK) return rc;
  const int64_t all = static_cast<int64_t>(s.ranges) * s.units;
  const int64_t ctas = s.local ? static_cast<int64_t>(p.n_seqs) * s.units : (all + v.warps - 1) / v.warps;
  const int warps = p.local ? p.local : v.warps;
  DKV_CUDA_CHECK(launch_overlapped(kernel, dim3(static_cast<unsigned>(ctas)), warps * 32, warps * kWarp, st, p));
  return DKV_OK;
}

template <int PT, int DT, int HD>
int launch_walk8(const Params &p, const Shape &s, cudaStream_t st) {
  if constexpr (heads8(DT == DKV_F32, HD, 16) == 16)
    if (s.g == 16) return launch_walk8<PT, DT, HD, 2>(p, s, st);
  return launch_walk8<PT, DT, HD, 1>(p, s, st);
}

template <int PT, int DT>
int launch8(const Params &p, const Shape &s, cudaStream_t st) {
  const int rc = s.hd_pad == 32    ? launch_walk8<PT, DT, 32>(p, s, st)
                 : s.hd_pad == 64  ? launch_walk8<PT, DT, 64>(p, s, st)
                 : s.hd_pad == 128 ? launch_walk8<PT, DT, 128>(p, s, st)
                                   : launch_walk8<PT, DT, 256>(p, s, st);
  return rc != DKV_OK ? rc : launch_join(DT, p, s, st);
}

template <int PT>
int launch8(int q_dtype, const Params &p, const Shape &s, cudaStream_t st) {
  switch (q_dtype) {
    case DKV_F32: return launch8<PT, DKV_F32>(p, s, st);
    case DKV_F16: return launch8<PT, DKV_F16>(p, s, st);
    default: return launch8<PT, DKV_BF16>(p, s, st);
  }
}
int launch8_int8(int q_dtype, const Params &p, const Shape &s, cudaStream_t st);  // paged_attn8_int8.cu

}  // namespace pattn
}  // namespace dkv
