// The walk of the paged decode attention over 8-bit pages (e4m3 or int8 codes, an fp32 scale for each block and KV head).
//
// For sequence b, query head h of KV head u, with codes c, d and scales k, v of the blocks:
//   s_i = scale k_i q.c_i,  m = max_i s_i,  l = sum_i exp(s_i - m),  out = sum_i exp(s_i - m) v_i d_i / l.
// A scale is one factor for a token's whole row, so it multiplies the row's score, or its weight, and the products run
// over the codes themselves: every e4m3 and int8 code is an f16 number, and
//   S^T [16 tokens x 8 heads] = C . Q^T,   O^T [16 columns x 8 heads] += D^T . W^T,   W_i = exp(s_i - m) v_i
// are mma.m16n8k16 in f16 with the tokens (columns) on the wide side, as in the 16-bit walk.  The weights W take V's
// scales, which differ from block to block, so they have a running maximum of their own: M = max_i (s_i + log2 of v_i's
// power of two) keeps the largest W between 1 and 2, as m keeps the largest exp(s_i - m) at 1; O is in units of
// 2^M and l of 2^m until a piece ends.
//
// Bytes to fragments: a lane's ldmatrix register holds four codes of one token's row, which become the k-indices
// (2t, 2t + 1) and (2t + 8, 2t + 9) of one product (any order of the head's columns gives the same score, as long as
// q's fragment has it too).  For V, ldmatrix.trans gives a lane the codes of two columns of two tokens; the columns are
// dealt so that a lane's rows g and g + 8 of O^T are neighbours, 16 k + 2 g and + 1, and outputs are stored in pairs.
//
// A K or V byte meets twice the arithmetic that it meets in a 16-bit page, so the issue of instructions counts here:
// q is one f16 term where it has 16 bits (exact: scaled by a power of two, 11 bits hold it) and two where it is fp32; W is one
// term where out is bf16 (off by 2^-11 of itself at most, where out's own rounding is 2^-8), else two (2^-22).
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
    lo = e4m3x2_to_f16x2(w), hi = e4m3x2_to_f16x2(w >> 16);
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

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Weights carry 2^13: they reach down to 2^-27 of the largest with all 11 bits, and stay below 2^15 in f16.
constexpr float kWeightBias = 13.f;

template <int DT, int HD, int kStages>
struct Walk8 {
  using O = typename Elem<DT>::T;
  using S = Stream<uint8_t, HD, kStages, kTile, O, true>;
};

template <int PT, int DT, int HD, int W, int kStages>
__global__ void __launch_bounds__(W * 32, 1) walk8_kernel(const __grid_constant__ Params p) {
  using S = typename Walk8<DT, HD, kStages>::S;
  using T = typename Elem<DT>::T;
  constexpr int kTerms = DT == DKV_F32 ? 2 : 1;    // of q
  constexpr int kWTerms = DT == DKV_BF16 ? 1 : 2;  // of a weight
  constexpr int kGroups = HD / 32;  // of 32 columns: one ldmatrix
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

  char *mine = smem + warp * S::kBytes;
  S stream(p, mine, u, h0, n_h, lane);
  stream.start(p.local ? local_walk(p, r, kTile, warp, p.local) : range_walk(p, win, ln, r, kTile, lane));

  const int g = lane >> 2, t = lane & 3;
  // ldmatrix rows: K as (token, half of 32 columns), V as (token half, 16 columns) of a 16 x 32 block
  const uint32_t k_at = smem_u32(mine) + (lane & 15) * S::kRow + (lane >> 4) * 16;
  const uint32_t v_at = k_at + kTile * S::kRow;
  uint32_t qf[kTerms][kGroups][2][2];
  float unit_q[2];  // what a score of heads 2t, 2t + 1 is in base 2, but for the token's scale
  float o[kSteps][4], m[2], l[2], top_w[2];
  auto clear = [&]() {
    m[0] = m[1] = top_w[0] = top_w[1] = kNegInf;
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
  auto unit_of = [&](int c) {  // O in units of 2^m (O is 0 where no weight was)
    return top_w[c] == kNegInf ? 0.f : ex2(top_w[c] - m[c] - kWeightBias);
  };
  auto load_q = [&](int b) {  // (lanes past the unit's heads repeat the last one; their results are not stored)
    const T *qr = reinterpret_cast<const T *>(p.q + b * p.q_seq + (h0 + min(g, n_h - 1)) * p.q_head);
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
    const int up = DT == DKV_F16 ? 0 : min(140 - static_cast<int>(__float_as_uint(top) >> 23), 126);
    const float by = exp2i(up);
#pragma unroll
    for (int k = 0; k < kGroups; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a = x[k][e][2 * i] * by, c = x[k][e][2 * i + 1] * by;
          const uint32_t w = pack_f16x2(a, c);
          qf[0][k][e][i] = w;
          if (kTerms == 2) qf[kTerms - 1][k][e][i] = pack_f16x2(a - f16lo(w), c - f16hi(w));
        }
    const float back = exp2i(-up) * p.scale_log2;
    unit_q[0] = __shfl_sync(0xffffffffu, back, t * 8), unit_q[1] = __shfl_sync(0xffffffffu, back, t * 8 + 4);
  };
  clear();

  for (int s = 0; s < kStages; ++s) stream.fill(s);
  for (int s = 0;; s = s + 1 == kStages ? 0 : s + 1) {
    __syncwarp();
    const uint4 mt = stream.meta[s];
    if (mt.w) break;
    const int b = mt.x;
    if (mt.y & kFirst) {
      load_q(b);
      clear();
    }
    cp_async_wait<kStages - 1>();  // after a first tile's q is on its way
    __syncwarp();
    float sc[2][4];  // two chains over the head
#pragma unroll
    for (int e = 0; e < 4; ++e) sc[0][e] = sc[1][e] = 0.f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      uint32_t c[4];
      ldmatrix_x4(c[0], c[1], c[2], c[3], k_at + s * S::kStage + k * 32);
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // tokens g and g + 8 of 16 columns
        uint32_t a[4];
        Pairs<PT>::in_order(c[2 * e], a[0], a[2]);
        Pairs<PT>::in_order(c[2 * e + 1], a[1], a[3]);
#pragma unroll
        for (int i = 0; i < kTerms; ++i)
          mma16816(sc[e], a[0], a[1], a[2], a[3], qf[i][k][e][0], qf[i][k][e][1]);
      }
    }
    // x: {token g, token g + 8} x {head 2t, head 2t + 1}
    const float *scales = stream.scales(s);
    const float ks[2] = {scales[g], scales[g + 8]}, vs[2] = {scales[kTile + g], scales[kTile + g + 8]};
    float x[4], y[4], v_rest[2];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (sc[0][e] + sc[1][e]) * ks[e >> 1] * unit_q[e & 1];
    if (mt.z != 0xffffu) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!((mt.z >> (g + (e & 2) * 4)) & 1)) x[e] = kNegInf;
    }
    // V's scales as a power of two and the rest, in [1, 2) (0 and subnormals below it, the very largest in [2, 4))
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t bits = min(max((__float_as_uint(vs[e]) >> 23) & 0xffu, 1u), 253u);
      v_rest[e] = vs[e] * __uint_as_float((254u - bits) << 23);
      const float power = __uint_as_float(0x4b000000u | bits) - 8388735.f;
      y[2 * e] = x[2 * e] + power, y[2 * e + 1] = x[2 * e + 1] + power;
    }
    // m and top_w are any values not far below the largest so far: they move (and l, O with them) only when
    // one passes them, which after the first tiles is rare
    const float top0 = fmaxf(x[0], x[2]), top1 = fmaxf(x[1], x[3]);
    const float tw0 = fmaxf(y[0], y[2]), tw1 = fmaxf(y[1], y[3]);
    if (__any_sync(0xffffffffu, top0 > m[0] || top1 > m[1] || tw0 > top_w[0] || tw1 > top_w[1])) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = c ? top1 : top0, tw = c ? tw1 : tw0;
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
          tw = fmaxf(tw, __shfl_xor_sync(0xffffffffu, tw, k));
        }
        top = fmaxf(top, m[c]), tw = fmaxf(tw, top_w[c]);
        l[c] *= ex2(m[c] - (top == kNegInf ? 0.f : top));
        const float keep = ex2(top_w[c] - (tw == kNegInf ? 0.f : tw));
        m[c] = top, top_w[c] = tw;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) o[k][c] *= keep, o[k][2 + c] *= keep;
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float base = m[c] == kNegInf ? 0.f : m[c];  // nothing seen yet: any finite base
      const float base_w = (top_w[c] == kNegInf ? 0.f : top_w[c]) - kWeightBias;
      l[c] += ex2(x[c] - base) + ex2(x[c + 2] - base);
      y[c] = ex2(y[c] - base_w) * v_rest[0];
      y[c + 2] = ex2(y[c + 2] - base_w) * v_rest[1];
    }
    uint32_t w[kWTerms][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t v = pack_f16x2(y[2 * c], y[2 * c + 1]);
      w[0][c] = transpose_8x8(v);
      if (kWTerms == 2) w[kWTerms - 1][c] = transpose_8x8(pack_f16x2(y[2 * c] - f16lo(v), y[2 * c + 1] - f16hi(v)));
    }
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      uint32_t c[4];
      ldmatrix_x4_trans(c[0], c[1], c[2], c[3], v_at + s * S::kStage + k * 32);
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // columns 32 k + 16 e + 2 g and + 1, tokens 2t, 2t + 1 and 2t + 8, 2t + 9
        uint32_t a[4];
        Pairs<PT>::crossed(c[2 * e], a[0], a[1]);
        Pairs<PT>::crossed(c[2 * e + 1], a[2], a[3]);
#pragma unroll
        for (int i = 0; i < kWTerms; ++i) mma16816(o[2 * k + e], a[0], a[1], a[2], a[3], w[i][0], w[i][1]);
      }
    }
    if (mt.y & kLast) {
      const bool whole = (mt.y & kFromStart) && (mt.y & kToEnd);
      const int64_t part = (static_cast<int64_t>(r) * p.units + unit) * 2 + (mt.y & kFromStart ? 1 : 0);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int in = t * 2 + c;
        const float sum = sum_of(c), by = unit_of(c);
        if (in >= n_h) continue;
        if (whole) {
          const float inv = sum == 0.f ? 0.f : by / sum;
          T *dst = reinterpret_cast<T *>(p.out + b * p.out_seq + (h0 + in) * p.out_head);
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const int d = k * 16 + 2 * g;
            const float lo = o[k][c] * inv, hi = o[k][2 + c] * inv;
            if (DT != DKV_F32 && p.pairs) {
              if (d < p.hd) *reinterpret_cast<uint32_t *>(dst + d) = DT == DKV_BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
            } else {
              if (d < p.hd) dst[d] = Elem<DT>::from_f(lo);
              if (d + 1 < p.hd) dst[d + 1] = Elem<DT>::from_f(hi);
            }
          }
          if (p.lse && g == 0) p.lse[static_cast<int64_t>(b) * p.heads + h0 + in] = (m[c] + log2f(sum)) * 0.6931471805599453f;
        } else {
          float *dst = p.part_o + (part * 8 + in) * p.hd;
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const int d = k * 16 + 2 * g;
            if (d < p.hd) dst[d] = o[k][c] * by;
            if (d + 1 < p.hd) dst[d + 1] = o[k][2 + c] * by;
          }
          if (g == 0) {
            p.part_ml[(part * 8 + in) * 2] = m[c];
            p.part_ml[(part * 8 + in) * 2 + 1] = sum;
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
    static_assert(sizeof(LocalState<HD, 8>) <= kStages * S::kStage, "the state fits the ring");
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int in = t * 2 + c;
      const float sum = sum_of(c), by = unit_of(c);
      if (g == 0) mine_out->m[in] = m[c], mine_out->l[in] = sum;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        mine_out->o[in][k * 16 + 2 * g] = o[k][c] * by;
        mine_out->o[in][k * 16 + 2 * g + 1] = o[k][2 + c] * by;
      }
    }
    local_join<DT, HD, 8>(p, smem, S::kBytes, p.local, r, h0, n_h);
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
// as many warps and stages as registers and shared memory allow
constexpr Variant variant8(bool f32, int hd) {
  if (hd == 256) return f32 ? Variant{8, 3, 16} : Variant{12, 2, 16};
  if (hd == 128) return f32 ? Variant{12, 4, 16} : Variant{16, 3, 16};
  return hd == 64 ? Variant{16, 5, 16} : Variant{16, 8, 16};
}

template <int PT, int DT, int HD>
int launch_walk8(const Params &p, const Shape &s, int grid, cudaStream_t st) {
  constexpr Variant v = variant8(DT == DKV_F32, HD);
  constexpr int kWarp = Walk8<DT, HD, v.stages>::S::kBytes;
  static_assert(v.warps * kWarp <= 227 * 1024, "shared memory of the walk");
  const auto kernel = walk8_kernel<PT, DT, HD, v.warps, v.stages>;
  const int rc = allow_smem<walk8_kernel<PT, DT, HD, v.warps, v.stages>>(v.warps * kWarp);
  if (rc != DKV_OK) return rc;
  const int warps = p.local ? p.local : v.warps;
  DKV_CUDA_CHECK(launch_overlapped(kernel, dim3(grid), warps * 32, warps * kWarp, st, p));
  return DKV_OK;
}

template <int PT, int DT>
int launch8(const Params &p, const Shape &s, cudaStream_t st) {
  const int64_t warps = static_cast<int64_t>(s.ranges) * s.units;
  const int grid = static_cast<int>(s.local ? static_cast<int64_t>(p.n_seqs) * s.units : (warps + s.warps - 1) / s.warps);
  const int rc = s.hd_pad == 32    ? launch_walk8<PT, DT, 32>(p, s, grid, st)
                 : s.hd_pad == 64  ? launch_walk8<PT, DT, 64>(p, s, grid, st)
                 : s.hd_pad == 128 ? launch_walk8<PT, DT, 128>(p, s, grid, st)
                                   : launch_walk8<PT, DT, 256>(p, s, grid, st);
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
