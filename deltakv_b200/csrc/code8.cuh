// The 8-bit codes of a paged cache: a value is its code (e4m3 or int8) times the fp32 scale of its block and KV head.
//
// The scale of a block's head that holds nothing is the least that its values fit: a power of two for e4m3 (a
// floating-point code loses nothing by that, every value is exact in bf16, and a scale that grows by powers of two
// moves codes without rounding them again, above the subnormals), amax times 1 / 127 in fp32 for int8.  A scale that is too small
// for values to come grows by the least power of two that lets them fit, and the codes that it held are rounded once
// more: by half a step of the scale after each of its growths, so by less than one step of the last scale in all.
#pragma once

#include "dkv_common.cuh"

namespace dkv {
namespace code8 {

template <int PT>
struct Code;
template <>
struct Code<DKV_E4M3> {
  static constexpr float kMost = 448.f;
  static constexpr float kFits = 448.f;  // the largest value, in steps, for which a held scale stays
  static __device__ __forceinline__ float first_scale(float top) {
    const float x = __fmul_rn(top, 1.f / kMost);
    if (!(x > 1.17549435e-38f)) return 1.17549435e-38f;
    const uint32_t b = __float_as_uint(x);
    return __uint_as_float(((b >> 23) + ((b & 0x7fffffu) != 0)) << 23);
  }
  // four values to four codes; they fit, NaN stays NaN
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
    uint32_t w;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(w)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return w;
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float (&x)[4]) {
    asm("{\n\t.reg .b16 l, h, a, b;\n\t.reg .b32 u, v;\n\tmov.b32 {l, h}, %4;\n\t"
        "cvt.rn.f16x2.e4m3x2 u, l;\n\tcvt.rn.f16x2.e4m3x2 v, h;\n\t"
        "mov.b32 {a, b}, u;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t"
        "mov.b32 {a, b}, v;\n\tcvt.f32.f16 %2, a;\n\tcvt.f32.f16 %3, b;\n\t}"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
        : "r"(w));
  }
};
template <>
struct Code<DKV_I8> {
  static constexpr float kMost = 127.f;
  static constexpr float kFits = 127.5f;  // up to there the nearest code is off by half a step at most
  static __device__ __forceinline__ float first_scale(float top) { return fmaxf(__fmul_rn(top, 1.f / kMost), 1.17549435e-38f); }
  // Whole numbers by way of fp32 numbers around 2^23, whose last place is 1: adding 1.5 x 2^23 rounds to the nearest one, ties
  // to even.  (The conversion instructions run at a quarter of the rate.)
  static __device__ __forceinline__ uint32_t one(float v) {
    return __float_as_uint(__fadd_rn(fminf(fmaxf(v, -127.f), 127.f), 12582912.f));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(one(a), one(b), 0x0040), __byte_perm(one(c), one(d), 0x0040), 0x5410);
  }
  static __device__ __forceinline__ void unpack(uint32_t w, float (&x)[4]) {
    w ^= 0x80808080u;  // 128 more, behind the exponent of 2^23
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __fsub_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | i)), 8388736.f);
  }
};

// The scale of a block's head whose values to store have the largest magnitude `top` (its bits; not finite: NaN),
// given the scale of what it keeps (0: nothing).
template <int PT>
__device__ __forceinline__ float scale_for(uint32_t top_bits, float held) {
  if (top_bits >= 0x7f800000u || held != held) return __uint_as_float(0x7fffffffu);
  const float top = __uint_as_float(top_bits);
  if (top == 0.f) return held > 0.f ? held : 0.f;
  const float first = Code<PT>::first_scale(top);
  if (!(held > 0.f)) return first;
  const float over = __fdiv_rn(top, __fmul_rn(Code<PT>::kFits, held));
  if (over <= 1.f) return held;
  const uint32_t b = __float_as_uint(over);
  if (b >= 0x7f800000u) return first;  // beyond any power of two of fp32
  return ldexpf(held, static_cast<int>(b >> 23) - 127 + ((b & 0x7fffffu) != 0));
}
// what values are multiplied by on the way to codes
__device__ __forceinline__ float inverse_of(float scale) { return scale == 0.f ? 0.f : __fdiv_rn(1.f, scale); }

}  // namespace code8
}  // namespace dkv
