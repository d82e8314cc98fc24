// 4-bit number formats shared by the row quantiser (fp4.cu) and the paged cache (paged.cu, paged_tc.cu): exact roundings to
// e2m1 (values 0, .5, 1, 1.5, 2, 3, 4, 6) under a block scale, and the layout of a cache page.
#pragma once
#include <cuda_fp4.h>

#include "common.cuh"

namespace fp4 {

// four e2m1 bytes -> four f16 pairs (low nibble first); cvt.rn.f16x2.e2m1x2 runs at the rate of a multiplication, a
// quarter of the instructions of taking the nibbles apart
__device__ __forceinline__ void e2m1x8_to_h2x4(uint32_t w, uint32_t o[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}
// (lo, hi) -> byte, round to nearest even, beyond 6 to 6
__device__ __forceinline__ uint32_t f2_to_e2m1x2(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(lo, hi), __NV_E2M1, cudaRoundNearest);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A double as a float that compares with every number of fewer than 24 significant bits as the double does: truncated, with
// the last bit set where something was cut off (the borders of a rounding to e4m3 or, times a scale, to e2m1 are such numbers).
__device__ __forceinline__ float sticky(double x) {
  const float f = __double2float_rz(x);
  return (double)f == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
// a / s in the same sense (a >= 0 finite, s > 0 a normal number, r = 1 / s rounded): a corrected quotient, and its remainder's
// sign tells on which side of it the true one lies
__device__ __forceinline__ float sticky_div(float a, float s, float r) {
  const float y0 = a * r;
  const float y = fmaf(fmaf(-y0, s, a), r, y0);
  const float rem = fmaf(-y, s, a);
  const uint32_t b = __float_as_uint(y);
  return rem == 0.f ? y : __uint_as_float((rem > 0.f ? b : b - 1u) | 1u);
}
// 16 values (sticky floats, finite) -> e4m3 scale max(amax / 6, 2^-6) rounded, and the values over it, ready for f2_to_e2m1x2.
// amax / 6 beyond 448 saturates, as the values do.
__device__ __forceinline__ uint8_t kv4_scale(const float x[16], float y[16]) {
  float am = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) am = fmaxf(am, fabsf(x[i]));
  // (amax below 2^-3 only needs the lower bound: no quotient of a tiny number is formed)
  const float q = am <= 0.09375f ? 0.015625f : am >= 2688.f ? 448.f : sticky_div(am, 6.f, 1.f / 6.f);
  const uint8_t sc = float_to_e4m3(q);
  const float s = e4m3_to_float(sc), r = __frcp_rn(s);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float a = fminf(fabsf(x[i]), 8.f * s);         // beyond 6 s all values are 6
    // below a quarter of the scale everything is zero, and a remainder of a tiny quotient could be lost
    const float v = a < 0.125f * s ? 0.f : sticky_div(a, s, r);
    y[i] = copysignf(v, x[i]);
  }
  return sc;
}

// ---------------------------------------------------------------------------------------------
// Cache pages.  A page holds 2^shift tokens; for every kv head a key block and a value block of `block` bytes each:
//   keys    [token][D / 2]      packed e2m1, even channel in the low nibble     then [token][D / 16]        e4m3 scales
//   values  [token / 2][D]      byte c: channel c of the even token in the low  then [token / 2][D / 16][2] e4m3 scales
//                               nibble, of the odd token in the high one
// Both products of the attention read a page without moving a nibble: a byte is two neighbours along the axis that the
// product sums over (channels of a key, tokens of a value), which is what one register of an MMA operand holds.
// ---------------------------------------------------------------------------------------------
struct Cache {
  uint8_t *k, *v;
  int pages, kv, shift, D;
  long block;                              // bytes of one head's keys (values) of a page
};
inline int page_shift(int page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

}  // namespace fp4
