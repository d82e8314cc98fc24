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
// Scale of a block of the cache: e4m3 of max(amax / 6, 2^-6), at most 448.  amax: sticky, finite.
__device__ __forceinline__ uint8_t kv4_scale(float amax) {
  // (an amax below 2^-3 only needs the lower bound: no quotient of a tiny number is formed)
  return float_to_e4m3(amax <= 0.09375f ? 0.015625f : amax >= 2688.f ? 448.f : sticky_div(amax, 6.f, 1.f / 6.f));
}
// 1 / s to 48 bits
struct Recip {
  float hi, lo;
};
__device__ __forceinline__ Recip recip(float s) {
  const float r = __frcp_rn(s);
  return {r, fmaf(-s, r, 1.f) * r};
}
// x / s, rounded; exact wherever the quotient is a border of the grid.  x has at most 11 bits and s 4: any other quotient is 2^-11
// or more away from all borders, so this one decides as the true one does.  Beyond the grid (infinity too): 6.
__device__ __forceinline__ float over(float x, Recip r) { return fmaf(x, r.hi, x * r.lo); }
// the same for a sticky x of 24 bits
__device__ __forceinline__ float over_sticky(float x, float s, float r) {
  return copysignf(sticky_div(fminf(fabsf(x), 8.f * s), s, r), x);
}
// four pairs (low, high nibble) -> four bytes
__device__ __forceinline__ uint32_t e2m1x8(const float lo[4], const float hi[4]) {
  const uint32_t a = f2_to_e2m1x2(lo[0], hi[0]), b = f2_to_e2m1x2(lo[1], hi[1]), c = f2_to_e2m1x2(lo[2], hi[2]), d = f2_to_e2m1x2(lo[3], hi[3]);
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
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
