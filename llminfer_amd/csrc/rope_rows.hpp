// Rotary arithmetic of the row rotation (rope_rows.hip) and of the paged
// append (paged_append.hip): the angle of a pair is position * frequency,
// its cosine and sine are taken in double and rounded once to fp32, and a
// pair (x, y) of fp16 values becomes fp16(x c - y s), fp16(y c + x s) with
// every product and sum of fp32 rounded on its own.
//
// Double, because an fp32 angle of position 10^6 is off by up to 0.03 rad;
// the product of a 31-bit position and a 24-bit frequency is exact up to
// position 2^29. Both files are compiled with -ffp-contract=off.
#pragma once

#include "exact_fp.hpp"
#include "hip_common.hpp"

#include <hip/hip_runtime.h>

namespace llmi {

// fp32(factor cos(pos f)), fp32(factor sin(pos f)). The angle in quarter
// turns is reduced by its nearest whole number k with 1/(2 pi) in two parts
// (off by less than 2^-53 of a turn); on the remainder, at most pi/4, the
// Taylor series to x^13 (sine) and x^14 (cosine) are within 2.1e-14.
__device__ __forceinline__ float2 rope_turn(int pos, float freq, float factor) {
  constexpr double kTurn = 0x1.45f306dc9c883p-3;     // 1 / (2 pi)
  constexpr double kTurnLow = -0x1.6b01ec5417056p-57;
  const double a = (double)pos * (double)freq;
  const double p = a * kTurn;
  const double low = __builtin_fma(a, kTurn, -p) + a * kTurnLow;
  const double k = __builtin_rint(4.0 * p);
  const double x = ((4.0 * p - k) + 4.0 * low) * 1.5707963267948966;
  const double x2 = x * x;
  double s = 1.0 / 6227020800.0, c = -1.0 / 87178291200.0;
  s = __builtin_fma(s, x2, -1.0 / 39916800.0);
  s = __builtin_fma(s, x2, 1.0 / 362880.0);
  s = __builtin_fma(s, x2, -1.0 / 5040.0);
  s = __builtin_fma(s, x2, 1.0 / 120.0);
  s = __builtin_fma(s, x2, -1.0 / 6.0);
  s = __builtin_fma(s * x2, x, x);
  c = __builtin_fma(c, x2, 1.0 / 479001600.0);
  c = __builtin_fma(c, x2, -1.0 / 3628800.0);
  c = __builtin_fma(c, x2, 1.0 / 40320.0);
  c = __builtin_fma(c, x2, -1.0 / 720.0);
  c = __builtin_fma(c, x2, 1.0 / 24.0);
  c = __builtin_fma(c, x2, -0.5);
  c = __builtin_fma(c, x2, 1.0);
  // the quarter turns left over: k mod 4, for any k
  const int quarter = (int)(k - 4.0 * __builtin_floor(0.25 * k));
  const double cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
  const double co = quarter == 1 || quarter == 2 ? -cc : cc;
  const double si = quarter >= 2 ? -ss : ss;
  return make_float2((float)(co * (double)factor), (float)(si * (double)factor));
}

// Sixteen bytes of a row: aligned (VEC) or at any element.
typedef uint32_t any4_t __attribute__((ext_vector_type(4), aligned(2)));
template <bool VEC> __device__ __forceinline__ uint4_t load_word(const uint16_t *x) {
  if constexpr (VEC)
    return *reinterpret_cast<const uint4_t *>(x);
  else
    return *reinterpret_cast<const any4_t *>(x);
}
template <bool VEC> __device__ __forceinline__ void store_word(uint16_t *x, uint4_t v) {
  if constexpr (VEC)
    *reinterpret_cast<uint4_t *>(x) = v;
  else
    *reinterpret_cast<any4_t *>(x) = v;
}

// The value, hidden from the optimiser like exact_fp.hpp's opaque(), but free
// to be moved: no product is folded into the rounding after it.
__device__ __forceinline__ float apart(float x) {
  asm("" : "+v"(x));
  return x;
}
// fp16(own c + other s): the first of a pair with -s, the second with s.
__device__ __forceinline__ uint16_t turn(float own, float other, float c, float s) {
  return f2h(apart(apart(own * c) + apart(other * s)));
}
__device__ __forceinline__ uint16_t turn_x(float x, float y, float2 cs) {
  return turn(x, y, cs.x, -cs.y);
}
__device__ __forceinline__ uint16_t turn_y(float x, float y, float2 cs) {
  return turn(y, x, cs.x, cs.y);
}

} // namespace llmi
