// The weight of a logit in a draw, in f64 (verify_kernels.hip).
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace vpa {

// 2^t for 0 >= t > -2^31 in f64, 0 below -1074: t = n + f, and for 2^f,
// |f| <= 1/2, the polynomial 1 + f g(f) with g through the 9 Chebyshev nodes of
// (2^f - 1) / f: within 4e-14 of the value. A draw among 150 000 tokens then has
// about one chance in 10^8 to see a border on its wrong side.
__device__ __forceinline__ double exp2_nonpos(double t) {
  const double n = __builtin_rint(t);
  const double f = t - n;
  double p = 1.02031210633917290e-07;
  p = __builtin_fma(p, f, 1.32552248786688168e-06);
  p = __builtin_fma(p, f, 1.52526868462677196e-05);
  p = __builtin_fma(p, f, 1.54034558524538382e-04);
  p = __builtin_fma(p, f, 1.33335581790431116e-03);
  p = __builtin_fma(p, f, 9.61812915940255843e-03);
  p = __builtin_fma(p, f, 5.55041086647604237e-02);
  p = __builtin_fma(p, f, 2.40226506958129887e-01);
  p = __builtin_fma(p, f, 6.93147180559945286e-01);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}
// The weights e^((l - m) / T) of logits l against a maximum m: 1 at the maximum
// (also an infinite one), 0 for -inf and NaN.
struct Scale {
  double c;  // log2 e / T
  double m64;
  float m;
  float floor;  // logits below it, and NaN, count as it: an exponent below every f64
  // Only the maximum's equals weigh: it is infinite, or the lowest number, or the next
  // number below it has no weight already (a step of 1e-6 below 10 at T = 1e-9, of 2e31
  // below a row of the 16-bit types' lowest value). Every other exponent is above -2^31:
  // a step's is at most 1100, so `floor` is less than 2000 T and a step away (T above
  // 1e30: all of f32 is 1e9 away).
  bool odd;
  __device__ __forceinline__ Scale(float max, float temp)
      // (T above 1e30 as 1e30: a masked logit's weight stays 0)
      : c(fmax(1.44269504088896340736 / (double)temp, 1e-30)),
        m64((double)max),
        m(max),
        floor(fmaxf(fminf(max - 2000.f * temp, below(max)), -FLT_MAX)),
        odd(!(max > -FLT_MAX && max < INFINITY) ||
            ((double)below(max) - (double)max) * c < -1100.0) {}
  // the next number below a finite one
  static __device__ __forceinline__ float below(float v) {
    const uint32_t u = __float_as_uint(v);
    return __uint_as_float(v > 0.f ? u - 1u : v < 0.f ? u + 1u : 0x80000001u);
  }
  __device__ __forceinline__ double exponent(float l) const {
    // (the difference first: logits of the lowest value have products whose
    // rounding alone would be a huge exponent)
    return ((double)fmaxf(l, floor) - m64) * c;
  }
  __device__ __forceinline__ double plain(float l) const { return exp2_nonpos(exponent(l)); }
  __device__ __forceinline__ double weight(float l) const {
    return odd ? (l == m && l > -INFINITY ? 1.0 : 0.0) : plain(l);
  }
};

}  // namespace vpa
