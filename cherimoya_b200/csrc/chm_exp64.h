// chm_exp64.h -- exp in 64 bits with a short chain of operations, on the device and the host.
#pragma once
#include <math.h>
#include <string.h>

#ifdef __CUDACC__
#define CHM_EXP64_FN __device__ __forceinline__
#else
#define CHM_EXP64_FN inline
#endif

namespace chm {
namespace lk {

// 2^k for -1023 < k < 1024, and inf
#ifdef __CUDACC__
CHM_EXP64_FN double power_of_two(int k) { return __hiloint2double((1023 + k) << 20, 0); }
CHM_EXP64_FN double inf64() { return (double)__int_as_float(0x7f800000); }
#else
CHM_EXP64_FN double power_of_two(int k) {
  const long long bits = (long long)(1023 + k) << 52;
  double v;
  memcpy(&v, &bits, sizeof v);
  return v;
}
CHM_EXP64_FN double inf64() { return HUGE_VAL; }
#endif

// exp in 64 bits, for masses that are added up and taken from 1: Cody and Waite's reduction
// x = n log 2 + r with |r| <= log(2) / 2, log 2 in the two parts that fdlibm's e_exp.c (Sun
// Microsystems, 1993) publishes, whose first has 32 bits, so that its product with n is exact;
// then the Taylor sum of e^r to r^11 in a tree (Estrin's scheme), since one call after the other
// waits for fp64's latency. The rest of the sum is r^12 / 12! and less, below 9.2e-15 of e^r;
// with the roundings the result is off by less than 1e-14 of itself.
// 0 below -700, where no mass is left; inf above 700.
CHM_EXP64_FN double exp64(double x) {
  const double n = rint(x * 1.4426950408889634);
  const double r = fma(n, -1.9082149292705877e-10, fma(n, -6.9314718036912382e-1, x));
  const double r2 = r * r, r4 = r2 * r2;
  const double a = fma(fma(1.0 / 6, r, 0.5), r2, 1.0 + r);
  const double b = fma(fma(1.0 / 5040, r, 1.0 / 720), r2, fma(1.0 / 120, r, 1.0 / 24));
  const double c = fma(fma(1.0 / 39916800, r, 1.0 / 3628800), r2,
                       fma(1.0 / 362880, r, 1.0 / 40320));
  const double e = fma(fma(c, r4, b), r4, a);
  const int k = (int)fmin(fmax(n, -1010.0), 1010.0);
  const double s = e * power_of_two(k);
  return x < -700.0 ? 0.0 : x > 700.0 ? inf64() : s;
}

}  // namespace lk
}  // namespace chm
