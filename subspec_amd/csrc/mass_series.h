// The part of an exponential that a sampled entry's mass is made of: 2^f for |f| <= 1/2, in 64 bits and in units of 2^-42.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace subspec {

constexpr int kMassBits = 42;
constexpr int kSeriesTerms = 11;

// Coefficients of f^0 .. f^10, scaled by 2^42: the Taylor series of e^(f ln 2), ln^k 2 / k!, with its eleventh power folded into the odd ones below it
// (economization, C. Lanczos, "Applied Analysis", 1956): x^11 = (2816 x^9 - 2816 x^7 + 1232 x^5 - 220 x^3 + 11 x + T_11(x)) / 1024 with x = 2 f,
// where |T_11| <= 1.  What is left out is ln^11 2 / 11! / 2^21 of T_11 and the twelfth power, (ln 2 / 2)^12 / 12! = 6.3e-15 or 0.028 of 2^-42; without the
// folding the eleventh power would be missing, 0.98 of it, one-sided, at the same cost.
struct SeriesTable { double c[kSeriesTerms]; };
constexpr SeriesTable series_table() {
  SeriesTable t{{1.0, 6.9314718055994531e-1, 2.4022650695910072e-1, 5.5504108664821580e-2, 9.6181291076284772e-3, 1.3333558146428443e-3,
                 1.5403530393381610e-4, 1.5252733804059841e-5, 1.3215486790144309e-6, 1.0178086009239699e-7, 7.0549116208011233e-9}};
  constexpr double eleventh = 4.4455382718708116e-10, odd[5] = {11.0, -220.0, 1232.0, -2816.0, 2816.0};
  double scale = eleventh / 2048.0 / 1024.0;                  // of x^11 = 2048 f^11
  for (int i = 0; i < 5; ++i) t.c[2 * i + 1] += scale * odd[i] * (double)(2ull << (2 * i));
  for (int k = 0; k < kSeriesTerms; ++k) t.c[k] *= (double)(1ull << kMassBits);
  return t;
}
__host__ __device__ __forceinline__ double series_value(const double (&c)[kSeriesTerms], double f) {
  double s = c[kSeriesTerms - 1];
#pragma unroll
  for (int k = kSeriesTerms - 2; k >= 0; --k) s = fma(s, f, c[k]);
  return s;
}

}  // namespace subspec
