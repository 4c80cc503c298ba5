// Rotary positions shared by the kernels that turn features: a pair of features at
// position p is turned by p f turns, of which whole ones are dropped in 64 bits (f32 angles
// are off by 6e-3 at position 10^5), and scaled by a magnitude.
#pragma once

#include <hip/hip_runtime.h>

#include "tfd_internal.hpp"

namespace tfd {

// The part of p f behind its nearest whole number. The product is rounded once by
// itself, so that the result is the same wherever it is taken.
__device__ __forceinline__ double turn_of(double p, double f) {
#pragma clang fp contract(off)
  const double t = p * f;
  return t - rint(t);
}

// Sine and cosine of t turns, |t| <= 1/2: the nearest quarter apart, the rest r, at most
// pi/4, by the first 8 and 9 terms of their series (the next ones are below 2^-53 of the
// result). A third of the operations of sincospi, and without branches, so that those of
// several features run into one another.
__device__ __forceinline__ void sincos_turns(double t, double &s, double &c) {
  const double q = rint(4.0 * t);
  const double r = fma(q, -0.25, t) * 6.283185307179586;
  const double z = r * r;
  double a = -1.0 / 1307674368000.0, b = 1.0 / 20922789888000.0;
  a = fma(a, z, 1.0 / 6227020800.0);
  b = fma(b, z, -1.0 / 87178291200.0);
  a = fma(a, z, -1.0 / 39916800.0);
  b = fma(b, z, 1.0 / 479001600.0);
  a = fma(a, z, 1.0 / 362880.0);
  b = fma(b, z, -1.0 / 3628800.0);
  a = fma(a, z, -1.0 / 5040.0);
  b = fma(b, z, 1.0 / 40320.0);
  a = fma(a, z, 1.0 / 120.0);
  b = fma(b, z, -1.0 / 720.0);
  a = fma(a, z, -1.0 / 6.0);
  b = fma(b, z, 1.0 / 24.0);
  a = fma(a * z, r, r);
  b = fma(fma(b, z, -0.5), z, 1.0);
  const int n = (int)q;
  const double u = n & 1 ? b : a, v = n & 1 ? a : b;
  s = n & 2 ? -u : u;
  c = (n + 1) & 2 ? -v : v;
}

// Features of pair i.
__device__ __forceinline__ int pair_first(const RotaryPlan &r, int i) {
  return r.interleaved ? 2 * i : i;
}
__device__ __forceinline__ int pair_second(const RotaryPlan &r, int i) {
  return r.interleaved ? 2 * i + 1 : i + r.pairs;
}

}  // namespace tfd
