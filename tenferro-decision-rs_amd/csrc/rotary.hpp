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

// Features of pair i.
__device__ __forceinline__ int pair_first(const RotaryPlan &r, int i) {
  return r.interleaved ? 2 * i : i;
}
__device__ __forceinline__ int pair_second(const RotaryPlan &r, int i) {
  return r.interleaved ? 2 * i + 1 : i + r.pairs;
}

}  // namespace tfd
