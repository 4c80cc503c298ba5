// Rotary positions of rows of heads.
//
// Per token t of row r at position p, for each of the first `pairs` pairs (a, b) of a
// head's features, with u = p f_i turns:
//   a' = m (a cos 2 pi u - b sin 2 pi u)
//   b' = m (a sin 2 pi u + b cos 2 pi u)
// (inverse: -u, the gradient's turn). The features behind the pairs are copied.
//
// Bound: memory, x once in and out once. Lanes go along the tokens, 16 bytes each of the
// pair's two features; the sines, a function of token and pair, are taken once for all
// heads that a workgroup walks. Measured: 2 rows of 8192 f32 tokens, 16 heads of 128 (268 MB) 45 us
// (46 to 51 from call to call), 5.9 TB/s; 8 such rows of bf16 tokens (537 MB) 104 us a call,
// 5.1 TB/s; 3 rows of 1003 bf16 tokens, 5 heads of 96 6.5 us; single tokens of 64 rows 3.0 us, where an
// empty launch takes 3.5 from one call to the next.
#include <hip/hip_ext.h>
#include <string.h>

#include "rotary.hpp"
#include "tfd_device.hpp"
#include "tfd_internal.hpp"

namespace tfd {
namespace {

template <typename T>
__device__ __forceinline__ float widen(T x) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(x);
  else
    return x;
}
template <typename T>
__device__ __forceinline__ T narrow(float x) {
  if constexpr (sizeof(T) == 2)
    return f32_to_bf16(x);
  else
    return x;
}

// A thread takes V tokens of one pair (or of two features behind the pairs) and walks
// over its share of the heads, which share the sine and cosine.
template <typename T, int V>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  struct Vec {
    T e[V];
  };
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  if (at >= (uint32_t)a.steps * a.groups) return;
  const int i = (int)(at / (uint32_t)a.steps), t0 = (int)(at - (uint32_t)i * a.steps) * V;
  const int r = blockIdx.z, L = a.L;
  const int n = min(V, L - t0);
  const bool turned = i < a.plan.pairs;
  int fa, fb;
  float c[V], s[V];
  if (turned) {
    fa = pair_first(a.plan, i);
    fb = pair_second(a.plan, i);
    const double f = a.plan.turns[i];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int t = t0 + (e < n ? e : 0);
      const int p = a.positions ? a.positions[(size_t)r * L + t] : t;
      sincospif(2.0f * (float)turn_of(p, f), &s[e], &c[e]);
      c[e] *= a.plan.magnitude;
      s[e] *= a.inverse ? -a.plan.magnitude : a.plan.magnitude;
    }
  } else {
    fa = 2 * i;
    fb = fa + 1;
  }
  const bool second = fb < a.hd;
  const T *x = static_cast<const T *>(a.x);
  T *out = static_cast<T *>(a.out);
  for (int h = blockIdx.y; h < a.heads; h += gridDim.y) {
    const size_t head = ((size_t)r * a.heads + h) * a.hd * L + t0;
    const size_t ia = head + (size_t)fa * L, ib = head + (size_t)fb * L;
    Vec va = {}, vb = {};
    if (n == V) {
      memcpy(&va, x + ia, sizeof(Vec));
      if (second) memcpy(&vb, x + ib, sizeof(Vec));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < n) {
          va.e[e] = x[ia + e];
          if (second) vb.e[e] = x[ib + e];
        }
    }
    if (turned) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float p = widen(va.e[e]), q = widen(vb.e[e]);
        va.e[e] = narrow<T>(fmaf(p, c[e], -(q * s[e])));
        vb.e[e] = narrow<T>(fmaf(p, s[e], q * c[e]));
      }
    }
    if (n == V) {
      memcpy(out + ia, &va, sizeof(Vec));
      if (second) memcpy(out + ib, &vb, sizeof(Vec));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < n) {
          out[ia + e] = va.e[e];
          if (second) out[ib + e] = vb.e[e];
        }
    }
  }
}

}  // namespace

hipError_t launch_rotary(RotaryArgs a, int rows, hipStream_t stream, const KernelEvents &ev) {
  const int v = rotary_vec(a);
  a.steps = (a.L + v - 1) / v;
  a.groups = (a.hd + 1) / 2;
  const size_t blocks = rotary_blocks(a);
  // Heads over several workgroups until the grid has eight a CU.
  const size_t wanted = (size_t)8 * a.cus;
  size_t shares = (wanted + blocks * rows - 1) / (blocks * rows);
  if (shares > (size_t)a.heads) shares = a.heads;
  const dim3 grid((unsigned)blocks, (unsigned)shares, (unsigned)rows);
#define TFD_ROTARY(T, V)                                                                         \
  hipExtLaunchKernelGGL((rotary_kernel<T, V>), grid, dim3(256), 0, stream, ev.start, ev.stop, 0, a)
  if (a.bf16 && v == 8)
    TFD_ROTARY(unsigned short, 8);
  else if (a.bf16)
    TFD_ROTARY(unsigned short, 1);
  else if (v == 4)
    TFD_ROTARY(float, 4);
  else
    TFD_ROTARY(float, 1);
#undef TFD_ROTARY
  return hipGetLastError();
}

}  // namespace tfd
