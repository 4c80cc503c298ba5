// Linear attention with a decay per head and an optional delta-rule write.
//
// Per row and value head, with a state S (key_dim x value_dim), for every
// active token t:
//   S <- e^(g_t) S
//   u  = v_t, or beta_t (v_t - S^T k_t) with the delta rule
//   S <- S + k_t u^T
//   o_t = scale S^T q_t
// Inactive tokens leave S as it is and give o_t = 0; what they hold (NaN, inf)
// is never read into a product.
#include <hip/hip_ext.h>
#include <math.h>

#include "tfd_device.hpp"
#include "tfd_internal.hpp"

namespace tfd {
namespace {

template <typename T>
__device__ __forceinline__ float load_as_f32(const void *p, size_t i) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(static_cast<const unsigned short *>(p)[i]);
  else
    return static_cast<const float *>(p)[i];
}

// The recurrence token by token, for single tokens and short prompts.
// Workgroup = 32 value columns of one (row, head): thread t holds columns
// 4 (t % 8) .. + 3 of the key rows t / 8 + 32 n, n < NI. Both products with the
// state (with k for the delta rule, with q for the output) are taken on the
// decayed state in one reduction, since
//   S_new^T q = S^T q + u (k . q).
// Single tokens are bound by reading and writing the states: 128 rows of 8 heads of
// 256 x 256 (539 MB) take 118 us, 4.6 TB/s (a copy reaches 5.1 TB/s). Both ways past
// the caches, which no state of a large batch comes back to in time: with plain
// loads 128 us, with plain stores as well 129 us. 64 columns a workgroup (256-byte
// pieces of the states' rows): 128 rows of 16 heads of 128 x 128 60 us against 56.
template <typename T, bool DELTA, int NI>
__global__ __launch_bounds__(256) void linear_recurrent_kernel(LinearArgs a) {
  __shared__ float part[2][4][8][9];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int quad = threadIdx.x & 7, ig = threadIdx.x >> 3;
  const int h = blockIdx.y, r = blockIdx.z, L = a.L;
  const int j0 = blockIdx.x * 32 + 4 * quad;
  const int nj = min(4, a.dv - j0);  // may be <= 0
  const size_t rh = (size_t)r * a.heads + h;
  const float *sin = a.state_in ? a.state_in + rh * a.dk * a.dv : nullptr;
  float *sout = a.state_out ? a.state_out + rh * a.dk * a.dv : nullptr;
  float S[NI][4];
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int i = ig + 32 * n;
#pragma unroll
    for (int c = 0; c < 4; ++c) S[n][c] = 0.0f;
    if (!sin || i >= a.dk || nj <= 0) continue;
    const float *p = sin + (size_t)i * a.dv + j0;
    if (a.state_vec) {
      const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(p));
#pragma unroll
      for (int c = 0; c < 4; ++c) S[n][c] = v[c];
    } else {
      for (int c = 0; c < nj; ++c) S[n][c] = p[c];
    }
  }
  const size_t kh = (size_t)h / a.group;
  const size_t key0 = ((size_t)r * a.key_heads + kh) * a.dk * L;
  const size_t val0 = rh * a.dv * L;
  const float *mask = a.mask ? a.mask + (size_t)r * L : nullptr;
  int turn = 0;
  for (int t = 0; t < L; ++t) {
    if (mask && mask[t] == 0.0f) {
      if (ig == 0)
        for (int c = 0; c < nj; ++c) a.out[val0 + (size_t)(j0 + c) * L + t] = 0.0f;
      continue;
    }
    const float decay = expf(a.log_decay[rh * L + t]);
    float k[NI], q[NI], red[9] = {};
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int i = ig + 32 * n;
      const bool in = i < a.dk;
      k[n] = in ? load_as_f32<T>(a.k, key0 + (size_t)i * L + t) : 0.0f;
      q[n] = in ? load_as_f32<T>(a.q, key0 + (size_t)i * L + t) : 0.0f;
    }
#pragma unroll
    for (int n = 0; n < NI; ++n) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        S[n][c] *= decay;
        red[c] = fmaf(S[n][c], q[n], red[c]);
        if (DELTA) red[4 + c] = fmaf(S[n][c], k[n], red[4 + c]);
      }
      red[8] = fmaf(k[n], q[n], red[8]);
    }
#pragma unroll
    for (int c = 0; c < 9; ++c) {
      if (!DELTA && c >= 4 && c < 8) continue;
#pragma unroll
      for (int o = 8; o < 64; o <<= 1) red[c] += __shfl_xor(red[c], o);
      if (lane < 8) part[turn][wave][quad][c] = red[c];
    }
    __syncthreads();
    auto sum = [&](int c) {
      return (part[turn][0][quad][c] + part[turn][1][quad][c]) +
             (part[turn][2][quad][c] + part[turn][3][quad][c]);
    };
    const float kq = sum(8);
    const float beta = DELTA ? a.beta[rh * L + t] : 1.0f;
    float u[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = c < nj ? load_as_f32<T>(a.v, val0 + (size_t)(j0 + c) * L + t) : 0.0f;
      if (DELTA) u[c] = beta * (u[c] - sum(4 + c));
      if (ig == 0 && c < nj)
        a.out[val0 + (size_t)(j0 + c) * L + t] = a.scale * fmaf(u[c], kq, sum(c));
    }
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) S[n][c] = fmaf(k[n], u[c], S[n][c]);
    turn ^= 1;
  }
  if (!sout) return;
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int i = ig + 32 * n;
    if (i >= a.dk || nj <= 0) continue;
    float *p = sout + (size_t)i * a.dv + j0;
    if (a.state_vec) {
      f32x4 v;
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = S[n][c];
      __builtin_nontemporal_store(v, reinterpret_cast<f32x4 *>(p));
    } else {
      for (int c = 0; c < nj; ++c) p[c] = S[n][c];
    }
  }
}

template <typename T, bool DELTA>
hipError_t launch_recurrent(const LinearArgs &a, hipStream_t stream, const KernelEvents &ev) {
  const dim3 grid((unsigned)((a.dv + 31) / 32), (unsigned)a.heads, (unsigned)a.rows);
  if (a.dk <= 32)
    hipExtLaunchKernelGGL((linear_recurrent_kernel<T, DELTA, 1>), grid, dim3(256), 0, stream,
                          ev.start, ev.stop, 0, a);
  else if (a.dk <= 64)
    hipExtLaunchKernelGGL((linear_recurrent_kernel<T, DELTA, 2>), grid, dim3(256), 0, stream,
                          ev.start, ev.stop, 0, a);
  else if (a.dk <= 128)
    hipExtLaunchKernelGGL((linear_recurrent_kernel<T, DELTA, 4>), grid, dim3(256), 0, stream,
                          ev.start, ev.stop, 0, a);
  else
    hipExtLaunchKernelGGL((linear_recurrent_kernel<T, DELTA, 8>), grid, dim3(256), 0, stream,
                          ev.start, ev.stop, 0, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_linear_recurrent(const LinearArgs &a, hipStream_t stream,
                                   const KernelEvents &ev) {
  if (a.bf16)
    return a.beta ? launch_recurrent<unsigned short, true>(a, stream, ev)
                  : launch_recurrent<unsigned short, false>(a, stream, ev);
  return a.beta ? launch_recurrent<float, true>(a, stream, ev)
                : launch_recurrent<float, false>(a, stream, ev);
}

}  // namespace tfd
