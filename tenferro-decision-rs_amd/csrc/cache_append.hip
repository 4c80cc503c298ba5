// Keys and values of new tokens into a paged cache of e4m3 codes with a power of two as
// scale for each block of 64 tokens and head.
//
// A key is normalized (x / sqrt(mean(x^2) + eps) (1 + w)) and turned to its place in the
// row; a value goes as it is. A block's scale is the smallest 2^e >= 2^-100 with
// |x| <= 448 * 2^e for every finite x in it, and it never falls while the block fills: where
// a new token needs a larger one, the codes of the earlier tokens are rounded again, which
// is exact for all but e4m3's subnormals, as both scales are powers of two. Codes are
// rounded to nearest even; NaN and inf become the code of NaN and count for no scale.
//
// Keys are computed in 64 bits, whose vector rate is that of 32 bits here: a code then does
// not depend on the order of a sum or on the shape of the launch, so tokens appended
// one by one leave the codes that a prompt of them leaves, as long as no scale grew between.
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

// x in 32 bits with the last bit set where it is not exact (round to odd): rounding the
// result again to at most 22 bits is then rounding x once.
__device__ __forceinline__ float odd_f32(double x) {
  const float f = (float)x;
  uint32_t u = __float_as_uint(f);
  const double back = (double)f;
  if (back != x && !(u & 1u)) u += fabs(back) > fabs(x) ? ~0u : 1u;
  return __uint_as_float(u);
}

// 1 / scale, a power of two from 2^-100 to 2^120.
__device__ __forceinline__ float inverse_of(float scale) {
  return __uint_as_float((254u << 23) - __float_as_uint(scale));
}

constexpr uint32_t kNanCode = 0x7f;

__device__ __forceinline__ float from_code(uint32_t c) {
  return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}
__device__ __forceinline__ uint32_t four_codes(const float (&x)[4]) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
}
// Codes of the nearest e4m3 values of |x| <= 448, of others (and of NaN) the code of NaN.
__device__ __forceinline__ uint32_t to_codes(const float (&x)[4]) {
  uint32_t c = four_codes(x);
  const float most = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  if (most > 448.0f || (((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u)) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(fabsf(x[e]) <= 448.0f)) c = (c & ~(0xffu << (8 * e))) | kNanCode << (8 * e);
  }
  return c;
}
// The same from 64 bits, rounded once: f32 is rounded to on the way, which can only change a
// code where it ends on the middle between two e4m3 values, whose significands have at most
// five bits.
__device__ __forceinline__ uint32_t to_codes(const double (&x)[4]) {
  float f[4];
  uint32_t least = ~0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = (float)x[e];
    least = min(least, __float_as_uint(f[e]) & 0x7ffffu);
  }
  if (least == 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = odd_f32(x[e]);
  }
  return to_codes(f);
}

// Smallest e with most <= 448 * 2^e, at least kCacheLowest.
__device__ __forceinline__ int need_exponent(float most) {
  if (!(most > 0.0f)) return kCacheLowest;
  int e;
  const float m = frexpf(most, &e);
  return min(127, max(kCacheLowest, e - 9 + (m > 0.875f ? 1 : 0)));
}
__device__ __forceinline__ int need_exponent(double most) {
  if (!(most > 0.0)) return kCacheLowest;
  int e;
  const double m = frexp(most, &e);
  return min(127, max(kCacheLowest, e - 9 + (m > 0.875 ? 1 : 0)));
}

// One block of one (row, kv head), its keys or its values. Thread tid holds the four
// slots 4 (tid % QUADS) .. + 3 of the feature pairs tid / QUADS + n * THREADS / QUADS,
// n < NP. QUADS 16: whole blocks; 1: one token a row.
template <typename T, int QUADS, int THREADS, int NP>
__global__ __launch_bounds__(THREADS) void append_kernel(AppendArgs a) {
  constexpr int LANES = THREADS / QUADS;  // feature pairs side by side
  constexpr int WAVES = THREADS / 64;
  __shared__ int need_s[WAVES];
  __shared__ double sums[WAVES][64], inv_s[64];
  // Codes by token, 256 features; rows four bytes apart, so that 16 quads are in 16 banks.
  __shared__ uint32_t rows_s[QUADS == 16 ? 64 * 65 : 1];
  const CacheView &cv = a.cache;
  const int r = blockIdx.z, h = blockIdx.y >> 1, L = cv.L, hd = cv.hd;
  const bool keys = (blockIdx.y & 1) == 0;
  int first, count;
  if (!cache_row(cv, r, first, count) || count == 0) return;
  const int b = (first >> 6) + blockIdx.x;
  if (b * 64LL >= (long long)first + count) return;
  // Slots [lo, hi) of the block are new; slot s is token t = s + shift.
  const int lo = max(first - b * 64, 0);
  const int hi = (int)min(64LL, (long long)first + count - b * 64LL);
  const long long shift = (long long)b * 64 - first + (L - count);
  const int quad = threadIdx.x % QUADS, lane0 = threadIdx.x / QUADS;
  const int s0 = QUADS == 16 ? 4 * quad : lo & ~3;
  const int wave = threadIdx.x >> 6;
  const int pairs = keys ? a.plan.pairs : 0;
  const int half = cv.wide / 2;
  const T *x = static_cast<const T *>(keys ? a.k : a.v) +
               ((size_t)r * cv.kv_heads + h) * hd * L;
  int fa[NP], fb[NP];
  float va[NP][4], vb[NP][4];
  const bool whole = s0 >= lo && s0 + 4 <= hi;
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const int i = lane0 + LANES * n;
    fa[n] = i < pairs ? pair_first(a.plan, i) : 2 * i;
    fb[n] = i < pairs ? pair_second(a.plan, i) : 2 * i + 1;
    struct {
      T e[4];
    } p = {}, q = {};
    const T *pa = x + (long long)fa[n] * L + (s0 + shift), *pb = x + (long long)fb[n] * L + (s0 + shift);
    if (whole) {
      if (fa[n] < hd) memcpy(&p, pa, sizeof p);
      if (fb[n] < hd) memcpy(&q, pb, sizeof q);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s0 + e >= lo && s0 + e < hi) {
          if (fa[n] < hd) p.e[e] = pa[e];
          if (fb[n] < hd) q.e[e] = pb[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      va[n][e] = widen(p.e[e]);
      vb[n][e] = widen(q.e[e]);
    }
  }
  const long long place = cache_block(cv, r, h, b);
  if (place < 0) return;
  float *scale_at = (keys ? cv.key_scales : cv.value_scales) + place;
  const float before = lo > 0 ? *scale_at : 0.0f;
  const size_t block0 = (size_t)place * 64 * cv.wide;
  uint8_t *codes = (keys ? cv.keys : cv.values) + block0;

  uint32_t ca[NP], cb[NP];  // four codes each
  int need;
  float scale;
  auto agree = [&](int mine) {  // the block's scale
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine = max(mine, __shfl_xor(mine, o));
    if ((threadIdx.x & 63) == 0) need_s[wave] = mine;
    __syncthreads();
    need = need_s[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) need = max(need, need_s[w]);
    const float s = ldexpf(1.0f, need);
    scale = fmaxf(s, before);
  };
  if (keys) {
    double ya[NP][4], yb[NP][4];
    double inv[4] = {1.0, 1.0, 1.0, 1.0};
    if (a.k_norm) {
      double sq[4] = {};
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const double p = va[n][e], q = vb[n][e];
          sq[e] = fma(p, p, fma(q, q, sq[e]));
        }
      // Lanes with the same quad: tid % QUADS.
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int o = QUADS; o < 64; o <<= 1) sq[e] += __shfl_xor(sq[e], o);
      if ((threadIdx.x & 63) < QUADS)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave][4 * quad + e] = sq[e];
      __syncthreads();
      if (threadIdx.x < 4 * QUADS) {  // each token's once: the root and its inverse cost 60 operations
        double t = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) t += sums[w][threadIdx.x];
        inv_s[threadIdx.x] = 1.0 / sqrt(t / hd + (double)a.eps);
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) inv[e] = inv_s[4 * quad + e];
    }
    double most = 0.0;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int i = lane0 + LANES * n;
      double wa = 1.0, wb = 1.0;
      if (a.k_norm) {
        wa = fa[n] < hd ? 1.0 + (double)a.k_norm[fa[n]] : 0.0;
        wb = fb[n] < hd ? 1.0 + (double)a.k_norm[fb[n]] : 0.0;
      }
      const double f = i < pairs ? a.plan.turns[i] : 0.0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double p = (double)va[n][e] * inv[e] * wa, q = (double)vb[n][e] * inv[e] * wb;
        if (i < pairs) {
          double c, s;
          sincospi(2.0 * turn_of((double)(b * 64LL + s0 + e), f), &s, &c);
          c *= (double)a.plan.magnitude;
          s *= (double)a.plan.magnitude;
          ya[n][e] = fma(p, c, -(q * s));
          yb[n][e] = fma(p, s, q * c);
        } else {
          ya[n][e] = fa[n] < hd ? p : 0.0;  // also beside a NaN in the token
          yb[n][e] = fb[n] < hd ? q : 0.0;
        }
        most = fmax(most, fmax(fabs(ya[n][e]), fabs(yb[n][e])));
      }
    }
    if (most > 1e300) {  // inf, which counts as little as NaN
      most = 0.0;
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (fabs(ya[n][e]) <= 1e300) most = fmax(most, fabs(ya[n][e]));
          if (fabs(yb[n][e]) <= 1e300) most = fmax(most, fabs(yb[n][e]));
        }
    }
    agree(need_exponent(most));
    const double to = (double)inverse_of(scale);
#pragma unroll
    for (int n = 0; n < NP; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ya[n][e] *= to;
        yb[n][e] *= to;
      }
      ca[n] = to_codes(ya[n]);
      cb[n] = to_codes(yb[n]);
    }
  } else {
    float most = 0.0f;
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        most = fmaxf(most, fmaxf(fabsf(va[n][e]), fabsf(vb[n][e])));
      }
    if (most > 3.402823466e38f) {
      most = 0.0f;
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (fabsf(va[n][e]) <= 3.402823466e38f) most = fmaxf(most, fabsf(va[n][e]));
          if (fabsf(vb[n][e]) <= 3.402823466e38f) most = fmaxf(most, fabsf(vb[n][e]));
        }
    }
    agree(need_exponent(most));
    const float to = inverse_of(scale);
#pragma unroll
    for (int n = 0; n < NP; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        va[n][e] *= to;
        vb[n][e] *= to;
      }
      ca[n] = to_codes(va[n]);
      cb[n] = to_codes(vb[n]);
    }
  }
  // Earlier tokens under a scale that grew.
  if (lo > 0 && scale != before) {
    const float again = before / scale;
    for (int j = threadIdx.x; j < lo * cv.wide; j += THREADS) {
      const int s = keys ? j / cv.wide : j % lo, f = keys ? j % cv.wide : j / lo;
      uint8_t *p = codes + (keys ? s * cv.wide + f : f * 64 + s);
      const uint32_t c = *p;
      const float x = from_code(c) * again;
      if ((c & 0x7f) != kNanCode)
        *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false);
    }
  }
  if (threadIdx.x == 0) *scale_at = scale;
  if (!keys) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int f = k ? fb[n] : fa[n];
        const uint32_t c = k ? cb[n] : ca[n];
        if (f >= hd) continue;
        uint8_t *p = codes + f * 64 + s0;
        if (whole) {
          *reinterpret_cast<uint32_t *>(p) = c;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s0 + e >= lo && s0 + e < hi) p[e] = (uint8_t)(c >> (8 * e));
        }
      }
    return;
  }
  if constexpr (QUADS == 1) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s0 + s >= lo && s0 + s < hi && lane0 + LANES * n < half) {
          codes[(s0 + s) * cv.wide + fa[n]] = (uint8_t)(ca[n] >> (8 * s));
          codes[(s0 + s) * cv.wide + fb[n]] = (uint8_t)(cb[n] >> (8 * s));
        }
  } else {
    // Through LDS, so that a token's features leave side by side.
    uint8_t *bytes = reinterpret_cast<uint8_t *>(rows_s);
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (lane0 + LANES * n < half)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bytes[(s0 + e) * (cv.wide + 4) + fa[n]] = (uint8_t)(ca[n] >> (8 * e));
          bytes[(s0 + e) * (cv.wide + 4) + fb[n]] = (uint8_t)(cb[n] >> (8 * e));
        }
    __syncthreads();
    uint32_t *to = reinterpret_cast<uint32_t *>(codes);
    const int row = cv.wide / 4;
    for (int j = threadIdx.x + lo * row; j < hi * row; j += THREADS) to[j] = rows_s[j + j / row];
  }
}

template <typename T>
hipError_t launch_append(const AppendArgs &a, int rows, hipStream_t stream,
                         const KernelEvents &ev) {
  const int L = a.cache.L, half = a.cache.wide / 2;
  // Blocks that L tokens from any slot on may touch.
  const unsigned blocks = (unsigned)((L + 62) / 64 + 1);
  const dim3 grid(blocks, (unsigned)a.cache.kv_heads * 2, (unsigned)rows);
#define TFD_APPEND(Q, N, P)                                                                     \
  hipExtLaunchKernelGGL((append_kernel<T, Q, N, P>), grid, dim3(N), 0, stream, ev.start, ev.stop, 0, a)
  if (L == 1)
    TFD_APPEND(1, 128, 1);
  else if (half <= 32)
    TFD_APPEND(16, 512, 1);
  else if (half <= 64)
    TFD_APPEND(16, 512, 2);
  else
    TFD_APPEND(16, 512, 4);
#undef TFD_APPEND
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_append(const AppendArgs &a, int rows, hipStream_t stream,
                               const KernelEvents &ev) {
  return a.bf16 ? launch_append<unsigned short>(a, rows, stream, ev)
                : launch_append<float>(a, rows, stream, ev);
}

}  // namespace tfd
