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
//
// A workgroup has one block of one head, as all of it decides the scale: loads are runs of
// tokens of a feature, a key's codes change to a token's features side by side in LDS.
// Measured: 4 rows of 8192 bf16 tokens, 4 heads of 128 features (66 MB read, 33 MB written):
// 67 us, 1.5 TB/s. Of it the values are 21 us and the keys the rest, whose loads alone take 26
// (runs of 128 bytes, 16 KB apart, that begin anywhere: lines shared with the next block's are
// read twice; neighbours on one XCD, which read them once, take 1 to 4 us more all the same),
// sines 15, norms, codes and stores the rest. 512 threads with 8 pairs of features each, held to
// 80 registers, three workgroups a CU, of which 6 spill: 67 us; in the 88 that they would take, two
// workgroups: 70; in 64: 88; 1024 threads with 4 pairs 71 to 93; 256 with 16: 73; sines
// before the norm, behind the loads: 74; a workgroup for all heads of a block, which takes sines once but
// holds them (over 126 registers): 91 to 117. For over 128 features 1024 threads and 512 measured
// the same (16 rows of up to 256 tokens: 14 us, a chain of waits). A single token of 64 rows:
// 5 us.
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

// 2^e, e from -100 to 127.
__device__ __forceinline__ float power_of_two(int e) {
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// 1 / scale, a power of two from 2^-100 to 2^126.
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
// The same of x * to from 64 bits, rounded once: f32 is rounded to on the way, which can only
// change a code where it ends on the middle between two e4m3 values, whose significands have
// at most five bits. (What f32 does not hold is far below the least code, or above the last.)
__device__ __forceinline__ uint32_t to_codes(const double (&x)[4], float to) {
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
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] *= to;
  return to_codes(f);
}

// Numbers ordered as |x|, with what the scale depends on: the exponent, and whether the
// significand is above 1.75.
__device__ __forceinline__ uint32_t size_of(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return ((uint32_t)(u >> 32) << 1) + ((uint32_t)u != 0);
}
__device__ __forceinline__ uint32_t size_of(float x) { return __float_as_uint(x) << 1; }
// Those of inf and NaN, which the scale does not count.
constexpr uint32_t kInfinite64 = 0x7ffu << 21, kInfinite32 = 0xffu << 24;
// Smallest e with |x| <= 448 * 2^e, in range.
__device__ __forceinline__ int need_exponent64(uint32_t size) {
  return min(127, max(kCacheLowest, (int)(size >> 21) - 1031 + ((size & 0x1fffff) > 0x180000)));
}
__device__ __forceinline__ int need_exponent32(uint32_t size) {
  return min(127, max(kCacheLowest, (int)(size >> 24) - 135 + ((size & 0xffffff) > 0xc00000)));
}

// One block of one (row, kv head): its keys, or (blockIdx.y behind the heads) its values.
// Thread tid holds the E slots E (tid % QUADS) .. + E - 1 of the feature pairs
// tid / QUADS + n * THREADS / QUADS, n < NP. QUADS 16, E 4: whole blocks; 1, 1: one token a row.
template <typename T, int QUADS, int THREADS, int NP>
__global__ __launch_bounds__(THREADS, THREADS == 512 ? 6 : 4) void append_kernel(AppendArgs a) {
  constexpr int LANES = THREADS / QUADS;  // feature pairs side by side
  constexpr int WAVES = THREADS / 64;
  constexpr int E = QUADS == 1 ? 1 : 4;
  __shared__ int need_s[WAVES];
  __shared__ double sums[WAVES][E * QUADS], inv_s[E * QUADS];
  // Codes by token, 256 features; rows four bytes apart, so that 16 quads are in 16 banks.
  __shared__ uint32_t rows_s[QUADS == 16 ? 64 * 65 : 1];
  const CacheView &cv = a.cache;
  const int r = blockIdx.z, L = cv.L, hd = cv.hd;
  const bool keys = blockIdx.y < (unsigned)cv.kv_heads;
  const int h = keys ? blockIdx.y : blockIdx.y - cv.kv_heads;
  int first, count;
  if (!cache_row(cv, r, first, count) || count == 0) return;
  const int b = (first >> 6) + blockIdx.x;
  if (b * 64LL >= (long long)first + count) return;
  // Slots [lo, hi) of the block are new; slot s is token t = s + shift.
  const int lo = max(first - b * 64, 0);
  const int hi = (int)min(64LL, (long long)first + count - b * 64LL);
  const long long shift = (long long)b * 64 - first + (L - count);
  const int quad = threadIdx.x % QUADS, lane0 = threadIdx.x / QUADS;
  const int s0 = QUADS == 16 ? 4 * quad : lo;
  const int wave = threadIdx.x >> 6;
  const int pairs = keys ? a.plan.pairs : 0;
  const int half = cv.wide / 2;
  const T *x = static_cast<const T *>(keys ? a.k : a.v) + ((size_t)r * cv.kv_heads + h) * hd * L;
  int fa[NP], fb[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const int i = lane0 + LANES * n;
    fa[n] = i < pairs ? pair_first(a.plan, i) : 2 * i;
    fb[n] = i < pairs ? pair_second(a.plan, i) : 2 * i + 1;
  }
  float va[NP][4] = {}, vb[NP][4] = {};
  const bool whole = s0 >= lo && s0 + E <= hi;
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    struct {
      T e[E];
    } p = {}, q = {};
    const T *pa = x + (long long)fa[n] * L + (s0 + shift);
    const T *pb = x + (long long)fb[n] * L + (s0 + shift);
    if (whole) {
      if (fa[n] < hd) memcpy(&p, pa, sizeof p);
      if (fb[n] < hd) memcpy(&q, pb, sizeof q);
    } else if constexpr (E > 1) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (s0 + e >= lo && s0 + e < hi) {
          if (fa[n] < hd) p.e[e] = pa[e];
          if (fb[n] < hd) q.e[e] = pb[e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      va[n][e] = widen(p.e[e]);
      vb[n][e] = widen(q.e[e]);
    }
  }
  const long long place = cache_block(cv, r, h, b);
  if (place < 0) return;
  float *scale_at = (keys ? cv.key_scales : cv.value_scales) + place;
  const float before = lo > 0 ? *scale_at : 0.0f;
  uint8_t *codes = (keys ? cv.keys : cv.values) + (size_t)place * 64 * cv.wide;
  uint32_t ca[NP], cb[NP];  // E codes each
  float scale;
  auto agree = [&](int mine) {  // the block's scale
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine = max(mine, __shfl_xor(mine, o));
    if ((threadIdx.x & 63) == 0) need_s[wave] = mine;
    __syncthreads();
    int need = need_s[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) need = max(need, need_s[w]);
    scale = fmaxf(power_of_two(need), before);
  };
  if (keys) {
    double ya[NP][4] = {}, yb[NP][4] = {};
    double inv[E];
#pragma unroll
    for (int e = 0; e < E; ++e) inv[e] = 1.0;
    if (a.k_norm) {
      double sq[E] = {};
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const double p = va[n][e], q = vb[n][e];
          sq[e] = fma(p, p, fma(q, q, sq[e]));
        }
      // Lanes with the same slots: tid % QUADS.
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int o = QUADS; o < 64; o <<= 1) sq[e] += __shfl_xor(sq[e], o);
      if ((threadIdx.x & 63) < QUADS)
#pragma unroll
        for (int e = 0; e < E; ++e) sums[wave][E * quad + e] = sq[e];
      __syncthreads();
      if (threadIdx.x < E * QUADS) {  // a token's once: root and inverse cost 60 operations
        double t = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) t += sums[w][threadIdx.x];
        inv_s[threadIdx.x] = 1.0 / sqrt(t / hd + (double)a.eps);
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) inv[e] = inv_s[E * quad + e];
    }
    uint32_t most = 0;
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
      for (int e = 0; e < E; ++e) {
        const double p = (double)va[n][e] * inv[e] * wa, q = (double)vb[n][e] * inv[e] * wb;
        double c, s;
        sincos_turns(turn_of((double)(b * 64LL + s0 + e), f), s, c);
        c *= (double)a.plan.magnitude;
        s *= (double)a.plan.magnitude;
        const double ta = fma(p, c, -(q * s)), tb = fma(p, s, q * c);
        // Features that are not turned: also beside a NaN in the token, and past the last.
        ya[n][e] = i < pairs ? ta : fa[n] < hd ? p : 0.0;
        yb[n][e] = i < pairs ? tb : fb[n] < hd ? q : 0.0;
        most = max(most, max(size_of(ya[n][e]), size_of(yb[n][e])));
      }
    }
    if (most >= kInfinite64) {
      most = 0;
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t sa = size_of(ya[n][e]), sb = size_of(yb[n][e]);
          most = max(most, max(sa < kInfinite64 ? sa : 0u, sb < kInfinite64 ? sb : 0u));
        }
    }
    agree(need_exponent64(most));
    float to = inverse_of(scale);
    if (scale >= 0x1p119f) {  // past what 32 bits hold
      to = 1.0f;
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          ya[n][e] *= 1.0 / (double)scale;
          yb[n][e] *= 1.0 / (double)scale;
        }
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      ca[n] = to_codes(ya[n], to);
      cb[n] = to_codes(yb[n], to);
    }
  } else {
    uint32_t most = 0;
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int e = 0; e < E; ++e) most = max(most, max(size_of(va[n][e]), size_of(vb[n][e])));
    if (most >= kInfinite32) {
      most = 0;
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t sa = size_of(va[n][e]), sb = size_of(vb[n][e]);
          most = max(most, max(sa < kInfinite32 ? sa : 0u, sb < kInfinite32 ? sb : 0u));
        }
    }
    agree(need_exponent32(most));
    const float to = inverse_of(scale);
#pragma unroll
    for (int n = 0; n < NP; ++n) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
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
      const float y = from_code(c) * again;
      if ((c & 0x7f) != kNanCode)
        *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
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
        if constexpr (E == 1) {
          *p = (uint8_t)c;
        } else if (whole) {
          *reinterpret_cast<uint32_t *>(p) = c;
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (s0 + e >= lo && s0 + e < hi) p[e] = (uint8_t)(c >> (8 * e));
        }
      }
  } else if constexpr (E == 1) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (lane0 + LANES * n < half) {
        codes[s0 * cv.wide + fa[n]] = (uint8_t)ca[n];
        codes[s0 * cv.wide + fb[n]] = (uint8_t)cb[n];
      }
  } else {
    // Through LDS, so that a token's features leave side by side.
    uint8_t *bytes = reinterpret_cast<uint8_t *>(rows_s);
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (lane0 + LANES * n < half)
#pragma unroll
        for (int e = 0; e < E; ++e) {
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
hipError_t launch_append(const AppendArgs &a, int rows, hipStream_t stream, const KernelEvents &ev) {
  const int L = a.cache.L, half = a.cache.wide / 2;
  const unsigned blocks = (unsigned)append_blocks(a);
  const dim3 grid(blocks, (unsigned)a.cache.kv_heads * 2, (unsigned)rows);
#define TFD_APPEND(Q, N, P)                                                                     \
  hipExtLaunchKernelGGL((append_kernel<T, Q, N, P>), grid, dim3(N), 0, stream, ev.start, ev.stop, 0, a)
  // For single tokens a thread for each pair of features; for runs 8 pairs and slots a
  // thread, or 4 where the features are few.
  if (L == 1)
    TFD_APPEND(1, 128, 1);
  else if (half <= 32)
    TFD_APPEND(16, 512, 1);
  else if (half <= 64)
    TFD_APPEND(16, 512, 2);
  else
    TFD_APPEND(16, 1024, 2);
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
