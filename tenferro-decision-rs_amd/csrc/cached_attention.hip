// Causal attention of new tokens over a paged cache of e4m3 keys and values.
//
// Per row, new token u (of count) and query head, with its queries normalized
// (x / sqrt(mean(x^2) + eps) (1 + w)) and turned to position first + u:
//   s_j = q . k_j / sqrt(hd) over the keys j <= first + u
//   o   = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), times sigmoid(gate)
// A code is exact in bf16, so a product with an f32 operand is three bf16 matrix products,
// one for each piece of the f32 one (split_bf16x3); the blocks' scales are applied to the
// scores and the probabilities.
//
// Tiles: the columns of a product are the (token, query head of the group) pairs of one
// (row, kv head), 16 a workgroup; its rows are keys, then features. S^T = K Q^T leaves lane
// (column l % 16, group g = l / 16) the keys 16 g + 4 t + i of accumulator i of key tile t,
// as the rows of tile t are taken in that order: 16 keys in a row, which are what the lane
// has to give to O^T = V^T P^T and what 16 bytes of a value's block hold. No value passes
// between lanes but a column's maximum and sum.
#include <hip/hip_ext.h>

#include "rotary.hpp"
#include "tfd_device.hpp"
#include "tfd_internal.hpp"

namespace tfd {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kCols = kCachedColumns;

// Eight e4m3 codes as bf16.
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t lo, uint32_t hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 0x80 in each byte of x that is the code of NaN.
__device__ __forceinline__ uint32_t nan_codes(uint32_t x) {
  return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

template <typename T>
__device__ __forceinline__ float load_as_f32(const void *p, size_t i) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(static_cast<const unsigned short *>(p)[i]);
  else
    return static_cast<const float *>(p)[i];
}

// Column c of a row: active tokens come first, in order, then the others.
struct Column {
  int token, head;  // of the row, of the group
  int place;        // active: index among the row's active tokens, else -1
};
__device__ __forceinline__ Column column_of(int c, int group, int L, int count) {
  const int u = c / group;
  return Column{u < count ? L - count + u : u - count, c - u * group, u < count ? u : -1};
}

struct Stats {
  float m, l;  // reference in log2 units and sum, of a column
};

// out of column `col` (of a tile whose first one is c0), features f .. f + 3.
template <typename T>
__device__ __forceinline__ void store_out(const CachedArgs &a, int r, int h, const Column &c, int f,
                                          f32x4 o, float inv) {
  const int L = a.cache.L, hd = a.cache.hd;
  const size_t at = (((size_t)r * a.heads + h * a.group + c.head) * hd + f) * L + c.token;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (f + i >= hd) continue;
    float y = o[i] * inv;
    if (a.gate) y *= fast_sigmoid(load_as_f32<T>(a.gate, at + (size_t)i * L));
    a.out[at + (size_t)i * L] = y;
  }
}

template <typename T, int W>
__global__ __launch_bounds__(256, 1) void cached_kernel(CachedArgs a) {
  constexpr int WIDE = 64 * W;
  __shared__ float q_s[kCols][WIDE + 4];
  __shared__ float o_s[kWaves][kCols][WIDE + 4];
  __shared__ Stats st_s[kWaves][kCols];
  const CacheView &cv = a.cache;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, grp = lane >> 4;
  const int part = blockIdx.x % a.parts, tile = blockIdx.x / a.parts;
  const int h = blockIdx.y, r = blockIdx.z, L = cv.L, hd = cv.hd, group = a.group;
  int first, count;
  const bool sound = cache_row(cv, r, first, count);
  if (!sound) first = count = 0;
  const int c0 = tile * kCols, columns = group * L;
  const int active = group * count;  // columns

  // Columns of tokens that are not active, and of rows whose pages do not hold them.
  if (part == 0 && c0 + kCols > active) {
    for (int c = wave; c < kCols; c += kWaves) {
      if (c0 + c < active || c0 + c >= columns) continue;
      const Column at = column_of(c0 + c, group, L, count);
      const size_t o = (((size_t)r * a.heads + h * group + at.head) * hd) * L + at.token;
      for (int f = lane; f < hd; f += 64)
        a.out[o + (size_t)f * L] = sound ? 0.0f : __builtin_nanf("");
    }
  }
  if (c0 >= active) return;
  const int last = min(c0 + kCols, active) - 1;  // last active column of the tile
  const int u0 = c0 / group, u1 = last / group;
  const int blocks = (first + u1) / 64 + 1;
  const int share = (blocks + a.parts - 1) / a.parts;
  const int b0 = part * share, b1 = min(blocks, b0 + share);
  const size_t item = (((size_t)r * cv.kv_heads + h) * a.tiles + tile) * a.parts + part;
  if (b0 >= b1) return;

  // Queries: a wave takes a column, its lanes the features.
  for (int c = wave; c < kCols; c += kWaves) {
    float x[W];
    const bool in = c0 + c <= last;
    const Column at = column_of(min(c0 + c, last), group, L, count);
    const size_t from = (((size_t)r * a.heads + h * group + at.head) * hd) * L + at.token;
    float sq = 0.0f;
#pragma unroll
    for (int n = 0; n < W; ++n) {
      const int f = lane + 64 * n;
      x[n] = in && f < hd ? load_as_f32<T>(a.q, from + (size_t)f * L) : 0.0f;
      sq = fmaf(x[n], x[n], sq);
    }
    if (a.q_norm) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sq += __shfl_xor(sq, o);
      const float inv = 1.0f / sqrtf(sq / (float)hd + a.eps);
#pragma unroll
      for (int n = 0; n < W; ++n) {
        const int f = lane + 64 * n;
        if (f < hd) x[n] *= inv * (1.0f + a.q_norm[f]);
      }
    }
#pragma unroll
    for (int n = 0; n < W; ++n) q_s[c][lane + 64 * n] = x[n];
    // The wave's own column: its LDS accesses are in order.
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int n = 0; n < (W + 1) / 2; ++n) {
      const int i = lane + 64 * n;
      if (i >= a.plan.pairs) continue;
      const int fa = pair_first(a.plan, i), fb = pair_second(a.plan, i);
      float s, k;
      sincospif(2.0f * (float)turn_of((double)(first + at.place), a.plan.turns[i]), &s, &k);
      s *= a.plan.magnitude;
      k *= a.plan.magnitude;
      const float p = q_s[c][fa], q = q_s[c][fb];
      q_s[c][fa] = fmaf(p, k, -(q * s));
      q_s[c][fb] = fmaf(p, s, q * k);
    }
  }
  __syncthreads();
  // Operand of step (j, half): features 64 j + 16 grp + 8 half .. + 7 of the lane's column.
  bf16x8 q[3][2 * W];
#pragma unroll
  for (int j = 0; j < 2 * W; ++j) {
    const float *p = &q_s[col][64 * (j >> 1) + 16 * grp + 8 * (j & 1)];
    const Bf16x3 lo = split_bf16x3(*reinterpret_cast<const f32x4 *>(p));
    const Bf16x3 hi = split_bf16x3(*reinterpret_cast<const f32x4 *>(p + 4));
#pragma unroll
    for (int i = 0; i < 3; ++i) q[i][j] = join_bf16(lo, hi, i);
  }
  // Last key that the lane's column sees; columns past the last see what it sees.
  const int mine = first + min(c0 + col, last) / group;
  const int seen_by_all = first + u0;

  f32x4 o[4 * W];
#pragma unroll
  for (int i = 0; i < 4 * W; ++i) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  for (int b = b0 + wave; b < b1; b += kWaves) {
    const long long place = cache_block(cv, r, h, b);
    const size_t base = (size_t)(place < 0 ? 0 : place) * 64 * WIDE;
    const uint8_t *kp = cv.keys + base + (16 * (col >> 2) + (col & 3)) * WIDE + 16 * grp;
    const uint8_t *vp = cv.values + base + col * 64 + 16 * grp;
    const float ks = place < 0 ? __builtin_nanf("") : cv.key_scales[place] * a.c1;
    const float vs = place < 0 ? 0.0f : cv.value_scales[place];
    u32x4 kr[4][W], vr[4 * W];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < W; ++j)
        kr[t][j] = *reinterpret_cast<const u32x4 *>(kp + 4 * t * WIDE + 64 * j);
#pragma unroll
    for (int f = 0; f < 4 * W; ++f) vr[f] = *reinterpret_cast<const u32x4 *>(vp + f * 16 * 64);
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 2 * W; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bf16x8 k = codes_bf16(kr[t][j >> 1][2 * (j & 1)], kr[t][j >> 1][2 * (j & 1) + 1]);
#pragma unroll
        for (int i = 0; i < 3; ++i) s[t] = mfma_16x16x32_bf16(k, q[2 - i][j], s[t]);
      }
    const bool masked = b * 64 + 63 > seen_by_all;
    const int limit = mine - b * 64 - 16 * grp;  // of the lane's 16 keys: those <= limit
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] *= ks;
        if (masked && 4 * t + i > limit) s[t][i] = -INFINITY;
        mx = fmaxf(mx, s[t][i]);
      }
    mx = pair_max(pair16_max(mx));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float alpha = m == -INFINITY ? 0.0f : fast_exp2(m - ref);
    m = mn;
    float rs = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = fast_exp2(s[t][i] - ref);
        rs += e;
        s[t][i] = e * vs;
      }
    l = l * alpha + rs;
#pragma unroll
    for (int f = 0; f < 4 * W; ++f) o[f] *= alpha;
    bf16x8 p[3][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Bf16x3 lo = split_bf16x3(s[2 * k]), hi = split_bf16x3(s[2 * k + 1]);
#pragma unroll
      for (int i = 0; i < 3; ++i) p[i][k] = join_bf16(lo, hi, i);
    }
    if (masked) {
      // What a column does not see must not reach it: the product of a probability of 0
      // and a NaN (a later token's, or what was in memory) is NaN. The tile's NaN codes
      // become 0, and the columns that do see one get it back.
      uint32_t any = 0;
#pragma unroll
      for (int f = 0; f < 4 * W; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= nan_codes(vr[f][e]);
      if (__any(any != 0)) {
        union {
          unsigned short u[8];
          bf16x8 v;
        } sees[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) sees[k].u[e] = 8 * k + e <= limit ? 0x3f80 : 0;
#pragma unroll
        for (int f = 0; f < 4 * W; ++f) {
          f32x4 n = {0, 0, 0, 0};
          u32x4 is;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t bad = nan_codes(vr[f][e]);
            is[e] = (bad >> 7) * 0x38u;  // e4m3's 1
            vr[f][e] &= ~((bad >> 7) * 0xffu);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
            n = mfma_16x16x32_bf16(codes_bf16(is[2 * k], is[2 * k + 1]), sees[k].v, n);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n[i] > 0.0f) o[f][i] = __builtin_nanf("");
        }
      }
    }
#pragma unroll
    for (int f = 0; f < 4 * W; ++f)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bf16x8 v = codes_bf16(vr[f][2 * k], vr[f][2 * k + 1]);
#pragma unroll
        for (int i = 0; i < 3; ++i) o[f] = mfma_16x16x32_bf16(v, p[2 - i][k], o[f]);
      }
  }
  l = pair_sum(pair16_sum(l));
  // The waves' sums, joined by all of them.
  if (grp == 0) st_s[wave][col] = Stats{m, l};
#pragma unroll
  for (int f = 0; f < 4 * W; ++f)
    *reinterpret_cast<f32x4 *>(&o_s[wave][col][16 * f + 4 * grp]) = o[f];
  __syncthreads();
  for (int at = threadIdx.x; at < kCols * (WIDE / 4); at += 256) {
    const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
    if (c0 + c > last || f >= hd) continue;
    float ref = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) ref = fmaxf(ref, st_s[w][c].m);
    const float safe = ref == -INFINITY ? 0.0f : ref;
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float k = fast_exp2(st_s[w][c].m - safe);
      total = fmaf(st_s[w][c].l, k, total);
      sum += *reinterpret_cast<const f32x4 *>(&o_s[w][c][f]) * k;
    }
    if (a.parts == 1) {
      store_out<T>(a, r, h, column_of(c0 + c, group, L, count), f, sum, 1.0f / total);
    } else {
      *reinterpret_cast<f32x4 *>(a.part_out + (item * kCols + c) * WIDE + f) = sum;
      if (f == 0) {
        a.part_stats[(item * kCols + c) * 2] = ref;
        a.part_stats[(item * kCols + c) * 2 + 1] = total;
      }
    }
  }
}

// Joins a tile's parts, four features a thread.
template <typename T, int W>
__global__ __launch_bounds__(256) void cached_join_kernel(CachedArgs a) {
  constexpr int WIDE = 64 * W;
  const CacheView &cv = a.cache;
  const int at_thread = blockIdx.x * 256 + threadIdx.x;
  const int c = at_thread / (16 * W), f = 4 * (at_thread % (16 * W));
  const int tile = c / kCols;
  const int h = blockIdx.y, r = blockIdx.z, L = cv.L, group = a.group;
  int first, count;
  if (!cache_row(cv, r, first, count)) return;
  const int active = group * count;
  if (c >= active || f >= cv.hd) return;
  const int u1 = (min((tile + 1) * kCols, active) - 1) / group;
  const int blocks = (first + u1) / 64 + 1;
  const int share = (blocks + a.parts - 1) / a.parts;
  const int parts = (blocks + share - 1) / share;
  const size_t item = (((size_t)r * cv.kv_heads + h) * a.tiles + tile) * a.parts;
  float ref = -INFINITY;
  for (int p = 0; p < parts; ++p)
    ref = fmaxf(ref, a.part_stats[((item + p) * kCols + c % kCols) * 2]);
  const float safe = ref == -INFINITY ? 0.0f : ref;
  f32x4 sum = {0, 0, 0, 0};
  float total = 0.0f;
  for (int p = 0; p < parts; ++p) {
    const size_t at = (item + p) * kCols + c % kCols;
    const float k = fast_exp2(a.part_stats[at * 2] - safe);
    total = fmaf(a.part_stats[at * 2 + 1], k, total);
    sum += *reinterpret_cast<const f32x4 *>(a.part_out + at * WIDE + f) * k;
  }
  store_out<T>(a, r, h, column_of(c, group, L, count), f, sum, 1.0f / total);
}

template <typename T, int W>
hipError_t launch_wide(const CachedArgs &a, int rows, hipStream_t stream, const KernelEvents &ev) {
  const dim3 grid((unsigned)(a.tiles * a.parts), (unsigned)a.cache.kv_heads, (unsigned)rows);
  hipExtLaunchKernelGGL((cached_kernel<T, W>), grid, dim3(256), 0, stream, ev.start,
                        a.parts == 1 ? ev.stop : nullptr, 0, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.parts == 1) return e;
  const size_t threads = (size_t)a.group * a.cache.L * 16 * W;
  hipExtLaunchKernelGGL((cached_join_kernel<T, W>),
                        dim3((unsigned)((threads + 255) / 256), grid.y, grid.z), dim3(256), 0,
                        stream, nullptr, ev.stop, 0, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const CachedArgs &a, int rows, hipStream_t stream, const KernelEvents &ev) {
  switch (a.cache.wide / 64) {
    case 1: return launch_wide<T, 1>(a, rows, stream, ev);
    case 2: return launch_wide<T, 2>(a, rows, stream, ev);
    case 3: return launch_wide<T, 3>(a, rows, stream, ev);
    default: return launch_wide<T, 4>(a, rows, stream, ev);
  }
}

}  // namespace

void cached_plan(CachedArgs &a, int rows) {
  a.tiles = (a.group * a.cache.L + kCols - 1) / kCols;
  const long long items = (long long)rows * a.cache.kv_heads * a.tiles;
  const long long most = ((long long)a.cache.per_row << a.cache.blocks_log2) / kWaves;
  long long parts = 2 * a.cus / items;
  if (parts > most) parts = most;
  a.parts = parts < 1 ? 1 : (int)parts;
}

size_t cached_work_bytes(const CachedArgs &a, int rows) {
  if (a.parts == 1) return 0;
  return (size_t)rows * a.cache.kv_heads * a.tiles * a.parts * kCols * (a.cache.wide + 2) *
         sizeof(float);
}

hipError_t launch_cached_attention(const CachedArgs &a, int rows, hipStream_t stream,
                                   const KernelEvents &ev) {
  return a.bf16 ? launch_typed<unsigned short>(a, rows, stream, ev)
                : launch_typed<float>(a, rows, stream, ev);
}

}  // namespace tfd
