// Causal attention of new tokens over a paged cache of e4m3 keys and values.
//
// Per row, new token u (of count) and query head, with its queries normalized
// (x / sqrt(mean(x^2) + eps) (1 + w)) and turned to position first + u:
//   s_j = q . k_j / sqrt(hd) over the keys j <= first + u
//   o   = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), times sigmoid(gate)
//
// Products. A code is exact in fp16, so a product with an f32 operand is two fp16 matrix
// products, one for each piece of the f32 one: hi the nearest fp16, lo that of the rest, 22
// significant bits. A column's queries are taken times a power of two that brings the largest
// to [2^13, 2^14), so that what fp16's range cuts off is below 2^-37 of the column's
// largest; probabilities (at most 1) times 2^15, which leaves 2^-40. The blocks' key scales
// are applied to the scores; the outputs are kept in units of the last block's value scale.
//
// Tiles. The columns of a product are (token, query head of the group) pairs of one
// (row, kv head), 16 of them; its rows are keys, then features. S^T = K Q^T leaves lane
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

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kCols = kCachedColumns;
constexpr int kJoin = 16;  // parts that are joined at once
// Workgroups that a launch deals parts to, at most: also a tile's parts.
constexpr int kMostParts = 512;
constexpr int kMostJoined = kMostParts / kJoin + 1;

// Eight e4m3 codes as fp16.
__device__ __forceinline__ f16x8 codes_f16(uint32_t lo, uint32_t hi) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Pieces of four f32 values.
struct F16x2 {
  f16x4 hi, lo;
};
__device__ __forceinline__ F16x2 split_f16x2(f32x4 v) {
  F16x2 s;
  s.hi = __builtin_convertvector(v, f16x4);
  s.lo = __builtin_convertvector(v - __builtin_convertvector(s.hi, f32x4), f16x4);
  return s;
}
__device__ __forceinline__ f16x8 join_f16(f16x4 a, f16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
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

// out of column c, features f .. f + 3.
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

// Partial results pass between workgroups of a launch, whose XCDs' caches do not see each
// other's: stores and loads that go past them (sc1). A writer waits for its stores (stored())
// before it says that they are there. Fences would write back and drop the caches' lines
// for all workgroups: 128 rows of 8192 tokens took 400 us with two a wave.
constexpr int kPastCaches = 16;
struct Parts {
  __amdgpu_buffer_rsrc_t out, stats;
  template <int WIDE>
  static __device__ __forceinline__ Parts of(const CachedArgs &a) {
    const uint32_t slots = a.slots;
    return Parts{buffer_rsrc(a.part_out, slots * kCols * WIDE * 4),
                 buffer_rsrc(a.part_stats, slots * kCols * 8)};
  }
};
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t r, f32x4 v, int at) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4v, v), r, at, 0, kPastCaches);
}
__device__ __forceinline__ f32x4 get4(__amdgpu_buffer_rsrc_t r, int at) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kPastCaches));
}
__device__ __forceinline__ void put2(__amdgpu_buffer_rsrc_t r, float x, float y, int at) {
  __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(x), __float_as_uint(y)}, r, at, 0,
                                        kPastCaches);
}
__device__ __forceinline__ u32x2 get2(__amdgpu_buffer_rsrc_t r, int at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, kPastCaches));
}
__device__ __forceinline__ void stored() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// What a workgroup of the rows kernel does: part `part` of `parts` of the blocks of one tile
// of columns of one (row, kv head).
struct Share {
  int r, h, tile, part, parts;
  int slot;  // of the first part's partial results, where there are several
  int first, count;
  bool sound;
};
// Blocks that a row's last token sees.
__device__ __forceinline__ int row_blocks(const CacheView &cv, int r) {
  int first, count;
  return cache_row(cv, r, first, count) && count ? ((first + count - 1) >> 6) + 1 : 0;
}
// The rows' blocks are dealt to the grid's workgroups: a part has at most `most` blocks, the
// least with which the parts are no more than the workgroups. Every wave finds its
// workgroup's share by itself, lane by row. False: no share is left for this workgroup.
__device__ __forceinline__ bool find_share(const CachedArgs &a, uint32_t w, Share &s) {
  const CacheView &cv = a.cache;
  const int lane = threadIdx.x & 63, per = cv.kv_heads * a.tiles;
  double all = 0.0;
  int mine = 0;
  for (int r0 = 0; r0 < a.rows; r0 += 64) {
    mine = r0 + lane < a.rows ? row_blocks(cv, r0 + lane) : 0;
    all += (double)wave_sum(mine);
  }
  // sum(ceil(blocks / most)) is at most sum(blocks) / most + items, which fits the grid
  // from twice the even share on where the items are at most half of it (spread 0), and
  // with an even share of the `spread` workgroups that there are beside the items.
  int most;
  if (a.spread) {
    most = max(a.least, (int)(all * per / a.spread) + 1);
  } else {
    const uint32_t room = gridDim.x;
    most = max(a.least, (int)(all * per / room) + 1);
    for (;;) {
      double n = 0.0;
      for (int r0 = 0; r0 < a.rows; r0 += 64) {
        if (a.rows > 64) mine = r0 + lane < a.rows ? row_blocks(cv, r0 + lane) : 0;
        n += (double)wave_sum(r0 + lane < a.rows ? max(1, (mine + most - 1) / most) : 0);
      }
      if (n * per <= room) break;
      most += max(1, most >> 4);
    }
  }
  uint32_t before = 0, slots = 0;  // workgroups and slots of the rows up to r0
  for (int r0 = 0; r0 < a.rows; r0 += 64) {
    if (a.rows > 64) mine = r0 + lane < a.rows ? row_blocks(cv, r0 + lane) : 0;
    const int parts = r0 + lane < a.rows ? max(1, (mine + most - 1) / most) : 0;
    uint32_t upto = (uint32_t)parts * per, split = parts > 1 ? upto : 0;
    const uint32_t own = upto, own_split = split;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(upto, o), v = __shfl_up(split, o);
      if (lane >= o) {
        upto += u;
        split += v;
      }
    }
    const uint64_t found = __ballot(w >= before + upto - own && w < before + upto);
    if (found) {
      const int at = __builtin_ctzll(found);
      const uint32_t in = w - before - (uint32_t)__builtin_amdgcn_readlane((int)(upto - own), at);
      s.r = r0 + at;
      s.parts = __builtin_amdgcn_readlane(parts, at);
      const uint32_t item = in / (uint32_t)s.parts;
      s.part = (int)(in - item * s.parts);
      s.h = (int)(item / (uint32_t)a.tiles);
      s.tile = (int)(item - (uint32_t)s.h * a.tiles);
      s.slot = (int)(slots + (uint32_t)__builtin_amdgcn_readlane((int)(split - own_split), at) +
                     item * s.parts);
      s.sound = cache_row(cv, s.r, s.first, s.count);
      if (!s.sound) s.first = s.count = 0;
      return true;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    slots += (uint32_t)__builtin_amdgcn_readlane((int)split, 63);
  }
  return false;
}

template <typename T, int W>
__global__ __launch_bounds__(256, 2) void cached_rows_kernel(CachedArgs a) {
  constexpr int WIDE = 64 * W;
  constexpr int QROW = WIDE + 8;  // halves of a column's piece in LDS
  __shared__ union {
    struct {
      float x[kCols][WIDE + 4];  // queries before they are split
      _Float16 q[2][kCols][QROW];
    };
    float o[kWaves][kCols][WIDE + 4];  // the waves' outputs
    struct {
      float weight[kMostJoined][kCols], total[kMostJoined][kCols];
    };
  } sh;
  __shared__ float scale_s[kCols];  // c1 over the column's power of two
  __shared__ float m_s[kWaves][kCols], l_s[kWaves][kCols], unit_s[kWaves];
  __shared__ int last_s;
  const CacheView &cv = a.cache;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  Share sh_;
  if (!find_share(a, blockIdx.x, sh_)) return;
  const int r = sh_.r, h = sh_.h, first = sh_.first, count = sh_.count;
  const int L = cv.L, hd = cv.hd, group = a.group;
  const int c0 = sh_.tile * kCols, columns = group * L;
  const int active = group * count;  // columns

  // Columns of tokens that are not active, and of rows whose pages do not hold them.
  if (sh_.part == 0 && c0 + kCols > active) {
    for (int c = wave; c < kCols; c += kWaves) {
      if (c0 + c < active || c0 + c >= columns) continue;
      const Column at = column_of(c0 + c, group, L, count);
      const size_t o = (((size_t)r * a.heads + h * group + at.head) * hd) * L + at.token;
      for (int f = lane; f < hd; f += 64)
        a.out[o + (size_t)f * L] = sh_.sound ? 0.0f : __builtin_nanf("");
    }
  }
  if (c0 >= active) return;
  const int last = min(c0 + kCols, active) - 1;  // last active column of the tile
  const int u0 = c0 / group, u1 = last / group;
  const int blocks = (first + u1) / 64 + 1;
  // Parts of a tile that ends before the row does may be empty.
  const int b0 = (int)((long long)blocks * sh_.part / sh_.parts);
  const int b1 = (int)((long long)blocks * (sh_.part + 1) / sh_.parts);

  u32x4 kr[4][W], vr[4 * W];
  float ks = 0.0f, vs = 0.0f;
  const int k_at = (16 * (col >> 2) + (col & 3)) * WIDE + 16 * grp;
  const int v_at = col * 64 + 16 * grp;
  auto load_keys = [&](long long place) {
    const uint8_t *p = cv.keys + (size_t)(place < 0 ? 0 : place) * 64 * WIDE + k_at;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < W; ++j)
        kr[t][j] = *reinterpret_cast<const u32x4 *>(p + 4 * t * WIDE + 64 * j);
    ks = place < 0 ? __builtin_nanf("") : cv.key_scales[place];
  };
  auto load_values = [&](long long place) {
    const uint8_t *p = cv.values + (size_t)(place < 0 ? 0 : place) * 64 * WIDE + v_at;
#pragma unroll
    for (int f = 0; f < 4 * W; ++f) 
      vr[f] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + f * 16 * 64));
    vs = place < 0 ? 1.0f : cv.value_scales[place];
  };
  // The first block is on its way while the queries are made.
  long long place = 0;
  if (b0 + wave < b1) {
    place = cache_block(cv, r, h, b0 + wave);
    load_keys(place);
    load_values(place);
  }

  // Queries: a wave takes a column, its lanes the features.
  for (int c = wave; c < kCols; c += kWaves) {
    float x[W];
    const bool in = c0 + c <= last;
    if (in) {
      const Column at = column_of(c0 + c, group, L, count);
      const size_t from = (((size_t)r * a.heads + h * group + at.head) * hd) * L + at.token;
      float sq = 0.0f;
#pragma unroll
      for (int n = 0; n < W; ++n) {
        const int f = lane + 64 * n;
        x[n] = f < hd ? load_as_f32<T>(a.q, from + (size_t)f * L) : 0.0f;
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
      if (a.plan.pairs > 0) {
#pragma unroll
        for (int n = 0; n < W; ++n) sh.x[c][lane + 64 * n] = x[n];
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
          const float p = sh.x[c][fa], q = sh.x[c][fb];
          sh.x[c][fa] = fmaf(p, k, -(q * s));
          sh.x[c][fb] = fmaf(p, s, q * k);
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < W; ++n) x[n] = sh.x[c][lane + 64 * n];
      }
    } else {
#pragma unroll
      for (int n = 0; n < W; ++n) x[n] = 0.0f;
    }
    float most = 0.0f;
#pragma unroll
    for (int n = 0; n < W; ++n) most = fmaxf(most, fabsf(x[n]));
    most = wave_max_f(most);
    int e = 0;
    if (most > 0.0f && most <= 3.402823466e38f) (void)frexpf(most, &e);
    e = 14 - max(-100, e);
#pragma unroll
    for (int n = 0; n < W; ++n) {
      const float y = ldexpf(x[n], e);
      const _Float16 hi = (_Float16)y;
      sh.q[0][c][lane + 64 * n] = hi;
      sh.q[1][c][lane + 64 * n] = (_Float16)(y - (float)hi);
    }
    if (lane == 0) scale_s[c] = ldexpf(a.c1, -e);
  }
  __syncthreads();
  const float c1 = scale_s[col];
  // Last key that the lane's column sees; columns past the last see what it sees.
  const int mine = first + min(c0 + col, last) / group;
  const int seen_by_all = first + u0;

  f32x4 o[4 * W];
#pragma unroll
  for (int i = 0; i < 4 * W; ++i) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f, unit = 1.0f, top = 0.0f;
  for (int b = b0 + wave; b < b1; b += kWaves) {
    const bool more = b + kWaves < b1;
    const long long next = more ? cache_block(cv, r, h, b + kWaves) : -1;
    // The queries' operands are read again for every block: kept, they would take the
    // registers of a second workgroup on the CU.
    asm volatile("" ::: "memory");
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 2 * W; ++j) {
      const int at = 64 * (j >> 1) + 16 * grp + 8 * (j & 1);
      const f16x8 hi = *reinterpret_cast<const f16x8 *>(&sh.q[0][col][at]);
      const f16x8 lo = *reinterpret_cast<const f16x8 *>(&sh.q[1][col][at]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f16x8 k = codes_f16(kr[t][j >> 1][2 * (j & 1)], kr[t][j >> 1][2 * (j & 1) + 1]);
        s[t] = mfma_16x16x32_f16(k, lo, s[t]);
        s[t] = mfma_16x16x32_f16(k, hi, s[t]);
      }
    }
    const float factor = ks * c1;
    // Not before the products that read the registers: they would be doubled.
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_keys(next);
    __builtin_amdgcn_sched_barrier(0);
    const bool masked = b * 64 + 63 > seen_by_all;
    const int limit = mine - b * 64 - 16 * grp;  // of the lane's 16 keys: those <= limit
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] *= factor;
        if (masked && 4 * t + i > limit) s[t][i] = -INFINITY;
        mx = fmaxf(mx, s[t][i]);
      }
    mx = pair_max(pair16_max(mx));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float alpha = m == -INFINITY ? 0.0f : fast_exp2(m - ref);
    m = mn;
    // The block's value scale becomes the unit, unless it is so far below the largest one
    // that the outputs could leave f32's range in it: then the probabilities carry the
    // difference.
    top = fmaxf(top, vs);
    const float to = fmaxf(vs, top * 0x1p-90f);
    const float turn = alpha * (unit / to), p15 = 0x1p15f * (vs / to);
    unit = to;
    float rs = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = fast_exp2(s[t][i] - ref);
        rs += e;
        s[t][i] = e * p15;
      }
    l = l * alpha + rs;
    if (__any(turn != 1.0f)) {
#pragma unroll
      for (int f = 0; f < 4 * W; ++f) o[f] *= turn;
    }
    f16x8 p[2][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const F16x2 lo = split_f16x2(s[2 * k]), hi = split_f16x2(s[2 * k + 1]);
      p[0][k] = join_f16(lo.hi, hi.hi);
      p[1][k] = join_f16(lo.lo, hi.lo);
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
        f16x8 sees[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) sees[k][e] = (_Float16)(8 * k + e <= limit ? 1.0f : 0.0f);
#pragma unroll
        for (int f = 0; f < 4 * W; ++f) {
          f32x4 n = {0, 0, 0, 0};
          u32x4 is;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t x = vr[f][e];
            asm("" : "+v"(x));  // taken again: kept from above, it would cost 16 W registers
            const uint32_t bad = nan_codes(x);
            is[e] = (bad >> 7) * 0x38u;  // e4m3's 1
            vr[f][e] &= ~((bad >> 7) * 0xffu);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
            n = mfma_16x16x32_f16(codes_f16(is[2 * k], is[2 * k + 1]), sees[k], n);
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
        const f16x8 v = codes_f16(vr[f][2 * k], vr[f][2 * k + 1]);
        o[f] = mfma_16x16x32_f16(v, p[1][k], o[f]);
        o[f] = mfma_16x16x32_f16(v, p[0][k], o[f]);
      }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_values(next);
  }
  l = pair_sum(pair16_sum(l));
  __syncthreads();  // the queries' place is the outputs'
  // The waves' sums, joined by all of them, in units of 1 and 2^-15 probabilities.
  if (grp == 0) {
    m_s[wave][col] = m;
    l_s[wave][col] = l;
  }
  if (lane == 0) unit_s[wave] = unit * 0x1p-15f;
  const int used = last - c0 + 1;
#pragma unroll
  for (int f = 0; f < 4 * W; ++f)
    if (col < used) *reinterpret_cast<f32x4 *>(&sh.o[wave][col][16 * f + 4 * grp]) = o[f];
  __syncthreads();
  const Parts parts = Parts::of<WIDE>(a);
  for (int at = threadIdx.x; at < used * (WIDE / 4); at += 256) {
    const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
    float ref = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) ref = fmaxf(ref, m_s[w][c]);
    const float safe = ref == -INFINITY ? 0.0f : ref;
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float k = fast_exp2(m_s[w][c] - safe);
      total = fmaf(l_s[w][c], k, total);
      sum += *reinterpret_cast<const f32x4 *>(&sh.o[w][c][f]) * (k * unit_s[w]);
    }
    if (sh_.parts == 1) {
      if (f < hd) store_out<T>(a, r, h, column_of(c0 + c, group, L, count), f, sum, 1.0f / total);
    } else {
      const int to = (sh_.slot + sh_.part) * kCols + c;
      put4(parts.out, sum, (to * WIDE + f) * 4);
      if (f == 0) put2(parts.stats, ref, total, to * 8);
    }
  }
  if (sh_.parts == 1) return;
  // The last workgroup of 16 parts to get here joins them, in the first one's place; the last
  // one of a tile's groups joins those. Each leaves its counter as it was.
  auto arrived_last = [&](unsigned *done, int of) {
    stored();
    __syncthreads();
    if (threadIdx.x == 0) {
      const unsigned n =
          __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last_s = n + 1 == (unsigned)of;
      if (last_s) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return last_s != 0;
  };
  // Slots from, from + step, .., n of them: the weights first, then the outputs.
  auto join = [&](int from, int step, int n, bool finish) {
    float(*weight)[kCols] = sh.weight;
    for (int at = threadIdx.x; at < n * used; at += 256) {
      const int p = at / used, c = at - p * used;
      const u32x2 s = get2(parts.stats, ((from + p * step) * kCols + c) * 8);
      weight[p][c] = __uint_as_float(s[0]);
      sh.total[p][c] = __uint_as_float(s[1]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < used; c += 256) {
      float ref = -INFINITY, total = 0.0f;
      for (int p = 0; p < n; ++p) ref = fmaxf(ref, weight[p][c]);
      const float safe = ref == -INFINITY ? 0.0f : ref;
      for (int p = 0; p < n; ++p) {
        const float k = fast_exp2(weight[p][c] - safe);
        weight[p][c] = k;
        total = fmaf(sh.total[p][c], k, total);
      }
      m_s[0][c] = ref;
      l_s[0][c] = total;
    }
    __syncthreads();
    for (int at = threadIdx.x; at < used * (WIDE / 4); at += 256) {
      const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
      f32x4 sum = {0, 0, 0, 0};
#pragma unroll 8
      for (int p = 0; p < n; ++p)
        sum += get4(parts.out, (((from + p * step) * kCols + c) * WIDE + f) * 4) * weight[p][c];
      if (finish) {
        if (f < hd)
          store_out<T>(a, r, h, column_of(c0 + c, group, L, count), f, sum, 1.0f / l_s[0][c]);
      } else {
        put4(parts.out, sum, ((from * kCols + c) * WIDE + f) * 4);
        if (f == 0) put2(parts.stats, m_s[0][c], l_s[0][c], (from * kCols + c) * 8);
      }
    }
  };
  const int lead = sh_.part & ~(kJoin - 1), members = min(kJoin, sh_.parts - lead);
  if (!arrived_last(a.part_done + sh_.slot + lead, members)) return;
  join(sh_.slot + lead, 1, members, sh_.parts <= kJoin);
  if (sh_.parts <= kJoin) return;
  const int groups = (sh_.parts + kJoin - 1) / kJoin;
  if (!arrived_last(a.part_done + a.slots + sh_.slot, groups)) return;
  join(sh_.slot, kJoin, groups, true);
}

template <typename T, int W>
hipError_t launch_wide(const CachedArgs &a, hipStream_t stream, const KernelEvents &ev) {
  hipExtLaunchKernelGGL((cached_rows_kernel<T, W>), dim3((unsigned)a.grid), dim3(256), 0, stream, ev.start,
                        ev.stop, 0, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const CachedArgs &a, hipStream_t stream, const KernelEvents &ev) {
  switch (a.cache.wide / 64) {
    case 1: return launch_wide<T, 1>(a, stream, ev);
    case 2: return launch_wide<T, 2>(a, stream, ev);
    case 3: return launch_wide<T, 3>(a, stream, ev);
    default: return launch_wide<T, 4>(a, stream, ev);
  }
}

}  // namespace

void cached_plan(CachedArgs &a) {
  a.tiles = (a.group * a.cache.L + kCols - 1) / kCols;
  // Two workgroups a CU are there at once. Up to half as many items are dealt to exactly
  // those: one more would run after them (128 rows of 8000 to 8192 tokens in 520 workgroups
  // 270 us, in 512 200).
  const size_t items = (size_t)a.rows * a.cache.kv_heads * a.tiles;
  const int here = a.cus < kMostParts / 2 ? 2 * a.cus : kMostParts;
  a.spread = 2 * items <= (size_t)here ? 0 : here;
  a.grid = (int)(a.spread ? items + here : here);
  a.least = 2 * kWaves;
  // Parts of tiles in several: all there are, or, as a tile in n > 1 parts has more than
  // (n - 1) most blocks and all have at most spread * most, 2 spread.
  a.slots = 2 * here;
}

CachedSpace cached_space(const CachedArgs &a) {
  return CachedSpace{2 * (size_t)a.slots * sizeof(unsigned), (size_t)a.slots * kCols * 2 * sizeof(float),
                     (size_t)a.slots * kCols * a.cache.wide * sizeof(float)};
}

hipError_t launch_cached_attention(const CachedArgs &a, hipStream_t stream,
                                   const KernelEvents &ev) {
  return a.bf16 ? launch_typed<unsigned short>(a, stream, ev)
                : launch_typed<float>(a, stream, ev);
}

}  // namespace tfd
