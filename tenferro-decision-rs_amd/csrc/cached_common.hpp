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
// largest; probabilities (at most 1) times 2^11 to 2^15, which leaves 2^-36. The blocks' key
// scales are applied to the scores, their value scales to the probabilities, against a unit
// that the outputs are kept in.
//
// Tiles. The columns of a product are (token, query head of the group) pairs of one
// (row, kv head), 16 of them; its rows are keys, then features. S^T = K Q^T leaves lane
// (column l % 16, group g = l / 16) the keys 16 g + 4 t + i of accumulator i of key tile t,
// as the rows of tile t are taken in that order: 16 keys in a row, which are what the lane
// has to give to O^T = V^T P^T and what 16 bytes of a value's block hold. No value passes
// between lanes but a column's maximum and sum.
//
// Two kernels: cached_rows.hip for few columns, whose time is the cache's way from memory, and
// cached_prompt.hip for many, whose time is the products.
#pragma once

#include <type_traits>

#include "rotary.hpp"
#include "tfd_device.hpp"
#include "tfd_internal.hpp"

namespace tfd {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kJoin = 16;  // parts that are joined at once; CachedArgs::cap of them by groups

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

// Partial results pass between workgroups of a launch, whose XCDs' caches do not see each
// other's: stores and loads that go past them (sc1). A writer waits for its stores (stored())
// before it says that they are there. Fences would write back and drop the caches' lines
// for all workgroups: 128 rows of 8192 tokens took 400 us with two a wave.
constexpr int kPastCaches = 16;
constexpr int kNonTemporal = 2;
struct Parts {
  __amdgpu_buffer_rsrc_t out, stats;
  template <int COLS, int WIDE>
  static __device__ __forceinline__ Parts of(const CachedArgs &a) {
    const uint32_t slots = a.slots;
    return Parts{buffer_rsrc(a.part_out, slots * COLS * WIDE * 4),
                 buffer_rsrc(a.part_stats, slots * COLS * 8)};
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

// Sum and maximum over the wave, the same in all lanes: within 16 lanes by DPP, then by lane
// swaps.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
      0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;
__device__ __forceinline__ float all_sum(float x) {
  x += dpp<kSwap1>(x);
  x += dpp<kSwap2>(x);
  x += dpp<kMirror8>(x);
  x += dpp<kMirror16>(x);
  return pair_sum(pair16_sum(x));
}
__device__ __forceinline__ float all_max(float x) {
  x = fmaxf(x, dpp<kSwap1>(x));
  x = fmaxf(x, dpp<kSwap2>(x));
  x = fmaxf(x, dpp<kMirror8>(x));
  x = fmaxf(x, dpp<kMirror16>(x));
  return pair_max(pair16_max(x));
}
__device__ __forceinline__ int all_sum_of(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, kSwap1, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, kSwap2, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, kMirror8, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, kMirror16, 0xf, 0xf, true);
  return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) +
         (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}
// Sum over the lanes up to this one: within 16 lanes, then their last lanes' sums on.
__device__ __forceinline__ uint32_t sum_upto(uint32_t x) {
  int v = (int)x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return (uint32_t)v;
}

// Reads at a place that all lanes share, by the scalar unit: they wait for no vector load
// that is on its way. For what no kernel writes while it is read: tables and scales.
template <typename T>
__device__ __forceinline__ T scalar_read(const T *p, long long i) {
  return ((const __attribute__((address_space(4))) T *)p)[i];
}
// cache_block of a row, head and block that all lanes share.
__device__ __forceinline__ long long shared_block(const CacheView &c, int r, int h, int b) {
  const int page = scalar_read(c.table, (long long)r * c.per_row + (b >> c.blocks_log2));
  if ((uint32_t)page >= (uint32_t)c.pages) return -1;
  return (((long long)page * c.kv_heads + h) << c.blocks_log2) + (b & ((1 << c.blocks_log2) - 1));
}

// Part `part` of `parts` of the blocks of one tile of columns of one (row, kv head).
struct Share {
  int r, h, tile, part, parts;
  int slot;  // of the first part's partial results, where there are several
};
// How a launch's workgroups share the rows' blocks: a tile's go in parts of at most `most`
// blocks. Every wave finds that out by itself, each lane for `each` rows in a row.
// An even share for every workgroup is `all` / workgroups. If parts of up to 5/16 more are no
// more than the workgroups (ragged lengths leave parts that are not full), that is it:
// the work then takes as long as one part. Otherwise parts are even shares, and some workgroups
// have one more: finer ones cost more in their beginnings and ends than a shorter last one
// saves (200 rows of 1500 tokens, 2 kv heads: 39 us, in halves 60, in quarters 70; 300 rows
// of 4096: 74, 76, 88).
struct Deal {
  int each, most;
  // By lane, in LDS between the shares: parts of the lanes up to this one, and of this one;
  // those of tiles in several parts.
  struct Lanes {
    uint32_t upto[64], own[64], split_upto[64], split_own[64];
  };

  // Blocks that row r's last token sees.
  static __device__ __forceinline__ int blocks(const CachedArgs &a, int r) {
    int first, count;
    return r < a.rows && cache_row(a.cache, r, first, count) && count ? ((first + count - 1) >> 6) + 1
                                                                       : 0;
  }
  __device__ __forceinline__ int parts(const CachedArgs &a, int r, int nb) const {
    return r < a.rows ? max(1, min(a.cap, (nb + most - 1) / most)) : 0;
  }
  // Every wave writes the same values.
  __device__ __forceinline__ void make(const CachedArgs &a, Lanes &lanes) {
    const int lane = threadIdx.x & 63, per = a.cache.kv_heads * a.tiles;
    each = (a.rows + 63) >> 6;
    const int r0 = lane * each;
    int nb = blocks(a, r0);  // of the lane's first row: the only one up to 64 rows
    float mine = (float)nb;
    for (int j = 1; j < each; ++j) mine += (float)blocks(a, r0 + j);
    const int room = (int)gridDim.x;
    // At least an even share, whatever f32 rounds, as the places for partial results are counted
    // by it; rows' blocks are at most 2^25.
    int even = (int)fminf(all_sum(mine) * (float)per / (float)room, 0x1p26f) + 1;
    even += even >> 16;
    most = max(a.least, even);
    bool fits = false;
    for (int step = 0; step < 6 && !fits && (size_t)a.rows * per <= (size_t)room; ++step) {
      if (step) most += max(1, even >> 4);
      int n = parts(a, r0, nb);
      for (int j = 1; j < each; ++j) n += parts(a, r0 + j, blocks(a, r0 + j));
      fits = (long long)all_sum_of(n) * per <= room;
    }
    if (!fits) most = max(a.least, even);
    uint32_t own = 0, split_own = 0;
    for (int j = 0; j < each; ++j) {
      const uint32_t n = (uint32_t)parts(a, r0 + j, j ? blocks(a, r0 + j) : nb) * per;
      own += n;
      if (n > (uint32_t)per) split_own += n;
    }
    lanes.own[lane] = own;
    lanes.split_own[lane] = split_own;
    lanes.upto[lane] = sum_upto(own);
    lanes.split_upto[lane] = sum_upto(split_own);
    __builtin_amdgcn_wave_barrier();
  }
  // Share w, false past the last.
  __device__ __forceinline__ bool find(const CachedArgs &a, const Lanes &lanes, uint32_t w,
                                       Share &s) const {
    const int lane = threadIdx.x & 63, per = a.cache.kv_heads * a.tiles;
    const uint32_t upto = lanes.upto[lane], own = lanes.own[lane];
    const uint32_t split_upto = lanes.split_upto[lane], split_own = lanes.split_own[lane];
    if (w >= (uint32_t)__builtin_amdgcn_readlane((int)upto, 63)) return false;
    auto of_lane = [](uint32_t v, int at) {
      return (uint32_t)__builtin_amdgcn_readlane((int)v, at);
    };
    int at = __builtin_ctzll(__ballot(w < upto));
    uint32_t in = w - of_lane(upto - own, at), slot = of_lane(split_upto - split_own, at);
    s.r = at * each;
    uint32_t n = of_lane(own, at);  // parts of row r
    if (each > 1) {
      for (int j0 = 0; j0 < each; j0 += 64) {
        const int r = s.r + j0 + lane;
        const uint32_t mine = j0 + lane < each ? (uint32_t)parts(a, r, blocks(a, r)) * per : 0;
        const uint32_t split = mine > (uint32_t)per ? mine : 0;
        const uint32_t x = sum_upto(mine), y = sum_upto(split);
        const uint64_t found = __ballot(in < x);
        if (found) {
          at = __builtin_ctzll(found);
          in -= of_lane(x - mine, at);
          slot += of_lane(y - split, at);
          n = of_lane(mine, at);
          s.r += j0 + at;
          break;
        }
        in -= of_lane(x, 63);
        slot += of_lane(y, 63);
      }
    }
    s.parts = (int)(n / (uint32_t)per);
    const uint32_t item = in / (uint32_t)s.parts;
    s.part = (int)(in - item * s.parts);
    s.h = (int)(item / (uint32_t)a.tiles);
    // The last tiles, which see most, first.
    s.tile = a.tiles - 1 - (int)(item - (uint32_t)s.h * a.tiles);
    s.slot = (int)(slot + item * s.parts);
    return true;
  }
};

// Keys on their way to the matrix operands: a block as it is in memory, from loads
// of 1 KB in a row straight into LDS (their lines are then whole: 7.0 TB/s, while the
// operands' 16 rows of 64 bytes a load reach 6.0), with a row's 16-byte pieces in an order
// that the row turns, so that the pieces of a tile's 16 rows are in different banks. Row
// 16 a + 4 t + b of the block is row 4 a + b of key tile t.
template <int W>
struct KeyStage {
  static constexpr int kPieces = 4 * W;  // of a row
  u32x4 piece[64 * kPieces];
  static __device__ __forceinline__ int turn(int a, int b) {
    return W == 4 ? 4 * a + b : W == 2 ? 2 * a + (b >> 1) : a;
  }
  // Byte behind 1024 i of the block that the lane's 16 bytes of load i come from.
  static __device__ __forceinline__ int source(int i, int lane) {
    const int at = 64 * i + lane, row = at / kPieces, c = at % kPieces;
    return 16 * (lane - c + (c ^ turn(row >> 4, row & 3)));
  }
  __device__ __forceinline__ u32x4 get(int t, int j, int col, int grp) const {
    const int a = col >> 2, b = col & 3;
    return piece[(16 * a + 4 * t + b) * kPieces + ((4 * j + grp) ^ turn(a, b))];
  }
};

// The kernel's arguments (its only ones), read again from here on: what is read once
// would be kept across the shares, in more scalar registers than there are.
__device__ __forceinline__ const CachedArgs &args_again() {
  auto p = (const __attribute__((address_space(4))) CachedArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const CachedArgs *)p;
}

// A tile of columns of a share.
struct Tile {
  int first, count;  // tokens of the row before the call, and of it
  int c0, used;      // its first column, those that are active
  int u0, u1;        // tokens of those, among the row's active ones
  int b0, b1;        // blocks of the share
};
// False where the tile has no active column. Columns of tokens that are not active, and of
// rows whose pages do not hold them, get their outputs here.
template <int COLS, int THREADS>
__device__ __forceinline__ bool open_tile(const CachedArgs &a, const Share &share, Tile &t) {
  const CacheView &cv = a.cache;
  const int L = cv.L, hd = cv.hd, group = a.group, r = share.r, h = share.h;
  t.first = cv.lengths ? scalar_read(cv.lengths, r) : 0;
  t.count = cv.counts ? scalar_read(cv.counts, r) : L;
  const bool sound = cache_holds(cv, t.first, t.count);
  if (!sound) t.first = t.count = 0;
  t.c0 = share.tile * COLS;
  const int columns = group * L, active = group * t.count;
  if (share.part == 0 && t.c0 + COLS > active) {
    const int lane = threadIdx.x & 63;
    for (int c = threadIdx.x >> 6; c < COLS; c += THREADS / 64) {
      if (t.c0 + c < active || t.c0 + c >= columns) continue;
      const Column at = column_of(t.c0 + c, group, L, t.count);
      const size_t o = (((size_t)r * a.heads + h * group + at.head) * hd) * L + at.token;
      for (int f = lane; f < hd; f += 64)
        a.out[o + (size_t)f * L] = sound ? 0.0f : __builtin_nanf("");
    }
  }
  if (t.c0 >= active) return false;
  t.used = min(COLS, active - t.c0);
  t.u0 = t.c0 / group;
  t.u1 = (t.c0 + t.used - 1) / group;
  const int blocks = (t.first + t.u1) / 64 + 1;
  // Parts of a tile that ends before the row does may be empty.
  t.b0 = (int)((long long)blocks * share.part / share.parts);
  t.b1 = (int)((long long)blocks * (share.part + 1) / share.parts);
  return true;
}

// Walks the (query head, feature) rows of a tile, V tokens a lane: use(first column of the
// tile, feature, place in rows x (L, heads * hd), tokens (1 to V; columns a group apart),
// load(that place, tokens)), with several loads on their way at once. A first or last token
// may have columns outside of the tile.
template <int THREADS, int V, typename F, typename G>
__device__ __forceinline__ void along_tokens(const CachedArgs &a, const Share &share, const Tile &t,
                                             F load, G use) {
  const int L = a.cache.L, hd = a.cache.hd, group = a.group;
  const int tokens = t.u1 - t.u0 + 1, runs = (tokens + V - 1) / V;
  const int bits = runs > 1 ? 32 - __builtin_clz(runs - 1) : 0;  // at most COLS of them
  const int u = V * (threadIdx.x & ((1 << bits) - 1)), step = THREADS >> bits;
  // Heads of a tile within one token.
  const int low = tokens == 1 ? t.c0 - t.u0 * group : 0;
  const int high = tokens == 1 ? low + t.used : group;
  int row = threadIdx.x >> bits, g = low;
  const int skip = row / hd;
  g += skip;
  row -= skip * hd;
  const size_t base = ((size_t)share.r * a.heads + share.h * group) * hd;
  const int token = L - t.count + t.u0 + u, n = min(V, tokens - u);
  const int jump = step / hd, rest = step - jump * hd;
  while (g < high) {
    constexpr int kBatch = V > 1 ? 4 : 8;
    int c[kBatch], f[kBatch];
    size_t at[kBatch];
    decltype(load(size_t(0), 0)) v[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      c[e] = (t.u0 + u) * group + g - t.c0;
      f[e] = row;
      at[e] = (base + (size_t)g * hd + row) * L + token;
      if (g >= high || n <= 0) c[e] = INT32_MAX;
      if (c[e] != INT32_MAX) v[e] = load(at[e], n);
      g += jump;
      row += rest;
      if (row >= hd) {
        row -= hd;
        ++g;
      }
    }
#pragma unroll
    for (int e = 0; e < kBatch; ++e)
      if (c[e] != INT32_MAX) use(c[e], f[e], at[e], n, v[e]);
  }
}
// V values side by side, at any alignment.
template <typename T, int V>
struct Run {
  T e[V];
  static __device__ __forceinline__ Run load(const void *p, size_t at, int n) {
    Run r;
    const T *from = static_cast<const T *>(p) + at;
    if (n == V) {
      __builtin_memcpy(&r, from, sizeof r);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < n) r.e[i] = from[i];
    }
    return r;
  }
};
__device__ __forceinline__ float as_f32(unsigned short x) { return bf16_to_f32(x); }
__device__ __forceinline__ float as_f32(float x) { return x; }

// One block's step of the online softmax of a lane's 16 scores (keys 16 grp + 4 t + i of its
// column; those > limit are not seen): the state moves on, and p becomes the pieces of the
// probabilities times 2^15.
template <int N>
struct Softmax {
  float m = -INFINITY, l = 0.0f;   // reference in log2 units and sum
  float unit = 1.0f, top = 0.0f;   // the outputs' unit, the largest so far
  f32x4 o[N];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int f = 0; f < N; ++f) o[f] = f32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void step(f32x4 (&s)[4], float factor, bool masked, int limit,
                                       float vs, f16x8 (&p)[2][2]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] *= factor;
    if (masked) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * t + i > limit) s[t][i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[t][i]);
    mx = pair_max(pair16_max(mx));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float alpha = m == -INFINITY ? 0.0f : fast_exp2(m - ref);
    m = mn;
    // The outputs' unit is a value scale that blocks have had: a block's own up to 16 times
    // smaller is made up for in the probabilities; another one becomes the unit, unless it is
    // so far below the largest that the outputs could leave f32's range in it. The largest is that
    // of all blocks, also of those that did not become the unit (the first ones within 1 to 1/16).
    // N <= 2^31 tokens add up to 2^15 448 N of it, below 2^55: 2^60 times that is in range.
    float turn = alpha;
    top = fmaxf(top, vs);
    if (vs > unit || vs < unit * 0x1p-4f) {
      const float to = fmaxf(fmaxf(vs, top * 0x1p-60f), 0x1p-126f);  // not 0, for a scale of 0
      turn = alpha * (unit / to);
      unit = to;
    }
    const float p15 = vs == unit ? 0x1p15f : 0x1p15f * (vs / unit);
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
      for (int f = 0; f < N; ++f) o[f] *= turn;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const F16x2 lo = split_f16x2(s[2 * k]), hi = split_f16x2(s[2 * k + 1]);
      p[0][k] = join_f16(lo.hi, hi.hi);
      p[1][k] = join_f16(lo.lo, hi.lo);
    }
  }
};

// Adds a block's values to a tile's outputs; raw(f): the lane's 16 bytes of features
// 16 f + lane % 16.
template <int N, typename F>
__device__ __forceinline__ void add_values(Softmax<N> &soft, F raw, bool masked, int limit,
                                           const f16x8 (&p)[2][2]) {
  auto multiply = [&](int f, u32x4 c) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const f16x8 v = codes_f16(c[2 * k], c[2 * k + 1]);
#pragma unroll
      for (int i = 1; i >= 0; --i) soft.o[f] = mfma_16x16x32_f16(v, p[i][k], soft.o[f]);
    }
  };
  if (!masked) {
    // Operands ahead of the products, which take long enough for them to arrive.
    constexpr int kAhead = 4;
    u32x4 c[kAhead], next[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) c[e] = raw(e);
#pragma unroll
    for (int f = 0; f < N; f += kAhead) {
#pragma unroll
      for (int e = 0; e < kAhead; ++e)
        if (f + kAhead < N) next[e] = raw(f + kAhead + e);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < kAhead; ++e) multiply(f + e, c[e]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < kAhead; ++e) c[e] = next[e];
    }
    return;
  }
  // What a column does not see must not reach it: the product of a probability of 0 and a
  // NaN (a later token's, or what was in memory) is NaN. The block's NaN codes become 0,
  // and the columns that do see one get it back.
#pragma unroll
  for (int f = 0; f < N; ++f) {
    u32x4 c = raw(f), bad;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bad[e] = nan_codes(c[e]) >> 7;
      c[e] &= ~(bad[e] * 0xffu);
    }
    multiply(f, c);
    if (__any((bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
      f32x4 n = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f16x8 sees;
#pragma unroll
        for (int e = 0; e < 8; ++e) sees[e] = (_Float16)(8 * k + e <= limit ? 1.0f : 0.0f);
        // 0x38: e4m3's 1.
        n = mfma_16x16x32_f16(codes_f16(bad[2 * k] * 0x38u, bad[2 * k + 1] * 0x38u), sees, n);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) soft.o[f][i] = n[i] > 0.0f ? __builtin_nanf("") : soft.o[f][i];
    }
  }
}

// What the waves of a share left in LDS (o, m, l and unit of PER waves a column) to its outputs
// or, where the tile has several parts, to its place, and the join by the last workgroup.
template <typename T, int W, int COLS, int PER, int THREADS, typename Lds>
__device__ __forceinline__ void finish_share(const Share &share, const Tile &t, Lds &sh) {
  constexpr int WIDE = 64 * W;
  const CachedArgs &a = args_again();
  const Parts parts = Parts::of<COLS, WIDE>(a);
  // Joined outputs, times the gate, from LDS to where they belong.
  auto give = [&](const float(&from)[COLS][WIDE + 4]) {
    auto run = [&](auto width) {
      constexpr int V = decltype(width)::value;
      along_tokens<THREADS, V>(
          a, share, t,
          [&](size_t at, int n) {
            return a.gate ? Run<T, V>::load(a.gate, at, n) : Run<T, V>{};
          },
          [&](int c, int f, size_t at, int n, const Run<T, V> &gate) {
            Run<float, V> y;
            bool whole = n == V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const int ci = c + i * a.group;
              const bool in = i < n && ci >= 0 && ci < t.used;
              whole = whole && in;
              y.e[i] = in ? from[ci][f] : 0.0f;
              if (a.gate) y.e[i] *= fast_sigmoid(as_f32(gate.e[i]));
            }
            if (whole) {
              __builtin_memcpy(a.out + at, &y, sizeof y);
            } else {
#pragma unroll
              for (int i = 0; i < V; ++i) {
                const int ci = c + i * a.group;
                if (i < n && ci >= 0 && ci < t.used) a.out[at + i] = y.e[i];
              }
            }
          });
    };
    if (t.u1 - t.u0 >= 4)
      run(std::integral_constant<int, 4>{});
    else
      run(std::integral_constant<int, 1>{});
  };
  for (int at = threadIdx.x; at < t.used * (WIDE / 4); at += THREADS) {
    const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
    float ref = -INFINITY;
#pragma unroll
    for (int w = 0; w < PER; ++w) ref = fmaxf(ref, sh.m[w][c]);
    const float safe = ref == -INFINITY ? 0.0f : ref;
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < PER; ++w) {
      const float k = fast_exp2(sh.m[w][c] - safe);
      total = fmaf(sh.l[w][c], k, total);
      sum += *reinterpret_cast<const f32x4 *>(&sh.o[w][c][f]) * (k * sh.unit[w][c]);
    }
    if (share.parts == 1) {
      *reinterpret_cast<f32x4 *>(&sh.o[0][c][f]) = sum * (1.0f / total);
    } else {
      const int to = (share.slot + share.part) * COLS + c;
      put4(parts.out, sum, (to * WIDE + f) * 4);
      if (f == 0) put2(parts.stats, ref, total, to * 8);
    }
  }
  if (share.parts == 1) {
    __syncthreads();
    give(sh.o[0]);
    return;
  }
  // The last workgroup of 16 parts to get here joins them, in the first one's place; the last
  // one of a tile's groups joins those. Each leaves its counter as it was.
  auto arrived_last = [&](unsigned *done, int of) {
    stored();
    __syncthreads();
    if (threadIdx.x == 0) {
      const unsigned n =
          __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sh.last = n + 1 == (unsigned)of;
      if (sh.last) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return sh.last != 0;
  };
  // Slots from, from + step, .., n of them: the weights first, then the outputs.
  auto join = [&](int from, int step, int n, bool finish) {
    for (int at = threadIdx.x; at < n * t.used; at += THREADS) {
      const int p = at / t.used, c = at - p * t.used;
      const u32x2 s = get2(parts.stats, ((from + p * step) * COLS + c) * 8);
      sh.weight[p][c] = __uint_as_float(s[0]);
      sh.total[p][c] = __uint_as_float(s[1]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < t.used; c += THREADS) {
      float ref = -INFINITY, total = 0.0f;
      for (int p = 0; p < n; ++p) ref = fmaxf(ref, sh.weight[p][c]);
      const float safe = ref == -INFINITY ? 0.0f : ref;
      for (int p = 0; p < n; ++p) {
        const float k = fast_exp2(sh.weight[p][c] - safe);
        sh.weight[p][c] = k;
        total = fmaf(sh.total[p][c], k, total);
      }
      sh.m[0][c] = ref;
      sh.l[0][c] = total;
    }
    __syncthreads();
    // Several places a thread at once, and of few of them several parts.
    constexpr int kPlaces = COLS > 16 ? 8 : 1;
    const int places = t.used * (WIDE / 4);
    for (int at0 = threadIdx.x; at0 < places; at0 += kPlaces * THREADS) {
      f32x4 sum[kPlaces];
#pragma unroll
      for (int i = 0; i < kPlaces; ++i) sum[i] = f32x4{0, 0, 0, 0};
#pragma unroll 8 / kPlaces
      for (int p = 0; p < n; ++p)
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) {
          const int at = min(at0 + i * THREADS, places - 1);
          const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
          sum[i] += get4(parts.out, (((from + p * step) * COLS + c) * WIDE + f) * 4) * sh.weight[p][c];
        }
#pragma unroll
      for (int i = 0; i < kPlaces; ++i) {
        const int at = at0 + i * THREADS;
        if (at >= places) break;
        const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
        if (finish) {
          *reinterpret_cast<f32x4 *>(&sh.joined[c][f]) = sum[i] * (1.0f / sh.l[0][c]);
        } else {
          put4(parts.out, sum[i], ((from * COLS + c) * WIDE + f) * 4);
          if (f == 0) put2(parts.stats, sh.m[0][c], sh.l[0][c], (from * COLS + c) * 8);
        }
      }
    }
    if (!finish) return;
    __syncthreads();
    give(sh.joined);
  };
  const int lead = share.part & ~(kJoin - 1), members = min(kJoin, share.parts - lead);
  if (!arrived_last(a.part_done + share.slot + lead, members)) return;
  join(share.slot + lead, 1, members, share.parts <= kJoin);
  if (share.parts <= kJoin) return;
  const int groups = (share.parts + kJoin - 1) / kJoin;
  if (!arrived_last(a.part_done + a.slots + share.slot, groups)) return;
  join(share.slot, kJoin, groups, true);
}

}  // namespace
}  // namespace tfd
