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

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = kCachedColumns;
constexpr int kJoin = 16;  // parts that are joined at once
constexpr int kMostGrid = 256;  // workgroups of a launch
// A tile's parts are at most 4 times as many (Deal), joined by groups.
constexpr int kMostJoined = 4 * kMostGrid / kJoin + 1;

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
constexpr int kNonTemporal = 2;
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
// the work then takes as long as one part. Otherwise quarters of an even share, one after
// another: one part more than even at the end.
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
    return r < a.rows ? max(1, (nb + most - 1) / most) : 0;
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
    const int even = (int)(all_sum(mine) * (float)per / (float)room) + 1;
    most = max(a.least, even);
    bool fits = false;
    for (int step = 0; step < 6 && !fits && (size_t)a.rows * per <= (size_t)room; ++step) {
      if (step) most += max(1, even >> 4);
      int n = parts(a, r0, nb);
      for (int j = 1; j < each; ++j) n += parts(a, r0 + j, blocks(a, r0 + j));
      fits = (long long)all_sum_of(n) * per <= room;
    }
    if (!fits) most = max(a.least, (even >> 2) + 1);
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
    s.tile = (int)(item - (uint32_t)s.h * a.tiles);
    s.slot = (int)(slot + item * s.parts);
    return true;
  }
};

// A wave's keys on their way to the matrix operands: a block as it is in memory, from loads
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
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, int lane) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int at = 64 * i + lane, row = at / kPieces, c = at % kPieces;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          from, (__attribute__((address_space(3))) void *)&piece[64 * i], 16,
          16 * (lane - c + (c ^ turn(row >> 4, row & 3))), 1024 * i, 0, kNonTemporal);
    }
  }
  __device__ __forceinline__ u32x4 get(int t, int j, int col, int grp) const {
    const int a = col >> 2, b = col & 3;
    return piece[(16 * a + 4 * t + b) * kPieces + ((4 * j + grp) ^ turn(a, b))];
  }
};

template <int W>
struct RowsLds {
  static constexpr int kQRow = 64 * W + 8;  // halves of a column's piece
  union {
    KeyStage<W> keys[kWaves];
    float o[kWaves][kCols][64 * W + 4];  // the waves' outputs
    struct {
      float weight[kMostJoined][kCols], total[kMostJoined][kCols];
    };
  };
  _Float16 q[2][kCols][kQRow];
  float x[kWaves][64 * W];   // queries before they are split
  float scale[kCols];        // c1 over the column's power of two
  float m[kWaves][kCols], l[kWaves][kCols], unit[kWaves];
  int last;
  Deal::Lanes lanes;
};

// The rows kernel's arguments (its only ones), read again from here on: what is read once
// would be kept across the shares, in more scalar registers than there are.
__device__ __forceinline__ const CachedArgs &args_again() {
  auto p = (const __attribute__((address_space(4))) CachedArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const CachedArgs *)p;
}

// What the waves of a share left in LDS to its outputs or, where the tile has several parts, to
// its place, and the join by the last workgroup.
template <typename T, int W>
__device__ __forceinline__ void finish_share(const Share &share, RowsLds<W> &sh, int c0, int used,
                                             int count) {
  constexpr int WIDE = 64 * W;
  const CachedArgs &a = args_again();
  const int hd = a.cache.hd, L = a.cache.L, group = a.group, r = share.r, h = share.h;
  const Parts parts = Parts::of<WIDE>(a);
  for (int at = threadIdx.x; at < used * (WIDE / 4); at += kThreads) {
    const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
    float ref = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) ref = fmaxf(ref, sh.m[w][c]);
    const float safe = ref == -INFINITY ? 0.0f : ref;
    f32x4 sum = {0, 0, 0, 0};
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float k = fast_exp2(sh.m[w][c] - safe);
      total = fmaf(sh.l[w][c], k, total);
      sum += *reinterpret_cast<const f32x4 *>(&sh.o[w][c][f]) * (k * sh.unit[w]);
    }
    if (share.parts == 1) {
      if (f < hd) store_out<T>(a, r, h, column_of(c0 + c, group, L, count), f, sum, 1.0f / total);
    } else {
      const int to = (share.slot + share.part) * kCols + c;
      put4(parts.out, sum, (to * WIDE + f) * 4);
      if (f == 0) put2(parts.stats, ref, total, to * 8);
    }
  }
  if (share.parts == 1) return;
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
    float(*weight)[kCols] = sh.weight;
    for (int at = threadIdx.x; at < n * used; at += kThreads) {
      const int p = at / used, c = at - p * used;
      const u32x2 s = get2(parts.stats, ((from + p * step) * kCols + c) * 8);
      weight[p][c] = __uint_as_float(s[0]);
      sh.total[p][c] = __uint_as_float(s[1]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < used; c += kThreads) {
      float ref = -INFINITY, total = 0.0f;
      for (int p = 0; p < n; ++p) ref = fmaxf(ref, weight[p][c]);
      const float safe = ref == -INFINITY ? 0.0f : ref;
      for (int p = 0; p < n; ++p) {
        const float k = fast_exp2(weight[p][c] - safe);
        weight[p][c] = k;
        total = fmaf(sh.total[p][c], k, total);
      }
      sh.m[0][c] = ref;
      sh.l[0][c] = total;
    }
    __syncthreads();
    for (int at = threadIdx.x; at < used * (WIDE / 4); at += kThreads) {
      const int f = 4 * (at % (WIDE / 4)), c = at / (WIDE / 4);
      f32x4 sum = {0, 0, 0, 0};
#pragma unroll 8
      for (int p = 0; p < n; ++p)
        sum += get4(parts.out, (((from + p * step) * kCols + c) * WIDE + f) * 4) * weight[p][c];
      if (finish) {
        if (f < hd)
          store_out<T>(a, r, h, column_of(c0 + c, group, L, count), f, sum, 1.0f / sh.l[0][c]);
      } else {
        put4(parts.out, sum, ((from * kCols + c) * WIDE + f) * 4);
        if (f == 0) put2(parts.stats, sh.m[0][c], sh.l[0][c], (from * kCols + c) * 8);
      }
    }
  };
  const int lead = share.part & ~(kJoin - 1), members = min(kJoin, share.parts - lead);
  if (!arrived_last(a.part_done + share.slot + lead, members)) return;
  join(share.slot + lead, 1, members, share.parts <= kJoin);
  if (share.parts <= kJoin) return;
  const int groups = (share.parts + kJoin - 1) / kJoin;
  if (!arrived_last(a.part_done + a.slots + share.slot, groups)) return;
  join(share.slot, kJoin, groups, true);
}

template <typename T, int W>
__device__ __forceinline__ void rows_share(const Share &share, RowsLds<W> &sh) {
  constexpr int WIDE = 64 * W;
  const CachedArgs &a = args_again();
  const CacheView &cv = a.cache;
  // Taken anew for every share: what is made of it would be kept across them, and the
  // registers spilt, whose loads wait for the keys and values on their way.
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int r = share.r, h = share.h;
  int first = cv.lengths ? scalar_read(cv.lengths, r) : 0;
  int count = cv.counts ? scalar_read(cv.counts, r) : cv.L;
  const bool sound = cache_holds(cv, first, count);
  if (!sound) first = count = 0;
  const int L = cv.L, hd = cv.hd, group = a.group;
  const int c0 = share.tile * kCols, columns = group * L;
  const int active = group * count;  // columns

  // Columns of tokens that are not active, and of rows whose pages do not hold them.
  if (share.part == 0 && c0 + kCols > active) {
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
  // Parts of a tile that ends before the row does may be empty.
  const int b0 = (int)((long long)blocks * share.part / share.parts);
  const int b1 = (int)((long long)blocks * (share.part + 1) / share.parts);

  u32x4 vr[4 * W];
  float ks = 0.0f, vs = 0.0f;
  KeyStage<W> &stage = sh.keys[wave];
  const int v_at = col * 64 + 16 * grp;
  auto load_keys = [&](long long place) {
    stage.load(buffer_rsrc(cv.keys + (size_t)(place < 0 ? 0 : place) * 64 * WIDE, 64 * WIDE), lane);
    ks = place < 0 ? __builtin_nanf("") : scalar_read(cv.key_scales, place);
  };
  auto load_values = [&](long long place) {
    const auto from =
        buffer_rsrc(cv.values + (size_t)(place < 0 ? 0 : place) * 64 * WIDE, 64 * WIDE);
#pragma unroll
    for (int f = 0; f < 4 * W; ++f)
      vr[f] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, v_at, 1024 * f,
                                                                              kNonTemporal));
    vs = place < 0 ? 1.0f : scalar_read(cv.value_scales, place);
  };
  // Queries: a wave takes two columns, its lanes the features. The first block's values are on
  // their way while they are made, behind what they need; its keys follow, as loads into
  // LDS would have to be there before the queries' LDS is read.
  // All without branches (a wave without a block loads another's): the waits then count
  // what is behind them on its way.
  constexpr int kEach = kCols / kWaves;
  float x[kEach][W], weight[W];
  double turns[(W + 1) / 2];
  const float *norm = a.q_norm ? a.q_norm : cv.key_scales;
#pragma unroll
  for (int n = 0; n < W; ++n) {
    const int f = lane + 64 * n;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int c = wave + kWaves * k;
      const Column at = column_of(min(c0 + c, last), group, L, count);
      const size_t from = (((size_t)r * a.heads + h * group + at.head) * hd) * L + at.token;
      x[k][n] = load_as_f32<T>(a.q, from + (size_t)(f < hd ? f : 0) * L);
    }
    weight[n] = norm[a.q_norm && f < hd ? f : 0];
  }
#pragma unroll
  for (int n = 0; n < (W + 1) / 2; ++n) turns[n] = a.plan.turns[lane + 64 * n];
  __builtin_amdgcn_sched_barrier(0);
  const long long place = shared_block(cv, r, h, max(0, min(b0 + wave, b1 - 1)));
  load_values(place);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int n = 0; n < W; ++n) {
    const bool in = lane + 64 * n < hd;
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      x[k][n] = in && c0 + wave + kWaves * k <= last ? x[k][n] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int c = wave + kWaves * k;
    if (c0 + c <= last) {
      if (a.q_norm) {
        float sq = 0.0f;
#pragma unroll
        for (int n = 0; n < W; ++n) sq = fmaf(x[k][n], x[k][n], sq);
        const float inv = 1.0f / sqrtf(all_sum(sq) / (float)hd + a.eps);
#pragma unroll
        for (int n = 0; n < W; ++n) x[k][n] *= inv * (1.0f + weight[n]);
      }
      if (a.plan.pairs > 0) {
        const int position = first + (c0 + c) / group;
#pragma unroll
        for (int n = 0; n < W; ++n) sh.x[wave][lane + 64 * n] = x[k][n];
        // The wave's own place: its LDS accesses are in order.
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < (W + 1) / 2; ++n) {
          const int i = lane + 64 * n;
          if (i >= a.plan.pairs) continue;
          const int fa = pair_first(a.plan, i), fb = pair_second(a.plan, i);
          float s, c;
          sincospif(2.0f * (float)turn_of((double)position, turns[n]), &s, &c);
          s *= a.plan.magnitude;
          c *= a.plan.magnitude;
          const float p = sh.x[wave][fa], q = sh.x[wave][fb];
          sh.x[wave][fa] = fmaf(p, c, -(q * s));
          sh.x[wave][fb] = fmaf(p, s, q * c);
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < W; ++n) x[k][n] = sh.x[wave][lane + 64 * n];
        __builtin_amdgcn_wave_barrier();
      }
    }
    float most = 0.0f;
#pragma unroll
    for (int n = 0; n < W; ++n) most = fmaxf(most, fabsf(x[k][n]));
    most = all_max(most);
    int e = 0;
    if (most > 0.0f && most <= 3.402823466e38f) (void)frexpf(most, &e);
    e = 14 - max(-100, e);
#pragma unroll
    for (int n = 0; n < W; ++n) {
      const float y = ldexpf(x[k][n], e);
      const _Float16 hi = (_Float16)y;
      sh.q[0][c][lane + 64 * n] = hi;
      sh.q[1][c][lane + 64 * n] = (_Float16)(y - (float)hi);
    }
    if (lane == 0) sh.scale[c] = ldexpf(a.c1, -e);
  }
  load_keys(place);
  __syncthreads();
  const float c1 = sh.scale[col];
  // Last key that the lane's column sees; columns past the last see what it sees.
  const int mine = first + min(c0 + col, last) / group;
  const int seen_by_all = first + u0;

  f32x4 o[4 * W];
#pragma unroll
  for (int i = 0; i < 4 * W; ++i) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f, unit = 1.0f, top = 0.0f;
  for (int b = b0 + wave; b < b1; b += kWaves) {
    const bool more = b + kWaves < b1;
    const long long next = more ? shared_block(cv, r, h, b + kWaves) : -1;
    // The queries' operands are read again for every block: kept, they would take the
    // registers of the SIMD's other wave.
    asm volatile("" ::: "memory");
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < W; ++j) {
      f16x8 hi[2], lo[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int at = 64 * j + 16 * grp + 8 * k;
        hi[k] = *reinterpret_cast<const f16x8 *>(&sh.q[0][col][at]);
        lo[k] = *reinterpret_cast<const f16x8 *>(&sh.q[1][col][at]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const u32x4 c = stage.get(t, j, col, grp);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f16x8 key = codes_f16(c[2 * k], c[2 * k + 1]);
          s[t] = mfma_16x16x32_f16(key, lo[k], s[t]);
          s[t] = mfma_16x16x32_f16(key, hi[k], s[t]);
        }
      }
    }
    const float factor = ks * c1;
    // The products have read the keys' place.
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
    sh.m[wave][col] = m;
    sh.l[wave][col] = l;
  }
  if (lane == 0) sh.unit[wave] = unit * 0x1p-15f;
  const int used = last - c0 + 1;
#pragma unroll
  for (int f = 0; f < 4 * W; ++f)
    if (col < used) *reinterpret_cast<f32x4 *>(&sh.o[wave][col][16 * f + 4 * grp]) = o[f];
  __syncthreads();
  finish_share<T, W>(share, sh, c0, used, count);
}

template <typename T, int W>
__global__ __launch_bounds__(512, 2) void cached_rows_kernel(CachedArgs a) {
  __shared__ RowsLds<W> sh;
  Deal deal;
  deal.make(a, sh.lanes);
  Share share;
  for (uint32_t w = blockIdx.x; deal.find(args_again(), sh.lanes, w, share); w += gridDim.x) {
    rows_share<T, W>(share, sh);
    __syncthreads();
  }
}

template <typename T, int W>
hipError_t launch_wide(const CachedArgs &a, hipStream_t stream, const KernelEvents &ev) {
  hipExtLaunchKernelGGL((cached_rows_kernel<T, W>), dim3((unsigned)a.grid), dim3(kThreads), 0, stream, ev.start,
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
  // One workgroup a CU is there at once.
  a.grid = a.cus < kMostGrid ? a.cus : kMostGrid;
  a.least = kWaves;
  // Parts of tiles in several: no more than the workgroups, or, as a tile in n > 1 parts has
  // more than (n - 1) most blocks and 4 grid most is at least all of them, 8 times that.
  a.slots = 8 * a.grid;
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
