// The attention over a paged 8-bit cache for few columns (cached_common.hpp): single tokens, and
// a few a row.
//
// Bound: the cache's way from memory, once for each tile of 16 columns. A block of 64 keys and
// 256 features is 32 KB, 1.2 us of a CU's share of the 7.1 TB/s that plain reads reach; its 128
// matrix instructions (two pieces, keys and values) are a quarter of a CU's 1 us.
//
// A workgroup of eight waves takes a share; wave w its blocks w, w + 8, ... with a softmax of its
// own, and the eight are joined in LDS. Two waves a SIMD, as one's loads are under way while
// the other multiplies: the next block's keys leave for LDS as soon as the products have
// read this one's, its values for registers behind the products. Keys by whole lines straight
// into LDS (KeyStage); values as the operands lie in memory, 16 runs of 64 bytes a
// load. Both nontemporal, as they are read once.
//
// Measured, 2 kv heads of 256 features in groups of 4: 128 rows of 8000 to 8192 tokens 169 us
// (1065 MB, 6.3 TB/s); 64 rows of 200 to 4000 tokens 38 us (139 MB, 3.6 TB/s); one row of 131000
// tokens 35 us (134 MB, 3.8 TB/s, with the join of 256 parts); one row of 300 tokens 14.5 us: launch 3.5,
// lengths, table, queries, a block and the outputs one after another. Before: four waves that
// kept all in registers 185, 44 and 41 us, one launch more for the join 238, 74 and 178.
#include <hip/hip_ext.h>

#include <type_traits>

#include "cached_common.hpp"

namespace tfd {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = 16;
constexpr int kRowsCap = 1024;

template <int W>
struct RowsLds {
  static constexpr int kQRow = 64 * W + 8;  // halves of a column's piece
  union {
    KeyStage<W> keys[kWaves];
    float o[kWaves][kCols][64 * W + 4];  // the waves' outputs
    struct {
      float weight[kRowsCap / kJoin][kCols], total[kRowsCap / kJoin][kCols];
      float joined[kCols][64 * W + 4];
    };
  };
  _Float16 q[2][kCols][kQRow];
  float x[kWaves][64 * W];   // queries before they are split
  float scale[kCols];        // c1 over the column's power of two
  float m[kWaves][kCols], l[kWaves][kCols], unit[kWaves][kCols];
  int last;
  Deal::Lanes lanes;
};

template <typename T, int W>
__device__ __forceinline__ void rows_share(const Share &share, RowsLds<W> &sh) {
  constexpr int WIDE = 64 * W;
  const CachedArgs &a = args_again();
  const CacheView &cv = a.cache;
  // Taken anew for every share: what is made of it would be kept across them, and the
  // registers spilt, whose loads wait for the keys and values on their way.
  int lane = threadIdx.x;
  asm volatile("" : "+v"(lane));
  lane &= 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int r = share.r, h = share.h, L = cv.L, hd = cv.hd, group = a.group;
  Tile tile;
  if (!open_tile<kCols, kThreads>(a, share, tile)) return;
  const int first = tile.first, count = tile.count, c0 = tile.c0;
  const int last = c0 + tile.used - 1, b0 = tile.b0, b1 = tile.b1;

  u32x4 vr[4 * W];
  float ks = 0.0f, vs = 0.0f;
  KeyStage<W> &stage = sh.keys[wave];
  const int v_at = col * 64 + 16 * grp;
  auto load_keys = [&](long long place) {
    const auto from = buffer_rsrc(cv.keys + (size_t)(place < 0 ? 0 : place) * 64 * WIDE, 64 * WIDE);
#pragma unroll
    for (int i = 0; i < 4 * W; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          from, (__attribute__((address_space(3))) void *)&stage.piece[64 * i], 16,
          KeyStage<W>::source(i, lane), 1024 * i, 0, kNonTemporal);
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
  // Loads into LDS are waited for by hand, here and before a block's keys are read: the
  // compiler does not see in a loop that those reads are of what the loads wrote.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const float c1 = sh.scale[col];
  // Last key that the lane's column sees; columns past the last see what it sees.
  const int mine = first + min(c0 + col, last) / group;
  const int seen_by_all = first + tile.u0;

  Softmax<4 * W> soft;
  soft.clear();
  // A wave's last block apart: the loads of another one without a branch, so that the waits
  // for the values count the next keys behind them (with it 64 ragged rows take 43 us and 128 of
  // 8192 tokens 190, without 38 and 170). No other block holds a key that some column does not see:
  // a tile's columns are 16 tokens at most, its blocks dealt to eight waves in turn.
  long long next = 0;  // place of the wave's next block
  auto block = [&](int b, auto is_last) {
    constexpr bool kLast = decltype(is_last)::value;
    // The block's keys are there when no more than the values' loads behind them are on their
    // way. (And the queries' operands are read again for every block: kept, they would take
    // the registers of the SIMD's other wave.)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * W) : "memory");
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
    if constexpr (!kLast) load_keys(next);
    __builtin_amdgcn_sched_barrier(0);
    const bool masked = kLast && b * 64 + 63 > seen_by_all;
    const int limit = mine - b * 64 - 16 * grp;  // of the lane's 16 keys: those <= limit
    f16x8 p[2][2];
    soft.step(s, factor, masked, limit, vs, p);
    add_values(soft, [&](int f) { return vr[f]; }, masked, limit, p);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!kLast) {
      load_values(next);
      next = shared_block(cv, r, h, min(b + 2 * kWaves, b1 - 1));
    }
  };
  int b = b0 + wave;
  if (b + kWaves < b1) next = shared_block(cv, r, h, b + kWaves);
  for (; b + kWaves < b1; b += kWaves) block(b, std::false_type{});
  if (b < b1) block(b, std::true_type{});
  const float l = pair_sum(pair16_sum(soft.l));
  __syncthreads();  // the keys' place is the outputs'
  // The waves' sums, joined by all of them, in units of 1 and 2^-15 probabilities.
  if (grp == 0) {
    sh.m[wave][col] = soft.m;
    sh.l[wave][col] = l;
    sh.unit[wave][col] = soft.unit * 0x1p-15f;
  }
#pragma unroll
  for (int f = 0; f < 4 * W; ++f)
    if (col < tile.used)
      *reinterpret_cast<f32x4 *>(&sh.o[wave][col][16 * f + 4 * grp]) = soft.o[f];
  __syncthreads();
  finish_share<T, W, kCols, kWaves, kThreads>(share, tile, sh);
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
  hipExtLaunchKernelGGL((cached_rows_kernel<T, W>), dim3((unsigned)a.grid), dim3(kThreads), 0,
                        stream, ev.start, ev.stop, 0, a);
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

// The rows kernel reads a row's blocks once for each tile of 16 columns, and gives every tile
// workgroups of its own; the prompt kernel takes 128 columns at once. The first is faster up to
// two tiles, and where there are few tiles in all (us, rows kernel and prompt kernel; heads of
// 128, groups of 8, tokens seen: 4096 by 32 rows and kv heads of 32 columns 23 and 34, of 40 44
// and 36, of 256 93 and 69; by 1 of 256 columns 300 15 and 27, 2048 16 and 32, 16384 19 and 48; by
// 2 of 1024 columns 2048 18 and 37, 16384 52 and 74; by 16 of 64 columns 16384 45 and
// 54). It loses where long rows are many: by 32 of 64 columns 2048 21 and 27, 16384 94 and
// 76. How long they are is in device memory.
void cached_plan(CachedArgs &a) {
  const long long columns = (long long)a.group * a.cache.L, tiles = (columns + 15) / 16;
  a.prompt = tiles > 2 && tiles * a.rows * a.cache.kv_heads > a.cus / 2;
  a.columns = a.prompt ? 128 : 16;
  a.tiles = (int)((columns + a.columns - 1) / a.columns);
  // One workgroup of eight waves for a CU is what it holds of either kernel at once.
  a.grid = a.cus < 256 ? a.cus : 256;
  // A part of fewer blocks costs more in its beginning and end than it saves: a block for each
  // wave (1 row of 65536 tokens: 16.3 us, from 4 blocks 18.6, from 16 19.1), or 4 that all
  // read (128 tokens of 2 kv heads at 1024: 31.7 us, from 2 blocks 32.7, from 8 38.8).
  a.least = a.prompt ? 4 : kWaves;
  a.cap = a.prompt ? 256 : kRowsCap;
  // Parts of tiles in several: a tile in n > 1 parts has more than (n - 1) most blocks, and
  // grid most is at least all blocks.
  a.slots = 2 * a.grid;
}

CachedSpace cached_space(const CachedArgs &a) {
  // As many counters for every call: what is behind them is not zero between calls.
  const size_t slots = (size_t)a.slots;
  return CachedSpace{2 * kCachedSlots * sizeof(unsigned), slots * a.columns * 2 * sizeof(float),
                     slots * a.columns * a.cache.wide * sizeof(float)};
}

hipError_t launch_cached_rows(const CachedArgs &a, hipStream_t stream, const KernelEvents &ev) {
  return a.bf16 ? launch_typed<unsigned short>(a, stream, ev)
                : launch_typed<float>(a, stream, ev);
}

hipError_t launch_cached_attention(const CachedArgs &a, hipStream_t stream,
                                   const KernelEvents &ev) {
  return a.prompt ? launch_cached_prompt(a, stream, ev) : launch_cached_rows(a, stream, ev);
}

}  // namespace tfd
