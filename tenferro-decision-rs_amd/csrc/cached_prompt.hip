// The attention over a paged 8-bit cache for many columns (cached_common.hpp): prompts behind
// what is cached.
//
// Bound: the SIMDs' issue. Per (column, key) 8 hd operations are done for the 4 hd of the formula,
// as f32 operands go in two fp16 pieces, and a code is converted by every wave that
// multiplies it; what a tile reads of the cache stays in L2.
//
// A workgroup of eight waves takes 128 columns, 16 a wave, whose queries' pieces and outputs
// stay in registers; all waves read each block from LDS, where it arrives as it is in memory
// while the one before is multiplied (two places). A code becomes fp16 on its way from LDS to
// the matrix unit: four conversions for two products, while the SIMD's other wave has products under way.
// Blocks that no column of a wave sees are not multiplied.
//
// Measured: 2 rows of 900 to 1024 tokens behind 8000 to 8192, 2 kv heads of 256 features in groups of 4
// (135 Gflop of the formula, 270 done): 301 to 345 us by the clock that the load leaves, 0.8 to 0.9
// Pflop/s of products, where a plain one of 8192 cubed reaches 1.2. The matrix unit is busy
// for 33% of the cycles, vector instructions are issued in 46% (4.5 for each product: 2
// conversions, softmax, pieces). Before: the rows kernel's order 450 us; four waves of 16 columns 360;
// 32 columns a wave, whose registers leave one wave a SIMD, 503.
#include <hip/hip_ext.h>

#include "cached_common.hpp"

namespace tfd {
namespace {

constexpr int kWaves = 8;  // of 16 columns each
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = 16 * kWaves;
constexpr int kPromptCap = 256;

// Values as keys (KeyStage): feature f's 64 tokens are four pieces, at places that f / 4 turns.
// Which quarter is first turned is chosen for the lanes that LDS serves at once, 0 to 3, 12 to
// 15 and 20 to 27 of 32.
template <int W>
struct ValueStage {
  u32x4 piece[64 * 4 * W];
  static __device__ __forceinline__ int turn(int quarter) {  // 0, 3, 1, 2
    return (0x9c >> (2 * quarter)) & 3;
  }
  static __device__ __forceinline__ int unturn(int place) {  // and back
    return (0x78 >> (2 * place)) & 3;
  }
  static __device__ __forceinline__ int source(int lane) {
    return 16 * ((lane & ~3) | unturn((lane & 3) ^ ((lane >> 4) & 3)));
  }
  __device__ __forceinline__ u32x4 get(int f, int col, int grp) const {
    return piece[64 * f + 4 * col + (turn(grp) ^ ((col >> 2) & 3))];
  }
};

template <int W>
struct PromptLds {
  union {
    struct {
      KeyStage<W> keys[2];
      ValueStage<W> values[2];
    };
    float x[kCols][64 * W + 4];     // queries before they are split
    float o[1][kCols][64 * W + 4];  // outputs
    struct {
      float weight[kPromptCap / kJoin][kCols], total[kPromptCap / kJoin][kCols];
      float joined[kCols][64 * W + 4];
    };
  };
  float m[1][kCols], l[1][kCols], unit[1][kCols];
  int last;
  Deal::Lanes lanes;
};

template <typename T, int W>
__device__ __forceinline__ void prompt_share(const Share &share, PromptLds<W> &sh) {
  constexpr int WIDE = 64 * W;
  const CachedArgs &a = args_again();
  const CacheView &cv = a.cache;
  int lane = threadIdx.x;
  asm volatile("" : "+v"(lane));  // taken anew for every share
  lane &= 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int r = share.r, h = share.h, hd = cv.hd, group = a.group;
  Tile tile;
  if (!open_tile<kCols, kThreads>(a, share, tile)) return;
  const int first = tile.first, b0 = tile.b0, b1 = tile.b1;

  // Queries to LDS, lanes along the tokens; a wave makes the operands of its 16 columns.
  if (tile.used < kCols || hd < WIDE) {
    for (int at = threadIdx.x; at < kCols * (WIDE / 4); at += kThreads)
      *reinterpret_cast<f32x4 *>(&sh.x[at / (WIDE / 4)][4 * (at % (WIDE / 4))]) = f32x4{0, 0, 0, 0};
    __syncthreads();
  }
  constexpr int kRun = sizeof(T) == 2 ? 8 : 4;
  along_tokens<kThreads, kRun>(
      a, share, tile, [&](size_t at, int n) { return Run<T, kRun>::load(a.q, at, n); },
      [&](int c, int f, size_t, int n, const Run<T, kRun> &v) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          const int ci = c + i * group;
          if (i < n && ci >= 0 && ci < tile.used) sh.x[ci][f] = as_f32(v.e[i]);
        }
      });
  __syncthreads();
  const int used = tile.used, w0 = 16 * wave;  // the wave's first column
  // Operand 2 j + k: features 64 j + 16 grp + 8 k .. + 7 of the lane's column; and the last
  // key that it sees (columns past the last: what that one sees).
  f16x8 high[2 * W], low[2 * W];
  float c1;
  int mine;
  {
    const int c = w0 + col;
    float *x = sh.x[c];
    mine = first + (tile.c0 + min(c, used - 1)) / group;
    f32x4 y[4 * W];
    if (a.q_norm) {
      // Each of the column's four lanes has a quarter of the features.
#pragma unroll
      for (int n = 0; n < 4 * W; ++n)
        y[n] = *reinterpret_cast<const f32x4 *>(x + 16 * W * grp + 4 * n);
      float sq = 0.0f;
#pragma unroll
      for (int n = 0; n < 4 * W; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sq = fmaf(y[n][e], y[n][e], sq);
      sq = pair_sum(pair16_sum(sq));
      const float inv = 1.0f / sqrtf(sq / (float)hd + a.eps);
#pragma unroll
      for (int n = 0; n < 4 * W; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int f = 16 * W * grp + 4 * n + e;
          y[n][e] *= inv * (1.0f + a.q_norm[f < hd ? f : 0]);
        }
        *reinterpret_cast<f32x4 *>(x + 16 * W * grp + 4 * n) = y[n];
      }
      __builtin_amdgcn_wave_barrier();
    }
    for (int i = grp; i < a.plan.pairs; i += 4) {
      const int fa = pair_first(a.plan, i), fb = pair_second(a.plan, i);
      float s, k;
      sincospif(2.0f * (float)turn_of((double)mine, a.plan.turns[i]), &s, &k);
      s *= a.plan.magnitude;
      k *= a.plan.magnitude;
      const float p = x[fa], r = x[fb];
      x[fa] = fmaf(p, k, -(r * s));
      x[fb] = fmaf(p, s, r * k);
    }
    __builtin_amdgcn_wave_barrier();
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        y[4 * j + n] = *reinterpret_cast<const f32x4 *>(x + 64 * j + 16 * grp + 4 * n);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(y[4 * j + n][e]));
      }
    most = pair_max(pair16_max(most));
    int e = 0;
    if (most > 0.0f && most <= 3.402823466e38f) (void)frexpf(most, &e);
    e = 14 - max(-100, e);
    c1 = ldexpf(a.c1, -e);
#pragma unroll
    for (int n = 0; n < 2 * W; ++n) {
      F16x2 s[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f32x4 v = y[2 * n + k];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = ldexpf(v[i], e);
        s[k] = split_f16x2(v);
      }
      high[n] = join_f16(s[0].hi, s[1].hi);
      low[n] = join_f16(s[0].lo, s[1].lo);
    }
  }
  // The wave's columns see keys up to here, all of them up to the first's.
  const int wave_sees = first + (tile.c0 + min(w0 + 15, used - 1)) / group;
  const int seen_by_all = first + (tile.c0 + min(w0, used - 1)) / group;

  // The waves bring a block together, 1 KB a load. The loads are waited for by hand: by all before
  // the barrier behind which they are read.
  float ks = 0.0f, vs = 1.0f;  // of the block that is on its way, then of the one that is read
  long long place = 0;         // of the next block to load
  auto look_up = [&](int b) { place = shared_block(cv, r, h, min(b, b1 - 1)); };
  auto load = [&](int to) {
    const size_t at = (size_t)(place < 0 ? 0 : place) * 64 * WIDE;
    const u32x4r keys = rsrc_words(cv.keys + at, 64 * WIDE);
    const u32x4r values = rsrc_words(cv.values + at, 64 * WIDE);
#pragma unroll
    for (int n = 0; n < (4 * W + kWaves - 1) / kWaves; ++n) {
      const int i = wave + kWaves * n;
      if (4 * W % kWaves && i >= 4 * W) break;
      load_lds16(keys, KeyStage<W>::source(i, lane), 1024 * i,
                 reinterpret_cast<unsigned char *>(&sh.keys[to].piece[64 * i]));
      load_lds16(values, ValueStage<W>::source(lane), 1024 * i,
                 reinterpret_cast<unsigned char *>(&sh.values[to].piece[64 * i]));
    }
  };
  auto scales = [&](float &k, float &v) {
    k = place < 0 ? __builtin_nanf("") : scalar_read(cv.key_scales, place);
    v = place < 0 ? 1.0f : scalar_read(cv.value_scales, place);
  };
  Softmax<4 * W> soft;
  soft.clear();
  __syncthreads();  // the queries' place is the blocks'
  float next_ks = 0.0f, next_vs = 1.0f;
  if (b0 < b1) {
    look_up(b0);
    load(0);
    scales(ks, vs);
    look_up(b0 + 1);
  }
  int at = 0;
  for (int b = b0; b < b1; ++b, at ^= 1) {
    // The block is there, and its reads of the place that the next one goes to are over.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (b > b0) {
      ks = next_ks;
      vs = next_vs;
    }
    // The next block, and what the one after it needs of the scales and the table, are asked for
    // behind the scores, where no LDS read (which would wait for the scalar ones) follows at
    // once.
    auto ahead = [&]() {
      if (b + 1 < b1) load(at ^ 1);
      scales(next_ks, next_vs);
      look_up(b + 2);
    };
    const bool sees = w0 < used && b * 64 <= wave_sees;
    if (!sees) {
      ahead();
      continue;
    }
    // Taken anew for every block: the places made of it would be kept, and spilt.
    int here = threadIdx.x;
    asm volatile("" : "+v"(here));
    const int row = here & 15, quarter = (here >> 4) & 3;
    const KeyStage<W> &keys = sh.keys[at];
    const ValueStage<W> &values = sh.values[at];
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = f32x4{0, 0, 0, 0};
    // Operands ahead of the products, as the values' (add_values).
    u32x4 c[4], next[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = keys.get(t, 0, row, quarter);
#pragma unroll
    for (int j = 0; j < W; ++j) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (j + 1 < W) next[t] = keys.get(t, j + 1, row, quarter);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f16x8 key = codes_f16(c[t][2 * k], c[t][2 * k + 1]);
          s[t] = mfma_16x16x32_f16(key, low[2 * j + k], s[t]);
          s[t] = mfma_16x16x32_f16(key, high[2 * j + k], s[t]);
        }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 4; ++t) c[t] = next[t];
    }
    ahead();
    const bool masked = b * 64 + 63 > seen_by_all;
    const int limit = mine - b * 64 - 16 * quarter;
    f16x8 p[2][2];
    soft.step(s, ks * c1, masked, limit, vs, p);
    add_values(soft, [&](int f) { return values.get(f, row, quarter); }, masked, limit, p);
  }
  __syncthreads();  // the blocks' place is the outputs'
  const int c = w0 + col;
  const float l = pair_sum(pair16_sum(soft.l));
  if (grp == 0) {
    sh.m[0][c] = soft.m;
    sh.l[0][c] = l;
    sh.unit[0][c] = soft.unit * 0x1p-15f;
  }
#pragma unroll
  for (int f = 0; f < 4 * W; ++f)
    *reinterpret_cast<f32x4 *>(&sh.o[0][c][16 * f + 4 * grp]) = soft.o[f];
  __syncthreads();
  finish_share<T, W, kCols, 1, kThreads>(share, tile, sh);
}

template <typename T, int W>
__global__ __launch_bounds__(kThreads, 2) void cached_prompt_kernel(CachedArgs a) {
  __shared__ PromptLds<W> sh;
  Deal deal;
  deal.make(a, sh.lanes);
  Share share;
  for (uint32_t w = blockIdx.x; deal.find(args_again(), sh.lanes, w, share); w += gridDim.x) {
    prompt_share<T, W>(share, sh);
    __syncthreads();
  }
}

template <typename T, int W>
hipError_t launch_wide(const CachedArgs &a, hipStream_t stream, const KernelEvents &ev) {
  hipExtLaunchKernelGGL((cached_prompt_kernel<T, W>), dim3((unsigned)a.grid), dim3(kThreads), 0,
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

hipError_t launch_cached_prompt(const CachedArgs &a, hipStream_t stream, const KernelEvents &ev) {
  return a.bf16 ? launch_typed<unsigned short>(a, stream, ev)
                : launch_typed<float>(a, stream, ev);
}

}  // namespace tfd
