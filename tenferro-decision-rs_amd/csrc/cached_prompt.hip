// The attention over a paged 8-bit cache for many columns (cached_common.hpp): prompts behind
// what is cached.
//
// TODO-COMMENT
#include <hip/hip_ext.h>

#include "cached_common.hpp"

namespace tfd {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kCols = 64;
constexpr int kPromptCap = 256;

// Values as keys (KeyStage): feature f's 64 tokens are four pieces, turned by f / 4.
template <int W>
struct ValueStage {
  u32x4 piece[64 * 4 * W];
  static __device__ __forceinline__ int source(int lane) {
    return 16 * ((lane & ~3) | ((lane & 3) ^ ((lane >> 4) & 3)));
  }
  __device__ __forceinline__ u32x4 get(int f, int col, int grp) const {
    return piece[64 * f + 4 * col + (grp ^ ((col >> 2) & 3))];
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
  along_tokens<kThreads>(a, share, tile,
                         [&](int c, int f, size_t at) { sh.x[c][f] = load_as_f32<T>(a.q, at); });
  __syncthreads();
  float *x = sh.x[16 * wave + col];
  const int c = 16 * wave + col, used = tile.used;
  const int own = min(c, used - 1);  // columns past the last see what it sees
  const int mine = first + (tile.c0 + own) / group;
  {
    // Each of the column's four lanes has a quarter of the features.
    f32x4 y[4 * W];
#pragma unroll
    for (int n = 0; n < 4 * W; ++n) y[n] = *reinterpret_cast<const f32x4 *>(x + 16 * W * grp + 4 * n);
    if (a.q_norm) {
      float sq = 0.0f;
#pragma unroll
      for (int n = 0; n < 4 * W; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sq = fmaf(y[n][e], y[n][e], sq);
      sq = pair_sum(pair16_sum(sq));
      const float inv = 1.0f / sqrtf(sq / (float)hd + a.eps);
#pragma unroll
      for (int n = 0; n < 4 * W; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int f = 16 * W * grp + 4 * n + e;
          y[n][e] *= inv * (1.0f + a.q_norm[f < hd ? f : 0]);
        }
#pragma unroll
      for (int n = 0; n < 4 * W; ++n) *reinterpret_cast<f32x4 *>(x + 16 * W * grp + 4 * n) = y[n];
    }
  }
  __builtin_amdgcn_wave_barrier();
  for (int i = grp; i < a.plan.pairs; i += 4) {
    const int fa = pair_first(a.plan, i), fb = pair_second(a.plan, i);
    float s, k;
    sincospif(2.0f * (float)turn_of((double)mine, a.plan.turns[i]), &s, &k);
    s *= a.plan.magnitude;
    k *= a.plan.magnitude;
    const float p = x[fa], q = x[fb];
    x[fa] = fmaf(p, k, -(q * s));
    x[fb] = fmaf(p, s, q * k);
  }
  __builtin_amdgcn_wave_barrier();
  // Operand of step (j, k): features 64 j + 16 grp + 8 k .. + 7 of the lane's column.
  f16x8 q[2][2 * W];
  float c1;
  {
    f32x4 y[4 * W];
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
      q[0][n] = join_f16(s[0].hi, s[1].hi);
      q[1][n] = join_f16(s[0].lo, s[1].lo);
    }
  }
  // The wave's columns see keys up to here, all of them up to the first's.
  const int wave_sees = first + (tile.c0 + min(16 * wave + 15, used - 1)) / group;
  const int seen_by_all = first + (tile.c0 + min(16 * wave, used - 1)) / group;

  // A wave brings a quarter of a block. The loads are waited for by hand: by all before
  // the barrier behind which they are read.
  float ks[2], vs[2];
  auto load = [&](int b, int to) {
    const long long place = shared_block(cv, r, h, b);
    const size_t at = (size_t)(place < 0 ? 0 : place) * 64 * WIDE;
    const u32x4r keys = rsrc_words(cv.keys + at, 64 * WIDE);
    const u32x4r values = rsrc_words(cv.values + at, 64 * WIDE);
#pragma unroll
    for (int n = 0; n < W; ++n) {
      const int i = wave * W + n;
      load_lds16(keys, KeyStage<W>::source(i, lane), 1024 * i,
                 reinterpret_cast<unsigned char *>(&sh.keys[to].piece[64 * i]));
      load_lds16(values, ValueStage<W>::source(lane), 1024 * i,
                 reinterpret_cast<unsigned char *>(&sh.values[to].piece[64 * i]));
    }
    ks[to] = place < 0 ? __builtin_nanf("") : scalar_read(cv.key_scales, place);
    vs[to] = place < 0 ? 1.0f : scalar_read(cv.value_scales, place);
  };
  Softmax<4 * W> soft;
  soft.clear();
  __syncthreads();  // the queries' place is the blocks'
  if (b0 < b1) load(b0, 0);
  auto step = [&](int b, int at) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (b + 1 < b1) load(b + 1, at ^ 1);
    if (16 * wave >= used || b * 64 > wave_sees) return;
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = f32x4{0, 0, 0, 0};
    u32x4 c[4], next[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) c[t] = sh.keys[at].get(t, 0, col, grp);
#pragma unroll
    for (int j = 0; j < W; ++j) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (j + 1 < W) next[t] = sh.keys[at].get(t, j + 1, col, grp);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f16x8 key = codes_f16(c[t][2 * k], c[t][2 * k + 1]);
          s[t] = mfma_16x16x32_f16(key, q[1][2 * j + k], s[t]);
          s[t] = mfma_16x16x32_f16(key, q[0][2 * j + k], s[t]);
        }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 4; ++t) c[t] = next[t];
    }
    const bool masked = b * 64 + 63 > seen_by_all;
    const int limit = mine - b * 64 - 16 * grp;
    f16x8 p[2][2];
    soft.step(s, ks[at] * c1, masked, limit, vs[at], p);
    soft.add([&](int f) { return sh.values[at].get(f, col, grp); }, masked, limit, p);
  };
  for (int b = b0; b < b1; b += 2) {
    step(b, 0);
    if (b + 1 < b1) step(b + 1, 1);
  }
  const float l = pair_sum(pair16_sum(soft.l));
  __syncthreads();  // the blocks' place is the outputs'
  if (grp == 0) {
    sh.m[0][c] = soft.m;
    sh.l[0][c] = l;
    sh.unit[0][c] = soft.unit * 0x1p-15f;
  }
#pragma unroll
  for (int f = 0; f < 4 * W; ++f) *reinterpret_cast<f32x4 *>(&sh.o[0][c][16 * f + 4 * grp]) = soft.o[f];
  __syncthreads();
  finish_share<T, W, kCols, 1, kThreads>(share, tile, sh);
}

template <typename T, int W>
__global__ __launch_bounds__(256, 2) void cached_prompt_kernel(CachedArgs a) {
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
