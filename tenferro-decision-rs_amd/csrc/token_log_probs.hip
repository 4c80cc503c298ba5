// Log probabilities of given tokens, the entropy and the largest logits of
// every position of a (vocab, positions) matrix of logits, in one pass.
//
// With m = max x, z = sum e^(x - m), a = sum e^(x - m) (x - m):
//   log p(i) = (x_i - m) - log z,   entropy = log z - a / z.
// Each lane keeps its own (m, z, a) and moves m by
//   z' = f z,  a' = f (a + (m - m') z),  f = e^(m - m'),
// so a position is read once, 16 bytes a lane, and the lanes, waves and parts
// of a position are joined in a fixed order (the same bits on every run). A
// NaN or +inf logit makes z NaN, no finite logit makes it 0: both end as NaN.
//
// The `top` largest logits: every wave keeps its best 64 so far sorted across
// its lanes, as unique 64-bit keys (value order, then the lower index first),
// and compares the 16 bytes' maximum, which the softmax needs anyway, with
// the top-th of them (of any of the position's waves: 1024 x 131072 bf16, top 5, 104
// us with each wave's own, 82 with the highest). What passes is collected in LDS and
// merged 64 at a time by a bitonic network; for logits in random order that is a few
// merges in a row of 10^5.
//
// Bound by reading the logits. A position goes to one wave up to 2048 logits,
// to one workgroup of four waves past that, and to several workgroups (joined
// by a second kernel) when there are too few positions to fill the chip.
#include <hip/hip_ext.h>
#include <math.h>

#include "tfd_device.hpp"
#include "tfd_internal.hpp"

namespace tfd {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
// Exponents are clamped here: e^-1e30 is 0, and 0 * -1e30 is 0, not NaN.
constexpr float kFar = -1.0e30f;

typedef unsigned long long u64;

// Value order of a logit: larger numbers have larger codes, -0 equals 0, a NaN
// ranks below every number.
__device__ __forceinline__ uint32_t value_code(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ float code_value(uint32_t c) {
  if (c == 0u) return NAN;
  return __uint_as_float(c & 0x80000000u ? c & 0x7fffffffu : ~c);
}
__device__ __forceinline__ u64 key_of(float x, uint32_t index) {
  return ((u64)value_code(x) << 32) | (uint32_t)~index;
}

// The value of lane l ^ O, by DPP within rows of 16 lanes and lane swaps across
// them: no trip through LDS.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, true);
}
template <int O>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v, int lane) {
  static_assert(O == 1 || O == 2 || O == 4 || O == 8 || O == 16 || O == 32 || O == 63, "");
  if constexpr (O == 1) return dpp<0xB1>(v);             // quad_perm 1 0 3 2
  if constexpr (O == 2) return dpp<0x4E>(v);             // quad_perm 2 3 0 1
  if constexpr (O == 4) return dpp<0x1B>(dpp<0x141>(v));  // 7 - l, then quad_perm 3 2 1 0
  if constexpr (O == 8) return dpp<0x128>(v);            // row_ror 8
  if constexpr (O == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  if constexpr (O == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
  if constexpr (O == 63) return xor_lane<32>(xor_lane<16>(dpp<0x140>(v), lane), lane);  // 15 - l
}
template <int O>
__device__ __forceinline__ u64 xor_lane(u64 v, int lane) {
  return (u64)xor_lane<O>((uint32_t)(v >> 32), lane) << 32 | xor_lane<O>((uint32_t)v, lane);
}

// Bitonic stages O, O / 2, .. 1 over the wave's lanes: blocks of N lanes sort
// downwards and upwards in turn (N = 128: all downwards).
template <int N, int O>
__device__ __forceinline__ u64 stages(u64 v, int lane) {
  const u64 w = xor_lane<O>(v, lane);
  v = (v > w) == (((lane & O) == 0) == ((lane & N) == 0)) ? v : w;
  if constexpr (O > 1)
    return stages<N, O / 2>(v, lane);
  else
    return v;
}
// Sorts one key a lane, largest in lane 0.
__device__ __forceinline__ u64 sort64(u64 v, int lane) {
  v = stages<2, 1>(v, lane);
  v = stages<4, 2>(v, lane);
  v = stages<8, 4>(v, lane);
  v = stages<16, 8>(v, lane);
  v = stages<32, 16>(v, lane);
  return stages<64, 32>(v, lane);
}
// The 64 largest of two sorted lists, sorted.
__device__ __forceinline__ u64 merge64(u64 a, u64 b, int lane) {
  const u64 r = xor_lane<63>(b, lane);
  return stages<128, 32>(a > r ? a : r, lane);
}
__device__ __forceinline__ u64 key_at(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}

// A wave's largest keys so far: `best` sorted over the lanes, `bar` a key that
// at least `top` of the keys seen reach (0: none yet), so that only keys from it on
// matter, and up to 64 keys waiting in LDS.
struct TopList {
  u64 best = 0, bar = 0;
  int held = 0, top;
  u64 *buf;
  __device__ __forceinline__ void flush(int lane) {
    const u64 fresh = lane < held ? buf[lane] : 0;
    best = merge64(best, sort64(fresh, lane), lane);
    const u64 b = key_at(best, top - 1);
    bar = b > bar ? b : bar;
    held = 0;
    __builtin_amdgcn_wave_barrier();
  }
  // The first keys: `most` is the largest of each lane's. The top-th of them
  // bounds the list from below before any key is kept.
  __device__ __forceinline__ void start(u64 most, int lane) {
    bar = key_at(sort64(most, lane), top - 1);
  }
  __device__ __forceinline__ void raise(u64 other) {
    other = key_at(other, 0);
    bar = other > bar ? other : bar;
  }
  // One key a lane (0: none). Keys are unique; the bar itself may still come.
  __device__ __forceinline__ void push(u64 key, int lane) {
    u64 pass = __ballot(key >= bar && key != 0);
    if (!pass) return;
    if (held + __popcll(pass) > 64) {
      flush(lane);
      pass = __ballot(key >= bar && key != 0);
    }
    if ((pass >> lane) & 1u) buf[held + __popcll(pass & (((u64)1 << lane) - 1))] = key;
    held += __popcll(pass);
    __builtin_amdgcn_wave_barrier();
  }
};

// Softmax statistics of part of a position.
struct Stats {
  float m, z, a;
};
__device__ __forceinline__ void move_reference(Stats &s, float m) {
  const float d = fmaxf(s.m - m, kFar);
  const float f = s.m == m ? 1.0f : fast_exp2(d * kLog2e);
  s.a = f * (s.a + d * s.z);
  s.z = f * s.z;
  s.m = m;
}
// e^(x - m) and its product with x - m for one logit. The exponent's product is rounded, by
// 2^-24 |d| log2 e: of the term, which is e^d, so of z by 2^-24 at most (|d| e^d <= 1 / e).
__device__ __forceinline__ void add_logit(Stats &s, float x) {
  float d = x - s.m;
  d = d < kFar ? kFar : d;  // keeps a NaN
  const float e = fast_exp2(d * kLog2e);
  s.z += e;
  s.a = fmaf(e, d, s.a);
}
__device__ __forceinline__ Stats wave_join(Stats s) {
  move_reference(s, wave_max_f(s.m));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s.z += __shfl_xor(s.z, o);
    s.a += __shfl_xor(s.a, o);
  }
  return s;
}

// What is left once a position's statistics and list are known (one wave).
__device__ __forceinline__ void write_position(const LogProbArgs &a, long pos, const Stats &s,
                                               u64 best, int lane) {
  const float logz = logf(s.z);
  if (lane == 0 && a.entropy) a.entropy[pos] = logz - s.a / s.z;
  if (lane < a.top) {
    a.top_tokens[pos * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)best;
    a.top_log_probs[pos * a.top + lane] = (code_value((uint32_t)(best >> 32)) - s.m) - logz;
  }
  for (int j = lane; j < a.per; j += 64) {
    const int64_t t = a.tokens[pos * a.per + j];
    float lp = 0.0f;
    if (t >= 0) {
      float x = NAN;
      if (t < (int64_t)a.vocab) {
        const size_t at = (size_t)pos * a.ld + (size_t)t;
        x = a.bf16 ? bf16_to_f32(static_cast<const unsigned short *>(a.logits)[at])
                   : static_cast<const float *>(a.logits)[at];
      }
      lp = (x - s.m) - logz;
    }
    a.log_probs[pos * a.per + j] = lp;
  }
}

// Workgroup = one part of one position; NW waves. Parts are whole numbers of
// 16-byte pieces of the position, counted from the 16-byte boundary at or
// before its first logit.
template <bool BF16, bool TOP, int NW>
__global__ __launch_bounds__(64 * NW) void log_probs_kernel(LogProbArgs a) {
  constexpr int E = BF16 ? 8 : 4;  // logits per 16 bytes
  constexpr int U = 4;             // 16-byte pieces in flight per lane
  __shared__ u64 buf[NW][64];
  __shared__ float stats[NW][3];
  __shared__ u64 bars;  // the highest of the waves' bars so far, a bar for all of them
  const int lane = threadIdx.x & 63, wave = NW == 1 ? 0 : threadIdx.x >> 6;
  const long pos = blockIdx.x / (unsigned)a.parts;
  const int part = (int)(blockIdx.x - (unsigned)pos * (unsigned)a.parts);
  const char *row = static_cast<const char *>(a.logits) + (size_t)pos * a.ld * (16 / E);
  const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / (16 / E));
  const char *base = row - skew * (16 / E);
  const int vocab = (int)a.vocab;
  // Pieces of this part: piece p holds logits E p - skew .. E p - skew + E - 1.
  const int pieces = (vocab + skew + E - 1) / E;
  const int p0 = min(part * a.part_pieces, pieces), p1 = min(p0 + a.part_pieces, pieces);

  Stats s{kLowest, 0.0f, 0.0f};
  TopList list;
  list.top = a.top;
  list.buf = buf[wave];
  bool begun = false;
  if constexpr (TOP && NW > 1) {
    if (threadIdx.x == 0) bars = 0;
    __syncthreads();
  }

  for (int p = p0 + wave * 64 + lane; p - lane < p1; p += 64 * NW * U) {
    float x[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int q = p + u * 64 * NW;
      const int first = q * E - skew;
      if (q < p1 && first >= 0 && first + E <= vocab) {
        if constexpr (BF16) {
          const u16x8 h = *reinterpret_cast<const u16x8 *>(base + (size_t)q * 16);
#pragma unroll
          for (int e = 0; e < E; ++e) x[u][e] = bf16_to_f32(h[e]);
        } else {
          const f32x4 h = *reinterpret_cast<const f32x4 *>(base + (size_t)q * 16);
#pragma unroll
          for (int e = 0; e < E; ++e) x[u][e] = h[e];
        }
      } else {
        // The row's first and last piece, and lanes past the part: -inf adds nothing.
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = first + e;
          x[u][e] = -INFINITY;
          if (q < p1 && i >= 0 && i < vocab) {
            if constexpr (BF16)
              x[u][e] = bf16_to_f32(reinterpret_cast<const unsigned short *>(row)[i]);
            else
              x[u][e] = reinterpret_cast<const float *>(row)[i];
          }
        }
      }
    }
    float mx[U], m = s.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mx[u] = x[u][0];
#pragma unroll
      for (int e = 1; e < E; ++e) mx[u] = fmaxf(mx[u], x[u][e]);
      m = fmaxf(m, mx[u]);
    }
    if (m > s.m) move_reference(s, m);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) add_logit(s, x[u][e]);
    if constexpr (TOP) {
      auto key = [&](int u, int e) -> u64 {
        const int q = p + u * 64 * NW, i = q * E - skew + e;
        return q < p1 && i >= 0 && i < vocab ? key_of(x[u][e], (uint32_t)i) : 0;
      };
      if (!begun) {
        u64 most = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const u64 k = key(u, e);
            most = k > most ? k : most;
          }
        list.start(most, lane);
        begun = true;
      }
      if constexpr (NW > 1) {
        if (lane == 0) atomicMax(&bars, list.bar);
        list.raise(*const_cast<volatile u64 *>(&bars));
      }
      // Values are compared first: few keys are ever made.
      const float bar_value = list.bar ? code_value((uint32_t)(list.bar >> 32)) : NAN;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!__any(p + u * 64 * NW < p1 && !(mx[u] < bar_value))) continue;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (__any(!(x[u][e] < bar_value))) list.push(key(u, e), lane);
      }
    }
  }
  s = wave_join(s);
  if constexpr (TOP) list.flush(lane);
  u64 best = list.best;
  if constexpr (NW > 1) {
    if constexpr (TOP) buf[wave][lane] = best;
    if (lane == 0) {
      stats[wave][0] = s.m;
      stats[wave][1] = s.z;
      stats[wave][2] = s.a;
    }
    __syncthreads();
    if (wave != 0) return;
    float m = s.m;
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, stats[w][0]);
    move_reference(s, m);
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      Stats t{stats[w][0], stats[w][1], stats[w][2]};
      move_reference(t, m);
      s.z += t.z;
      s.a += t.a;
      if constexpr (TOP) best = merge64(best, buf[w][lane], lane);
    }
  }
  if (a.parts == 1) {
    write_position(a, pos, s, best, lane);
    return;
  }
  if (lane == 0) {
    float *o = a.part_stats + 4 * (size_t)blockIdx.x;
    o[0] = s.m;
    o[1] = s.z;
    o[2] = s.a;
  }
  if (TOP && lane < a.top) a.part_keys[(size_t)blockIdx.x * a.top + lane] = best;
}

// Joins the parts of a position: lane l takes parts l, l + 64, ... (one wave).
template <bool TOP>
__global__ __launch_bounds__(64) void log_probs_join_kernel(LogProbArgs a) {
  const long pos = blockIdx.x;
  const int lane = threadIdx.x;
  Stats s{kLowest, 0.0f, 0.0f};
  for (int p = lane; p < a.parts; p += 64) {
    const float *o = a.part_stats + 4 * ((size_t)pos * a.parts + p);
    Stats t{o[0], o[1], o[2]};
    const float m = fmaxf(s.m, t.m);
    move_reference(s, m);
    move_reference(t, m);
    s.z += t.z;
    s.a += t.a;
  }
  s = wave_join(s);
  TopList list;
  if constexpr (TOP) {
    __shared__ u64 buf[64];
    list.top = a.top;
    list.buf = buf;
    const size_t n = (size_t)a.parts * a.top;
    const u64 *keys = a.part_keys + (size_t)pos * n;
    constexpr int U = 8;  // loads in flight
    for (size_t i = 0; i < n; i += 64 * U) {
      u64 k[U], most = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) k[u] = i + 64 * u + lane < n ? keys[i + 64 * u + lane] : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) most = k[u] > most ? k[u] : most;
      if (i == 0) list.start(most, lane);
#pragma unroll
      for (int u = 0; u < U; ++u) list.push(k[u], lane);
    }
    list.flush(lane);
  }
  write_position(a, pos, s, list.best, lane);
}

template <bool BF16, bool TOP>
void launch_parts(const LogProbArgs &a, int waves, hipStream_t stream, const KernelEvents &ev) {
  const dim3 grid((unsigned)(a.positions * (size_t)a.parts));
  hipEvent_t stop = a.parts == 1 ? ev.stop : nullptr;
  if (waves == 1)
    hipExtLaunchKernelGGL((log_probs_kernel<BF16, TOP, 1>), grid, dim3(64), 0, stream, ev.start,
                          stop, 0, a);
  else
    hipExtLaunchKernelGGL((log_probs_kernel<BF16, TOP, 4>), grid, dim3(256), 0, stream, ev.start,
                          stop, 0, a);
  if (a.parts == 1) return;
  hipExtLaunchKernelGGL((log_probs_join_kernel<TOP>), dim3((unsigned)a.positions), dim3(64), 0,
                        stream, nullptr, ev.stop, 0, a);
}

}  // namespace

// Positions of up to so many 16-byte pieces stay whole: the join is a launch more, 2.6 us of
// the host's time a call, and a wave that reads what the others left. Whole and in parts, us
// per call (eager ones one after another, from Python; in brackets replays of a graph, where
// the launch costs least):
//   4096 pieces f32,  1 position 8.0, 10.6 (4.8, 4.9), 256: 8.0, 10.6 (5.6, 6.8)
//   4096 pieces bf16, 1 position 8.0, 10.7 (7.3, 5.6), 256: 9.7, 10.3 (9.8, 8.3)
//   8192 pieces f32,  1 position 8.0, 10.6 (7.3, 4.9), 256: 9.0, 10.2 (9.3, 9.2)
//   8192 pieces bf16, 1 position 12.0, 10.5 (12.1, 5.5), 256: 15.4, 13.3 (15.6, 13.7)
//   16384 pieces f32, 1 position 12.1, 10.4 (12.2, 4.9), 256: 16.8, 14.7 (17.3, 15.1)
// With top 5:
//   2048 pieces f32,  1 position 10.9, 13.5 (9.0, 11.4), 256: 11.0, 13.7 (10.1, 13.1)
//   2048 pieces bf16, 1 position 11.9, 14.1 (11.5, 13.4), 256: 12.9, 15.7 (13.3, 15.7)
//   4096 pieces f32,  1 position 11.1, 13.7 (12.2, 11.5), 256: 14.1, 15.4 (14.4, 15.1)
//   4096 pieces bf16, 1 position 16.7, 14.1 (16.4, 13.4), 256: 20.3, 19.0 (20.1, 19.2)
// With top 20 replays of 2048 pieces bf16 take 15.2 and 15.7 (1 position), 17.6 and 17.7
// (256), of 4096 24.1 and 16.0, 27.5 and 22.6. The limits are where eager calls of both
// types are about even.
constexpr size_t kLogProbWhole = 8192, kLogProbWholeTop = 2048;
// Fewest pieces of a part: one step of a workgroup's four waves. Fewer spread
// a position further, but every wave has to find its first `top` and the joining
// wave reads them all (bf16, 100003 logits, top 20: 21.0 us with 256 pieces, 19.0 with
// 512, 19.6 with 1024, 22.5 with 2048; 4 x 151936 f32, top 50: 61, 44, 30, 27).
constexpr size_t kLogProbPart = 1024;

void log_probs_plan(LogProbArgs &a, int cus) {
  const size_t per_piece = a.bf16 ? 8 : 4;
  const size_t pieces = (a.vocab + 2 * (per_piece - 1)) / per_piece;  // at any skew
  a.parts = 1;
  a.part_pieces = (int)pieces;
  if (a.vocab <= kLogProbWaveVocab || pieces <= (a.top ? kLogProbWholeTop : kLogProbWhole)) return;
  // Parts of kLogProbPart pieces or more, until every CU has two workgroups.
  const size_t want = a.positions ? (2 * (size_t)cus + a.positions - 1) / a.positions : 1;
  const size_t most = (pieces + kLogProbPart - 1) / kLogProbPart;
  size_t parts = want < most ? want : most;
  if (parts <= 1) return;
  const size_t len = (pieces + parts - 1) / parts;
  a.part_pieces = (int)len;
  a.parts = (int)((pieces + len - 1) / len);
}

// Positions of one launch: 2^30 threads of the 2^32 that a grid may have.
constexpr size_t kLogProbLaunch = (size_t)1 << 22;

hipError_t launch_log_probs(const LogProbArgs &a, hipStream_t stream, const KernelEvents &ev) {
  const int waves = a.vocab <= kLogProbWaveVocab ? 1 : 4;
  for (size_t p0 = 0; p0 < a.positions; p0 += kLogProbLaunch) {
    LogProbArgs b = a;
    b.positions = a.positions - p0 < kLogProbLaunch ? a.positions - p0 : kLogProbLaunch;
    b.logits = static_cast<const char *>(a.logits) + (a.bf16 ? 2 : 4) * a.ld * p0;
    if (a.per) {
      b.tokens = a.tokens + a.per * p0;
      b.log_probs = a.log_probs + a.per * p0;
    }
    if (a.entropy) b.entropy = a.entropy + p0;
    if (a.top) {
      b.top_tokens = a.top_tokens + a.top * p0;
      b.top_log_probs = a.top_log_probs + a.top * p0;
    }
    const KernelEvents e{p0 ? nullptr : ev.start,
                         p0 + b.positions < a.positions ? nullptr : ev.stop};
    if (a.bf16)
      a.top ? launch_parts<true, true>(b, waves, stream, e)
            : launch_parts<true, false>(b, waves, stream, e);
    else
      a.top ? launch_parts<false, true>(b, waves, stream, e)
            : launch_parts<false, false>(b, waves, stream, e);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace tfd
