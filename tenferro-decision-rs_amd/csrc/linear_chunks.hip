// Linear attention over prompts, 64 tokens at a time (the formulas of
// linear_attention.hip; D_ts = e^(g_(s+1) + .. + g_t) for s <= t, d_t = D from the
// chunk's start, e_s = D to its end, S0 the state before the chunk):
//   M_ts = beta_t D_ts (k_t . k_s) for s < t,   T = (I + M)^-1
//   U    = T (beta (V - d K S0))                 (plain: U = V)
//   O    = scale (d Q S0 + (D . Q K^T) U)
//   S0  <- e^G S0 + K^T (e U)
// Three kernels, the last and the first parallel over the chunks:
//   linear_solve_kernel   T of every chunk (delta rule only)
//   linear_walk_kernel    along each (row, head): U and the states S0
//   linear_output_kernel  O of every chunk
//
// Products run on the bf16 matrix cores with f32 accumulation, f32 operands as
// three bf16 pieces (six products, tfd_device.hpp), bf16 operands as they are:
// nothing is rounded to bf16. Decays are factors of f32 values, never of the
// operands that are exact in bf16.
//
// Operands live in fragment order: block (tile, step, piece) of 1 KB holds 16
// bytes for each lane l of the wavefront, element e of row 16 tile + l % 16 at
// contraction index 32 step + slot_index(l / 16, e). That order is the one in which
// the accumulators of two row tiles (4 (l / 16) + r of each) come out, so a
// product's result is the next product's operand without leaving its lane:
// S0, V - d K S0 and U are never moved between lanes.
#include <hip/hip_ext.h>
#include <math.h>

#include "tfd_device.hpp"
#include "tfd_internal.hpp"

namespace tfd {
namespace {

constexpr int kC = kLinearChunk;  // 64 tokens
constexpr double kLog2eD = 1.4426950408889634;
// log_decay below this is e^g = 0 in f32: the state is forgotten, and such terms
// stay out of the sums, where they would drown the others.
constexpr float kForget = -104.0f;

typedef bf16x8 frag;

// Contraction index of element e (0..7) of lane group g within a step of 32.
__device__ __forceinline__ int slot_index(int g, int e) { return 16 * (e >> 2) + 4 * g + (e & 3); }

// Pieces of two accumulator quads as one operand.
__device__ __forceinline__ void split8(f32x4 lo, f32x4 hi, frag (&p)[3]) {
  const Bf16x3 a = split_bf16x3(lo), b = split_bf16x3(hi);
#pragma unroll
  for (int i = 0; i < 3; ++i) p[i] = join_bf16(a, b, i);
}

// c += a b with all pieces whose product counts in f32, small ones first.
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const frag (&a)[NA], const frag (&b)[NB], f32x4 c) {
  if constexpr (NA == 3 && NB == 3) {
    c = mfma_16x16x32_bf16(a[0], b[2], c);
    c = mfma_16x16x32_bf16(a[2], b[0], c);
    c = mfma_16x16x32_bf16(a[1], b[1], c);
    c = mfma_16x16x32_bf16(a[0], b[1], c);
    c = mfma_16x16x32_bf16(a[1], b[0], c);
  } else if constexpr (NB == 3) {
    c = mfma_16x16x32_bf16(a[0], b[2], c);
    c = mfma_16x16x32_bf16(a[0], b[1], c);
  } else if constexpr (NA == 3) {
    c = mfma_16x16x32_bf16(a[2], b[0], c);
    c = mfma_16x16x32_bf16(a[1], b[0], c);
  }
  return mfma_16x16x32_bf16(a[0], b[0], c);
}

template <int NP>
__device__ __forceinline__ void load_frag(const unsigned char *block, int lane, frag (&p)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i)
    p[i] = *reinterpret_cast<const frag *>(block + 1024 * i + 16 * lane);
}
template <int NP>
__device__ __forceinline__ void store_frag(unsigned char *block, int lane, const frag (&p)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) *reinterpret_cast<frag *>(block + 1024 * i + 16 * lane) = p[i];
}

// Operand elements: f32 as three pieces, bf16 as itself.
template <typename T>
struct Pieces {
  static constexpr int n = sizeof(T) == 4 ? 3 : 1;
};

template <typename T>
__device__ __forceinline__ float as_f32(T x) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(x);
  else
    return x;
}

template <typename T>
__device__ __forceinline__ void to_frag(const T (&v)[8], frag (&p)[Pieces<T>::n]) {
  if constexpr (sizeof(T) == 2) {
    u16x8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = v[e];
    p[0] = __builtin_bit_cast(frag, h);
  } else {
    split8(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]}, p);
  }
}

// Four consecutive tokens of a feature row, 0 where `act` (bit = token of the
// chunk) is not set; at = chunk token of the first one. Inactive tokens are
// only read inside the row (vec: 16 or 8 byte pieces, length % 4 == 0).
template <typename T>
__device__ __forceinline__ void load4(const T *row, int at, uint64_t act, int n, bool vec, T (&v)[4]) {
  const unsigned on = (unsigned)(act >> at) & 15u;
  if (vec) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    vec4 x = {};
    if (at < n) x = *reinterpret_cast<const vec4 *>(row + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (on >> e) & 1u ? x[e] : T(0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (on >> e) & 1u ? row[at + e] : T(0);
  }
}

// ------------------------------------------------------------------ a chunk

struct ChunkScan {
  double cum[kC];   // log2 of the decay from the chunk's start through token t
  int forget[kC];   // last token <= t that forgets the state, or -1
  float from_start[kC], to_end[kC], beta[kC];
};

// The chunk's decays, by one wavefront (lane = token). The sums are held in 64
// bits: a difference of sums is then good to 2^-24 of the terms between them,
// whatever came before.
__device__ __forceinline__ void scan_chunk(const LinearArgs &a, size_t rh, int t0, int n,
                                           uint64_t act, int lane, ChunkScan &c) {
  const bool on = (act >> lane) & 1u;
  const float g = on ? a.log_decay[rh * a.L + t0 + lane] : 0.0f;
  const bool forgets = g < kForget;
  double x = forgets ? 0.0 : (double)g * kLog2eD;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  const uint64_t f = __ballot(forgets);
  const uint64_t upto = f & (~0ull >> (63 - lane));
  const int p = upto ? 63 - __clzll((long long)upto) : -1;
  const double all = __shfl(x, 63);
  const int last = f ? 63 - __clzll((long long)f) : -1;
  c.cum[lane] = x;
  c.forget[lane] = p;
  c.from_start[lane] = p >= 0 ? 0.0f : fast_exp2((float)x);
  c.to_end[lane] = last > lane ? 0.0f : fast_exp2((float)(all - x));
  c.beta[lane] = on && a.beta ? a.beta[rh * a.L + t0 + lane] : 0.0f;
}

__device__ __forceinline__ float decay_between(const ChunkScan &c, int t, int s) {
  return c.forget[t] > s ? 0.0f : fast_exp2((float)(c.cum[t] - c.cum[s]));
}

// Bit t: token t0 + t is there and active (one wavefront's lanes).
__device__ __forceinline__ uint64_t active_tokens(const LinearArgs &a, int r, int t0, int lane) {
  const int t = t0 + lane;
  return __ballot(t < a.L && (!a.mask || a.mask[(size_t)r * a.L + t] != 0.0f));
}

// Token-major operand (rows = tokens, contraction = features f0 ..): blocks
// [token tile 4][step][piece] of `steps` steps, by the whole workgroup. Lanes
// read along the tokens, eight features each.
template <typename T>
__device__ __forceinline__ void stage_tokens(unsigned char *dst, const T *src, int L, int f0, int dk,
                                             int steps, uint64_t act, int thread, int threads) {
  constexpr int NP = Pieces<T>::n;
  const int t = thread & 63, tile = t >> 4;
  const bool on = (act >> t) & 1u;
  for (int o = thread >> 6; o < 4 * steps; o += threads >> 6) {
    const int kk = o >> 2, g = o & 3;
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int f = f0 + 32 * kk + slot_index(g, e);
      v[e] = on && f < dk ? src[(size_t)f * L + t] : T(0);
    }
    frag p[NP];
    to_frag<T>(v, p);
    store_frag<NP>(dst + 1024 * NP * (tile * steps + kk), 16 * g + (t & 15), p);
  }
}

// Feature-major operand (rows = features f0 .., contraction = tokens): blocks
// [feature tile][step 2][piece] of `tiles` tiles.
template <typename T>
__device__ __forceinline__ void stage_features(unsigned char *dst, const T *src, int L, int f0,
                                               int dk, int tiles, uint64_t act, int n, bool vec,
                                               int thread, int threads) {
  constexpr int NP = Pieces<T>::n;
  const int lane = thread & 63, g = lane >> 4;
  for (int b = thread >> 6; b < 2 * tiles; b += threads >> 6) {
    const int tile = b >> 1, ks = b & 1;
    const int f = f0 + 16 * tile + (lane & 15);
    T lo[4] = {}, hi[4] = {};
    if (f < dk) {
      load4<T>(src + (size_t)f * L, 32 * ks + 4 * g, act, n, vec, lo);
      load4<T>(src + (size_t)f * L, 32 * ks + 16 + 4 * g, act, n, vec, hi);
    }
    const T v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    frag p[NP];
    to_frag<T>(v, p);
    store_frag<NP>(dst + 1024 * NP * (2 * tile + ks), lane, p);
  }
}

// ------------------------------------------------------------------ T

// Workgroup = one chunk of one (row, head), four waves. K K^T by row tiles, then
// (I + M)^-1 by 16 x 16 blocks: the diagonal blocks by substitution (one wave
// each), the others by T_ij = -T_ii sum_(j <= k < i) M_ik T_kj on the f32 matrix
// cores, one distance i - j after the other.
template <typename T>
__global__ __launch_bounds__(256) void linear_solve_kernel(LinearArgs a, unsigned char *solve) {
  constexpr int NP = Pieces<T>::n;
  constexpr int kS = 68;  // floats per row: 16-byte rows, rows 4 banks apart
  __shared__ __attribute__((aligned(16))) unsigned char kpl[8 * NP * 1024];
  __shared__ __attribute__((aligned(16))) float M[kC * kS], X[kC * kS];
  __shared__ ChunkScan sc;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
  const int chunk = blockIdx.x, h = blockIdx.y, r = blockIdx.z, nch = gridDim.x;
  const size_t rh = (size_t)r * a.heads + h;
  const int t0 = chunk * kC, n = min(kC, a.L - t0);
  const uint64_t act = active_tokens(a, r, t0, lane);
  if (wave == 0) scan_chunk(a, rh, t0, n, act, lane, sc);
  const T *k = static_cast<const T *>(a.k) +
               ((size_t)r * a.key_heads + h / a.group) * a.dk * a.L + t0;
  f32x4 acc[4] = {};
  for (int f0 = 0; f0 < a.dk; f0 += 64) {
    if (f0) __syncthreads();
    stage_tokens<T>(kpl, k, a.L, f0, a.dk, 2, act, threadIdx.x, 256);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      frag x[NP];
      load_frag<NP>(kpl + 1024 * NP * (2 * wave + kk), lane, x);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (st > wave) continue;
        frag y[NP];
        load_frag<NP>(kpl + 1024 * NP * (2 * st + kk), lane, y);
        acc[st] = mma<NP, NP>(x, y, acc[st]);
      }
    }
  }
#pragma unroll
  for (int st = 0; st < 4; ++st)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 16 * wave + 4 * g + e, s = 16 * st + c16;
      if (st <= wave) M[t * kS + s] = s < t ? sc.beta[t] * decay_between(sc, t, s) * acc[st][e] : 0.0f;
      X[t * kS + s] = 0.0f;
    }
  __syncthreads();
  // Diagonal block: lane c holds column c of the inverse.
  {
    const float *m = M + 16 * wave * kS + 16 * wave;
    float x[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      float v = t == c16 ? 1.0f : 0.0f;
#pragma unroll
      for (int s = 0; s < t; ++s) v = fmaf(-m[t * kS + s], x[s], v);
      x[t] = v;
    }
    if (lane < 16)
#pragma unroll
      for (int t = 0; t < 16; ++t) X[(16 * wave + t) * kS + 16 * wave + c16] = x[t];
  }
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    __syncthreads();
    const int i = wave + d, j = wave;
    if (i < 4) {
      f32x4 w = {};
      for (int b = j; b < i; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s)
          w = mfma_16x16x4(M[(16 * i + c16) * kS + 16 * b + 4 * s + g],
                           X[(16 * b + 4 * s + g) * kS + 16 * j + c16], w);
      f32x4 v = {};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        v = mfma_16x16x4(-X[(16 * i + c16) * kS + 16 * i + 4 * g + s], w[s], v);
#pragma unroll
      for (int s = 0; s < 4; ++s) X[(16 * i + 4 * g + s) * kS + 16 * j + c16] = v[s];
    }
  }
  __syncthreads();
  // Six operand blocks: steps past the diagonal hold nothing.
  unsigned char *dst = solve + (rh * nch + chunk) * kLinearSolveBytes;
  for (int b = wave; b < 6; b += 4) {
    const int tt = b < 2 ? b : 2 + ((b - 2) >> 1), ks = b < 2 ? 0 : (b - 2) & 1;
    const float *x = X + (16 * tt + c16) * kS + 32 * ks + 4 * g;
    frag p[3];
    split8(*reinterpret_cast<const f32x4 *>(x), *reinterpret_cast<const f32x4 *>(x + 16), p);
    store_frag<3>(dst + 3072 * b, lane, p);
  }
}

// Operand block of T's row tile tt at step ks.
__device__ __forceinline__ int solve_block(int tt, int ks) { return tt < 2 ? tt : 2 * tt - 2 + ks; }

// ------------------------------------------------------------------ the walk

// Workgroup = up to 8 waves of one (row, head), a wave = 16 value columns with their
// whole state in accumulators (feature 16 n + 4 (lane / 16) + e, column lane % 16).
// The waves share the chunk's keys (both orders) and T in LDS.
template <typename T, bool DELTA, int NI>
__global__ __launch_bounds__(512) void linear_walk_kernel(LinearArgs a, const unsigned char *solve,
                                                          float *states, float *writes) {
  constexpr int NP = Pieces<T>::n;
  constexpr int SI = NI < 8 ? NI : 8;      // feature tiles per slab of the keys
  constexpr int SK = SI / 2, NS = NI / SI;  // contraction steps per slab, slabs
  __shared__ __attribute__((aligned(16))) unsigned char kt[2 * SI * NP * 1024];
  __shared__ __attribute__((aligned(16))) unsigned char kpl[DELTA ? 4 * SK * NP * 1024 : 16];
  __shared__ __attribute__((aligned(16))) unsigned char tpl[DELTA ? kLinearSolveBytes : 16];
  __shared__ ChunkScan sc;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
  const int threads = blockDim.x;
  const int h = blockIdx.y, r = blockIdx.z;
  const int jt = blockIdx.x * (threads >> 6) + wave, j = 16 * jt + c16;
  const bool here = 16 * jt < a.dv, col = j < a.dv;
  const size_t rh = (size_t)r * a.heads + h;
  const int nch = (a.L + kC - 1) / kC, jtiles = (a.dv + 15) / 16;
  const T *k = static_cast<const T *>(a.k) + ((size_t)r * a.key_heads + h / a.group) * a.dk * a.L;
  const T *v = static_cast<const T *>(a.v) + (rh * a.dv + (col ? j : 0)) * a.L;

  f32x4 S[NI] = {};
  if (a.state_in && col) {
    const float *p = a.state_in + rh * a.dk * a.dv + j;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int f = 16 * i + 4 * g + e;
        S[i][e] = f < a.dk ? p[(size_t)f * a.dv] : 0.0f;
      }
  }
  for (int chunk = 0; chunk < nch; ++chunk) {
    const int t0 = chunk * kC, n = min(kC, a.L - t0);
    const uint64_t act = active_tokens(a, r, t0, lane);
    __syncthreads();  // the last chunk's operands are read
    if (wave == 0) scan_chunk(a, rh, t0, n, act, lane, sc);
    stage_features<T>(kt, k + t0, a.L, 0, a.dk, SI, act, n, a.vec_k, threadIdx.x, threads);
    if constexpr (DELTA) {
      stage_tokens<T>(kpl, k + t0, a.L, 0, a.dk, SK, act, threadIdx.x, threads);
      const unsigned char *src = solve + (rh * nch + chunk) * kLinearSolveBytes;
      for (int i = threadIdx.x * 16; i < kLinearSolveBytes; i += threads * 16)
        *reinterpret_cast<f32x4 *>(tpl + i) = *reinterpret_cast<const f32x4 *>(src + i);
    }
    __syncthreads();
    if (here) {  // S0 for the outputs, in fragment order
      float *o = states + ((rh * nch + chunk) * jtiles + jt) * (size_t)(NI / 2) * 512 + 8 * lane;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        *reinterpret_cast<f32x4 *>(o + (i >> 1) * 512 + 4 * (i & 1)) = S[i];
    }
    f32x4 U[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      T x[4] = {};
      if (col) load4<T>(v + t0, 16 * tt + 4 * g, act, n, a.vec_v, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) U[tt][e] = as_f32<T>(x[e]);
    }
    if constexpr (DELTA) {
      f32x4 X[4] = {};
#pragma unroll
      for (int slab = 0; slab < NS; ++slab) {
        if (slab) {
          __syncthreads();
          stage_tokens<T>(kpl, k + t0, a.L, 16 * SI * slab, a.dk, SK, act, threadIdx.x, threads);
          __syncthreads();
        }
#pragma unroll
        for (int kk = 0; kk < SK; ++kk) {
          frag s[3];
          split8(S[SI * slab + 2 * kk], S[SI * slab + 2 * kk + 1], s);
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            frag x[NP];
            load_frag<NP>(kpl + 1024 * NP * (tt * SK + kk), lane, x);
            X[tt] = mma<NP, 3>(x, s, X[tt]);
          }
        }
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = 16 * tt + 4 * g + e;
          X[tt][e] = sc.beta[t] * fmaf(-sc.from_start[t], X[tt][e], U[tt][e]);
        }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) U[tt] = f32x4{};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        frag x[3];
        split8(X[2 * ks], X[2 * ks + 1], x);
#pragma unroll
        for (int tt = 2 * ks; tt < 4; ++tt) {
          frag s[3];
          load_frag<3>(tpl + 3072 * solve_block(tt, ks), lane, s);
          U[tt] = mma<3, 3>(s, x, U[tt]);
        }
      }
      if (here) {
        float *o = writes + ((rh * nch + chunk) * jtiles + jt) * (size_t)1024 + 8 * lane;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
          *reinterpret_cast<f32x4 *>(o + (tt >> 1) * 512 + 4 * (tt & 1)) = U[tt];
      }
    }
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int e = 0; e < 4; ++e) U[tt][e] *= sc.to_end[16 * tt + 4 * g + e];
    const float whole = sc.from_start[kC - 1];
    frag u[2][3];
    split8(U[0], U[1], u[0]);
    split8(U[2], U[3], u[1]);
#pragma unroll
    for (int slab = 0; slab < NS; ++slab) {
      if (slab) {
        __syncthreads();
        stage_features<T>(kt, k + t0, a.L, 16 * SI * slab, a.dk, SI, act, n, a.vec_k, threadIdx.x,
                          threads);
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < SI; ++i) {
        f32x4 s = S[SI * slab + i] * whole;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          frag x[NP];
          load_frag<NP>(kt + 1024 * NP * (2 * i + ks), lane, x);
          s = mma<NP, 3>(x, u[ks], s);
        }
        S[SI * slab + i] = s;
      }
    }
  }
  if (a.state_out && col) {
    float *p = a.state_out + rh * a.dk * a.dv + j;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int f = 16 * i + 4 * g + e;
        if (f < a.dk) p[(size_t)f * a.dv] = S[i][e];
      }
  }
}

// ------------------------------------------------------------------ outputs

// Workgroup = one chunk of one (row, head), four waves, up to 4 JW column tiles.
// Wave w forms the scores of token tile w, then the outputs of columns tiles
// w, w + 4, .. (of the group) for all tokens.
template <typename T, bool DELTA, int JW>
__global__ __launch_bounds__(256) void linear_output_kernel(LinearArgs a, const float *states,
                                                            const float *writes, int steps) {
  constexpr int NP = Pieces<T>::n;
  constexpr int NU = DELTA ? 3 : NP;  // pieces of what is written
  constexpr int kHalf = 8 * 3 * 1024;
  __shared__ __attribute__((aligned(16))) unsigned char qpl[8 * NP * 1024];
  __shared__ __attribute__((aligned(16))) unsigned char kpl[kHalf];  // keys, then scores
  __shared__ ChunkScan sc;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
  const int nch = (a.L + kC - 1) / kC, jtiles = (a.dv + 15) / 16;
  const int chunk = blockIdx.x % nch, group = blockIdx.x / nch, h = blockIdx.y, r = blockIdx.z;
  const size_t rh = (size_t)r * a.heads + h;
  const int t0 = chunk * kC, n = min(kC, a.L - t0);
  const uint64_t act = active_tokens(a, r, t0, lane);
  if (wave == 0) scan_chunk(a, rh, t0, n, act, lane, sc);
  const size_t key = ((size_t)r * a.key_heads + h / a.group) * a.dk * a.L + t0;
  const T *q = static_cast<const T *>(a.q) + key, *k = static_cast<const T *>(a.k) + key;
  const int jt0 = group * 4 * JW + wave;
  f32x4 score[4] = {}, O[JW][4] = {};
  for (int f0 = 0; f0 < a.dk; f0 += 64) {
    if (f0) __syncthreads();
    stage_tokens<T>(qpl, q, a.L, f0, a.dk, 2, act, threadIdx.x, 256);
    stage_tokens<T>(kpl, k, a.L, f0, a.dk, 2, act, threadIdx.x, 256);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      if (f0 + 32 * kk >= a.dk) continue;
      frag y[NP];
      load_frag<NP>(qpl + 1024 * NP * (2 * wave + kk), lane, y);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (st > wave) continue;
        frag x[NP];
        load_frag<NP>(kpl + 1024 * NP * (2 * st + kk), lane, x);
        score[st] = mma<NP, NP>(x, y, score[st]);
      }
#pragma unroll
      for (int w = 0; w < JW; ++w) {
        const int jt = jt0 + 4 * w;
        if (jt >= jtiles) continue;
        const float *s0 = states + (((rh * nch + chunk) * jtiles + jt) * (size_t)steps +
                                    (f0 / 32 + kk)) * 512 + 8 * lane;
        frag s[3];
        split8(*reinterpret_cast<const f32x4 *>(s0), *reinterpret_cast<const f32x4 *>(s0 + 4), s);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          frag x[NP];
          load_frag<NP>(qpl + 1024 * NP * (2 * tt + kk), lane, x);
          O[w][tt] = mma<3, NP>(s, x, O[w][tt]);
        }
      }
    }
  }
  __syncthreads();  // the keys are read: their place takes the scores
  const int t = 16 * wave + c16;
#pragma unroll
  for (int st = 0; st < 4; ++st)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int s = 16 * st + 4 * g + e;
      score[st][e] = s <= t ? score[st][e] * decay_between(sc, t, s) : 0.0f;
    }
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    frag p[3];
    split8(score[2 * ks], score[2 * ks + 1], p);
    store_frag<3>(kpl + 3072 * (2 * wave + ks), lane, p);
  }
  __syncthreads();
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) {
    const float d = sc.from_start[16 * tt + c16];
#pragma unroll
    for (int w = 0; w < JW; ++w) O[w][tt] *= d;
  }
#pragma unroll
  for (int w = 0; w < JW; ++w) {
    const int jt = jt0 + 4 * w;
    if (jt >= jtiles) continue;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      frag u[NU];
      if constexpr (DELTA) {
        const float *p = writes + ((rh * nch + chunk) * jtiles + jt) * (size_t)1024 + 512 * ks + 8 * lane;
        split8(*reinterpret_cast<const f32x4 *>(p), *reinterpret_cast<const f32x4 *>(p + 4), u);
      } else {
        const int j = 16 * jt + c16;
        T lo[4] = {}, hi[4] = {};
        if (j < a.dv) {
          const T *row = static_cast<const T *>(a.v) + (rh * a.dv + j) * a.L + t0;
          load4<T>(row, 32 * ks + 4 * g, act, n, a.vec_v, lo);
          load4<T>(row, 32 * ks + 16 + 4 * g, act, n, a.vec_v, hi);
        }
        const T v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        to_frag<T>(v, u);
      }
#pragma unroll
      for (int tt = 2 * ks; tt < 4; ++tt) {
        frag x[3];
        load_frag<3>(kpl + 3072 * (2 * tt + ks), lane, x);
        O[w][tt] = mma<NU, 3>(u, x, O[w][tt]);
      }
    }
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 16 * jt + 4 * g + e, tok = 16 * tt + c16;
        if (j < a.dv && tok < n) a.out[(rh * a.dv + j) * a.L + t0 + tok] = a.scale * O[w][tt][e];
      }
  }
}

template <typename T, bool DELTA, int NI>
hipError_t launch_walk(const LinearArgs &a, const unsigned char *solve, float *states,
                       float *writes, hipStream_t stream, hipEvent_t start) {
  const int jtiles = (a.dv + 15) / 16;
  int nw = 8;
  while (nw > 1 && nw / 2 >= jtiles) nw /= 2;
  const dim3 grid((unsigned)((jtiles + nw - 1) / nw), (unsigned)a.heads, (unsigned)a.rows);
  hipExtLaunchKernelGGL((linear_walk_kernel<T, DELTA, NI>), grid, dim3(64 * nw), 0, stream, start,
                        nullptr, 0, a, solve, states, writes);
  return hipGetLastError();
}

template <typename T, bool DELTA>
hipError_t launch_chunks(const LinearArgs &a, unsigned char *ws, hipStream_t stream,
                         const KernelEvents &ev) {
  const LinearSpace sp = linear_space(a);
  float *states = reinterpret_cast<float *>(ws);
  float *writes = reinterpret_cast<float *>(ws + sp.states);
  unsigned char *solve = ws + sp.states + sp.writes;
  const unsigned nch = (unsigned)((a.L + kC - 1) / kC);
  hipError_t e = hipSuccess;
  hipEvent_t start = ev.start;
  if (DELTA) {
    hipExtLaunchKernelGGL((linear_solve_kernel<T>), dim3(nch, a.heads, a.rows), dim3(256), 0,
                          stream, start, nullptr, 0, a, solve);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    start = nullptr;
  }
  const int steps = linear_steps(a.dk);
  switch (steps) {
    case 1: e = launch_walk<T, DELTA, 2>(a, solve, states, writes, stream, start); break;
    case 2: e = launch_walk<T, DELTA, 4>(a, solve, states, writes, stream, start); break;
    case 4: e = launch_walk<T, DELTA, 8>(a, solve, states, writes, stream, start); break;
    default: e = launch_walk<T, DELTA, 16>(a, solve, states, writes, stream, start); break;
  }
  if (e != hipSuccess) return e;
  const int jtiles = (a.dv + 15) / 16;
  const int jw = jtiles <= 4 ? 1 : (jtiles <= 8 ? 2 : 4);
  const dim3 grid(nch * (unsigned)((jtiles + 4 * jw - 1) / (4 * jw)), (unsigned)a.heads,
                  (unsigned)a.rows);
  if (jw == 1)
    hipExtLaunchKernelGGL((linear_output_kernel<T, DELTA, 1>), grid, dim3(256), 0, stream, nullptr,
                          ev.stop, 0, a, states, writes, steps);
  else if (jw == 2)
    hipExtLaunchKernelGGL((linear_output_kernel<T, DELTA, 2>), grid, dim3(256), 0, stream, nullptr,
                          ev.stop, 0, a, states, writes, steps);
  else
    hipExtLaunchKernelGGL((linear_output_kernel<T, DELTA, 4>), grid, dim3(256), 0, stream, nullptr,
                          ev.stop, 0, a, states, writes, steps);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_linear_chunks(const LinearArgs &a, void *ws, hipStream_t stream,
                                const KernelEvents &ev) {
  unsigned char *w = static_cast<unsigned char *>(ws);
  if (a.bf16)
    return a.beta ? launch_chunks<unsigned short, true>(a, w, stream, ev)
                  : launch_chunks<unsigned short, false>(a, w, stream, ev);
  return a.beta ? launch_chunks<float, true>(a, w, stream, ev)
                : launch_chunks<float, false>(a, w, stream, ev);
}

}  // namespace tfd
