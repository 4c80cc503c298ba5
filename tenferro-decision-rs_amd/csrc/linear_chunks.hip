// Linear attention over prompts, 64 tokens at a time (the formulas of
// linear_attention.hip; D_ts = e^(g_(s+1) + .. + g_t) for s <= t, d_t = D from the
// chunk's start, e_s = D to its end, S0 the state before the chunk):
//   M_ts = beta_t D_ts (k_t . k_s) for s < t,   T = (I + M)^-1
//   U    = T (beta (V - d K S0))                 (plain: U = V)
//   O    = scale (d Q S0 + (D . Q K^T) U)
//   S0  <- e^G S0 + K^T (e U)
// Two kernels follow each other:
//   linear_pairs_kernel, over all chunks at once: the decays, D . Q K^T and T
//   one that walks along each (row, head): U, O and the state, which stays in the
//   accumulators from the first chunk to the last (linear_delta_kernel,
//   linear_delta_path_kernel, linear_plain_kernel)
// Chunks without an active token are skipped by both.
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
constexpr int kPieces = 3 * 1024;  // bytes of a block's three pieces

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

// The pieces (of a, of b) of product number x of the NA x NB that count, small first.
template <int NA, int NB>
struct Products {
  static constexpr int n = NA == 3 && NB == 3 ? 6 : (NA == 3 || NB == 3 ? 3 : 1);
  static constexpr int a(int x) {
    constexpr int six[6] = {0, 2, 1, 0, 1, 0};
    return NA == 1 ? 0 : (NB == 1 ? 2 - x : six[x]);
  }
  static constexpr int b(int x) {
    constexpr int six[6] = {2, 0, 1, 1, 0, 0};
    return NB == 1 ? 0 : (NA == 1 ? 2 - x : six[x]);
  }
};
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

// Operand elements: f32 as three pieces, bf16 as itself. In memory the keys and
// queries lie in fragment order as they are: f32 as two blocks of 1 KB (a lane's first
// and last four elements), split when they are used, bf16 as one.
template <typename T>
struct Pieces {
  static constexpr int n = sizeof(T) == 4 ? 3 : 1, blocks = sizeof(T) == 4 ? 2 : 1;
};
template <typename T>
struct Stored {
  f32x4 b[Pieces<T>::blocks];
};
template <typename T>
__device__ __forceinline__ void load_stored(const unsigned char *block, int lane, Stored<T> &s) {
#pragma unroll
  for (int i = 0; i < Pieces<T>::blocks; ++i)
    s.b[i] = *reinterpret_cast<const f32x4 *>(block + 1024 * i + 16 * lane);
}
template <typename T>
__device__ __forceinline__ void to_frag(const Stored<T> &s, frag (&p)[Pieces<T>::n]) {
  if constexpr (sizeof(T) == 4)
    split8(s.b[0], s.b[1], p);
  else
    p[0] = __builtin_bit_cast(frag, s.b[0]);
}

// Loads go through a buffer resource of the head's (feature, token) matrix: one
// 32-bit offset, no branch; past its end they give 0 (offsets stay below 2^31, so a
// feature past key_dim is past the end, never wrapped). Rows before
// the end run into the next one (tokens behind the sequence), and inactive tokens
// hold anything: both are dropped where the values are used, so that nothing
// waits for a load before that.
typedef __amdgpu_buffer_rsrc_t Rsrc;
constexpr int kNowhere = (int)0x80000000u;  // past every resource's end

// Eight values as loaded: f32, or bf16 in a register each.
struct Raw {
  uint32_t d[8];
};

template <typename T>
__device__ __forceinline__ uint32_t load_one(Rsrc m, int off) {
  if constexpr (sizeof(T) == 4)
    return __builtin_amdgcn_raw_buffer_load_b32(m, off, 0, 0);
  else
    return __builtin_amdgcn_raw_buffer_load_b16(m, off, 0, 0);
}
// Four consecutive tokens (16-byte loads need 4-byte alignment only). bf16 stays 16 bits
// until it is used: a value widened across a loop's edge is waited for there.
template <typename T>
struct Four {
  unsigned short d[4];
};
template <>
struct Four<float> {
  f32x4 v;
};
template <typename T>
__device__ __forceinline__ void load_four(Rsrc m, int off, Four<T> &x) {
  if constexpr (sizeof(T) == 4) {
    x.v = buffer_load4(m, off, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x.d[e] = (unsigned short)load_one<T>(m, off + 2 * e);
  }
}
template <typename T>
__device__ __forceinline__ f32x4 values_of(const Four<T> &x) {
  if constexpr (sizeof(T) == 4) {
    return x.v;
  } else {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float((uint32_t)x.d[e] << 16);
    return v;
  }
}

// In fragment order, 0 where not `on`.
template <typename T>
__device__ __forceinline__ Stored<T> stored(const Raw &v, bool on) {
  Stored<T> s;
  if constexpr (sizeof(T) == 2) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = on ? __builtin_amdgcn_perm(v.d[2 * i + 1], v.d[2 * i], 0x05040100u) : 0u;
    s.b[0] = __builtin_bit_cast(f32x4, w);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s.b[0][e] = on ? __uint_as_float(v.d[e]) : 0.0f;
      s.b[1][e] = on ? __uint_as_float(v.d[4 + e]) : 0.0f;
    }
  }
  return s;
}
template <typename T>
__device__ __forceinline__ void store_stored(unsigned char *block, int slot, const Stored<T> &s) {
#pragma unroll
  for (int i = 0; i < Pieces<T>::blocks; ++i)
    *reinterpret_cast<f32x4 *>(block + 1024 * i + 16 * slot) = s.b[i];
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
// log_decay, beta: of token `lane`, as they are in memory.
__device__ __forceinline__ void scan_chunk(float log_decay, float beta, uint64_t act, int lane,
                                           ChunkScan &c) {
  const bool on = (act >> lane) & 1u;
  const float g = on ? log_decay : 0.0f;
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
  c.beta[lane] = on ? beta : 0.0f;
}

// Token-major operand (rows = tokens, contraction = features f0 ..): blocks
// [token tile 4][step][piece] of `steps` steps. Lanes read along the tokens, eight
// features each; octet o of the slab is step o / 4, lane group o % 4.
template <typename T>
__device__ __forceinline__ void load_octet(Rsrc m, int L, int t0, int f0, int o, int t, Raw &v) {
  const int es = sizeof(T);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int f = f0 + 32 * (o >> 2) + slot_index(o & 3, e);
    v.d[e] = load_one<T>(m, (t0 + t) * es + f * L * es);
  }
}
// Byte offset of octet o's block of `size` bytes for token t, and the token's slot in it.
__device__ __forceinline__ int octet_block(int size, int steps, int o, int t) {
  return size * ((t >> 4) * steps + (o >> 2));
}
__device__ __forceinline__ int octet_slot(int o, int t) { return 16 * (o & 3) + (t & 15); }

// The keys by features (rows = features of tile i, contraction = tokens of step ks):
// f32 from the matrix itself, where the lane's feature is its row and its tokens
// lie side by side, bf16 out of the slab's token-major blocks in LDS, where
// ds_read_b64_tr_b16 hands element e of lane j of a group of 16 the value 16 e + j
// of their 16 x 8 bytes: lane c of the group reads the four features 4 (c % 4) .. of
// token 4 g + c / 4.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 read_transposed(const unsigned char *lo, const unsigned char *hi) {
  typedef __attribute__((address_space(3))) s16x4 *Lds;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (Lds)(uintptr_t)(__attribute__((address_space(3))) void *)lo);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (Lds)(uintptr_t)(__attribute__((address_space(3))) void *)hi);
  return __builtin_bit_cast(f32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
// 0 for the inactive among a lane's tokens of step ks.
__device__ __forceinline__ void drop_inactive(uint64_t act, int ks, int g, f32x4 (&b)[2]) {
  const uint32_t on = (uint32_t)(act >> (32 * ks)) >> (4 * g);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    b[0][e] = (on >> e) & 1u ? b[0][e] : 0.0f;
    b[1][e] = (on >> (16 + e)) & 1u ? b[1][e] : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ Stored<T> keys_by_feature(Rsrc m, int L, int t0, int f0, uint64_t act,
                                                     const unsigned char *blocks, int i, int ks,
                                                     int lane) {
  Stored<T> s;
  const int g = lane >> 4, c = lane & 15;
  if constexpr (sizeof(T) == 4) {
    const int off = (c * L + 4 * g) * 4 + ((f0 + 16 * i) * L + t0 + 32 * ks) * 4;
    s.b[0] = buffer_load4(m, off, 0);
    s.b[1] = buffer_load4(m, off + 64, 0);
    drop_inactive(act, ks, g, s.b);
  } else {
    const unsigned char *at = blocks + 1024 * (4 * ks + (i >> 1)) +
                              16 * (16 * (c & 3) + 4 * g + (c >> 2)) + 8 * (i & 1);
    s.b[0] = read_transposed(at, at + 2048);
  }
  return s;
}

// Barrier for LDS only: outstanding global loads and stores stay outstanding.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Six operand blocks of a lower triangular 64 x 64 matrix (row tile tt, step ks):
// the steps past the diagonal hold nothing.
constexpr int kTri = kLinearTriBytes;
__device__ __forceinline__ int tri_block(int tt, int ks) { return tt < 2 ? tt : 2 * tt - 2 + ks; }

// ------------------------------------------------------------------ pairs

// Workgroup = one chunk of one (row, head), four waves. Wave w forms the scores
// of token tile w against the tiles up to it, transposed, which is the order the
// walk reads them in; with the delta rule also K K^T the same way and (I + M)^-1
// by 16 x 16 blocks: the diagonal blocks by substitution (one wave each), the others
// by T_ij = -T_ii sum_(j <= k < i) M_ik T_kj on the f32 matrix cores, one distance
// i - j after the other. The first head of a key head's group also leaves the
// keys and queries behind in fragment order, the keys both ways: the walk's column
// groups then each read whole lines with few loads. This kernel and the walk take 15 + 95
// us for 8 x 1024 tokens with 8 heads of 256 x 256 in bf16, 89 + 342 for 2 x 8192 with 16
// heads of 128 x 128; the walks before them, on which the order was decided, 20 + 94 and 109
// + 424 with it, 14 + 222 and 62 + 586 from the original order, where a wave's token tile is
// 32 or 64 bytes of a feature row.
// All loads are issued before anything waits for the first of them.
template <typename T, bool DELTA, bool FEATURES>
__global__ __launch_bounds__(256) void linear_pairs_kernel(LinearArgs a, LinearWork ws) {
  constexpr int NP = Pieces<T>::n;
  constexpr int kS = 68;  // floats per row: 16-byte rows, rows 4 banks apart
  constexpr int kOperands = 16 * NP * 1024, kMatrices = DELTA ? 2 * kC * kS * 4 : 0;
  __shared__ __attribute__((aligned(16))) unsigned char
      smem[kOperands > kMatrices ? kOperands : kMatrices];
  __shared__ ChunkScan sc;
  unsigned char *qpl = smem, *kpl = smem + 8 * NP * 1024;
  const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = blockIdx.x, h = blockIdx.y, r = blockIdx.z, nch = gridDim.x;
  const size_t rh = (size_t)r * a.heads + h, at = rh * nch + chunk;
  const int t0 = chunk * kC, n = min(kC, a.L - t0);
  const int steps = linear_steps(a.dk), parts = 1 + DELTA + FEATURES;
  const size_t kh = (size_t)r * a.key_heads + h / a.group;
  const uint32_t bytes = (uint32_t)a.dk * a.L * sizeof(T);
  const Rsrc q = buffer_rsrc(static_cast<const T *>(a.q) + kh * a.dk * a.L, bytes);
  const Rsrc k = buffer_rsrc(static_cast<const T *>(a.k) + kh * a.dk * a.L, bytes);
  const int t = min(t0 + lane, a.L - 1);
  float mask = 1.0f, log_decay = 0.0f, beta = 0.0f;
  if (a.mask) mask = a.mask[(size_t)r * a.L + t];
  if (wave == 0) {
    log_decay = a.log_decay[rh * a.L + t];
    if (DELTA) beta = a.beta[rh * a.L + t];
  }
  Raw x[2][2], y[2][2];  // two slabs of 64 features
  auto fetch = [&](int f0, Raw (&x)[2], Raw (&y)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load_octet<T>(q, a.L, t0, f0, wave + 4 * i, lane, x[i]);
      load_octet<T>(k, a.L, t0, f0, wave + 4 * i, lane, y[i]);
    }
  };
  fetch(0, x[0], y[0]);
  if (a.dk > 64) fetch(64, x[1], y[1]);
  const uint64_t act = __ballot(lane < n && mask != 0.0f);
  if (h == 0 && threadIdx.x == 0) ws.active[(size_t)r * nch + chunk] = act;
  if (act == 0) {
    for (int j = wave; j < a.dv; j += 4)
      if (lane < n) a.out[(rh * a.dv + j) * a.L + t0 + lane] = 0.0f;
    return;
  }
  if (wave == 0) {
    scan_chunk(log_decay, beta, act, lane, sc);
    float *v = ws.factors + at * 3 * kC;
    v[lane] = sc.from_start[lane];
    v[kC + lane] = sc.to_end[lane];
    v[2 * kC + lane] = sc.beta[lane];
  }
  const bool first = h % a.group == 0;
  constexpr int SB = Pieces<T>::blocks * 1024;
  const size_t part = (size_t)4 * steps * SB;
  unsigned char *pq = ws.packed + (kh * nch + chunk) * parts * part;
  unsigned char *pk = pq + part, *pt = pq + (1 + DELTA) * part;
  f32x4 score[4] = {}, keys[4] = {};
  auto slab = [&](int f0, Raw (&x)[2], Raw (&y)[2]) {
    if (f0) lds_barrier();
    const bool on = (act >> lane) & 1u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int o = wave + 4 * i, whole = 4 * (f0 / 32) + o;  // octet of all features
      const bool keep = first && whole < 4 * steps;
      frag p[NP];
      const Stored<T> qs = stored<T>(x[i], on);
      to_frag<T>(qs, p);
      store_frag<NP>(qpl + octet_block(NP * 1024, 2, o, lane), octet_slot(o, lane), p);
      if (keep) store_stored<T>(pq + octet_block(SB, steps, whole, lane), octet_slot(o, lane), qs);
      const Stored<T> ks = stored<T>(y[i], on);
      to_frag<T>(ks, p);
      store_frag<NP>(kpl + octet_block(NP * 1024, 2, o, lane), octet_slot(o, lane), p);
      if (DELTA && keep)
        store_stored<T>(pk + octet_block(SB, steps, whole, lane), octet_slot(o, lane), ks);
    }
    lds_barrier();
    const int tile = f0 / 16 + wave;
    if (FEATURES && first && tile < 2 * steps)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        store_stored<T>(pt + SB * (2 * tile + b), lane,
                        keys_by_feature<T>(k, a.L, t0, f0, act, kpl, wave, b, lane));
    if (f0 + 128 < 32 * steps) fetch(f0 + 128, x, y);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      if (f0 + 32 * kk >= a.dk) continue;
      frag qf[NP], kf[NP];
      load_frag<NP>(qpl + 1024 * NP * (2 * wave + kk), lane, qf);
      if (DELTA) load_frag<NP>(kpl + 1024 * NP * (2 * wave + kk), lane, kf);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (st > wave) continue;
        frag s[NP];
        load_frag<NP>(kpl + 1024 * NP * (2 * st + kk), lane, s);
        score[st] = mma<NP, NP>(s, qf, score[st]);
        if (DELTA) keys[st] = mma<NP, NP>(s, kf, keys[st]);
      }
    }
  };
  for (int f0 = 0; f0 < 32 * steps; f0 += 128) {
    slab(f0, x[0], y[0]);
    if (f0 + 64 < 32 * steps) slab(f0 + 64, x[1], y[1]);
  }
  lds_barrier();  // the decays are there, the operands read
  unsigned char *planes = ws.planes + at * (DELTA ? 2 * kTri : kTri);
  float *M = reinterpret_cast<float *>(smem), *X = M + kC * kS;
  {  // lane = token 16 wave + c16, its partners 16 st + 4 g + e
    const int t = 16 * wave + c16;
    const double cum_t = sc.cum[t];
    const int forget_t = sc.forget[t];
    const float beta_t = sc.beta[t];
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      double cum_s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) cum_s[e] = sc.cum[16 * st + 4 * g + e];
      f32x4 m;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int s = 16 * st + 4 * g + e;
        const float d = forget_t > s || s > t ? 0.0f : fast_exp2((float)(cum_t - cum_s[e]));
        // Not 0 times a score past the diagonal, which may not be finite.
        score[st][e] = s <= t ? score[st][e] * d : 0.0f;
        m[e] = s < t ? beta_t * d * keys[st][e] : 0.0f;
      }
      if constexpr (DELTA) {
        *reinterpret_cast<f32x4 *>(M + t * kS + 16 * st + 4 * g) = m;
        *reinterpret_cast<f32x4 *>(X + t * kS + 16 * st + 4 * g) = f32x4{};
      }
    }
  }
  if constexpr (DELTA) lds_barrier();
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    if (ks && wave < 2) continue;
    frag p[3];
    split8(score[2 * ks], score[2 * ks + 1], p);
    store_frag<3>(planes + kPieces * tri_block(wave, ks), lane, p);
  }
  if constexpr (DELTA) {
    {  // diagonal block: lane c16 holds that column of the inverse
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
      lds_barrier();
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
    lds_barrier();
    for (int b = wave; b < 6; b += 4) {
      const int tt = b < 2 ? b : 2 + ((b - 2) >> 1), ks = b < 2 ? 0 : (b - 2) & 1;
      const float *x = X + (16 * tt + c16) * kS + 32 * ks + 4 * g;
      frag p[3];
      split8(*reinterpret_cast<const f32x4 *>(x), *reinterpret_cast<const f32x4 *>(x + 16), p);
      store_frag<3>(planes + kTri + kPieces * b, lane, p);
    }
  }
}

// ------------------------------------------------------------------ the walk

// f32 keys of up to 128 features are read by features where they are, whole lines of
// 32 tokens each (16 rows of 1024 tokens, 16 heads of 128 x 128: 404 us, packed 438; 8 x
// 2048 with 16 heads of 64 x 64: 235, 256; plain 2 x 8192: 449, 477; only the delta rule
// on a small grid, 3 x 777 with 6 heads of 96 x 80, prefers packed ones, 56 against 59).
// Keys of more features take packed ones (4 x 1024 with 8 heads of 256 x 256 on 2 key
// heads: 169, in place 179).
template <typename T>
constexpr bool keys_packed(int NI) {
  return linear_keys_packed(sizeof(T) == 2, NI / 2);
}

// A row's chunks with an active token, 64 at a time.
struct Chunk {
  int at;  // -1: none
  uint64_t act;
};
struct ActiveChunks {
  const uint64_t *active;
  int nch, lane, base = -64;
  uint64_t word = 0, live = 0;
  __device__ __forceinline__ ActiveChunks(const uint64_t *active, int nch, int lane)
      : active(active), nch(nch), lane(lane) {}
  __device__ __forceinline__ Chunk next() {
    while (!live) {
      base += 64;
      if (base >= nch) return Chunk{-1, 0};
      word = base + lane < nch ? active[base + lane] : 0;
      live = __ballot(word != 0);
    }
    const int b = __ffsll((unsigned long long)live) - 1;
    live &= live - 1;
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)word, b);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(word >> 32), b);
    return Chunk{base + b, (uint64_t)hi << 32 | lo};
  }
};

// Half of a fragment block: quad x of the lanes as pieces, half `half` of the block.
__device__ __forceinline__ void put_half(unsigned char *block, int lane, int half, f32x4 x) {
  const Bf16x3 p = split_bf16x3(x);
#pragma unroll
  for (int i = 0; i < 3; ++i)
    *reinterpret_cast<u32x2 *>(block + 1024 * i + 16 * lane + 8 * half) = p.p[i];
}

// A wave of a workgroup on CT tiles of 16 value columns of one (row, head), its token
// tile w of the chunks' operands and outputs.
template <typename T, bool DELTA, int NI, int CT>
struct Walk {
  static constexpr int NP = Pieces<T>::n, NK = NI / 2, SB = Pieces<T>::blocks * 1024;
  static constexpr int kPart = 4 * NK * SB, kParts = 1 + DELTA + keys_packed<T>(NI);
  static constexpr int kPlanes = DELTA ? 2 * kTri : kTri;
  enum { kQueries, kKeys, kByFeature = 1 + DELTA };  // parts of `packed`
  enum { kScores, kSolve };              // of `planes`
  typedef unsigned char State[NK * kPieces], Tokens[2 * kPieces];  // LDS, a column tile's

  int lane, g, c16, wave, w, nch, L;
  int r, h, j;  // row, head, first value column
  size_t rh, kh;
  const unsigned char *packed, *planes;
  const float *factors;  // the lane's four tokens'
  int row_off;           // elements: the lane's column and first token
  uint32_t mine;         // of the columns
  size_t col0;

  __device__ __forceinline__ Walk(const LinearArgs &a, const LinearWork &ws) {
    lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
    L = a.L, nch = (L + kC - 1) / kC;
    // Column groups of a (row, head) go to one XCD (workgroups are dealt to the eight
    // in turn) and share its L2.
    const unsigned groups = ((a.dv + 15) / 16 + CT - 1) / CT, heads = (unsigned)(a.rows * a.heads);
    const unsigned set = blockIdx.x / (8 * groups), in = blockIdx.x - set * 8 * groups;
    const unsigned width = min(8u, heads - 8 * set), cols = in / width;
    rh = 8 * set + (in - cols * width);
    r = (int)(rh / a.heads), h = (int)(rh - (size_t)r * a.heads), j = (int)(16 * CT * cols);
    kh = (size_t)r * a.key_heads + h / a.group;
    packed = ws.packed + kh * nch * ((size_t)kParts * kPart);
    planes = ws.planes + rh * nch * kPlanes;
    factors = ws.factors + rh * nch * 3 * kC + 16 * w + 4 * g;
    row_off = c16 * L + 16 * w + 4 * g;
    mine = (uint32_t)min(16 * CT, a.dv - j) * L;
    col0 = (rh * a.dv + j) * L;
  }
  __device__ __forceinline__ ActiveChunks chunks(const LinearWork &ws) const {
    return ActiveChunks(ws.active + (size_t)r * nch, nch, lane);
  }
  __device__ __forceinline__ Rsrc values(const LinearArgs &a) const {
    return buffer_rsrc(static_cast<const T *>(a.v) + col0, mine * sizeof(T));
  }
  __device__ __forceinline__ Rsrc outputs(const LinearArgs &a) const {
    return buffer_rsrc(a.out + col0, mine * 4);
  }
  __device__ __forceinline__ void fetch_rows(int at, int part, Stored<T> (&rows)[NK]) const {
    const unsigned char *p = packed + (size_t)at * (kParts * kPart) + part * kPart + SB * NK * w;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) load_stored<T>(p + SB * kk, lane, rows[kk]);
  }
  __device__ __forceinline__ void fetch_tri(int at, int which, frag (&f)[2][3]) const {
    const unsigned char *p = planes + (size_t)at * kPlanes + which * kTri;
    frag first[3];  // stored behind the branch, which would else wait for it
    load_frag<3>(p + kPieces * tri_block(w, 0), lane, first);
    if (w >= 2) load_frag<3>(p + kPieces * tri_block(w, 1), lane, f[1]);
#pragma unroll
    for (int i = 0; i < 3; ++i) f[0][i] = first[i];
  }
  // Factor 0: from the chunk's start, 1: to its end, 2: beta.
  __device__ __forceinline__ f32x4 factor(int at, int which) const {
    return *reinterpret_cast<const f32x4 *>(factors + (size_t)at * 3 * kC + which * kC);
  }
  __device__ __forceinline__ void fetch_values(Rsrc v, int at, bool on, Four<T> (&x)[CT]) const {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      load_four<T>(v, on ? (row_off + at * kC + 16 * ct * L) * (int)sizeof(T) : kNowhere, x[ct]);
  }
  // The values of the lane's active tokens.
  __device__ __forceinline__ f32x4 active_values(const Four<T> &x, uint64_t act) const {
    const unsigned on = (unsigned)(act >> (16 * w + 4 * g));
    f32x4 v = values_of<T>(x);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (on >> e) & 1u ? v[e] : 0.0f;
    return v;
  }
  __device__ __forceinline__ void put_tokens(Tokens *to, int ct, f32x4 x) const {
    put_half(to[ct] + kPieces * (w >> 1), lane, w & 1, x);
  }
  // rows S0, the steps in XA accumulators.
  __device__ __forceinline__ void times_state(const Stored<T> (&rows)[NK], const State *spl,
                                              f32x4 (&Y)[CT]) const {
    constexpr int XA = CT == 1 && NK >= 4 ? 4 : (NK >= 2 ? 2 : 1);
    f32x4 X[XA][CT] = {};
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      frag s[CT][3], f[NP];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) load_frag<3>(spl[ct] + kPieces * kk, lane, s[ct]);
      to_frag<T>(rows[kk], f);
      typedef Products<NP, 3> P;
#pragma unroll
      for (int p = 0; p < P::n; ++p)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          X[kk % XA][ct] = mfma_16x16x32_bf16(f[P::a(p)], s[ct][P::b(p)], X[kk % XA][ct]);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      Y[ct] = X[0][ct];
#pragma unroll
      for (int i = 1; i < XA; ++i) Y[ct] += X[i][ct];
    }
  }
  // U += tri x, x of NB pieces in LDS; with one column tile each step in accumulators of
  // its own.
  template <int NB>
  __device__ __forceinline__ void add_tri(const frag (&tri)[2][3], const unsigned char *from,
                                          int stride, f32x4 (&U)[CT]) const {
    f32x4 A[CT] = {};
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks && w < 2) continue;
      frag x[CT][NB];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        load_frag<NB>(from + ct * stride + 1024 * NB * ks, lane, x[ct]);
      typedef Products<3, NB> P;
#pragma unroll
      for (int p = 0; p < P::n; ++p)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          f32x4 &to = ks && CT == 1 ? A[ct] : U[ct];
          to = mfma_16x16x32_bf16(tri[ks][P::a(p)], x[ct][P::b(p)], to);
        }
    }
    if constexpr (CT == 1) U[0] += A[0];
  }
  // 0 for inactive tokens, whose queries are 0, but 0 times a state that is not finite is not.
  __device__ __forceinline__ void store(Rsrc out, const Chunk &c, float scale,
                                        const f32x4 (&O)[CT]) const {
    const int t0 = c.at * kC, n = L - t0 - 16 * w - 4 * g;
    const unsigned on = (unsigned)(c.act >> (16 * w + 4 * g));
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int off = (row_off + t0 + 16 * ct * L) * 4;
      f32x4 y = O[ct] * scale;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (on >> e) & 1u ? y[e] : 0.0f;
      if (t0 + kC <= L) {
        buffer_store4(y, out, off, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) buffer_store1(y[e], out, e < n ? off + 4 * e : kNowhere, 0);
      }
    }
  }
};

// A wave's feature tiles tile0 .. tile0 + TI - 1 of the state (feature 16 i + 4 (lane / 16)
// + e, column lane % 16, in accumulators), with what the next chunk multiplies in.
template <typename T, bool DELTA, int NI, int CT, int WAVES>
struct StateTiles {
  typedef Walk<T, DELTA, NI, CT> W;
  static constexpr int TI = NI >= WAVES ? NI / WAVES : 1, NP = W::NP;
  static constexpr bool kKeysPacked = keys_packed<T>(NI);
  f32x4 S[CT][TI];
  Stored<T> t[TI][2];
  float whole;
  int tile0, voff[CT], step;
  Rsrc keys;
  uint32_t bytes;

  __device__ __forceinline__ bool owner() const { return NI >= WAVES || tile0 < NI; }
  __device__ __forceinline__ StateTiles(const W &k, const LinearArgs &a) {
    tile0 = TI * k.wave, step = a.dv * 4;
    keys = buffer_rsrc(static_cast<const T *>(a.k) + k.kh * a.dk * a.L,
                       (uint32_t)a.dk * a.L * sizeof(T));
    bytes = (uint32_t)a.dk * a.dv * 4;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int j = k.j + 16 * ct + k.c16;
      voff[ct] = j < a.dv ? ((16 * tile0 + 4 * k.g) * a.dv + j) * 4 : kNowhere;
#pragma unroll
      for (int i = 0; i < TI; ++i) S[ct][i] = f32x4{};
    }
    if (!a.state_in || !owner()) return;
    const Rsrc from = buffer_rsrc(a.state_in + k.rh * a.dk * a.dv, bytes);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          S[ct][i][e] = buffer_load1(from, voff[ct] + (16 * i + e) * step, 0);
  }
  __device__ __forceinline__ void store(const W &k, const LinearArgs &a) const {
    if (!a.state_out || !owner()) return;
    const Rsrc to = buffer_rsrc(a.state_out + k.rh * a.dk * a.dv, bytes);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          buffer_store1(S[ct][i][e], to, voff[ct] + (16 * i + e) * step, 0);
  }
  __device__ __forceinline__ void fetch(const W &k, const LinearWork &ws, int at) {
    whole = ws.factors[(k.rh * k.nch + at) * 3 * kC + kC - 1];
    if (!owner()) return;
    const unsigned char *p = k.packed + (size_t)at * (W::kParts * W::kPart) +
                             W::kByFeature * W::kPart + 2 * W::SB * tile0;
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if constexpr (kKeysPacked) {
          load_stored<T>(p + W::SB * (2 * i + ks), k.lane, t[i][ks]);
        } else {
          const int off = ((16 * (tile0 + i) + k.c16) * k.L + at * kC + 32 * ks + 4 * k.g) * 4;
          t[i][ks].b[0] = buffer_load4(keys, off, 0);
          t[i][ks].b[1] = buffer_load4(keys, off + 64, 0);
        }
      }
  }
  // S <- e^G S + K^T (e U), e U in LDS; with one column tile the steps in accumulators
  // of their own. `taken` runs when the keys have been split.
  template <typename F>
  __device__ __forceinline__ void update(const W &k, const typename W::Tokens *epl, uint64_t act,
                                         F taken) {
    frag tf[TI][2][NP];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if constexpr (!kKeysPacked) drop_inactive(act, ks, k.g, t[i][ks].b);
        to_frag<T>(t[i][ks], tf[i][ks]);
      }
    const float decay = whole;
    taken();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      frag e[2][3];
      load_frag<3>(epl[ct], k.lane, e[0]);
      load_frag<3>(epl[ct] + kPieces, k.lane, e[1]);
      f32x4 D[TI] = {};
#pragma unroll
      for (int i = 0; i < TI; ++i) S[ct][i] *= decay;
      typedef Products<NP, 3> P;
#pragma unroll
      for (int p = 0; p < P::n; ++p)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int i = 0; i < TI; ++i) {
            f32x4 &to = ks && CT == 1 ? D[i] : S[ct][i];
            to = mfma_16x16x32_bf16(tf[i][ks][P::a(p)], e[ks][P::b(p)], to);
          }
      if constexpr (CT == 1)
#pragma unroll
        for (int i = 0; i < TI; ++i) S[ct][i] += D[i];
    }
  }
  __device__ __forceinline__ void put(const W &k, typename W::State *spl) const {
    if (!owner()) return;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < TI; ++i)
        put_half(spl[ct] + kPieces * ((tile0 + i) >> 1), k.lane, (tile0 + i) & 1, S[ct][i]);
  }
};

// In all of the kernels below, operands are fetched for the next chunk as soon as the
// present one has been multiplied, each line by one wave, straight into registers.
// Behind the last chunk its operands come again, for nothing: a branch around the loads
// makes the compiler wait for them at its end.

// The delta rule with the work of a chunk, which is what every later chunk waits for,
// shared by four waves: wave w has token tile w of U and O, and the feature tiles TI w ..
// of the state. Three times a chunk they hand their part to the others as operand
// pieces in LDS: the state for K S0 and Q S0, V - d K S0 for U, U for O and the state.
// Two or more workgroups a CU hide each other's exchanges; then the operands bound it (16
// rows of 512 tokens with 16 heads of 128 x 128 in bf16: the workgroups load 744 MB, most of
// it out of L2, in 114 us, 6.5 TB/s).
// On eight waves the first four are on the path from one state to the next (K S0, V - d
// K S0 and U), the others beside it (Q S0 and O, which nothing waits for), and the
// state's tiles are dealt to all eight. `path` and `side` are both true on four.
template <typename T, int NI, int CT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || (NI <= 8 && CT < 4) ? 2 : 1)
void linear_delta_kernel(LinearArgs a, LinearWork ws) {
  typedef Walk<T, true, NI, CT> W;
  constexpr bool kRoles = WAVES == 8;
  constexpr int NP = W::NP, NK = W::NK;
  __shared__ __attribute__((aligned(16))) typename W::State spl[CT];
  __shared__ __attribute__((aligned(16))) typename W::Tokens xpl[CT], upl[CT], epl[CT];
  const W k(a, ws);
  const bool path = !kRoles || k.wave < 4, side = !kRoles || k.wave >= 4;
  const Rsrc v = k.values(a), out = k.outputs(a);
  StateTiles<T, true, NI, CT, WAVES> state(k, a);
  ActiveChunks chunks = k.chunks(ws);
  Chunk cur = chunks.next(), next = chunks.next();
  // With roles `rows` and `tri` are keys and the solve operand, or queries and scores.
  Stored<T> rows[NK], krows[kRoles ? 1 : NK];
  frag tri[2][3], solve[2][3];
  f32x4 start, end, beta;
  Four<T> values[CT];
  auto fetch_rows = [&](int at) {
    k.fetch_rows(at, kRoles && path ? W::kKeys : W::kQueries, rows);
    if constexpr (!kRoles) k.fetch_rows(at, W::kKeys, krows);
  };
  auto fetch_tri = [&](int at) { k.fetch_tri(at, kRoles && path ? W::kSolve : W::kScores, tri); };
  auto fetch_values = [&](int at) {
    start = k.factor(at, 0), end = k.factor(at, 1), beta = k.factor(at, 2);
    k.fetch_values(v, at, path, values);
  };
  if (cur.at >= 0) {
    fetch_rows(cur.at);
    fetch_values(cur.at);
    if (!kRoles) k.fetch_tri(cur.at, W::kSolve, solve);
    fetch_tri(cur.at);
    state.fetch(k, ws, cur.at);
  }
  state.put(k, spl);
  lds_barrier();
  while (cur.at >= 0) {
    const int far = next.at >= 0 ? next.at : cur.at;
    f32x4 X[2][CT] = {}, O[2][CT] = {};  // K S0 and Q S0, even and odd steps
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      frag s[CT][3], f[NP], fk[NP];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) load_frag<3>(spl[ct] + kPieces * kk, k.lane, s[ct]);
      to_frag<T>(rows[kk], f);
      if constexpr (!kRoles) to_frag<T>(krows[kk], fk);
      typedef Products<NP, 3> P;
#pragma unroll
      for (int p = 0; p < P::n; ++p)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          if constexpr (!kRoles)
            X[kk & 1][ct] = mfma_16x16x32_bf16(fk[P::a(p)], s[ct][P::b(p)], X[kk & 1][ct]);
          O[kk & 1][ct] = mfma_16x16x32_bf16(f[P::a(p)], s[ct][P::b(p)], O[kk & 1][ct]);
        }
    }
    fetch_rows(far);
    f32x4 U[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      O[0][ct] = start * (O[0][ct] + O[1][ct]);
      const f32x4 x = kRoles ? O[0][ct] : start * (X[0][ct] + X[1][ct]);
      if (path) k.put_tokens(xpl, ct, beta * (k.active_values(values[ct], cur.act) - x));
      U[ct] = f32x4{};
    }
    lds_barrier();
    if (path) k.template add_tri<3>(kRoles ? tri : solve, xpl[0], sizeof(xpl[0]), U);
    if constexpr (!kRoles) k.fetch_tri(far, W::kSolve, solve);
    if (path)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        k.put_tokens(upl, ct, U[ct]);
        k.put_tokens(epl, ct, U[ct] * end);
      }
    lds_barrier();
    fetch_values(far);
    // The state first: the next chunk waits for it.
    state.update(k, epl, cur.act, [] {});
    __builtin_amdgcn_sched_barrier(0);  // the loads find the keys' registers free
    state.fetch(k, ws, far);
    if (kRoles) {  // only the side waits for what comes next
      state.put(k, spl);
      lds_barrier();
    }
    if (side) k.template add_tri<3>(tri, upl[0], sizeof(upl[0]), O[0]);
    if (!kRoles) state.put(k, spl);
    fetch_tri(far);
    if (side) k.store(out, cur, a.scale, O[0]);
    if (!kRoles) lds_barrier();
    cur = next;
    next = chunks.next();
  }
  state.store(k, a);
}

// The delta rule with every wave at one kind of work, for grids that leave a CU to one
// workgroup: waves 0 to 3 are on the path from one state to the next (token tile w of
// K S0, of V - d K S0 and of U, feature tiles TI w .. of the state), waves 4 to 7 are a
// chunk behind them with token tile w of Q S0 and O, between the barriers of the path.
// The state and U are in two buffers for that. Sums on the path run in several
// accumulators, whose latency nothing else hides.
// Bound by the path: 4700 cycles a chunk in bf16 with 128 x 128 and one tile, of which
// the products are 580. Against four waves that do both, two chunks ahead (us): bf16, 16
// heads of 128 x 128, 2 x 8192 tokens 404 and 417, 1 x 4096 158 and 165; f32 4 x 512 on two
// tiles 58 and 73.
template <typename T, int NI, int CT>
__global__ __launch_bounds__(512, 2) void linear_delta_path_kernel(LinearArgs a, LinearWork ws) {
  typedef Walk<T, true, NI, CT> W;
  __shared__ __attribute__((aligned(16))) typename W::State spl[2][CT];
  __shared__ __attribute__((aligned(16))) typename W::Tokens xpl[CT], epl[CT], upl[2][CT];
  const W k(a, ws);
  ActiveChunks chunks = k.chunks(ws);
  Chunk cur = chunks.next(), next = chunks.next();
  int ahead = next.at >= 0 ? next.at : cur.at;
  auto advance = [&] {
    cur = next;
    next = chunks.next();
    if (next.at >= 0) ahead = next.at;
  };
  Stored<T> rows[W::NK];
  frag tri[2][3];
  f32x4 start;
  if (k.wave < 4) {
    const Rsrc v = k.values(a);
    StateTiles<T, true, NI, CT, 4> state(k, a);
    Four<T> values[CT];
    f32x4 end, beta;
    auto fetch_values = [&](int at) {
      start = k.factor(at, 0), beta = k.factor(at, 2);
      k.fetch_values(v, at, true, values);
    };
    if (cur.at >= 0) {
      k.fetch_rows(cur.at, W::kKeys, rows);
      fetch_values(cur.at);
      k.fetch_tri(cur.at, W::kSolve, tri);
      end = k.factor(cur.at, 1);
      state.fetch(k, ws, cur.at);
    }
    state.put(k, spl[0]);
    lds_barrier();
    for (int b = 0; cur.at >= 0; b ^= 1) {
      f32x4 X[CT], U[CT] = {};
      k.times_state(rows, spl[b], X);
      k.fetch_rows(ahead, W::kKeys, rows);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        k.put_tokens(xpl, ct, beta * (k.active_values(values[ct], cur.act) - start * X[ct]));
      lds_barrier();
      fetch_values(ahead);
      k.template add_tri<3>(tri, xpl[0], sizeof(xpl[0]), U);
      k.fetch_tri(ahead, W::kSolve, tri);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        k.put_tokens(epl, ct, U[ct] * end);
        k.put_tokens(upl[b], ct, U[ct]);
      }
      lds_barrier();
      end = k.factor(ahead, 1);
      state.update(k, epl, cur.act, [] {});
      __builtin_amdgcn_sched_barrier(0);  // the loads find the keys' registers free
      state.fetch(k, ws, ahead);
      state.put(k, spl[b ^ 1]);
      lds_barrier();
      advance();
    }
    state.store(k, a);
  } else {
    const Rsrc out = k.outputs(a);
    // A chunk's outputs, between the barriers of the next one.
    auto outputs = [&](int b, auto between) {
      f32x4 O[CT];
      k.times_state(rows, spl[b], O);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) O[ct] = start * O[ct];
      k.fetch_rows(ahead, W::kQueries, rows);
      start = k.factor(ahead, 0);
      between();
      k.template add_tri<3>(tri, upl[b][0], sizeof(upl[b][0]), O);
      k.fetch_tri(ahead, W::kScores, tri);
      between();
      k.store(out, cur, a.scale, O);
      between();
      advance();
    };
    if (cur.at >= 0) {
      k.fetch_rows(cur.at, W::kQueries, rows);
      start = k.factor(cur.at, 0);
      k.fetch_tri(cur.at, W::kScores, tri);
    }
    lds_barrier();
    if (cur.at < 0) return;
    for (int i = 0; i < 3; ++i) lds_barrier();  // the first chunk's
    int b = 0;
    for (; next.at >= 0; b ^= 1) outputs(b, [] { lds_barrier(); });
    outputs(b, [] {});
  }
}

// Without the delta rule the state needs no product with itself: S <- e^G S + K^T (e U)
// with U = V is a chain of products in the accumulators, and only Q S0 reads it from LDS.
// Workgroup = eight waves on CT column tiles, one barrier a chunk, what they hand over
// in two buffers. Waves 0 to 3 have the feature tiles TI w .. of the state, and put it and
// token tile w of U and e U of the next chunk into LDS; waves 4 to 7 have token tile w
// of Q S0 and of O. (On four waves that did both, with two barriers: 3 x 777 tokens with 6
// heads of 96 x 80 48 us, now 38; 2 x 8192 with 16 heads of 128 x 128 442, now 400, in bf16
// 307, now 269; 8 x 1024 with 8 heads of 256 x 256 231, now 194.)
// Bound by the operands' way through L2 and LDS: 2 x 8192 in bf16 move 540 MB in and
// out of both kernels, 2 TB/s.
template <typename T, int NI, int CT>
__global__ __launch_bounds__(512, 2) void linear_plain_kernel(LinearArgs a, LinearWork ws) {
  typedef Walk<T, false, NI, CT> W;
  constexpr int NP = W::NP;
  __shared__ __attribute__((aligned(16))) typename W::State spl[2][CT];
  __shared__ __attribute__((aligned(16))) unsigned char upl[2][CT][2 * NP * 1024];
  __shared__ __attribute__((aligned(16))) typename W::Tokens epl[2][CT];
  const W k(a, ws);
  ActiveChunks chunks = k.chunks(ws);
  Chunk cur = chunks.next(), next = chunks.next();
  int ahead = next.at >= 0 ? next.at : cur.at;
  auto advance = [&] {
    cur = next;
    next = chunks.next();
    if (next.at >= 0) ahead = next.at;
  };
  if (k.wave < 4) {
    const Rsrc v = k.values(a);
    StateTiles<T, false, NI, CT, 4> state(k, a);
    Four<T> values[CT];
    f32x4 end;
    auto fetch_values = [&](int at) {
      end = k.factor(at, 1);
      k.fetch_values(v, at, true, values);
    };
    auto put_values = [&](int b, uint64_t act) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const f32x4 u = k.active_values(values[ct], act);
        unsigned char *p = upl[b][ct] + 1024 * NP * (k.w >> 1);
        if constexpr (NP == 3)
          put_half(p, k.lane, k.w & 1, u);
        else  // exact: the values are bf16
          *reinterpret_cast<u32x2 *>(p + 16 * k.lane + 8 * (k.w & 1)) =
              __builtin_bit_cast(u32x2, __builtin_convertvector(u, bf16x4));
        k.put_tokens(epl[b], ct, u * end);
      }
    };
    if (cur.at >= 0) {
      fetch_values(cur.at);
      state.fetch(k, ws, cur.at);
      put_values(0, cur.act);
      fetch_values(ahead);
    }
    state.put(k, spl[0]);
    lds_barrier();
    for (int b = 0; cur.at >= 0; b ^= 1) {
      state.update(k, epl[b], cur.act, [&] { state.fetch(k, ws, ahead); });
      put_values(b ^ 1, next.act);
      advance();
      fetch_values(ahead);
      state.put(k, spl[b ^ 1]);
      lds_barrier();
    }
    state.store(k, a);
  } else {
    const Rsrc out = k.outputs(a);
    Stored<T> rows[W::NK];
    frag scores[2][3];
    f32x4 start;
    if (cur.at >= 0) {
      k.fetch_rows(cur.at, W::kQueries, rows);
      start = k.factor(cur.at, 0);
      k.fetch_tri(cur.at, W::kScores, scores);
    }
    lds_barrier();
    for (int b = 0; cur.at >= 0; b ^= 1) {
      f32x4 O[CT];
      k.times_state(rows, spl[b], O);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) O[ct] = start * O[ct];
      k.fetch_rows(ahead, W::kQueries, rows);
      start = k.factor(ahead, 0);
      k.template add_tri<NP>(scores, upl[b][0], sizeof(upl[b][0]), O);
      k.fetch_tri(ahead, W::kScores, scores);
      k.store(out, cur, a.scale, O);
      lds_barrier();
      advance();
    }
  }
}

// Kernel and column tiles per workgroup by how the grid fills the CUs (us for prompts of
// 512 tokens, 16 heads of 128 x 128 unless stated, both kernels). With the delta rule
//   the path kernel with one tile if every workgroup then has a CU to itself (2 x 8192 in
//   bf16: 404, two tiles 511), with two while one tile would put two on a CU (4 rows: 58,
//   one 75, four waves 73) and for bf16 keys over 128 wide (8 x 1024 with 8 heads of 256 x
//   256: 181, four waves 195);
//   beyond that four waves, two or more workgroups a CU: every operand is loaded and
//   split for four tiles at once with f32 keys of 65 to 128, where the splitting weighs
//   most (16 rows: 220, two tiles 343, which spill, the path kernel 238), for two
//   otherwise (16 rows in bf16: 160, four tiles 171, the path kernel 173; 32 rows of 64 x
//   64 f32: 214, 210, 213);
//   f32 keys over 128 wide, whose state is half the work, on eight waves that share it
//   (8 x 1024 with 8 heads of 256 x 256: 279, the path kernel 311; 1 x 4096 306 and 318).
// Without it one tile each if every workgroup has a CU to itself (2 x 8192: 404 us, two
// tiles 448; bf16 275 and 355), else two (4 rows: 43, one 51; 16 rows: 167, 195; 8 x 1024
// with 8 heads of 256 x 256 bf16: 111, 124); two chunks ahead brought nothing.
template <typename T, bool DELTA, int NI>
hipError_t launch(const LinearArgs &a, const LinearWork &ws, hipStream_t stream,
                  const KernelEvents &ev) {
  constexpr bool f32 = sizeof(T) == 4;
  const size_t jtiles = (size_t)((a.dv + 15) / 16), heads = (size_t)a.rows * a.heads;
  auto grid = [&](int tiles) { return dim3((unsigned)(heads * ((jtiles + tiles - 1) / tiles))); };
  const bool few = heads * jtiles <= (size_t)a.cus, some = heads * jtiles <= 2 * (size_t)a.cus;
  const dim3 chunks((unsigned)((a.L + kC - 1) / kC), (unsigned)a.heads, (unsigned)a.rows);
  hipExtLaunchKernelGGL((linear_pairs_kernel<T, DELTA, keys_packed<T>(NI)>), chunks, dim3(256),
                        0, stream, ev.start, nullptr, 0, a, ws);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  auto walk = [&](auto kernel, int waves, int tiles) {
    hipExtLaunchKernelGGL(kernel, grid(tiles), dim3(64 * waves), 0, stream, nullptr, ev.stop, 0, a,
                          ws);
    return hipGetLastError();
  };
  if constexpr (!DELTA) {
    if (few) return walk(linear_plain_kernel<T, NI, 1>, 8, 1);
    return walk(linear_plain_kernel<T, NI, 2>, 8, 2);
  } else if constexpr (f32 && NI > 8) {
    if (few) return walk(linear_delta_kernel<T, NI, 1, 8>, 8, 1);
    return walk(linear_delta_kernel<T, NI, 2, 8>, 8, 2);
  } else {
    if (few) return walk(linear_delta_path_kernel<T, NI, 1>, 8, 1);
    if (some || NI > 8) return walk(linear_delta_path_kernel<T, NI, 2>, 8, 2);
    if constexpr (NI <= 8) {
      constexpr int kTiles = f32 && NI == 8 ? 4 : 2;
      return walk(linear_delta_kernel<T, NI, kTiles, 4>, 4, kTiles);
    }
  }
}

template <typename T, bool DELTA>
hipError_t launch_chunks(const LinearArgs &a, unsigned char *mem, hipStream_t stream,
                         const KernelEvents &ev) {
  const LinearSpace sp = linear_space(a);
  LinearWork ws;
  ws.packed = mem;
  ws.planes = ws.packed + sp.packed;
  ws.factors = reinterpret_cast<float *>(ws.planes + sp.planes);
  ws.active = reinterpret_cast<uint64_t *>(ws.planes + sp.planes + sp.factors);
  if (a.dk <= 32) return launch<T, DELTA, 2>(a, ws, stream, ev);
  if (a.dk <= 64) return launch<T, DELTA, 4>(a, ws, stream, ev);
  if (a.dk <= 128) return launch<T, DELTA, 8>(a, ws, stream, ev);
  return launch<T, DELTA, 16>(a, ws, stream, ev);
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
