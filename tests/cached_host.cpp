// Host side of the rotary positions, the cache append and the attention over a cache, on the CPU: the
// C entries of tfd_host.cpp with a HIP runtime and launchers that only record (the device is host
// memory). Each check prints its name; the exit code is the number of those that failed.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "tfd_attention.h"
#include "tfd_internal.hpp"

namespace {
bool g_fill_fails = false, g_capturing = false;
int g_fills = 0, g_attends = 0, g_dirty = 0;
// Launches of turns and appends: their rows, and where their operands are.
struct Launch {
  size_t rows, threads;
  const char *x, *out;
  const int32_t *positions, *table, *lengths, *counts;
};
std::vector<Launch> g_launches;
}  // namespace

extern "C" {
hipError_t hipGetDeviceCount(int *n) { return *n = 1, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "planned"; }
const char *hipGetErrorName(hipError_t) { return "planned"; }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) {
  return *s = reinterpret_cast<hipStream_t>(0x100), hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
  return *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) {
  *p = malloc(n);
  memset(*p, 0xAB, n);  // what was in memory
  return hipSuccess;
}
hipError_t hipFree(void *p) { return free(p), hipSuccess; }
}

namespace tfd {
hipError_t launch_fill_zero(float *out, size_t n, hipStream_t) {
  ++g_fills;
  if (g_fill_fails) return hipErrorLaunchFailure;
  memset(out, 0, n * sizeof(float));
  return hipSuccess;
}
void cached_plan(CachedArgs &a) {
  a.prompt = a.cache.L > 1;
  a.columns = a.prompt ? 128 : 16;
  a.slots = 512;
}
CachedSpace cached_space(const CachedArgs &a) {
  return CachedSpace{2 * kCachedSlots * sizeof(unsigned), (size_t)a.slots * a.columns * 8,
                     (size_t)a.slots * a.columns * a.cache.wide * 4};
}
hipError_t launch_cached_attention(const CachedArgs &a, hipStream_t, const KernelEvents &) {
  ++g_attends;
  for (size_t i = 0; i < 2 * kCachedSlots; ++i) g_dirty += a.part_done[i] != 0;
  return hipSuccess;
}
hipError_t launch_rotary(RotaryArgs a, int rows, hipStream_t, const KernelEvents &) {
  g_launches.push_back({(size_t)rows, rotary_blocks(a) * 256, (const char *)a.x, (const char *)a.out,
                        a.positions, nullptr, nullptr, nullptr});
  return hipSuccess;
}
hipError_t launch_cache_append(const AppendArgs &a, int rows, hipStream_t, const KernelEvents &) {
  g_launches.push_back({(size_t)rows, append_blocks(a) * a.cache.kv_heads * 2 * append_threads(a),
                        (const char *)a.k, (const char *)a.v, nullptr, a.cache.table, a.cache.lengths,
                        a.cache.counts});
  return hipSuccess;
}
}  // namespace tfd

namespace {

int check(const char *name, bool good) {
  printf("%s %s\n", good ? "ok  " : "FAIL", name);
  return !good;
}

alignas(16) char g_memory[64];  // operands that are not read

constexpr unsigned kDevice = TFD_DEVICE_PTRS | TFD_ASYNC;

int attend(tfd_ctx *c, size_t length, size_t head_dim, size_t rows = 1, size_t kv_heads = 1,
           size_t group = 1) {
  const tfd_paged_cache cache = {(uint8_t *)g_memory, (uint8_t *)g_memory, (float *)g_memory,
                                 (float *)g_memory, 1, 64};
  return tfd_jeff_cached_attention_f32(c, rows, length, group * kv_heads, kv_heads, head_dim, 0,
                                       (float *)g_memory, nullptr, nullptr, nullptr, 0, 0, &cache,
                                       (int32_t *)g_memory, 1, nullptr, nullptr, (float *)g_memory,
                                       kDevice);
}

// The counters are zero at every launch, also where the launch that zeroes them failed before.
int counters() {
  int bad = 0;
  tfd_ctx *c = nullptr;
  tfd_ctx_create(0, &c);
  for (size_t length : {1, 2}) {  // the workspace's first size, and a larger one
    const int fills = g_fills, attends = g_attends;
    g_fill_fails = true;
    bad += check("a call whose zeroing fails is refused", attend(c, length, 64) == TFD_EHIP);
    bad += check("and launches nothing", g_attends == attends);
    g_fill_fails = false;
    g_capturing = true;
    bad += check("a capture does not begin on what is not zeroed",
                 attend(c, length, 64) == TFD_EUNSUPPORTED && g_attends == attends);
    g_capturing = false;
    bad += check("the next call runs", attend(c, length, 64) == TFD_OK && g_attends == attends + 1);
    bad += check("on zeroed counters", g_dirty == 0);
    bad += check("zeroed by it", g_fills == fills + 2);
    bad += check("another one does not zero again", attend(c, length, 64) == TFD_OK &&
                                                        g_fills == fills + 2);
    g_capturing = true;
    bad += check("and a capture runs", attend(c, length, 64) == TFD_OK && g_fills == fills + 2);
    g_capturing = false;
  }
  tfd_ctx_destroy(c);
  return bad;
}

// Whether the launches have all rows once and in order, each within a grid, their operands
// `at(row)` as the first one's.
template <typename F>
bool covers(size_t rows, F at) {
  size_t r = 0;
  for (const Launch &l : g_launches) {
    if (l.rows == 0 || l.rows > 65535 || l.rows * l.threads >> 32 || !at(l, r)) return false;
    r += l.rows;
  }
  return r == rows;
}

// Rows that one grid does not hold go in several launches; what no launch holds is refused.
int rows() {
  int bad = 0;
  tfd_ctx *c = nullptr;
  tfd_ctx_create(0, &c);
  char *const x = (char *)((size_t)1 << 44), *const y = (char *)((size_t)1 << 45);  // never read
  int32_t *const p = (int32_t *)((size_t)1 << 43), *const t = p + ((size_t)1 << 32),
                 *const u = p + ((size_t)1 << 33);
  const struct {
    size_t rows, length, heads, hd, launches;
  } turns[] = {{1, 1, 1, 1, 1},          {65535, 1, 8, 256, 1},      {65536, 1, 1, 2, 2},
               {200000, 3, 2, 10, 4},    {70000, 8192, 1, 512, 9},  {1, 1, 70000, 2, 1},
               {3, 1 << 28, 1, 60, 2},   {2, 1 << 28, 1, 125, 2}};
  for (const auto &s : turns)
    for (int bf16 = 0; bf16 < 2; ++bf16)
      for (int with = 0; with < 2; ++with) {
        g_launches.clear();
        const int rc = bf16 ? tfd_rotary_rows_bf16(c, s.rows, s.length, s.heads, s.hd, 0, (uint16_t *)x,
                                                   with ? p : nullptr, nullptr, 0, (uint16_t *)y, kDevice)
                            : tfd_rotary_rows_f32(c, s.rows, s.length, s.heads, s.hd, 0, (float *)x,
                                                  with ? p : nullptr, nullptr, 0, (float *)y, kDevice);
        const size_t row = s.length * s.heads * s.hd * (bf16 ? 2 : 4);
        bad += check("turns: every row once", rc == TFD_OK && covers(s.rows, [&](const Launch &l, size_t r) {
                                                return l.x == x + r * row && l.out == y + r * row &&
                                                       l.positions == (with ? p + r * s.length : nullptr);
                                              }));
        bad += check("turns: launches", bf16 || g_launches.size() == s.launches);
      }
  g_launches.clear();
  bad += check("turns: a row past a grid is refused",
               tfd_rotary_rows_f32(c, 1, 1 << 28, 1, 127, 0, (float *)x, nullptr, nullptr, 0, (float *)y,
                                   kDevice) == TFD_EUNSUPPORTED && g_launches.empty());
  const struct {
    size_t rows, length, heads, hd, launches;
  } appends[] = {{1, 1, 1, 8, 1},       {65535, 1, 17, 8, 1},    {65535, 1, 300, 8, 2},
                 {65535, 130, 8, 256, 1}, {65535, 1000, 8, 256, 5}, {4096, 8192, 8, 64, 2},
                 {9, 1 << 24, 3, 256, 5}};
  for (const auto &s : appends)
    for (int with = 0; with < 2; ++with) {
      g_launches.clear();
      const tfd_paged_cache cache = {(uint8_t *)g_memory, (uint8_t *)g_memory, (float *)g_memory,
                                     (float *)g_memory, 1 << 20, 64};
      const size_t per_row = s.length / 64 + 2, row = s.length * s.heads * s.hd * 2;
      const int rc = tfd_jeff_cache_append_bf16(c, s.rows, s.length, s.heads, s.hd, 0, (uint16_t *)x,
                                                (uint16_t *)y, nullptr, nullptr, 0, 0, &cache, p, per_row,
                                                with ? t : nullptr, with ? u : nullptr, kDevice);
      bad += check("appends: every row once", rc == TFD_OK && covers(s.rows, [&](const Launch &l, size_t r) {
                                                return l.x == x + r * row && l.out == y + r * row &&
                                                       l.table == p + r * per_row &&
                                                       l.lengths == (with ? t + r : nullptr) &&
                                                       l.counts == (with ? u + r : nullptr);
                                              }));
      bad += check("appends: launches", g_launches.size() == s.launches);
    }
  g_launches.clear();
  const tfd_paged_cache one = {(uint8_t *)g_memory, (uint8_t *)g_memory, (float *)g_memory,
                               (float *)g_memory, 1, 64};
  bad += check("appends: a row past a grid is refused",
               tfd_jeff_cache_append_bf16(c, 1, 1 << 24, 8, 256, 0, (uint16_t *)x, (uint16_t *)y, nullptr,
                                          nullptr, 0, 0, &one, p, 1 << 20, nullptr, nullptr,
                                          kDevice) == TFD_EUNSUPPORTED && g_launches.empty());
  // The attention's grid does not go by its rows.
  const int attends = g_attends;
  bad += check("attention: many tiles", attend(c, 1, 8, 65535, 65) == TFD_OK);
  bad += check("attention: many columns", attend(c, 1 << 24, 8, 1, 1, 64) == TFD_OK);
  bad += check("attention: both launched", g_attends == attends + 2);
  bad += check("attention: columns past 32-bit counts", attend(c, 1 << 24, 8, 1, 1, 65) == TFD_EUNSUPPORTED);
  bad += check("attention: tiles past 32-bit counts",
               attend(c, 1, 8, 65535, 16385) == TFD_EUNSUPPORTED && g_attends == attends + 2);
  tfd_ctx_destroy(c);
  return bad;
}

}  // namespace

int main() {
  int bad = counters();
  bad += rows();
  return bad;
}
