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
}  // namespace tfd

namespace {

int check(const char *name, bool good) {
  printf("%s %s\n", good ? "ok  " : "FAIL", name);
  return !good;
}

alignas(16) char g_memory[64];  // operands that are not read

int attend(tfd_ctx *c, size_t length, size_t head_dim, unsigned flags = TFD_DEVICE_PTRS | TFD_ASYNC) {
  const tfd_paged_cache cache = {(uint8_t *)g_memory, (uint8_t *)g_memory, (float *)g_memory,
                                 (float *)g_memory, 1, 64};
  return tfd_jeff_cached_attention_f32(c, 1, length, 1, 1, head_dim, 0, (float *)g_memory, nullptr,
                                       nullptr, nullptr, 0, 0, &cache, (int32_t *)g_memory, 1, nullptr,
                                       nullptr, (float *)g_memory, flags);
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

}  // namespace

int main() {
  int bad = counters();
  return bad;
}
