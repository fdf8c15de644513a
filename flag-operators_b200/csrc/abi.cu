// Library-wide pieces of the C ABI: error strings, version, device queries.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "common.cuh"

namespace fo {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

void clear_error() { g_err[0] = '\0'; }

int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s: %s", what, cudaGetErrorString(e));
    return FO_ECUDA;
  }
  return FO_OK;
}

int num_sms() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cache[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    cache[dev] = n;
  }
  return cache[dev];
}

cudaError_t allow_shared(const void* kernel, int bytes) {
  // Kernels whose limit is raised already, with the device in the top bits; a full table only costs
  // the call again.
  static std::atomic<uint64_t> done[1024];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t key = (uint64_t)(uintptr_t)kernel ^ (uint64_t)(dev + 1) << 56;
  const unsigned at = (unsigned)((key * 0x9E3779B97F4A7C15ull) >> 54);
  for (unsigned i = 0; i < 16; ++i) {
    std::atomic<uint64_t>& slot = done[(at + i) % 1024];
    uint64_t seen = slot.load(std::memory_order_acquire);
    if (seen == key) return cudaSuccess;
    if (seen != 0) continue;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) slot.compare_exchange_strong(seen, key, std::memory_order_release);
    return e;
  }
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

}  // namespace fo

extern "C" const char* fo_last_error(void) { return fo::g_err; }

extern "C" int fo_abi_version(void) { return 1; }
