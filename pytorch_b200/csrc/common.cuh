// Host-side helpers shared by the C-ABI translation units.
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>
#include <mutex>
#include <utility>

#include "../../include/b200q.h"

namespace b200q {

// Stores the calling thread's last error message and returns `status`.
int fail(int status, const char* fmt, ...);
void clear_error();

// Number of SMs of the current device (cached per device).
int sm_count();

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

#define B200Q_REQUIRE(cond, status, ...)            \
  do {                                              \
    if (!(cond)) return ::b200q::fail((status), __VA_ARGS__); \
  } while (0)

// Call after a kernel launch: turns a launch error into B200Q_ERR_LAUNCH.
inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return B200Q_OK;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Raises the dynamic shared-memory limit of kernel `Kern` to `bytes`, once per device.  The per-device
// record is guarded by a mutex, so concurrent first calls from several host threads are safe.
template <auto Kern>
int ensure_dynamic_smem(int bytes, const char* what) {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= 0 && done[dev]) return B200Q_OK;
  cudaError_t err = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(err));
  if (dev >= 0) done[dev] = true;
  return B200Q_OK;
}

// Allows kernel `Kern` clusters of more than eight CTAs, once per device.
template <auto Kern>
int ensure_wide_clusters(const char* what) {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= 0 && done[dev]) return B200Q_OK;
  cudaError_t err = cudaFuncSetAttribute(Kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (err != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(err));
  if (dev >= 0) done[dev] = true;
  return B200Q_OK;
}

// CTAs of `threads` threads of kernel `Kern` (no dynamic shared memory) that an SM of the current device holds at once.
// The query costs more than a launch, so its answer is kept per device and size.
template <auto Kern>
int resident_ctas(int threads) {
  static std::atomic<int> cached[64][33];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
  const int size = threads / 32;
  if (dev >= 0 && size <= 32)
    if (const int n = cached[dev][size].load(std::memory_order_relaxed)) return n;
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kern, threads, 0) != cudaSuccess || n < 1) n = 1;
  if (dev >= 0 && size <= 32) cached[dev][size].store(n, std::memory_order_relaxed);
  return n;
}

// Launches a kernel that may start before the kernel in front of it on the stream has finished (programmatic
// dependent launch): it must not touch what that kernel writes before wait_for_primary() and reads it by ld_of_primary(_cached), and the
// kernel in front must itself be an ordinary launch, so that everything before it is complete.
template <typename... Params, typename... Args>
int launch_dependent(void (*kern)(Params...), unsigned grid, int threads, cudaStream_t st, const char* what, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
  if (err != cudaSuccess) return fail(B200Q_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(err));
  return check_launch(what);
}

}  // namespace b200q
