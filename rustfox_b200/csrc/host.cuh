// Host-side helpers shared by the library's translation units: the error
// message, device properties, the shared-memory opt-in and the device error
// word of kernel-level calls.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "../../include/foxcuda.h"

namespace fox {

// ---------------------------------------------------------------------------
// errors: thread-local message, status codes of upstream fox_status

inline thread_local char g_err[512];

inline foxcuda_status fail(foxcuda_status st, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof g_err, fmt, ap);
  va_end(ap);
  return st;
}

inline foxcuda_status cuda_fail(cudaError_t e, const char* what) {
  return fail(e == cudaErrorMemoryAllocation ? FOXCUDA_ERR_NOMEM : FOXCUDA_ERR_INTERNAL,
              "%s: %s", what, cudaGetErrorString(e));
}

#define CK(call, what)                                   \
  do {                                                   \
    cudaError_t e_ = (call);                             \
    if (e_ != cudaSuccess) return cuda_fail(e_, what);   \
  } while (0)

inline int sm_count(int dev) {
  static int cached[64] = {0};
  if (dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cached[dev] = n;
  }
  return cached[dev];
}

inline int current_sms() {
  int d = 0;
  cudaGetDevice(&d);
  return sm_count(d);
}

// The dynamic shared-memory opt-in is a property of a kernel on one device,
// so each launcher keeps its high-water mark per device (`marks` has one
// slot per device ordinal). The attribute only ever rises, under a lock, so
// two threads cannot leave it below a mark that another thread relies on.
constexpr int kMaxDevices = 64;
inline std::mutex g_smem_mu;

template <typename K>
inline cudaError_t opt_in_smem(K kern, size_t smem, size_t* marks) {
  if (smem <= 48 * 1024) return cudaSuccess;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lk(g_smem_mu);
  if (smem <= marks[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  marks[dev] = smem;
  return cudaSuccess;
}

// The device error word of kernel-level calls on the current device
// (foxcuda_kernel_errors reads and clears it); null when it cannot be found.
int* kernel_err_ptr();

// Its codes: a bounded wait that gave up, and a row, position or page that a
// device-side array placed outside its bounds (the access was skipped).
enum KernelErr : int { KERR_WAIT = 1, KERR_PAGES = 16 };

}  // namespace fox
