// Host-side helpers shared by the library's translation units: the error
// message, device properties, the shared-memory opt-in and the device error
// word of kernel-level calls.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
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

// n rows of `row` bytes, `stride` bytes apart (memory without rows: one). None
// where the pointer is null.
struct Rows {
  const void* p;
  size_t row, n = 1, stride = 0;
};
// Rows of one stride may stand between one another's; of different strides their
// whole ranges count.
inline bool overlap(const Rows& a, const Rows& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  if (!x || !y || !a.n || !b.n || !a.row || !b.row) return false;
  if (x >= y + (b.n - 1) * b.stride + b.row || y >= x + (a.n - 1) * a.stride + a.row) return false;
  if (a.n < 2 || b.n < 2 || a.stride != b.stride) return true;
  const size_t d = x < y ? (y - x) % a.stride : (a.stride - (x - y) % a.stride) % a.stride;  // from a row of a to the next of b
  return d < a.row || d + b.row > a.stride;
}
inline bool overlap(const Rows& a, std::initializer_list<Rows> others) {
  for (const Rows& b : others)
    if (overlap(a, b)) return true;
  return false;
}
// The device error word of kernel-level calls on the current device
// (foxcuda_kernel_errors reads and clears it); null when it cannot be found.
int* kernel_err_ptr();

// Its codes: a bounded wait that gave up (or another code below 16 of a kernel
// whose output is not valid), and the bit of a row, position or page that a
// device-side array placed outside its bounds (the access was skipped). The bit
// is added to what is there, and the graver code is what a call reports.
enum KernelErr : int { KERR_WAIT = 1, KERR_PAGES = 16 };

inline foxcuda_status kernel_err_status(int code) {
  const char* outside =
      "a call named a row, position or page outside its arrays (a position beyond the tables, a cached length beyond "
      "the block table, a page outside the cache, a row_start that falls or names more rows); what lay outside was "
      "skipped";
  if (code & ~KERR_PAGES)
    return fail(FOXCUDA_ERR_INTERNAL, "device: a bounded wait of a kernel-level tensor-core call gave up (code %d); "
                "that call's output is not valid%s%s", code & ~KERR_PAGES, code & KERR_PAGES ? "; and " : "",
                code & KERR_PAGES ? outside : "");
  return code ? fail(FOXCUDA_ERR_ARG, "device: %s", outside) : FOXCUDA_OK;
}

}  // namespace fox
