// What the stateless host entry points (batch.cpp, lora.cpp) share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/spec_b200.h"
#include "model.h"

namespace specb200 {

inline int fail(int rc, const char* msg) {
  set_thread_error(msg);
  return rc;
}
template <class... A>
int fail(int rc, const char* fmt, A... a) {
  char msg[256];
  snprintf(msg, sizeof msg, fmt, a...);
  set_thread_error(msg);
  return rc;
}
inline int fail_cuda(cudaError_t e, const char* what) {
  cudaGetLastError();  // reported here: the next launch's check is not to find it
  return fail(e == cudaErrorMemoryAllocation ? SPEC_ERR_OOM : SPEC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// The call's device is current during a call; the caller's comes back.
struct Current {
  int prev = -1, device;
  int rc = SPEC_OK;
  Current(int d, const char* what) : device(d) {
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != d) e = cudaSetDevice(d);
    if (e != cudaSuccess) rc = fail_cuda(e, what);
  }
  ~Current() {
    if (prev >= 0 && prev != device) cudaSetDevice(prev);
  }
  Current(const Current&) = delete;
  Current& operator=(const Current&) = delete;
};

constexpr int64_t kMaxStride = INT64_C(1) << 40;

inline bool misaligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

// Whether rows of `a` and of `b` share memory: n rows of a, `step_a` bytes apart and `wide_a` long, and n of b.
inline bool rows_meet(const void* a, int64_t step_a, int64_t wide_a, const void* b, int64_t step_b, int64_t wide_b, int64_t n) {
  const int64_t pa = (int64_t)reinterpret_cast<intptr_t>(a), pb = (int64_t)reinterpret_cast<intptr_t>(b);
  if (n <= 0 || pa + (n - 1) * step_a + wide_a <= pb || pb + (n - 1) * step_b + wide_b <= pa) return false;
  if (n == 1) return true;
  // A row of b that starts after `at - wide_b` and before `at + wide_a` meets a's row at `at`.
  auto meets = [&](int64_t at, int64_t first, int64_t last) {
    const int64_t lo = at - wide_b - pb, hi = at + wide_a - pb;  // lo < j step_b < hi
    if (step_b == 0) return first <= last && lo < 0 && hi > 0;
    const int64_t j = lo < 0 && lo % step_b != 0 ? lo / step_b : lo / step_b + 1;  // the first j past lo
    const int64_t k = j > first ? j : first;
    return k <= last && k * step_b < hi;
  };
  if (step_a == step_b) return meets(pa, 1 - n, n - 1);  // only the rows' distance counts
  for (int64_t i = 0; i < (step_a ? n : 1); ++i)
    if (meets(pa + i * step_a, 0, n - 1)) return true;
  return false;
}

// Multiprocessors of a device.
inline cudaError_t multiprocessors(int device, int* sms) {
  return cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device);
}

}  // namespace specb200
