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

// Multiprocessors of a device.
inline cudaError_t multiprocessors(int device, int* sms) {
  return cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device);
}

}  // namespace specb200
