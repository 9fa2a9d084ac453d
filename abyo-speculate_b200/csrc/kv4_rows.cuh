// Reading and writing 8 channels of the callers' rows (any type, any stride).
#pragma once

#include "common.cuh"
#include "kv4.h"

namespace specb200 {
namespace kv4 {

// 8 consecutive elements at element offset `at`.
SPEC_DEV void load8(const Rows& r, long long at, bool wide, float (&x)[8]) {
  if (r.dtype == T_F32) {
    const float* p = static_cast<const float*>(r.ptr) + at;
    if (wide) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
    return;
  }
  const uint16_t* p = static_cast<const uint16_t*>(r.ptr) + at;
  uint32_t w[4];
  if (wide) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r.dtype == T_BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// Each rounded once to the rows' type.
SPEC_DEV void store8(const Rows& r, long long at, bool wide, const float (&x)[8]) {
  if (r.dtype == T_F32) {
    float* p = static_cast<float*>(r.ptr) + at;
    if (wide) {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r.dtype == T_BF16) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  uint16_t* p = static_cast<uint16_t*>(r.ptr) + at;
  if (wide) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[2 * i] = (uint16_t)w[i];
      p[2 * i + 1] = (uint16_t)(w[i] >> 16);
    }
  }
}

// Launches a kernel that may start while the kernel before it on the stream
// still runs: it reads nothing but the plan, and writes nothing, before its
// griddepcontrol.wait.
template <class K, class P>
cudaError_t launch_overlapping(K* kernel, dim3 grid, int threads, int smem, cudaStream_t s, const P& p) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace kv4
}  // namespace specb200
