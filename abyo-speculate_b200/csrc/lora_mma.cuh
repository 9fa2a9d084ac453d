// What the kernels of the low-rank adapters share: products on mma.sync from
// 16-byte pieces, parts that f32 numbers are split into, and clusters.
//
// A product's sum may run in any order, so a lane takes 8 consecutive elements of
// its row for two instructions of 16 (its 2t, 2t + 1, 2t + 8, 2t + 9 of each).
//
// The tensor core drops what lies below its accumulator's last bit, so that a sum
// of many instructions ends too small: x A^T of 14336 channels by 0.8e-5 of itself (448
// instructions in a row) to 3e-5 (3584).  So few of them run in a row (2 or 8, 16 on
// tcgen05), the smaller of two parts first, and their sums meet in f32 additions,
// which round: 2e-7 to 6e-7 of the adapters' share in all (f32 library products 1.5e-6 to 2e-6).
#pragma once

#include "common.cuh"
#include "kv4_rows.cuh"
#include "lora.h"

namespace specb200 {
namespace lora {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

SPEC_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
SPEC_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
SPEC_DEV int cluster_rank() {
  int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
SPEC_DEV int cluster_size() {
  int r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
SPEC_DEV float remote_float(const float* p, int rank) {
  uint32_t at;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}

SPEC_DEV float4 remote_float4(const float* p, int rank) {
  uint32_t at;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}

SPEC_DEV void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// Waits until at most n (up to 4) of this thread's groups of copies are under way.
SPEC_DEV void cp_async_wait_for(int n) {
  switch (n) {
    case 0: cp_async_wait<0>(); break;
    case 1: cp_async_wait<1>(); break;
    case 2: cp_async_wait<2>(); break;
    case 3: cp_async_wait<3>(); break;
    default: cp_async_wait<4>(); break;
  }
}

// Asks for `n` elements from `p` on to be brought to L2 (whole 16-byte pieces of
// them, up to 64 KB).
template <class E>
SPEC_DEV void prefetch(const E* p, long long n) {
  const uintptr_t a = (reinterpret_cast<uintptr_t>(p) + 15) / 16 * 16, e = reinterpret_cast<uintptr_t>(p + n) / 16 * 16;
  if (e > a) tma_prefetch_l2(reinterpret_cast<const void*>(a), (uint32_t)(e - a < 65536 ? e - a : 65536));
}
// The same of rows n0 .. n1 - 1 of B, in pieces of 32 KB a thread, where all of a
// row is wanted or the row is no longer than the memory's 64 bytes.
template <class T>
SPEC_DEV void prefetch_b(const Params& p, const T* B, int n0, int n1) {
  if (p.ranks && p.b_row > 32) return;
  if (p.b_row > 2 * p.rank || !p.rank) return;
  const long long begin = n0 * p.b_row, end = n1 * p.b_row - (p.b_row - p.rank), piece = 32768 / (int)sizeof(T);
  for (long long at = begin + threadIdx.x * piece; at < end; at += blockDim.x * piece) prefetch(B + at, end - at < piece ? end - at : piece);
}

SPEC_DEV void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                    const __half*) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
SPEC_DEV void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                    const __nv_bfloat16*) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
SPEC_DEV void mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
SPEC_DEV uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}

SPEC_DEV float rest(float x, uint32_t hi) { return fabsf(x) < INFINITY ? x - __uint_as_float(hi) : 0.f; }

// Words of 8 consecutive 16-bit elements from `k` on; those at `n` and behind are zeros.
template <class T>
SPEC_DEV uint4 load8(const T* p, int k, int n, bool wide) {
  if (wide && k + 8 <= n) return *reinterpret_cast<const uint4*>(p + k);
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (k + 2 * i < n ? q[k + 2 * i] : 0u) | (k + 2 * i + 1 < n ? (uint32_t)q[k + 2 * i + 1] << 16 : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The words' elements before place n (of 8), zeros for the others.
SPEC_DEV uint4 first_of(const uint4& v, int n) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = n >= 2 * i + 2 ? w[i] : n == 2 * i + 1 ? w[i] & 0xffffu : 0u;
  return make_uint4(o[0], o[1], o[2], o[3]);
}
SPEC_DEV void load8(const float* p, int k, int n, bool wide, float (&x)[8]) {
  if (wide && k + 8 <= n) {
    const float4 a = *reinterpret_cast<const float4*>(p + k), b = *reinterpret_cast<const float4*>(p + k + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = k + i < n ? p[k + i] : 0.f;
}
SPEC_DEV void widen(const uint4& v, float (&x)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
SPEC_DEV void widen(const uint4& v, float (&x)[8], const __half*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
SPEC_DEV uint32_t pack2(float lo, float hi, const __half*) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
SPEC_DEV uint32_t pack2(float lo, float hi, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
SPEC_DEV uint16_t bits(__half h) { return __half_as_ushort(h); }
SPEC_DEV uint16_t bits(__nv_bfloat16 h) { return __bfloat16_as_ushort(h); }
SPEC_DEV float to_float(float x) { return x; }
SPEC_DEV float to_float(__half x) { return __half2float(x); }
SPEC_DEV float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
SPEC_DEV void from_float(float x, float* p) { *p = x; }
SPEC_DEV void from_float(float x, __half* p) { *p = __float2half_rn(x); }
SPEC_DEV void from_float(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }

// Numbers of type T that t, an f32 sum, is split into: all 24 bits in bf16, for
// results in bf16 too, where two (16 bits) show when y and the adapter's share
// nearly cancel (64 adapters of 64 rows, rank 64: 86 us, 79 with two); in f16 22 bits of
// the row's largest, 2^-23 of which is less than sums of k terms in f32 are off by.
__host__ __device__ constexpr int parts_of(const __half*) { return 2; }
__host__ __device__ constexpr int parts_of(const __nv_bfloat16*) { return 3; }

// The power of two that a row of t is divided by before it goes to f16.
SPEC_DEV int exponent(float top, const __half*) {
  return top > 0.f && top < INFINITY ? min(max((__float_as_int(top) >> 23) - 127, -100), 126) : 0;
}
SPEC_DEV int exponent(float, const __nv_bfloat16*) { return 0; }
SPEC_DEV float pow2i(int e) { return __int_as_float((127 + e) << 23); }

template <class K, class Q>
cudaError_t launch_clusters(K* kernel, int n, int size, int threads, int smem, cudaStream_t s, const Q& p) {
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = size;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n * size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Blocks a cluster of a kernel whose limit of shared memory is set: 8, fewer where n
// clusters are not resident at once (a GPC's SMs hold whole clusters: of 8, with a block an SM, a B200
// holds 15, not 18).
template <class K>
cudaError_t cluster_for(K* kernel, int n, int threads, int smem, int* size) {
  for (*size = 8; *size > 1; *size /= 2) {
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = *size;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(*size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int resident = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&resident, kernel, &cfg);
    if (e != cudaSuccess) return e;
    if (n <= resident) break;
  }
  return cudaSuccess;
}

}  // namespace
}  // namespace lora
}  // namespace specb200
