// Low-rank adapters of many requests beside a shared projection:
//
//   out = y + s (x A^T) B^T,   A [r x K], B [N x r] of the row's own adapter
//
// A cluster takes the rows of one adapter (up to 8), so that A and B are
// read once for all of them.  Each block forms the part of t = x A^T over its
// share of K; the parts meet in distributed shared memory, and each block
// then adds t B^T for its share of N.  Both products are taken transposed, so
// that the adapter is the 16-row operand of mma.sync and the rows are its 8
// columns:
//   T^T [16 ranks x 8 rows] += A [16 x 32] X^T,   Y^T [16 n x 8 rows] += B [16 x 32] T^T
// A product's sum may run in any order, so a lane takes 8 consecutive elements of
// its row for two instructions of 16 (its 2t, 2t + 1, 2t + 8, 2t + 9 of each):
// every operand comes by 16-byte loads from where it lies, without shared memory.
//
// f32 rows enter as two tf32 numbers, hi + lo, off by 2^-24.  t stays f32;
// for the second product it is split into bf16 numbers (three, 24 bits, for an
// f32 result; two, 16 bits, for a bf16 one, which itself has 8), or two f16
// numbers of t 2^-e, 2^e about the row's largest (22 bits).  All sums are f32.
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
SPEC_DEV uint16_t bits(__half h) { return __half_as_ushort(h); }
SPEC_DEV uint16_t bits(__nv_bfloat16 h) { return __bfloat16_as_ushort(h); }
SPEC_DEV float to_float(float x) { return x; }
SPEC_DEV float to_float(__half x) { return __half2float(x); }
SPEC_DEV float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
SPEC_DEV void from_float(float x, float* p) { *p = x; }
SPEC_DEV void from_float(float x, __half* p) { *p = __float2half_rn(x); }
SPEC_DEV void from_float(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }

// Numbers of type T that t is split into.
template <class TY>
__host__ __device__ constexpr int parts_of(const __half*) {
  return 2;
}
template <class TY>
__host__ __device__ constexpr int parts_of(const __nv_bfloat16*) {
  return sizeof(TY) == 4 ? 3 : 2;
}

// The power of two that a row of t is divided by before it goes to f16.
SPEC_DEV int exponent(float top, const __half*) {
  return top > 0.f && top < INFINITY ? min(max((__float_as_int(top) >> 23) - 127, -100), 126) : 0;
}
SPEC_DEV int exponent(float, const __nv_bfloat16*) { return 0; }
SPEC_DEV float pow2i(int e) { return __int_as_float((127 + e) << 23); }

struct Smem {
  float part[16 * kNarrowRows * 16];         // [k part x rank tile][row][16 ranks]
  float t[kNarrowRows][kMaxRank];            // this block's share of x A^T
  uint16_t frag[3][kMaxRank / 32][32 * 8];   // t's parts as the second product takes them
  float factor[kNarrowRows];
};

template <class T, class TX, class TY>
__global__ void __launch_bounds__(kThreads) narrow_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) Smem sm;
  constexpr bool kSplitX = sizeof(TX) == 4;
  constexpr int P = parts_of<TY>((const T*)nullptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = cluster_rank(), size = cluster_size();
  pdl_launch_dependents();
  pdl_wait();
  const Unit u = p.units[blockIdx.x / size];
  const int* rows = p.order + u.first;
  const int n_per = ((p.N + size * 16 - 1) / (size * 16)) * 16, n0 = min(rank * n_per, p.N), n1 = min(n0 + n_per, p.N);
  if (u.adapter < 0) {  // rows without an adapter: y as it is
    for (int i = 0; i < u.n_rows; ++i) {
      const long long row = rows[i];
      for (int n = n0 + threadIdx.x; n < n1; n += kThreads)
        static_cast<TY*>(p.out)[row * p.out_row + n] = static_cast<const TY*>(p.y)[row * p.y_row + n];
    }
    return;
  }
  const int r = p.ranks ? min(max(p.ranks[u.adapter], 0), p.rank) : p.rank;
  const T* A = static_cast<const T*>(p.a) + u.adapter * p.a_adapter;
  const T* B = static_cast<const T*>(p.b) + u.adapter * p.b_adapter;
  const int tiles = (r + 15) / 16, kparts = tiles ? max(kWarps / tiles, 1) : 1;

  // This block's part of T^T: warps share the rank tiles and the K steps.
  {
    const int k_per = ((p.K + size * 32 - 1) / (size * 32)) * 32, k0 = min(rank * k_per, p.K), k1 = min(k0 + k_per, p.K);
    const TX* x = static_cast<const TX*>(p.x) + (g < u.n_rows ? rows[g] : 0) * p.x_row;
    const int part = tiles ? warp / tiles : 0;
    for (int tile = tiles ? warp % tiles : 0; tile < tiles && part < kparts; tile += kWarps) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
      const int j0 = tile * 16 + g, j1 = j0 + 8;
      const T *a0 = A + j0 * p.a_row, *a1 = A + j1 * p.a_row;
#pragma unroll 2
      for (int k = k0 + part * 32; k < k1; k += kparts * 32) {
        const int at = k + 8 * t;
        const uint4 v0 = load8(a0, at, j0 < r ? k1 : 0, p.a_wide), v1 = load8(a1, at, j1 < r ? k1 : 0, p.a_wide);
        const int end = g < u.n_rows ? k1 : 0;
        if constexpr (kSplitX) {
          float f0[8], f1[8], xv[8];
          widen(v0, f0, A);
          widen(v1, f1, A);
          load8(x, at, end, p.x_wide, xv);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const uint32_t h0 = tf32(xv[i]), h1 = tf32(xv[i + 1]);
            const uint32_t l0 = tf32(rest(xv[i], h0)), l1 = tf32(rest(xv[i + 1], h1));
            const uint32_t w0 = __float_as_uint(f0[i]), w1 = __float_as_uint(f1[i]);
            const uint32_t w2 = __float_as_uint(f0[i + 1]), w3 = __float_as_uint(f1[i + 1]);
            mma8(d, w0, w1, w2, w3, h0, h1);
            mma8(d, w0, w1, w2, w3, l0, l1);
          }
        } else {
          const uint4 xv = load8(reinterpret_cast<const T*>(x), at, end, p.x_wide);
          mma16(d, v0.x, v1.x, v0.y, v1.y, xv.x, xv.y, A);
          mma16(d, v0.z, v1.z, v0.w, v1.w, xv.z, xv.w, A);
        }
      }
      float* o = sm.part + (part * tiles + tile) * (kNarrowRows * 16);
      o[2 * t * 16 + g] = d[0];
      o[(2 * t + 1) * 16 + g] = d[1];
      o[2 * t * 16 + g + 8] = d[2];
      o[(2 * t + 1) * 16 + g + 8] = d[3];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kNarrowRows * tiles * 16; i += kThreads) {
    const int row = i / (tiles * 16), j = i % (tiles * 16);
    float s = 0.f;
    for (int q = 0; q < kparts; ++q) s += sm.part[((q * tiles + j / 16) * kNarrowRows + row) * 16 + j % 16];
    sm.t[row][j] = s;
  }
  cluster_arrive();
  cluster_wait();

  // All of t, a warp a row, split into parts.
  const int steps = (r + 31) / 32;
  {
    const int row = warp;
    const float scale = p.scales ? p.scales[u.adapter] : 1.f;
    float v[kMaxRank / 32], top = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxRank / 32; ++i) {
      const int j = i * 32 + lane;
      v[i] = 0.f;
      if (j < r)
        for (int q = 0; q < size; ++q) v[i] += remote_float(&sm.t[row][j], q);
      v[i] *= scale;
      top = fmaxf(top, fabsf(v[i]));
    }
    cluster_arrive();  // nothing of the other blocks is read any more
    const int e = exponent(warp_max(top), A);
    const float down = pow2i(-e);
    if (lane == 0) sm.factor[row] = pow2i(e);
#pragma unroll
    for (int i = 0; i < kMaxRank / 32; ++i) {
      if (i >= steps) break;
      float left = v[i] * down;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        T h;
        from_float(left, &h);
        left = fabsf(left) < INFINITY ? left - to_float(h) : 0.f;
        sm.frag[q][i][(row * 4 + lane / 8) * 8 + lane % 8] = bits(h);
      }
    }
  }
  __syncthreads();

  // Y^T += B T^T over this block's columns.
  const int ra = 2 * t, rb = 2 * t + 1;
  const bool has_a = ra < u.n_rows, has_b = rb < u.n_rows;
  const long long row_a = has_a ? rows[ra] : 0, row_b = has_b ? rows[rb] : 0;
  const TY *ya = static_cast<const TY*>(p.y) + row_a * p.y_row, *yb = static_cast<const TY*>(p.y) + row_b * p.y_row;
  TY *oa = static_cast<TY*>(p.out) + row_a * p.out_row, *ob = static_cast<TY*>(p.out) + row_b * p.out_row;
  const float fa = sm.factor[ra], fb = sm.factor[rb];
#pragma unroll 2
  for (int n = n0 + warp * 16; n < n1; n += kWarps * 16) {
    const int m0 = n + g, m1 = m0 + 8;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    if (has_a && m0 < n1) y[0] = to_float(ya[m0]);
    if (has_b && m0 < n1) y[1] = to_float(yb[m0]);
    if (has_a && m1 < n1) y[2] = to_float(ya[m1]);
    if (has_b && m1 < n1) y[3] = to_float(yb[m1]);
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    const T *b0 = B + m0 * p.b_row, *b1 = B + m1 * p.b_row;
#pragma unroll 2
    for (int s = 0; s < steps; ++s) {
      const int at = s * 32 + 8 * t;
      const uint4 v0 = load8(b0, at, m0 < n1 ? r : 0, p.b_wide), v1 = load8(b1, at, m1 < n1 ? r : 0, p.b_wide);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const uint4 w = *reinterpret_cast<const uint4*>(&sm.frag[q][s][lane * 8]);
        mma16(d, v0.x, v1.x, v0.y, v1.y, w.x, w.y, A);
        mma16(d, v0.z, v1.z, v0.w, v1.w, w.z, w.w, A);
      }
    }
    if (has_a && m0 < n1) from_float(fmaf(d[0], fa, y[0]), oa + m0);
    if (has_b && m0 < n1) from_float(fmaf(d[1], fb, y[1]), ob + m0);
    if (has_a && m1 < n1) from_float(fmaf(d[2], fa, y[2]), oa + m1);
    if (has_b && m1 < n1) from_float(fmaf(d[3], fb, y[3]), ob + m1);
  }
  cluster_wait();
}

template <class T, class TX, class TY>
cudaError_t run(const Params& p, int n_units, int size, cudaStream_t s) {
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = size;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n_units * size);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, narrow_kernel<T, TX, TY>, p);
}
template <class T>
cudaError_t run(const Params& p, bool x_f32, bool y_f32, int n_units, int size, cudaStream_t s) {
  if (x_f32) return y_f32 ? run<T, float, float>(p, n_units, size, s) : run<T, float, T>(p, n_units, size, s);
  return y_f32 ? run<T, T, float>(p, n_units, size, s) : run<T, T, T>(p, n_units, size, s);
}

}  // namespace

cudaError_t launch(const Params& p, int type, bool x_f32, bool y_f32, int n_units, int size, cudaStream_t s) {
  if (n_units <= 0) return cudaSuccess;
  return type == T_BF16 ? run<__nv_bfloat16>(p, x_f32, y_f32, n_units, size, s)
                        : run<__half>(p, x_f32, y_f32, n_units, size, s);
}

}  // namespace lora
}  // namespace specb200
