// Low-rank adapters, many rows of one adapter: out = y + s (x A^T) B^T for up to
// 64 rows a cluster of blocks.
//
// First product, T [64 x r] = X [64 x K] A^T: the blocks of a cluster share K.  A
// block copies stages of 128 columns of its rows and of A asynchronously into
// shared memory; its warps share the rows (32 each), the ranks (8 NT each) and a
// stage's four slices of 32 columns, and add up what the slices gave at the end.
// The blocks' parts meet in distributed shared memory, each adding up a slice of T
// and all of them collecting the slices.  Second product, Y += T B^T: the
// blocks share N; T's parts are the 16-row operand from shared memory, B comes by
// 16-byte loads, 32 columns a warp and step, arranged so that a lane ends with 8
// columns of its rows behind one another.
//
// A slice lies as [row][64 bytes], slices 64 bytes apart, so that neither the
// copies (16 bytes a thread along a row) nor the operands' loads (16 bytes a lane)
// meet in a bank; f32 rows as two such halves of 16 columns a slice.
#include "lora_mma.cuh"

namespace specb200 {
namespace lora {
namespace {

constexpr int kSlices = 4;  // of 32 columns a stage
constexpr int kRows = kWideRows;

// Byte sizes of the shared memory, from the ranks' capacity RA (a multiple of 8 NT).
template <class TX>
__host__ __device__ constexpr int x_slice() {
  return kRows * (sizeof(TX) == 4 ? 128 : 64) + 64;
}
__host__ __device__ constexpr int a_slice(int RA) { return RA * 64 + 64; }
template <class TX>
__host__ __device__ constexpr int stage_bytes(int RA) {
  return kSlices * (x_slice<TX>() + a_slice(RA));
}

struct WideParams {
  Params p;
  int RA, stages;
};

SPEC_DEV void cp_async16(uint32_t dst, const void* src, int bytes) {  // the rest of the 16 is zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
SPEC_DEV uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// 16 bytes of row `src` from column k on to shared memory; zeros from `end` on.
template <class E>
SPEC_DEV void copy16(uint8_t* dst, const E* src, int k, int end, bool wide) {
  constexpr int N = 16 / sizeof(E);
  const int left = min(max(end - k, 0), N);
  if (wide) {
    cp_async16(smem_u32(dst), left ? src + k : src, left * (int)sizeof(E));
  } else {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) {
        if constexpr (N == 4) w[i] = reinterpret_cast<const uint32_t*>(src)[k + i];
        else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[k + i] << (i % 2 * 16);
      }
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <class T, class TX, class TY, int NT>
__global__ void __launch_bounds__(kThreads, 2) wide_kernel(const __grid_constant__ WideParams wp) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_factor[kRows];
  const Params& p = wp.p;
  constexpr bool kSplitX = sizeof(TX) == 4;
  constexpr int P = parts_of<TY>((const T*)nullptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = cluster_rank(), size = cluster_size(), RA = wp.RA, stages = wp.stages;
  pdl_launch_dependents();
  pdl_wait();
  const Unit u = p.units[blockIdx.x / size];
  const int* rows = p.order + u.first;
  const int r = p.ranks ? min(max(p.ranks[u.adapter], 0), p.rank) : p.rank;
  const T* A = static_cast<const T*>(p.a) + u.adapter * p.a_adapter;
  const T* B = static_cast<const T*>(p.b) + u.adapter * p.b_adapter;
  // Warps: row groups of 32, rank blocks of 8 NT, and the rest takes slices in turn.
  const int groups = u.n_rows > 32 ? 2 : 1, blocks = max((r + 8 * NT - 1) / (8 * NT), 1), turns = kWarps / (groups * blocks);
  const int W = blocks * 8 * NT;  // columns of T
  const int mg = warp % groups, nb = warp / groups % blocks, kg = warp / (groups * blocks);

  // ---- T ----
  float d[2][NT][4] = {};
  {
    const int k_per = ((p.K + size * 128 - 1) / (size * 128)) * 128, k0 = min(rank * k_per, p.K), k1 = min(k0 + k_per, p.K);
    const int n_steps = r ? (k1 - k0 + 127) / 128 : 0;
    const int xs = x_slice<TX>(), as = a_slice(RA), sb = stage_bytes<TX>(RA);
    constexpr int XC = kSplitX ? 32 : 16, XR = kThreads / XC, XN = kRows / XR;  // pieces a row; rows a pass; passes
    const int xc = threadIdx.x % XC, xr = threadIdx.x / XC, ac = threadIdx.x % 16, ar = threadIdx.x / 16;
    const TX* xp[XN];
#pragma unroll
    for (int i = 0; i < XN; ++i) {
      const int row = xr + i * XR;
      xp[i] = static_cast<const TX*>(p.x) + rows[row < u.n_rows ? row : 0] * p.x_row;
    }
    // f32: piece c of a slice is columns 4 c ..; half c % 2, place c / 2 of its row.
    const int x_at = kSplitX ? xc / 8 * xs + xc % 2 * (kRows * 64) + xc % 8 / 2 * 16 : xc / 4 * xs + xc % 4 * 16;
    const int a_at = kSlices * xs + ac / 4 * as + ac % 4 * 16;
    auto fetch = [&](int step) {
      uint8_t* st = smem + step % stages * sb;
      const int k = k0 + step * 128;
#pragma unroll
      for (int i = 0; i < XN; ++i)
        copy16(st + x_at + (xr + i * XR) * 64, xp[i], k + xc * (16 / (int)sizeof(TX)), xr + i * XR < u.n_rows ? k1 : 0, p.x_wide);
      for (int j = ar; j < W; j += kThreads / 16)
        copy16(st + a_at + j * 64, A + min(j, r - 1) * p.a_row, k + ac * 8, j < r ? k1 : 0, p.a_wide);
    };
    for (int s = 0; s < stages - 1; ++s) {
      if (s < n_steps) fetch(s);
      cp_async_commit();
    }
#pragma unroll 1
    for (int step = 0; step < n_steps; ++step) {
      if (stages == 2) cp_async_wait<0>();
      else if (stages == 3) cp_async_wait<1>();
      else cp_async_wait<2>();
      __syncthreads();
      if (step + stages - 1 < n_steps) fetch(step + stages - 1);
      cp_async_commit();
      const uint8_t* st = smem + step % stages * sb;
      for (int i = 0; i < kSlices; ++i) {
        if ((step * kSlices + i) % turns != kg) continue;
        const uint8_t* xb = st + i * xs + (mg * 32 + g) * 64 + t * 16;
        const uint8_t* ab = st + kSlices * xs + i * as + (nb * NT * 8 + g) * 64 + t * 16;
        if constexpr (kSplitX) {
          // Columns 8 t .. 8 t + 7 of two rows a tile: hi and lo.
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            float x0[8], x1[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float4 v = *reinterpret_cast<const float4*>(xb + h * (kRows * 64) + m * 1024);
              const float4 w = *reinterpret_cast<const float4*>(xb + h * (kRows * 64) + m * 1024 + 512);
              x0[h * 4] = v.x, x0[h * 4 + 1] = v.y, x0[h * 4 + 2] = v.z, x0[h * 4 + 3] = v.w;
              x1[h * 4] = w.x, x1[h * 4 + 1] = w.y, x1[h * 4 + 2] = w.z, x1[h * 4 + 3] = w.w;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float a[8];
              widen(lds128(ab + n * 512), a, A);
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                const uint32_t h0 = tf32(x0[e]), h1 = tf32(x1[e]), h2 = tf32(x0[e + 1]), h3 = tf32(x1[e + 1]);
                mma8(d[m][n], h0, h1, h2, h3, __float_as_uint(a[e]), __float_as_uint(a[e + 1]));
                mma8(d[m][n], tf32(rest(x0[e], h0)), tf32(rest(x1[e], h1)), tf32(rest(x0[e + 1], h2)), tf32(rest(x1[e + 1], h3)),
                     __float_as_uint(a[e]), __float_as_uint(a[e + 1]));
              }
            }
          }
        } else {
          uint4 x[2][2];
#pragma unroll
          for (int m = 0; m < 2; ++m) x[m][0] = lds128(xb + m * 1024), x[m][1] = lds128(xb + m * 1024 + 512);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 a = lds128(ab + n * 512);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              mma16(d[m][n], x[m][0].x, x[m][1].x, x[m][0].y, x[m][1].y, a.x, a.y, A);
              mma16(d[m][n], x[m][0].z, x[m][1].z, x[m][0].w, x[m][1].w, a.z, a.w, A);
            }
          }
        }
      }
    }
    cp_async_wait<0>();
    __syncthreads();
  }

  // ---- the parts of T join ----
  // `part`: this block's T; `all`: the cluster's; then, in part's place, the
  // numbers that T is split into.
  float* part = reinterpret_cast<float*>(smem);
  float* all = reinterpret_cast<float*>(smem + kRows * RA * 6);
  const int live = groups * 32 * W;
  if (kg < turns) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* o = part + kg * live + (mg * 32 + m * 16 + g) * W + nb * NT * 8 + n * 8 + 2 * t;
        *reinterpret_cast<float2*>(o) = make_float2(d[m][n][0], d[m][n][1]);
        *reinterpret_cast<float2*>(o + 8 * W) = make_float2(d[m][n][2], d[m][n][3]);
      }
  }
  __syncthreads();
  for (int i = threadIdx.x * 4; i < live; i += kThreads * 4) {
    float4 s = *reinterpret_cast<const float4*>(part + i);
    for (int q = 1; q < turns; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(part + q * live + i);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    *reinterpret_cast<float4*>(part + i) = s;
  }
  __syncthreads();
  if (size > 1) {
    cluster_arrive();
    cluster_wait();
    const int share = (live / 4 + size - 1) / size * 4;
    for (int i = rank * share + threadIdx.x * 4; i < min((rank + 1) * share, live); i += kThreads * 4) {
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < size; ++q) {
        const float4 v = remote_float4(part + i, q);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      *reinterpret_cast<float4*>(all + i) = s;
    }
    cluster_arrive();
    cluster_wait();
    for (int i = threadIdx.x * 4; i < live; i += kThreads * 4)
      if (i / share != rank) *reinterpret_cast<float4*>(all + i) = remote_float4(all + i, i / share);
    cluster_arrive();  // nothing of the other blocks is read any more
  } else {
    for (int i = threadIdx.x * 4; i < live; i += kThreads * 4) *reinterpret_cast<float4*>(all + i) = *reinterpret_cast<float4*>(part + i);
  }
  __syncthreads();
  const int steps = (r + 31) / 32, frag = kRows * 64;  // bytes of one part's 32 ranks
  if (threadIdx.x < groups * 32 * 4) {                 // four threads a row
    const int row = threadIdx.x / 4, c = threadIdx.x % 4;
    const float scale = p.scales ? p.scales[u.adapter] : 1.f;
    float top = 0.f;
    for (int j = c * 8; j < r; j += 32)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (j + k < r) top = fmaxf(top, fabsf(all[row * W + j + k] * scale));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = exponent(top, A);
    const float down = pow2i(-e);
    if (c == 0) s_factor[row] = pow2i(e);
    for (int s = 0; s < steps; ++s) {
      const int j = s * 32 + c * 8;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = j + k < r ? all[row * W + j + k] * scale * down : 0.f;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w[k] = pack2(v[2 * k], v[2 * k + 1], A);
          T h[2];
          *reinterpret_cast<uint32_t*>(h) = w[k];
          v[2 * k] = fabsf(v[2 * k]) < INFINITY ? v[2 * k] - to_float(h[0]) : 0.f;
          v[2 * k + 1] = fabsf(v[2 * k + 1]) < INFINITY ? v[2 * k + 1] - to_float(h[1]) : 0.f;
        }
        *reinterpret_cast<uint4*>(smem + (q * steps + s) * frag + row * 64 + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  __syncthreads();

  // ---- Y ----
  {
    const int n_per = ((p.N + size * 32 - 1) / (size * 32)) * 32, n0 = min(rank * n_per, p.N), n1 = min(n0 + n_per, p.N);
    const int ways = kWarps / groups, ng = warp / groups, first = (warp % groups) * 32 + g;
    long long at[4];
    float factor[4];
    bool has[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = first + i * 8;
      has[i] = row < u.n_rows;
      at[i] = has[i] ? rows[row] : 0;
      factor[i] = has[i] ? s_factor[row] : 0.f;
    }
#pragma unroll 1
    for (int n = n0 + ng * 32; n < n1; n += ways * 32) {
      float y[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (has[i]) load8(static_cast<const TY*>(p.y) + at[i] * p.y_row, n + 8 * t, n1, p.y_wide, y[i]);
      float d2[2][4][4] = {};
      const int column = n + g / 2 * 8 + g % 2;
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        uint4 b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          b[j] = load8(B + (column + 2 * j) * p.b_row, s * 32 + 8 * t, column + 2 * j < n1 ? r : 0, p.b_wide);
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const uint8_t* f = smem + (q * steps + s) * frag + first * 64 + t * 16;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const uint4 x0 = lds128(f + m * 1024), x1 = lds128(f + m * 1024 + 512);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma16(d2[m][j], x0.x, x1.x, x0.y, x1.y, b[j].x, b[j].y, A);
              mma16(d2[m][j], x0.z, x1.z, x0.w, x1.w, b[j].z, b[j].w, A);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!has[i]) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y[i][2 * j] = fmaf(d2[i / 2][j][i % 2 * 2], factor[i], y[i][2 * j]);
          y[i][2 * j + 1] = fmaf(d2[i / 2][j][i % 2 * 2 + 1], factor[i], y[i][2 * j + 1]);
        }
        store8(static_cast<TY*>(p.out) + at[i] * p.out_row, n + 8 * t, n1, p.out_wide, y[i]);
      }
    }
  }
  if (size > 1) cluster_wait();
}

template <class T, class TX, class TY, int NT>
cudaError_t run(const Params& p, int n_units, int size, cudaStream_t s) {
  constexpr int B = 8 * NT;
  WideParams w{p, ((p.rank > 1 ? p.rank : 1) + B - 1) / B * B, 0};
  const int stage = stage_bytes<TX>(w.RA);
  // As many stages, up to 4, as let an SM hold two blocks; two at least.
  w.stages = 112 * 1024 / stage;
  w.stages = w.stages > 4 ? 4 : w.stages < 2 ? 2 : w.stages;
  int bytes = w.stages * stage;
  // The warps' parts of T: 32 rows and a block of ranks each; T whole, and the numbers it is split into.
  if (bytes < kWarps * 32 * B * 4) bytes = kWarps * 32 * B * 4;
  if (bytes < kRows * w.RA * 10) bytes = kRows * w.RA * 10;
  const cudaError_t e = cudaFuncSetAttribute(wide_kernel<T, TX, TY, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  return launch_clusters(wide_kernel<T, TX, TY, NT>, n_units, size, kThreads, bytes, s, w);
}
template <class T, class TX, class TY>
cudaError_t run(const Params& p, int n_units, int size, cudaStream_t s) {
  return p.rank <= 32 ? run<T, TX, TY, 4>(p, n_units, size, s) : run<T, TX, TY, 8>(p, n_units, size, s);
}
template <class T>
cudaError_t run(const Params& p, bool x_f32, bool y_f32, int n_units, int size, cudaStream_t s) {
  if (x_f32) return y_f32 ? run<T, float, float>(p, n_units, size, s) : run<T, float, T>(p, n_units, size, s);
  return y_f32 ? run<T, T, float>(p, n_units, size, s) : run<T, T, T>(p, n_units, size, s);
}

}  // namespace

cudaError_t launch_wide(const Params& p, int type, bool x_f32, bool y_f32, int n_units, int size, cudaStream_t s) {
  if (n_units <= 0) return cudaSuccess;
  return type == T_BF16 ? run<__nv_bfloat16>(p, x_f32, y_f32, n_units, size, s)
                        : run<__half>(p, x_f32, y_f32, n_units, size, s);
}

}  // namespace lora
}  // namespace specb200
