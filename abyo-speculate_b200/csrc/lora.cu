// Low-rank adapters of many requests beside a shared projection:
//
//   out = y + s (x A^T) B^T,   A [r x K], B [N x r] of the row's own adapter
//
// A cluster takes the rows of one adapter (up to 8), so that A and B are
// read once for all of them.  Each block forms the part of t = x A^T over its
// share of K; the parts meet in distributed shared memory, and each block
// then adds t B^T for its share of N; a warp has its stages of B under way
// from the start.  Both products are taken transposed, so
// that the adapter is the 16-row operand of mma.sync and the rows are its 8
// columns:
//   T^T [16 ranks x 8 rows] += A [16 x 32] X^T,   Y^T [16 n x 8 rows] += B [16 x 32] T^T
// A product's sum may run in any order, so a lane takes 8 consecutive elements of
// its row for two instructions of 16 (its 2t, 2t + 1, 2t + 8, 2t + 9 of each):
// x and A come by 16-byte loads from where they lie, without shared memory.
//
// f32 rows enter as two tf32 numbers of 11 bits, hi + lo, off by at most 2^-23.  t stays f32;
// for the second product it is split into three bf16 numbers (24 bits), or two f16
// numbers of t 2^-e, 2^e about the row's largest (22 bits).  All sums are f32.
//
// Bound by latency: 64 rows of 64 adapters of rank 32 and less, 3584 to 18944 in f16
// with f32 results, 26 us of which 40 MB take 6 at the copy rate; 21 warps an SM read A, then B, in turn.
// Stages of 32 columns and three blocks an SM (80 registers) took 30 to 26 us.
#include "lora_mma.cuh"

namespace specb200 {
namespace lora {
namespace {

constexpr int kStages = 4;   // of B a warp has under way
constexpr int kColumns = 32;  // of a stage, by 32 ranks
constexpr int kStageBytes = kColumns * 64;

// A lane ends with four columns of its rows behind one another, 4 g + i; in a stage,
// column c lies where tile c % 4 / 2 of the product takes it.
SPEC_DEV int place_of(int c) { return c % 4 * 8 + c / 4; }

template <class TY>
SPEC_DEV void load4(const TY* p, int k, int n, bool wide, float (&x)[4]) {
  if (wide && k + 4 <= n) {
    if constexpr (sizeof(TY) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + k);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p + k);
      const TY* e = reinterpret_cast<const TY*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = to_float(e[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = k + i < n ? to_float(p[k + i]) : 0.f;
}
template <class TY>
SPEC_DEV void store4(TY* p, int k, int n, bool wide, const float (&x)[4]) {
  if (wide && k + 4 <= n) {
    if constexpr (sizeof(TY) == 4) *reinterpret_cast<float4*>(p + k) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2*>(p + k) = make_uint2(pack2(x[0], x[1], p), pack2(x[2], x[3], p));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (k + i < n) from_float(x[i], p + k + i);
}

struct Smem {
  uint8_t ring[kWarps][kStages][kStageBytes];
  union {
    float part[kWarps * kNarrowRows * 16];      // [k part x rank tile][row][16 ranks]
    uint16_t frag[3][kMaxRank / 32][32 * 8];    // then t's parts as the second product takes them
  };
  float t[kNarrowRows][kMaxRank];               // this block's share of x A^T
  float factor[kNarrowRows];
};

template <class T, class TX, class TY>
__global__ void __launch_bounds__(kThreads, 3) narrow_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  Smem& sm = *reinterpret_cast<Smem*>(smem);
  constexpr bool kSplitX = sizeof(TX) == 4;
  constexpr int P = parts_of((const T*)nullptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = cluster_rank(), size = cluster_size();
  pdl_launch_dependents();
  // The plan is older than any kernel that this one may overlap, and what L2 holds
  // follows later writes: B is asked for before the wait.
  const Unit& u = p.units[blockIdx.x / size];
  const int* rows = u.row;
  const int n_per = (p.N + size * kColumns - 1) / (size * kColumns) * kColumns, n0 = min(rank * n_per, p.N), n1 = min(n0 + n_per, p.N);
  if (u.adapter >= 0) prefetch_b(p, static_cast<const T*>(p.b) + u.adapter * p.b_adapter, n0, n1);
  pdl_wait();
  if (u.adapter < 0) {  // a row without an adapter: y as it is
    const TY* y = static_cast<const TY*>(p.y) + rows[0] * p.y_row;
    TY* o = static_cast<TY*>(p.out) + rows[0] * p.out_row;
    constexpr int V = 16 / sizeof(TY);
    const int vectors = p.y_wide && p.out_wide ? (n1 - n0) / V : 0;  // n0 is a multiple of V
#pragma unroll 4
    for (int i = threadIdx.x; i < vectors; i += kThreads)
      reinterpret_cast<uint4*>(o + n0)[i] = reinterpret_cast<const uint4*>(y + n0)[i];
#pragma unroll 4
    for (int n = n0 + vectors * V + threadIdx.x; n < n1; n += kThreads) o[n] = y[n];
    return;
  }
  const int r = p.ranks ? min(max(p.ranks[u.adapter], 0), p.rank) : p.rank;
  const T* A = static_cast<const T*>(p.a) + u.adapter * p.a_adapter;
  const T* B = static_cast<const T*>(p.b) + u.adapter * p.b_adapter;
  const int tiles = (r + 15) / 16, kparts = tiles ? max(kWarps / tiles, 1) : 1;

  // The stream of B's stages of this warp: chunks of 32 columns, in each the ranks
  // by 32.  It starts before x A^T is known.
  const int steps = (r + 31) / 32;
  int next_n = n0 + warp * kColumns, next_s = 0, next_slot = 0;  // the next stage to fetch
  auto fetch = [&]() {
    if (steps && next_n < n1) {
      const int k = next_s * 32 + 8 * t;
      uint8_t* to = sm.ring[warp][next_slot] + t * 16;
      if (k < r) {
        const T* b = B + k;
        if (p.b_wide && k + 8 <= p.rank) {
#pragma unroll
          for (int j = 0; j < kColumns / 8; ++j) cp_async16(to + place_of(j * 8 + g) * 64, b + min(next_n + j * 8 + g, n1 - 1) * p.b_row);
        } else {
#pragma unroll 1
          for (int j = 0; j < kColumns / 8; ++j)
            *reinterpret_cast<uint4*>(to + place_of(j * 8 + g) * 64) = load8(B + min(next_n + j * 8 + g, n1 - 1) * p.b_row, k, r, false);
        }
      }
      next_slot = next_slot + 1 == kStages ? 0 : next_slot + 1;
      if (++next_s == steps) next_s = 0, next_n += kWarps * kColumns;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch();

  // This block's part of T^T: warps share the rank tiles and the K steps.
  {
    const int k_per = ((p.K + size * 32 - 1) / (size * 32)) * 32, k0 = min(rank * k_per, p.K), k1 = min(k0 + k_per, p.K);
    const TX* x = static_cast<const TX*>(p.x) + (g < u.n_rows ? rows[g] : 0) * p.x_row;
    const int part = tiles ? warp / tiles : 0;
    for (int tile = tiles ? warp % tiles : 0; tile < tiles && part < kparts; tile += kWarps) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      const int j0 = tile * 16 + g, j1 = j0 + 8;
      const T *a0 = A + j0 * p.a_row, *a1 = A + j1 * p.a_row;
#pragma unroll 4
      for (int k = k0 + part * 32; k < k1; k += kparts * 32) {
        const int at = k + 8 * t;
        const uint4 v0 = load8(a0, at, j0 < r ? k1 : 0, p.a_wide), v1 = load8(a1, at, j1 < r ? k1 : 0, p.a_wide);
        const int end = g < u.n_rows ? k1 : 0;
        float d[4] = {0.f, 0.f, 0.f, 0.f};
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
            mma8(d, w0, w1, w2, w3, l0, l1);
            mma8(d, w0, w1, w2, w3, h0, h1);
          }
        } else {
          const uint4 xv = load8(reinterpret_cast<const T*>(x), at, end, p.x_wide);
          mma16(d, v0.x, v1.x, v0.y, v1.y, xv.x, xv.y, A);
          mma16(d, v0.z, v1.z, v0.w, v1.w, xv.z, xv.w, A);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += d[i];
      }
      float* o = sm.part + (part * tiles + tile) * (kNarrowRows * 16);
      o[2 * t * 16 + g] = sum[0];
      o[(2 * t + 1) * 16 + g] = sum[1];
      o[2 * t * 16 + g + 8] = sum[2];
      o[(2 * t + 1) * 16 + g + 8] = sum[3];
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
  {
    const int row = warp;
    const float scale = p.scales ? p.scales[u.adapter] : 1.f;
    float v[kMaxRank / 32], top = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxRank / 32; ++i) {
      const int j = i * 32 + lane;
      v[i] = 0.f;
      if (j < r) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < size) v[i] += remote_float(&sm.t[row][j], q);
      }
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

  // Y^T += B T^T over this block's columns, 32 a warp and step.
  const int ra = 2 * t, rb = 2 * t + 1;
  const bool has_a = ra < u.n_rows, has_b = rb < u.n_rows;
  const float fa = sm.factor[ra], fb = sm.factor[rb];
  const TY* py[2] = {static_cast<const TY*>(p.y) + (has_a ? rows[ra] : 0) * p.y_row,
                     static_cast<const TY*>(p.y) + (has_b ? rows[rb] : 0) * p.y_row};
  TY* po[2] = {static_cast<TY*>(p.out) + (has_a ? rows[ra] : 0) * p.out_row,
               static_cast<TY*>(p.out) + (has_b ? rows[rb] : 0) * p.out_row};
  const bool cut = r % 32 != 0;  // what lies behind the rank is cut off
  int slot = 0;
  float ya[4], yb[4];  // of the next columns
  auto load_y = [&](int m) {
    if (has_a && m < n1) load4(py[0], m, n1, p.y_wide, ya);
    if (has_b && m < n1) load4(py[1], m, n1, p.y_wide, yb);
  };
  load_y(n0 + warp * kColumns + 4 * g);
#pragma unroll 1
  for (int n = n0 + warp * kColumns; n < n1; n += kWarps * kColumns) {
    const int m = n + 4 * g;
    float d[2][4] = {};
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(sm.ring[warp][slot] + (j * 8 + g) * 64 + t * 16);
      if (cut) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = first_of(v[j], r - s * 32 - 8 * t);
      }
#pragma unroll
      for (int q = P - 1; q >= 0; --q) {
        const uint4 f = *reinterpret_cast<const uint4*>(&sm.frag[q][s][lane * 8]);
#pragma unroll
        for (int j = 0; j < 2; ++j) mma16(d[j], v[2 * j].x, v[2 * j + 1].x, v[2 * j].y, v[2 * j + 1].y, f.x, f.y, A);
#pragma unroll
        for (int j = 0; j < 2; ++j) mma16(d[j], v[2 * j].z, v[2 * j + 1].z, v[2 * j].w, v[2 * j + 1].w, f.z, f.w, A);
      }
      slot = slot + 1 == kStages ? 0 : slot + 1;
      __syncwarp();
      fetch();
    }
    const float oa[4] = {fmaf(d[0][0], fa, ya[0]), fmaf(d[0][2], fa, ya[1]), fmaf(d[1][0], fa, ya[2]), fmaf(d[1][2], fa, ya[3])};
    const float ob[4] = {fmaf(d[0][1], fb, yb[0]), fmaf(d[0][3], fb, yb[1]), fmaf(d[1][1], fb, yb[2]), fmaf(d[1][3], fb, yb[3])};
    load_y(m + kWarps * kColumns);
    if (has_a) store4(po[0], m, n1, p.out_wide, oa);
    if (has_b) store4(po[1], m, n1, p.out_wide, ob);
  }
  cp_async_wait<0>();
  cluster_wait();
}

template <class T, class TX, class TY>
cudaError_t run(const Params& p, int n_units, int size, cudaStream_t s) {
  const int bytes = (int)sizeof(Smem);
  const cudaError_t e = cudaFuncSetAttribute(narrow_kernel<T, TX, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  return launch_clusters(narrow_kernel<T, TX, TY>, n_units, size, kThreads, bytes, s, p);
}
template <class T>
cudaError_t run(const Params& p, bool x_f32, bool y_f32, int n_units, int size, cudaStream_t s) {
  if (x_f32) return y_f32 ? run<T, float, float>(p, n_units, size, s) : run<T, float, T>(p, n_units, size, s);
  return y_f32 ? run<T, T, float>(p, n_units, size, s) : run<T, T, T>(p, n_units, size, s);
}

}  // namespace

cudaError_t launch_narrow(const Params& p, int type, bool x_f32, bool y_f32, int n_units, int size, cudaStream_t s) {
  if (n_units <= 0) return cudaSuccess;
  return type == T_BF16 ? run<__nv_bfloat16>(p, x_f32, y_f32, n_units, size, s)
                        : run<__half>(p, x_f32, y_f32, n_units, size, s);
}

}  // namespace lora
}  // namespace specb200
