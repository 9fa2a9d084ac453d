// Low-rank adapters, many rows of one adapter: out = y + s (x A^T) B^T for up to
// 64 rows a cluster of blocks.
//
// First product, T [64 x r] = X [64 x K] A^T: the blocks of a cluster share K.  A
// block copies stages of 128 columns of its rows and of A asynchronously into
// shared memory; its warps share the rows (32 each), the ranks (8 NT each) and a
// stage's four slices of 32 columns, and add up what the slices gave at the end.
// The blocks' parts meet in distributed shared memory, each adding up a slice of T
// and all of them collecting the slices.  Second product, Y += T B^T: the
// blocks share N; y and B come in stages of 128 columns in the same way, T's parts
// are the 16-row operand, and B's columns are taken in an order that leaves a lane
// with 8 columns of its rows behind one another.
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
  int RA, stages, bytes;  // ranks' capacity; stages of the first product; of shared memory
};

SPEC_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
SPEC_DEV uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
SPEC_DEV float2 widen2(uint32_t w, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
SPEC_DEV float2 widen2(uint32_t w, const __half*) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Up to 16 bytes from `src`, of which `left` elements are there, to shared memory; zeros behind them.
template <class E>
SPEC_DEV void copy16(uint8_t* dst, const E* src, int left, bool wide) {
  constexpr int N = 16 / sizeof(E);
  if (wide && left >= N) {
    cp_async16(smem_u32(dst), src);
    return;
  }
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < left) {
      if constexpr (N == 4) w[i] = reinterpret_cast<const uint32_t*>(src)[i];
      else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[i] << (i % 2 * 16);
    }
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <class T, class TX, class TY, int NT>
__global__ void __launch_bounds__(kThreads, 2) wide_kernel(const __grid_constant__ WideParams wp) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_factor[kRows];
  __shared__ const void* s_row[kRows];  // the rows of x, from this block's first column on
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
    // Rows behind the last one are copies of it, T's columns behind the adapter's
    // rank whatever the memory holds: neither is used.
    if (threadIdx.x < kRows)
      s_row[threadIdx.x] = static_cast<const TX*>(p.x) + rows[min((int)threadIdx.x, u.n_rows - 1)] * p.x_row + k0;
    __syncthreads();
    const TX* const* xp = reinterpret_cast<const TX* const*>(s_row) + xr;
    const T* ap = A + ar * p.a_row + k0 + ac * 8;
    const long long a_pass = p.a_row * (kThreads / 16);
    // f32: piece c of a slice is columns 4 c ..; half c % 2, place c / 2 of its row.
    const int x_at = xr * 64 + (kSplitX ? xc / 8 * xs + xc % 2 * (kRows * 64) + xc % 8 / 2 * 16 : xc / 4 * xs + xc % 4 * 16);
    const int a_at = ar * 64 + kSlices * xs + ac / 4 * as + ac % 4 * 16;
    const uint32_t base = smem_u32(smem);
    const bool fast = p.x_wide && p.a_wide;
    const int width = k1 - k0;
    int at = 0, k = 0;  // of the next stage to fetch: its offset, its first column
    auto fetch = [&]() {
      const int xk = k + xc * (16 / (int)sizeof(TX));
      const T* a = ap + k;
      if (fast && k + 128 <= width) {
#pragma unroll
        for (int i = 0; i < XN; ++i) cp_async16(base + at + x_at + i * XR * 64, xp[i * XR] + xk);
        for (int j = ar, o = at + a_at; j < r; j += kThreads / 16, o += kThreads / 16 * 64, a += a_pass) cp_async16(base + o, a);
      } else {
#pragma unroll
        for (int i = 0; i < XN; ++i) copy16(smem + at + x_at + i * XR * 64, xp[i * XR] + xk, width - xk, p.x_wide);
        for (int j = ar, o = at + a_at; j < r; j += kThreads / 16, o += kThreads / 16 * 64, a += a_pass)
          copy16(smem + o, a, width - k - ac * 8, p.a_wide);
      }
      k += 128;
      at = at + sb == stages * sb ? 0 : at + sb;
    };
    for (int s = 0; s < stages - 1; ++s) {
      if (s < n_steps) fetch();
      cp_async_commit();
    }
    // Slices of this warp: every turns-th, of 8 turns one of every other stage.
    const int i0 = kg % kSlices, di = turns < kSlices ? turns : kSlices, xo = (mg * 32 + g) * 64 + t * 16,
              ao = kSlices * xs + (nb * NT * 8 + g) * 64 + t * 16;
    const uint8_t* st = smem;
#pragma unroll 1
    for (int step = 0; step < n_steps; ++step) {
      if (stages == 2) cp_async_wait<0>();
      else if (stages == 3) cp_async_wait<1>();
      else cp_async_wait<2>();
      __syncthreads();
      if (step + stages - 1 < n_steps) fetch();
      cp_async_commit();
      if (kg < turns && (turns <= kSlices || (step ^ kg / kSlices) % 2 == 0)) {
#pragma unroll 1
        for (int i = i0; i < kSlices; i += di) {
          const uint8_t *xb = st + i * xs + xo, *ab = st + i * as + ao;
          if constexpr (kSplitX) {
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += 4) {  // four rank tiles at a time
              uint4 a[4];
#pragma unroll
              for (int n = 0; n < 4; ++n) a[n] = lds128(ab + (n0 + n) * 512);
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                // Columns 8 t .. 8 t + 7 of two rows, as hi and lo.
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint4 v = lds128(xb + h * (kRows * 64) + m * 1024), w = lds128(xb + h * (kRows * 64) + m * 1024 + 512);
                  const float x[8] = {__uint_as_float(v.x), __uint_as_float(w.x), __uint_as_float(v.y), __uint_as_float(w.y),
                                      __uint_as_float(v.z), __uint_as_float(w.z), __uint_as_float(v.w), __uint_as_float(w.w)};
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) hi[c] = tf32(x[e * 4 + c]), lo[c] = tf32(rest(x[e * 4 + c], hi[c]));
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                      const uint32_t pair = h ? (e ? a[n].w : a[n].z) : (e ? a[n].y : a[n].x);
                      const float2 f = widen2(pair, A);
                      mma8(d[m][n0 + n], hi[0], hi[1], hi[2], hi[3], __float_as_uint(f.x), __float_as_uint(f.y));
                      mma8(d[m][n0 + n], lo[0], lo[1], lo[2], lo[3], __float_as_uint(f.x), __float_as_uint(f.y));
                    }
                  }
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
      st = st + sb == smem + stages * sb ? smem : st + sb;
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
    // Stages of 128 columns behind T's parts, laid out as those of the first
    // product: y's rows in slices of 32 columns, and for each 32 ranks B's 128
    // columns.  A warp takes the slices of its rows in turn.
    const int ys = x_slice<TY>(), bs = a_slice(128), sb = kSlices * ys + steps * bs;
    uint8_t* ring = smem + (P * steps * frag + 127) / 128 * 128;
    const int stages = min((wp.bytes - (int)(ring - smem)) / sb, 4), n_steps = (n1 - n0 + 127) / 128;
    constexpr int YC = sizeof(TY) == 4 ? 32 : 16, YR = kThreads / YC, YN = kRows / YR;
    const int yc = threadIdx.x % YC, yr = threadIdx.x / YC;
    const int y_at = yr * 64 + (sizeof(TY) == 4 ? yc / 8 * ys + yc % 2 * (kRows * 64) + yc % 8 / 2 * 16 : yc / 4 * ys + yc % 4 * 16);
    const TY* const* yp = reinterpret_cast<const TY* const*>(s_row) + yr;
    if (threadIdx.x < kRows) s_row[threadIdx.x] = static_cast<const TY*>(p.y) + rows[min((int)threadIdx.x, u.n_rows - 1)] * p.y_row + n0;
    __syncthreads();
    const bool fast = p.y_wide && p.b_wide && r % 8 == 0;
    const int width = n1 - n0, pieces = steps * 4;  // of a column of B
    int at = 0, k = 0;
    auto fetch = [&]() {
      const int yk = k + yc * (16 / (int)sizeof(TY));
      const bool whole = fast && k + 128 <= width;
#pragma unroll
      for (int i = 0; i < YN; ++i) {
        uint8_t* to = ring + at + y_at + i * YR * 64;
        if (yr + i * YR >= u.n_rows) continue;
        if (whole) cp_async16(smem_u32(to), yp[i * YR] + yk);
        else copy16(to, yp[i * YR] + yk, width - yk, p.y_wide);
      }
      for (int i = threadIdx.x; i < 128 * pieces; i += kThreads) {
        const int column = i / pieces, piece = i - column * pieces;
        uint8_t* to = ring + at + kSlices * ys + piece / 4 * bs + column * 64 + piece % 4 * 16;
        const T* from = B + (n0 + min(k + column, width - 1)) * p.b_row + piece * 8;
        if (whole && piece * 8 < r) cp_async16(smem_u32(to), from);
        else copy16(to, from, r - piece * 8, p.b_wide);
      }
      k += 128;
      at = at + sb == stages * sb ? 0 : at + sb;
    };
    for (int s = 0; s < stages - 1; ++s) {
      if (s < n_steps) fetch();
      cp_async_commit();
    }
    const int ways = kWarps / groups, ng = warp / groups, first = (warp % groups) * 32 + g;
    TY* op[4];
    float factor[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = first + i * 8;
      op[i] = row < u.n_rows ? static_cast<TY*>(p.out) + rows[row] * p.out_row : nullptr;
      factor[i] = row < u.n_rows ? s_factor[row] : 0.f;
    }
    const uint8_t* st = ring;
#pragma unroll 1
    for (int step = 0; step < n_steps; ++step) {
      if (stages == 2) cp_async_wait<0>();
      else if (stages == 3) cp_async_wait<1>();
      else cp_async_wait<2>();
      __syncthreads();
      if (step + stages - 1 < n_steps) fetch();
      cp_async_commit();
      for (int slice = ng; slice < kSlices; slice += ways) {
        const int n = n0 + step * 128 + slice * 32;
        if (n >= n1) break;
        float d2[2][4][4] = {};
        const uint8_t* bb = st + kSlices * ys + (slice * 32 + g / 2 * 8 + g % 2) * 64 + t * 16;
#pragma unroll 1
        for (int s = 0; s < steps; ++s, bb += bs) {
          uint4 b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = lds128(bb + j * 128);
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
          if (!op[i]) continue;
          float y[8];
          const uint8_t* yb = st + slice * ys + (first + i * 8) * 64 + t * 16;
          if constexpr (sizeof(TY) == 4) {
            const float4 v = *reinterpret_cast<const float4*>(yb), w = *reinterpret_cast<const float4*>(yb + kRows * 64);
            y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w, y[4] = w.x, y[5] = w.y, y[6] = w.z, y[7] = w.w;
          } else {
            widen(lds128(yb), y, A);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[2 * j] = fmaf(d2[i / 2][j][i % 2 * 2], factor[i], y[2 * j]);
            y[2 * j + 1] = fmaf(d2[i / 2][j][i % 2 * 2 + 1], factor[i], y[2 * j + 1]);
          }
          store8(op[i], n + 8 * t, n1, p.out_wide, y);
        }
      }
      st = st + sb == ring + stages * sb ? ring : st + sb;
    }
    cp_async_wait<0>();
  }
  if (size > 1) cluster_wait();
}

template <class T, class TX, class TY, int NT>
cudaError_t run(const Params& p, int n_units, int size, cudaStream_t s) {
  constexpr int B = 8 * NT;
  WideParams w{p, ((p.rank > 1 ? p.rank : 1) + B - 1) / B * B, 0, 0};
  const int stage = stage_bytes<TX>(w.RA);
  // As many stages, up to 4, as let an SM hold two blocks; two at least.
  w.stages = 112 * 1024 / stage;
  w.stages = w.stages > 4 ? 4 : w.stages < 2 ? 2 : w.stages;
  int bytes = w.stages * stage;
  // The warps' parts of T: 32 rows and a block of ranks each; T whole, and the numbers it is split into.
  if (bytes < kWarps * 32 * B * 4) bytes = kWarps * 32 * B * 4;
  if (bytes < kRows * w.RA * 10) bytes = kRows * w.RA * 10;
  // The numbers that T is split into, and two stages of the second product at least.
  const int steps = (w.RA + 31) / 32, second = kSlices * x_slice<TY>() + steps * a_slice(128);
  if (bytes < 3 * steps * kRows * 64 + 2 * second) bytes = 3 * steps * kRows * 64 + 2 * second;
  w.bytes = bytes;
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
