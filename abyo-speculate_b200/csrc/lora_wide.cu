// Low-rank adapters, many rows of one adapter: out = y + s (x A^T) B^T for up to
// 32 rows a cluster of blocks.
//
// First product, T [32 x r] = X [32 x K] A^T: the blocks of a cluster share K, and
// the warps of a block share the ranks (8 NT each) and its columns, 32 at a time.  Every warp copies what it needs
// asynchronously into a ring of its own and waits for nobody else; the warps add
// up at the end.  The blocks' parts meet in distributed shared memory, each adding up
// a slice of T and all of them collecting the slices.  Second product, Y += T
// B^T: the blocks share N, the warps columns, 32 at a time; T's parts are the
// 16-row operand, from shared memory, B and y come straight to registers a tile
// ahead, and B's columns are taken in an order that leaves a lane with 16 bytes of
// its rows next to its neighbour's.  Up to 16 ranks a lane takes 4 of B, not 8 with
// every second one zero.
//
// Pieces of the first product lie as [row][64 bytes], areas 64 bytes further apart
// than they are long, so that neither the copies (16 bytes a lane along a row) nor
// the operands' loads (16 bytes a lane) meet in a bank; f32 rows as two such
// halves, 16-byte pieces in turn.
//
// Two blocks an SM leave 128 registers, of which 12 to 92 bytes a thread spill, and the one
// block of f32 rows of rank above 32 255 (32 bytes).
//
// Bound by latency: 24 requests of 5 to 60 f32 rows (870 in all), rank 16, 4096 to
// 14336: 50 to 55 us, 18 at the copy rate.  x A^T takes about 11, its join 4, the rest moves
// y at 4 TB/s; 64 when y and B came through the warps' rings as well.
#include "lora_mma.cuh"

namespace specb200 {
namespace lora {
namespace {

constexpr int kArea = 32 * 64 + 64;  // 32 rows of 64 bytes
__host__ __device__ constexpr int area(int rows) { return rows * 64 + 64; }

// Shared memory of a block at most; bytes of a slot of a warp's ring; blocks that an SM
// holds by that, two slots a warp at least (f32 rows of rank above 32: 131 KB, one).
constexpr int kMost = 224 * 1024;
template <class TX, int NT>
__host__ __device__ constexpr int slot_bytes() {
  return (int)sizeof(TX) / 2 * kArea + area(8 * NT);
}
template <class TX, int NT>
__host__ __device__ constexpr int blocks_an_sm() {
  return kWarps * 2 * slot_bytes<TX, NT>() <= kMost / 2 ? 2 : 1;
}

struct WideParams {
  Params p;
  int RA, ring, bytes;  // ranks' capacity (a multiple of 8 NT); bytes of a warp's ring in the first product, of shared memory
};

constexpr int kMaxSlots = 6;

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
    cp_async16(dst, src);
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
// Where 16-byte piece c of a row lies: f32 pieces alternate between two halves.
template <class E>
SPEC_DEV int piece_at(int c) {
  return sizeof(E) == 4 ? c % 2 * kArea + c / 2 * 16 : c / 4 * kArea + c % 4 * 16;
}

// 16 bytes of a row from element k on, of n; what lies behind them is left.
template <class E>
SPEC_DEV uint4 load_piece(const E* p, int k, int n) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(E); ++i)
    if (k + i < n) {
      if constexpr (sizeof(E) == 4) w[i] = reinterpret_cast<const uint32_t*>(p)[k + i];
      else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[k + i] << (i % 2 * 16);
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <class E>
SPEC_DEV void store_piece(E* p, int k, int n, const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(E); ++i)
    if (k + i < n) {
      if constexpr (sizeof(E) == 4) reinterpret_cast<uint32_t*>(p)[k + i] = w[i];
      else reinterpret_cast<uint16_t*>(p)[k + i] = (uint16_t)(w[i / 2] >> (i % 2 * 16));
    }
}

template <class T, class TX, class TY, int NT>
__global__ void __launch_bounds__(kThreads, blocks_an_sm<TX, NT>()) wide_kernel(const __grid_constant__ WideParams wp) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_factor[kWideRows];
  __shared__ const void* s_row[kWideRows];  // the rows of x, from this block's first column on
  const Params& p = wp.p;
  constexpr bool kSplitX = sizeof(TX) == 4;
  constexpr int P = parts_of((const T*)nullptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = cluster_rank(), size = cluster_size(), RA = wp.RA;
  pdl_launch_dependents();
  // The plan is older than any kernel that this one may overlap, and what L2 holds
  // follows later writes: B is asked for before the wait, y once x is there.
  const Unit& u = p.units[blockIdx.x / size];
  const int* rows = p.order + u.first;
  const int n_rows = u.n_rows;
  const int n_per = (p.N + size * 32 - 1) / (size * 32) * 32, n0 = min(rank * n_per, p.N), n1 = min(n0 + n_per, p.N), width = n1 - n0;
  prefetch_b(p, static_cast<const T*>(p.b) + u.adapter * p.b_adapter, n0, n1);
  pdl_wait();
  const int r = p.ranks ? min(max(p.ranks[u.adapter], 0), p.rank) : p.rank;
  const T* A = static_cast<const T*>(p.a) + u.adapter * p.a_adapter;
  const T* B = static_cast<const T*>(p.b) + u.adapter * p.b_adapter;
  // Warps: rank blocks of 8 NT, and the rest takes columns in turn.
  const int blocks = max((r + 8 * NT - 1) / (8 * NT), 1), turns = kWarps / blocks;
  const int W = blocks * 8 * NT;  // columns of T
  const int nb = warp % blocks, kg = warp / blocks;

  // ---- T ----
  float d[2][NT][4] = {};
  {
    constexpr int C = 32, XP = C * (int)sizeof(TX) / 16, XR = 32 / XP;  // columns of a piece of work; 16-byte pieces of a row; rows a pass
    constexpr int XA = XP / 4 * kArea, kSlot = slot_bytes<TX, NT>();
    const int k_per = (p.K + size * C - 1) / (size * C) * C, k0 = min(rank * k_per, p.K), k1 = min(k0 + k_per, p.K), length = k1 - k0;
    if (threadIdx.x < kWideRows)
      s_row[threadIdx.x] = static_cast<const TX*>(p.x) + rows[min((int)threadIdx.x, n_rows - 1)] * p.x_row + k0;
    __syncthreads();
    // Rows behind the last one are copies of it, T's columns behind the adapter's
    // rank whatever the memory holds: neither is used.
    const TX* const* xp = reinterpret_cast<const TX* const*>(s_row) + lane / XP;
    constexpr int AP = C / 8, AR = 32 / AP;  // 16-byte pieces of a rank's columns; ranks a pass
    const int ranks = min(r - nb * NT * 8, NT * 8);
    const T* ap = A + (nb * NT * 8 + lane / AP) * p.a_row + k0 + lane % AP * 8;
    uint8_t* ring = smem + warp * wp.ring;
    const int slots = min(wp.ring / kSlot, kMaxSlots);
    const bool fast = p.x_wide && p.a_wide;
    int next = kg < turns && r ? kg * C : length, at = 0;  // the next to fetch: its first column, its slot
    auto fetch = [&]() {
      if (next < length) {
        uint8_t* to = ring + at + piece_at<TX>(lane % XP) + lane / XP * 64;
        const int xk = next + lane % XP * (16 / (int)sizeof(TX));
        uint8_t* ta = ring + at + XA + lane % AP * 16 + lane / AP * 64;
        const T* a = ap + next;
        if (fast && next + C <= length) {
#pragma unroll
          for (int i = 0; i < XP; ++i) cp_async16(to + i * XR * 64, xp[i * XR] + xk);
#pragma unroll
          for (int i = 0; i < NT * 8 / AR; ++i)
            if (lane / AP + i * AR < ranks) cp_async16(ta + i * AR * 64, a + i * AR * p.a_row);
        } else {
#pragma unroll 1
          for (int i = 0; i < XP; ++i) copy16(to + i * XR * 64, xp[i * XR] + xk, length - xk, p.x_wide);
#pragma unroll 1
          for (int i = 0; i < NT * 8 / AR; ++i)
            if (lane / AP + i * AR < ranks) copy16(ta + i * AR * 64, a + i * AR * p.a_row, length - next - lane % AP * 8, p.a_wide);
        }
        next += turns * C;
        at = at + kSlot == slots * kSlot ? 0 : at + kSlot;
      }
      cp_async_commit();
    };
    for (int i = 0; i < slots - 1; ++i) fetch();
    const uint8_t* st = ring;
#pragma unroll 1
    for (int k = kg < turns && r ? kg * C : length; k < length; k += turns * C) {
      cp_async_wait_for(slots - 2);
      __syncwarp();
      fetch();
      const uint8_t *xb = st + g * 64 + t * 16, *ab = st + XA + g * 64 + t * 16;
      if constexpr (kSplitX) {
#pragma unroll
        for (int n0 = 0; n0 < NT; n0 += 4) {  // four rank tiles at a time
          uint4 a[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) a[n] = lds128(ab + (n0 + n) * 512);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            // Columns 8 t .. 8 t + 7 of two rows, as hi and lo.
            float sum[4][4] = {};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 v = lds128(xb + h * kArea + m * 1024), w = lds128(xb + h * kArea + m * 1024 + 512);
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
                  mma8(sum[n], lo[0], lo[1], lo[2], lo[3], __float_as_uint(f.x), __float_as_uint(f.y));
                  mma8(sum[n], hi[0], hi[1], hi[2], hi[3], __float_as_uint(f.x), __float_as_uint(f.y));
                }
              }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) d[m][n0 + n][i] += sum[n][i];
          }
        }
      } else {
        uint4 x[2][2];
#pragma unroll
        for (int m = 0; m < 2; ++m) x[m][0] = lds128(xb + m * 1024), x[m][1] = lds128(xb + m * 1024 + 512);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 a = lds128(ab + n * 512);
          float sum[2][4] = {};
#pragma unroll
          for (int m = 0; m < 2; ++m) mma16(sum[m], x[m][0].x, x[m][1].x, x[m][0].y, x[m][1].y, a.x, a.y, A);
#pragma unroll
          for (int m = 0; m < 2; ++m) mma16(sum[m], x[m][0].z, x[m][1].z, x[m][0].w, x[m][1].w, a.z, a.w, A);
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[m][n][i] += sum[m][i];
        }
      }
      __syncwarp();
      st = st + kSlot == ring + slots * kSlot ? ring : st + kSlot;
    }
    cp_async_wait<0>();
    if (threadIdx.x < n_rows) prefetch(static_cast<const TY*>(p.y) + rows[threadIdx.x] * p.y_row + n0, width);
    __syncthreads();
  }

  // ---- the parts of T join ----
  // `part`: this block's T; `all`: the cluster's; then, in part's place, the
  // numbers that T is split into.
  float* part = reinterpret_cast<float*>(smem);
  float* all = reinterpret_cast<float*>(smem + kWideRows * RA * 6);
  const int live = kWideRows * W;
  if (kg < turns) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* o = part + kg * live + (m * 16 + g) * W + nb * NT * 8 + n * 8 + 2 * t;
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
  const int steps = (r + 31) / 32, frag = kWideRows * 64;  // bytes of one part's 32 ranks
  if (threadIdx.x < kWideRows * 4) {                 // four threads a row
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

  if (size > 1) cluster_wait();  // nor anything of this one: the rings may take its place

  // ---- Y ----
  {
    constexpr int V = (int)sizeof(TY) / 2;  // 16-byte pieces of 8 columns
    const bool half = r <= 16, cut = r % (half ? 4 : 8) != 0, b_fast = p.b_wide && p.rank % 8 == 0;
    const int per = half ? 4 : 8;  // ranks a lane takes of a step
    const TY* y0 = static_cast<const TY*>(p.y) + n0;
    TY* out0 = static_cast<TY*>(p.out) + n0;
    int at[4];  // the lane's rows, -1: none
    float factor[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = g + i * 8;
      at[i] = row < n_rows ? rows[row] : -1;
      factor[i] = s_factor[row];
    }
    // Where a lane's 8 columns of a row lie: 8 t .. (16-bit), or 4 t .. and 16 + 4 t .. (f32);
    // and so the column of B that is its operand of tile j.
    auto column_of = [&](int j) {
      return sizeof(TY) == 4 ? j / 2 * 16 + g / 2 * 4 + j % 2 * 2 + g % 2 : g / 2 * 8 + j * 2 + g % 2;
    };
    uint4 y[4][V], b[4];  // of the next tile of 32 columns, of the next 32 ranks of it
    auto load_y = [&](int n) {
      if (n >= width) return;
      if (p.y_wide && n + 32 <= width) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (at[i] >= 0) y[i][v] = *reinterpret_cast<const uint4*>(y0 + at[i] * p.y_row + n + (V == 2 ? 16 * v + 4 * t : 8 * t));
        return;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (at[i] >= 0) y[i][v] = load_piece(y0 + at[i] * p.y_row, n + (V == 2 ? 16 * v + 4 * t : 8 * t), width);
    };
    auto load_b = [&](int n, int s) {
      const int k = s * 32 + per * t;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        b[j] = make_uint4(0u, 0u, 0u, 0u);
        if (k >= r || n >= width) continue;
        const T* q = B + (n0 + min(n + column_of(j), width - 1)) * p.b_row;
        if (!b_fast) {
          b[j] = load8(q, k, min(r, k + per), false);
        } else if (half) {
          const uint2 w = *reinterpret_cast<const uint2*>(q + k);
          b[j].x = w.x, b[j].y = w.y;
        } else {
          b[j] = *reinterpret_cast<const uint4*>(q + k);
        }
      }
    };
    const int begin = warp * 32;
    load_b(begin, 0);
    load_y(begin);
#pragma unroll 1
    for (int n = begin; n < width; n += kWarps * 32) {
      float d2[2][4][4] = {};
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        if (cut) {
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = first_of(b[j], r - s * 32 - per * t);
        }
#pragma unroll
        for (int q = P - 1; q >= 0; --q) {
          const uint8_t* f = smem + (q * steps + s) * frag + g * 64 + per * 2 * t;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            if (half) {
              const uint2 x0 = *reinterpret_cast<const uint2*>(f + m * 1024), x1 = *reinterpret_cast<const uint2*>(f + m * 1024 + 512);
#pragma unroll
              for (int j = 0; j < 4; ++j) mma16(d2[m][j], x0.x, x1.x, x0.y, x1.y, b[j].x, b[j].y, A);
            } else {
              const uint4 x0 = lds128(f + m * 1024), x1 = lds128(f + m * 1024 + 512);
#pragma unroll
              for (int j = 0; j < 4; ++j) mma16(d2[m][j], x0.x, x1.x, x0.y, x1.y, b[j].x, b[j].y, A);
#pragma unroll
              for (int j = 0; j < 4; ++j) mma16(d2[m][j], x0.z, x1.z, x0.w, x1.w, b[j].z, b[j].w, A);
            }
          }
        }
        if (s + 1 < steps) load_b(n, s + 1);
        else load_b(n + kWarps * 32, 0);
      }
      const bool whole = p.out_wide && n + 32 <= width;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[8];
        if constexpr (sizeof(TY) == 4) {
#pragma unroll
          for (int h = 0; h < V; ++h) {
            v[4 * h] = __uint_as_float(y[i][h].x), v[4 * h + 1] = __uint_as_float(y[i][h].y);
            v[4 * h + 2] = __uint_as_float(y[i][h].z), v[4 * h + 3] = __uint_as_float(y[i][h].w);
          }
        } else {
          widen(y[i][0], v, A);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = fmaf(d2[i / 2][j][i % 2 * 2], factor[i], v[2 * j]);
          v[2 * j + 1] = fmaf(d2[i / 2][j][i % 2 * 2 + 1], factor[i], v[2 * j + 1]);
        }
        if constexpr (sizeof(TY) == 4) {
#pragma unroll
          for (int h = 0; h < V; ++h)
            y[i][h] = make_uint4(__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3]));
        } else {
          y[i][0] = make_uint4(pack2(v[0], v[1], A), pack2(v[2], v[3], A), pack2(v[4], v[5], A), pack2(v[6], v[7], A));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < V; ++h) {
          const int c = n + (V == 2 ? 16 * h + 4 * t : 8 * t);
          if (at[i] < 0) continue;
          TY* o = out0 + at[i] * p.out_row;
          if (whole) *reinterpret_cast<uint4*>(o + c) = y[i][h];
          else store_piece(o, c, width, y[i][h]);
        }
      load_y(n + kWarps * 32);
    }
  }
}

template <class T, class TX, class TY, int NT>
cudaError_t run(const Params& p, int n_units, int sms, cudaStream_t s) {
  constexpr int B = 8 * NT, kFit = blocks_an_sm<TX, NT>();
  WideParams w{p, ((p.rank > 1 ? p.rank : 1) + B - 1) / B * B, 0, 0};
  // Two blocks an SM where they fit and there are many: alone on an SM, clusters of 8
  // leave part of a GPC's SMs empty (16 of them, one an SM: 20 us, two 11).  Clusters for two
  // where one fits run as two waves (f32 rows, 16 adapters of 128 rows of rank 64: 86 us,
  // 78 so; 16 of 64 rows of rank 128: 117, 71).  Besides the rings a block holds
  // the warps' parts of T, 32 rows and a block of ranks each; T whole behind the numbers
  // that it is split into.
  static_assert(kWarps * 2 * slot_bytes<TX, NT>() <= kMost && kWarps * 32 * B * 4 <= kMost / 2 &&
                kWideRows * kMaxRank * 10 <= kMost / 2 && 3 * kWideRows * kMaxRank * 2 <= kMost / 2, "");
  // The kernel's limit is the process's: one number, which no other thread's call lowers before the launch.
  cudaError_t e = cudaFuncSetAttribute(wide_kernel<T, TX, TY, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
  int size = 1;
  if (e == cudaSuccess) e = cluster_for(wide_kernel<T, TX, TY, NT>, n_units, kThreads, kMost / kFit, &size);
  if (e != cudaSuccess) return e;
  const int bytes = kFit == 2 && (long long)n_units * size * 2 > sms ? kMost / 2 : kMost;
  w.ring = bytes / kWarps / 16 * 16;
  w.bytes = bytes;
  return launch_clusters(wide_kernel<T, TX, TY, NT>, n_units, size, kThreads, bytes, s, w);
}
template <class T, class TX, class TY>
cudaError_t run(const Params& p, int n_units, int sms, cudaStream_t s) {
  return p.rank <= 32 ? run<T, TX, TY, 4>(p, n_units, sms, s) : run<T, TX, TY, 8>(p, n_units, sms, s);
}
template <class T>
cudaError_t run(const Params& p, bool x_f32, bool y_f32, int n_units, int sms, cudaStream_t s) {
  if (x_f32) return y_f32 ? run<T, float, float>(p, n_units, sms, s) : run<T, float, T>(p, n_units, sms, s);
  return y_f32 ? run<T, T, float>(p, n_units, sms, s) : run<T, T, T>(p, n_units, sms, s);
}

}  // namespace

cudaError_t launch_wide(const Params& p, int type, bool x_f32, bool y_f32, int n_units, int sms, cudaStream_t s) {
  if (n_units <= 0) return cudaSuccess;
  return type == T_BF16 ? run<__nv_bfloat16>(p, x_f32, y_f32, n_units, sms, s)
                        : run<__half>(p, x_f32, y_f32, n_units, sms, s);
}

}  // namespace lora
}  // namespace specb200
