// Low-rank adapters, very many rows of one adapter: out = y + s (x A^T) B^T for up
// to 128 rows a cluster of blocks, on tcgen05 with accumulators in tensor memory.
//
// First product, T [128 x N] = X [128 x K] A^T (N: the rank up to a multiple of
// 16): the blocks of a cluster share K; stages of 128 columns of the rows and of A
// are copied asynchronously into the K-major operand layout of 128-byte rows
// whose 16-byte pieces are swizzled (piece c of row i lies at c ^ (i % 8)), so that
// 8 lanes copy 128 bytes of one row, and one thread issues the stage's 8 products;
// their operands' addresses are sums with constants, as each step of arithmetic there delays
// the whole block (put together anew: 16 us of the case below).
// An accumulator adds up two stages, two accumulators in turn, and goes from there to
// f32 additions in registers (the case below: error 3.3e-7 of the adapters' share;
// one stage 2.5e-7 and 2.5 us longer; all of them 81e-7 and 2 us less).  The blocks'
// parts join as in the kernel for fewer rows.  Second product: T's numbers are the
// 128-row operand, in tensor memory (in shared memory 126 us, not 120, and 237, not 206,
// for 14336 output channels), B's 64 columns a stage the other; while a stage's products
// run, all threads add the stage before it to y, which came with B into rows 16
// bytes further apart than they are long, and store it along the rows.
//
// x has the adapters' type.  8100 rows of rank 64, 14336 to 4096 channels in bf16: 120
// us (55 at the copy rate), about 75 of them the first product, which brings 350 MB of x and
// A at 4.7 TB/s, bound by the copies' 16-byte pieces in the load units; in the
// second, 133 MB of y and out and the load units again.  On mma.sync 146 us.
#include "lora_mma.cuh"

namespace specb200 {
namespace lora {
namespace {

constexpr int kTallThreads = 512, kTallWarps = kTallThreads / 32;
constexpr int kStep = 128;        // columns of a stage of the first product
constexpr int kCols = 64;         // and of the second
constexpr int kMaxStages = 6;
constexpr int kChain = 2;         // stages that one accumulator adds up
// Columns of tensor memory: two accumulators of the first product, in whose place two of
// the second come, then the numbers that T is split into, two a column.
constexpr int kTmem = 512, kParts = 256;

struct TallParams {
  Params p;
  unsigned* err;
  int N, stages, stages2, all_at;  // ring sizes; where T whole lies
};

// Operands lie in blocks of 64 columns: rows of 128 bytes.
SPEC_DEV int swizzled(int row, int piece) { return row * 128 + (piece ^ (row & 7)) * 16; }
// Descriptor of a block: 8-row groups 1024 bytes apart, 128-byte swizzle; 16
// columns further on are 32 bytes.
SPEC_DEV uint64_t block_desc(uint32_t at) { return umma_desc_kmajor(at, 16, 1024) | (2ull << 61); }
__host__ __device__ constexpr int blocks_of(int N) { return (N + 63) / 64; }

template <class TY>
__host__ __device__ constexpr int y_pitch() {
  return kCols * (int)sizeof(TY) + 16;
}
template <class TY>
__host__ __device__ constexpr int stage2(int N) {
  return (kTallRows * y_pitch<TY>() + 1023) / 1024 * 1024 + blocks_of(N) * kCols * 128;
}
__host__ __device__ constexpr int stage1(int N) { return kStep / 64 * (kTallRows * 128 + (N * 128 + 1023) / 1024 * 1024); }

SPEC_DEV uint32_t idesc(int N, const __nv_bfloat16*) { return umma_idesc_bf16(128, N); }
SPEC_DEV uint32_t idesc(int N, const __half*) { return umma_idesc_bf16(128, N) & ~((7u << 7) | (7u << 10)); }  // formats 0: f16

// 8 columns of tensor memory of this thread's row, there after tmem_wait_ld.
SPEC_DEV void tmem_ld8(uint32_t at, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(at)
               : "memory");
}
SPEC_DEV void tmem_st4(uint32_t at, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}
SPEC_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (+)= A B^T with A [128 x 16] in tensor memory, a row a lane, two numbers a column.
SPEC_DEV void umma_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
SPEC_DEV void publish_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Up to 8 elements from `src`, of which `left` are there, to shared memory; zeros behind them.
template <class T>
SPEC_DEV void copy8(uint8_t* dst, const T* src, int left, bool wide) {
  if (wide && left >= 8) {
    cp_async16(dst, src);
    return;
  }
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[i] << (i % 2 * 16);
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

SPEC_DEV void unpack16(const uint8_t* p, float (&x)[4], const float*) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <class T>
SPEC_DEV void unpack16(const uint8_t* p, float (&x)[8], const T* tag) {
  widen(*reinterpret_cast<const uint4*>(p), x, tag);
}
SPEC_DEV void pack16(uint8_t* p, const float (&x)[4], const float*) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <class T>
SPEC_DEV void pack16(uint8_t* p, const float (&x)[8], const T* tag) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1], tag), pack2(x[2], x[3], tag), pack2(x[4], x[5], tag), pack2(x[6], x[7], tag));
}

template <class T, class TY>
__global__ void __launch_bounds__(kTallThreads, 1) tall_kernel(const __grid_constant__ TallParams tp) {
  extern __shared__ __align__(128) uint8_t dynamic[];
  uint8_t* smem = dynamic + (1024 - smem_u32(dynamic) % 1024) % 1024;  // the same in every block of the cluster
  __shared__ uint64_t s_free[kMaxStages], s_done[2];
  __shared__ uint32_t s_tmem;
  __shared__ const TY* s_row[kTallRows];
  const Params& p = tp.p;
  constexpr int P = parts_of((const T*)nullptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), size = cluster_size(), N = tp.N;
  pdl_launch_dependents();
  pdl_wait();
  const Unit& u = p.units[blockIdx.x / size];
  const int* rows = p.order + u.first;
  const int n_rows = u.n_rows;
  const int r = p.ranks ? min(max(p.ranks[u.adapter], 0), p.rank) : p.rank;
  const T* A = static_cast<const T*>(p.a) + u.adapter * p.a_adapter;
  const T* B = static_cast<const T*>(p.b) + u.adapter * p.b_adapter;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxStages; ++i) mbar_init(&s_free[i], 1);
    mbar_init(&s_done[0], 1);
    mbar_init(&s_done[1], 1);
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(&s_tmem, kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  bool ok = true;  // no wait gave up

  // ---- T ----
  float* part = reinterpret_cast<float*>(smem);
  const int Wp = N + 4;  // floats between T's rows
  {
    const int k_per = (p.K + size * kStep - 1) / (size * kStep) * kStep, k0 = min(rank * k_per, p.K), k1 = min(k0 + k_per, p.K);
    const int width = k1 - k0, n_steps = r ? (width + kStep - 1) / kStep : 0, stages = tp.stages, sb = stage1(N);
    constexpr int xb = kTallRows * 128;             // bytes of a block of x, and of A
    const int ab = (N * 128 + 1023) / 1024 * 1024;
    // Rows of this lane: two of the warp's 8.  Rows behind the last one are
    // copies of it, T's columns behind the adapter's rank whatever the memory
    // holds: neither is used.
    const int row0 = warp * 8 + lane / 8, piece = lane % 8;
    const T* x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      x[i] = static_cast<const T*>(p.x) + rows[min(row0 + i * 4, n_rows - 1)] * p.x_row + k0 + piece * 8;
    const int a_row = warp * 4 + lane / 8;
    const T* a0 = A + a_row * p.a_row + k0 + piece * 8;
    const bool fast = p.x_wide && p.a_wide;
    int next = 0, at = 0;  // of the next stage to fetch: its first column, its offset
    auto fetch = [&]() {
      const bool whole = fast && next + kStep <= width;
#pragma unroll
      for (int q = 0; q < kStep / 64; ++q) {
        const int k = next + q * 64, left = width - k - piece * 8;
        uint8_t* to = smem + at + q * xb;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (whole) cp_async16(to + swizzled(row0 + i * 4, piece), x[i] + k);
          else copy8(to + swizzled(row0 + i * 4, piece), x[i] + k, left, p.x_wide);
        }
        to = smem + at + kStep / 64 * xb + q * ab;
        const T* a = a0 + k;
        for (int j = a_row; j < r; j += kTallWarps * 4, a += kTallWarps * 4 * p.a_row) {
          if (whole) cp_async16(to + swizzled(j, piece), a);
          else copy8(to + swizzled(j, piece), a, left, p.a_wide);
        }
      }
      next += kStep;
      at = at + sb == stages * sb ? 0 : at + sb;
    };
    for (int s = 0; s < stages - 1; ++s) {
      if (s < n_steps) fetch();
      cp_async_commit();
    }
    const uint32_t id = idesc(N, A), base = smem_u32(smem);
    // A warp adds up 32 rows, 8 columns in 32, of two accumulators in turn.
    float sum[kMaxRank / 32][8] = {};
    const uint32_t lanes = tmem + ((uint32_t)(warp % 4 * 32) << 16) + warp / 4 * 8;
    auto add = [&](int chain) {
      tc_fence_after();
      const uint32_t from = lanes + chain % 2 * 128;
#pragma unroll
      for (int i = 0; i < kMaxRank / 32; i += 2) {
        if (i * 32 >= N) break;
        uint32_t v[2][8];
        tmem_ld8(from + i * 32, v[0]);
        tmem_ld8(from + i * 32 + 32, v[1]);
        tmem_wait_ld();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            asm volatile("" : "+r"(v[h][k]));
            sum[i + h][k] += __uint_as_float(v[h][k]);
          }
      }
      tc_fence_before();
    };
    int slot = 0, phase = 0;  // of this step; phase: of the slot before it
#pragma unroll 1
    for (int step = 0; step < n_steps; ++step) {
      cp_async_wait_for(stages - 2);
      publish_smem();
      ok = __syncthreads_and(ok);
      if (!ok) break;
      if (threadIdx.x == 0) {
        tc_fence_after();
        const uint64_t xs = block_desc(base + slot * sb), as = block_desc(base + slot * sb + kStep / 64 * xb);
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k)
          umma_bf16(tmem + step / kChain % 2 * 128, xs + (k / 4 * xb + k % 4 * 32) / 16, as + (k / 4 * ab + k % 4 * 32) / 16, id, step % kChain | k);
        umma_commit(&s_free[slot]);
      }
      // The slot before this one is filled again once its products are done.
      if (step > 0) {
        const int before = slot ? slot - 1 : stages - 1;
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_free[before], phase, tp.err));
        if (before == stages - 1) phase ^= 1;
      }
      if (step + stages - 1 < n_steps && ok) fetch();
      cp_async_commit();
      if (step > 0 && step % kChain == 0) add(step / kChain - 1);
      slot = slot + 1 == stages ? 0 : slot + 1;
    }
    ok = __syncthreads_and(ok);
    if (n_steps && ok) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_free[slot ? slot - 1 : stages - 1], phase, tp.err));
      add((n_steps - 1) / kChain);
    }
    cp_async_wait<0>();
    ok = __syncthreads_and(ok);
    float* o = part + (warp % 4 * 32 + lane) * Wp + warp / 4 * 8;
#pragma unroll
    for (int i = 0; i < kMaxRank / 32; ++i) {
      if (warp / 4 * 8 + i * 32 >= N) break;
      *reinterpret_cast<float4*>(o + i * 32) = make_float4(sum[i][0], sum[i][1], sum[i][2], sum[i][3]);
      *reinterpret_cast<float4*>(o + i * 32 + 4) = make_float4(sum[i][4], sum[i][5], sum[i][6], sum[i][7]);
    }
    __syncthreads();
  }

  // ---- the parts of T join ----
  float* all = reinterpret_cast<float*>(smem + tp.all_at);
  const int live = kTallRows * Wp;
  cluster_arrive();
  cluster_wait();
  const int share = (live / 4 + size - 1) / size * 4;
  for (int i = rank * share + threadIdx.x * 4; i < min((rank + 1) * share, live); i += kTallThreads * 4) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < size; ++q) {
      const float4 v = remote_float4(part + i, q);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    *reinterpret_cast<float4*>(all + i) = s;
  }
  cluster_arrive();
  cluster_wait();
  for (int i = threadIdx.x * 4; i < live; i += kTallThreads * 4)
    if (i / share != rank) *reinterpret_cast<float4*>(all + i) = remote_float4(all + i, i / share);
  cluster_arrive();  // nothing of the other blocks is read any more
  __syncthreads();
  // The numbers that T is split into, four threads a row, to tensor memory.
  const int my_row = warp % 4 * 32 + lane;
  float factor;
  {
    const int h = warp / 4;
    const float scale = p.scales ? p.scales[u.adapter] : 1.f;
    float* mine = all + my_row * Wp;
    float top = 0.f;
    for (int j = h * 8; j < r; j += 32)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (j + k < r) top = fmaxf(top, fabsf(mine[j + k] * scale));
    mine[N + h] = top;  // the rows' pads: nothing else of them is read
    __syncthreads();
    top = fmaxf(fmaxf(mine[N], mine[N + 1]), fmaxf(mine[N + 2], mine[N + 3]));
    const int e = exponent(top, A);
    const float down = pow2i(-e);
    factor = pow2i(e);
    const uint32_t to = tmem + ((uint32_t)(warp % 4 * 32) << 16) + kParts;
    for (int j = h * 8; j < N; j += 32) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = j + k < r ? mine[j + k] * scale * down : 0.f;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w[k] = pack2(v[2 * k], v[2 * k + 1], A);
          T hl[2];
          *reinterpret_cast<uint32_t*>(hl) = w[k];
          v[2 * k] = fabsf(v[2 * k]) < INFINITY ? v[2 * k] - to_float(hl[0]) : 0.f;
          v[2 * k + 1] = fabsf(v[2 * k + 1]) < INFINITY ? v[2 * k + 1] - to_float(hl[1]) : 0.f;
        }
        tmem_st4(to + (q * N + j) / 2, w);
      }
    }
    tmem_wait_st();
    tc_fence_before();
  }
  cluster_wait();  // nor anything of this one
  __syncthreads();

  // ---- Y ----
  if (ok) {
    const int n_per = (p.N + size * kCols - 1) / (size * kCols) * kCols, n0 = min(rank * n_per, p.N), n1 = min(n0 + n_per, p.N);
    const int width = n1 - n0, n_steps = (width + kCols - 1) / kCols, stages = tp.stages2, sb = stage2<TY>(N);
    constexpr int YP = kCols * (int)sizeof(TY) / 16, YR = 32 / YP, YN = kTallRows / kTallWarps / YR, E = 16 / (int)sizeof(TY);
    uint8_t* ring = smem;  // `all` is not used any more
    if (threadIdx.x < kTallRows) s_row[threadIdx.x] = static_cast<const TY*>(p.y) + rows[min((int)threadIdx.x, n_rows - 1)] * p.y_row + n0;
    __syncthreads();
    TY* out[YN];  // where this thread stores
#pragma unroll
    for (int i = 0; i < YN; ++i) {
      const int row = warp * (kTallRows / kTallWarps) + lane / YP + i * YR;
      out[i] = row < n_rows ? static_cast<TY*>(p.out) + rows[row] * p.out_row + n0 + lane % YP * E : nullptr;
    }
    const bool fast = p.y_wide && p.b_wide && r % 8 == 0;
    constexpr int yb = (kTallRows * y_pitch<TY>() + 1023) / 1024 * 1024;  // bytes of a stage's y
    const int y_row = warp * (kTallRows / kTallWarps) + lane / YP, y_at = y_row * y_pitch<TY>() + lane % YP * 16;
    int next = 0, at = 0;
    auto fetch = [&]() {
      const bool whole = fast && next + kCols <= width;
      const int yk = next + lane % YP * E;
#pragma unroll
      for (int i = 0; i < YN; ++i) {
        uint8_t* to = ring + at + y_at + i * YR * y_pitch<TY>();
        const TY* from = s_row[y_row + i * YR] + yk;
        if (whole) {
          cp_async16(to, from);
        } else if (p.y_wide && yk + E <= width) {
          cp_async16(to, from);
        } else {
#pragma unroll 1
          for (int e = 0; e < E; ++e)
            if (yk + e < width) reinterpret_cast<TY*>(to)[e] = from[e];
        }
      }
      // B: ranks behind the adapter's are zeros, columns behind the last one copies of it.
      for (int i = warp * 4 + lane / 8; i < blocks_of(N) * kCols; i += kTallWarps * 4) {
        const int k = i / kCols * 64 + lane % 8 * 8, column = i % kCols;
        if (k >= N) continue;
        const T* from = B + (n0 + min(next + column, width - 1)) * p.b_row + k;
        uint8_t* to = ring + at + yb + i / kCols * (kCols * 128) + swizzled(column, lane % 8);
        if (whole && k < r) cp_async16(to, from);
        else copy8(to, from, r - k, p.b_wide);
      }
      next += kCols;
      at = at + sb == stages * sb ? 0 : at + sb;
    };
    for (int s = 0; s < stages - 2; ++s) {
      if (s < n_steps) fetch();
      cp_async_commit();
    }
    const uint32_t id = idesc(kCols, A);
    int slot = 0;
    // One step more than there are stages: the last one only finishes.
#pragma unroll 1
    for (int step = 0; step <= n_steps; ++step) {
      cp_async_wait_for(stages - 3);
      publish_smem();
      ok = __syncthreads_and(ok);  // also: the stage before is stored
      if (!ok) break;
      if (threadIdx.x == 0 && step < n_steps && r) {
        tc_fence_after();
        const uint32_t to = tmem + step % 2 * kCols;
        const uint64_t b = block_desc(smem_u32(ring) + slot * sb + yb);
#pragma unroll
        for (int q = P - 1; q >= 0; --q) {  // the small parts first
          const uint32_t from = tmem + kParts + q * N / 2;
          int k = 0;
#pragma unroll 1
          for (; k + 64 <= N; k += 64)
#pragma unroll
            for (int i = 0; i < 4; ++i) umma_from_tmem(to, from + k / 2 + i * 8, b + k * (kCols * 2) / 16 + i * 2, id, q < P - 1 || k + i);
#pragma unroll 1
          for (; k < N; k += 16) umma_from_tmem(to, from + k / 2, b + k / 64 * (kCols * 128 / 16) + k % 64 / 8, id, q < P - 1 || k);
        }
        umma_commit(&s_done[step % 2]);
      }
      // The slot of two steps ago is free.
      if (step + stages - 2 < n_steps) fetch();
      cp_async_commit();
      if (step > 0) {
        const int before = slot ? slot - 1 : stages - 1, n = (step - 1) * kCols;
        uint8_t* st = ring + before * sb;
        if (r) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_done[(step - 1) % 2], (step - 1) / 2 % 2, tp.err));
          tc_fence_after();
          uint32_t v[16];
          tmem_ld16(tmem + ((uint32_t)(warp % 4 * 32) << 16) + (step - 1) % 2 * kCols + warp / 4 * 16, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(v[i])::"memory");
          tc_fence_before();
          uint8_t* y = st + my_row * y_pitch<TY>() + warp / 4 * 16 * (int)sizeof(TY);
#pragma unroll
          for (int i = 0; i < 16 / E; ++i) {
            float f[E];
            unpack16(y + i * 16, f, (const TY*)nullptr);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = fmaf(__uint_as_float(v[i * E + e]), factor, f[e]);
            pack16(y + i * 16, f, (const TY*)nullptr);
          }
        }
        __syncthreads();
        const bool whole = p.out_wide && n + kCols <= width;
#pragma unroll
        for (int i = 0; i < YN; ++i) {
          if (!out[i]) continue;
          TY* o = out[i] + n;
          const uint8_t* v = st + y_at + i * YR * y_pitch<TY>();
          if (whole) {
            *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(v);
          } else {
#pragma unroll 1
            for (int e = 0; e < E; ++e)
              if (n + lane % YP * E + e < width) o[e] = reinterpret_cast<const TY*>(v)[e];
          }
        }
      }
      slot = slot + 1 == stages ? 0 : slot + 1;
    }
    cp_async_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, kTmem);
}

// Shared memory for N columns of T, besides what aligns it to 1024 bytes.
constexpr int kMost = 222 * 1024;
__host__ __device__ constexpr int whole(int N) { return kTallRows * (N + 4) * 4; }
template <class TY>
TallParams plan_memory(const Params& p, unsigned* err, int N) {
  static_assert(kMost >= 2 * stage1(kMaxRank) && kMost >= 3 * stage2<TY>(kMaxRank) && kMost >= 2 * whole(kMaxRank), "");
  const int stages = kMost / stage1(N), stages2 = kMost / stage2<TY>(N);
  return TallParams{p, err, N, stages < kMaxStages ? stages : kMaxStages, stages2 < kMaxStages ? stages2 : kMaxStages, whole(N)};
}

// Taken where the clusters, resident all at once, have at least half of the SMs; two waves
// of them, or a few, are slower than units of 32 rows, two an SM.  us of units of 128 / of 32, for rank 64
// 8192 to 2048 channels, the same 14336 to 4096, and rank 16 4096 to 4096, in bf16: 8 units of 128 25 /
// 21, 38 / 30, 22 / 19; 10 25 / 31, 38 / 47, 22 / 22; 16 in clusters of 8 49 / 31, 74 / 47, 43 / 23; 20
// in clusters of 4 39 / 50, 65 / 82, 36 / 35; 36 so 77 / 51, 127 / 85, 70 / 39; 50 69 / 86, 119 / 152, 65 / 66.
template <class T, class TY>
cudaError_t run(const Params& p, unsigned* err, int n_units, int sms, cudaStream_t s, bool* taken) {
  const TallParams t = plan_memory<TY>(p, err, p.rank > 16 ? (p.rank + 15) / 16 * 16 : 16);
  constexpr int bytes = kMost + 1024;
  cudaError_t e = cudaFuncSetAttribute(tall_kernel<T, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  int size = 1;
  if (e == cudaSuccess) e = cluster_for(tall_kernel<T, TY>, n_units, kTallThreads, bytes, &size);
  if (e != cudaSuccess) return e;
  *taken = (long long)n_units * size * 2 >= sms;
  if (!*taken) return cudaSuccess;
  return launch_clusters(tall_kernel<T, TY>, n_units, size, kTallThreads, bytes, s, t);
}

}  // namespace

cudaError_t launch_tall(const Params& p, unsigned* err, int type, bool y_f32, int n_units, int sms, cudaStream_t s, bool* taken) {
  if (type == T_BF16)
    return y_f32 ? run<__nv_bfloat16, float>(p, err, n_units, sms, s, taken) : run<__nv_bfloat16, __nv_bfloat16>(p, err, n_units, sms, s, taken);
  return y_f32 ? run<__half, float>(p, err, n_units, sms, s, taken) : run<__half, __half>(p, err, n_units, sms, s, taken);
}

}  // namespace lora
}  // namespace specb200
