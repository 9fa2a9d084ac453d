// Softmax attention over the 4-bit paged KV cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m)
//
// over the slots a row sees, in one pass with a running maximum m and sum.
// One block a (row, query head); its warps take tokens in turn and join their
// (m, l, o) through shared memory.
#include "common.cuh"
#include "kv4.h"

namespace specb200 {
namespace kv4 {
namespace {

constexpr int kWarps = 4;

SPEC_DEV float load1(const Rows& r, long long at) {
  if (r.dtype == T_F32) return static_cast<const float*>(r.ptr)[at];
  if (r.dtype == T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(r.ptr)[at]);
  return __half2float(static_cast<const __half*>(r.ptr)[at]);
}
SPEC_DEV void store1(const Rows& r, long long at, float x) {
  if (r.dtype == T_F32) static_cast<float*>(r.ptr)[at] = x;
  else if (r.dtype == T_BF16) static_cast<__nv_bfloat16*>(r.ptr)[at] = __float2bfloat16_rn(x);
  else static_cast<__half*>(r.ptr)[at] = __float2half_rn(x);
}

SPEC_DEV float value_of(const uint8_t* code_byte, int nibble, const uint8_t* scale) {
  const __half2 so = *reinterpret_cast<const __half2*>(scale);
  const int c = (*code_byte >> (4 * nibble)) & 15;
  return fmaf(__low2float(so), 1.f + c * 0.0625f, __high2float(so));
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const __grid_constant__ AttendParams p) {
  constexpr int CH = D / 32;
  const int row = blockIdx.x, head = blockIdx.y, kvh = head / (p.n_heads / p.n_kv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const SeqDev sq = p.seqs[p.row_seq[row]];
  const int i = row - sq.row0, T = sq.kv_len + sq.n_rows;
  const unsigned long long mask = p.masks ? p.masks[row] : 0ull;
  float q[CH], o[CH], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    q[c] = load1(p.q, row * p.q.row_stride + head * p.q.head_stride + lane * CH + c);
    o[c] = 0.f;
  }
  for (int t = warp; t < T; t += kWarps) {
    const int w = t - sq.kv_len;
    if (w >= 0 && !(p.masks ? (mask >> w) & 1ull : w <= i)) continue;
    const int j = t % p.P;
    const uint8_t* blk = p.pool + ((long long)p.table[sq.table + t / p.P] * p.n_kv + kvh) * block_bytes(p.P, D);
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int ch = lane * CH + c;
      s += q[c] * value_of(blk + j * (D / 2) + ch / 2, ch & 1, blk + k_scales_at(p.P, D) + (j * (D / 32) + ch / 32) * 4);
    }
    s = warp_sum(s) * p.scale;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float a = expf(m - base), e = expf(s - base);
    m = mn;
    l = l * a + e;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int ch = lane * CH + c;
      const float v = value_of(blk + v_codes_at(p.P, D) + v_piece_at(D, j, ch / 64) + (ch % 64) / 2, ch & 1,
                               blk + v_scales_at(p.P, D) + (j / 2) * (D / 32) * 8 + (ch / 32) * 8 + (j & 1) * 4);
      o[c] = o[c] * a + e * v;
    }
  }
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) so[warp][lane * CH + c] = o[c];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w]);
  const float base = M == -INFINITY ? 0.f : M;
  for (int w = 0; w < kWarps; ++w) L += sl[w] * expf(sm[w] - base);
  for (int ch = threadIdx.x; ch < D; ch += kWarps * 32) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w) x += so[w][ch] * expf(sm[w] - base);
    store1(p.out, row * p.out.row_stride + head * p.out.head_stride + ch, L == 0.f ? 0.f : x / L);
  }
}

}  // namespace

cudaError_t launch_attend(const AttendParams& p, int head_dim, cudaStream_t s) {
  if (p.n_rows <= 0) return cudaSuccess;
  const dim3 grid(p.n_rows, p.n_heads);
  if (head_dim == 128) attend_kernel<128><<<grid, kWarps * 32, 0, s>>>(p);
  else attend_kernel<64><<<grid, kWarps * 32, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace kv4
}  // namespace specb200
