// Appending rows to the 4-bit paged KV cache, the rotation applied on the way.
//
// Per row and head: x' = R(pos) x (rotate-half or neighbour pairs), then per
// group of 32 channels lo / hi, s = f16((hi - lo) * 16/15), o = f16(lo - s),
// code = clamp(round((x' - o) * (16 / s) - 16), 0, 15).  Every operation is
// rounded by itself (no fused multiply-add), so the stored bytes are a
// function of the inputs that a host restatement reproduces bit for bit.
//
// D/8 threads share a head, 8 channels each: one 16-byte load (two for f32),
// the rotate-half partner D/16 lanes away (four shuffles of 16-bit pairs; a
// second load of the partner's half was slower, 74 us against 68), a group's 4
// lanes for lo / hi, one 4-byte store of codes.
//
// Bound by instruction issue (77 % of the slots): 8192 rows of 32 query and 8
// kv heads of 128, bf16 in and out with the stored values, 50 us, 4.3 TB/s of
// the 216 MB it reads and writes; 64 rows 2.3 us.
#include "common.cuh"
#include "kv4.h"
#include "kv4_rows.cuh"

namespace specb200 {
namespace kv4 {
namespace {

SPEC_DEV float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
SPEC_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr int kThreads = 128;

// 8 channels of a row as the lanes hold them: raw 16-bit pairs or f32.
template <int T>
struct Raw {
  uint32_t w[T == T_BF16 || T == T_F16 ? 4 : 8];
  // T < 0: any type, any alignment.
  SPEC_DEV void load(const Rows& r, long long at, bool wide) {
    if constexpr (T == T_BF16 || T == T_F16) {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(r.ptr) + at);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
      float x[8];
      if constexpr (T == T_F32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(r.ptr) + at);
        const float4 a = p[0], b = p[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
      } else {
        load8(r, at, wide, x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(x[i]);
    }
  }
  SPEC_DEV void get(float (&x)[8]) const {
    if constexpr (T == T_BF16 || T == T_F16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = T == T_BF16 ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u))
                                     : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    }
  }
  // The rotate-half partner's channels, `lanes` away.
  SPEC_DEV Raw other(int lanes) const {
    Raw o;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 4); ++i) o.w[i] = __shfl_xor_sync(0xffffffffu, w[i], lanes);
    return o;
  }
};

// Block (row, part).  A row's work is chunks of SLOTS heads, q's first, then
// k's, then v's (so what a chunk is does not diverge); part y takes chunks y,
// y + gridDim.y, ...
template <int D, int T>
__global__ void __launch_bounds__(kThreads, 8) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int TPH = D / 8;             // threads of a head
  constexpr int SLOTS = kThreads / TPH;  // heads in flight
  const int l = threadIdx.x % TPH, slot = threadIdx.x / TPH;
  const int row = blockIdx.x;
  pdl_launch_dependents();
  const RowDev rd = p.rows[row];  // the plan is older than any kernel this one may overlap
  const int nq = p.q.ptr ? (p.n_heads + SLOTS - 1) / SLOTS : 0, nk = (p.n_kv + SLOTS - 1) / SLOTS;
  const bool rotate = p.cos != nullptr;

  pdl_wait();

  // This thread's 8 channels of the rotation: cos / sin of pair index
  // c mod D/2 (rotate-half, sin negated in the first half) or c / 2
  // (neighbours, 4 pairs).
  float cs[8], sn[8];
  if (rotate && (int)blockIdx.y < nq + nk) {
    const float* c = p.cos + (size_t)rd.pos * (D / 2);
    const float* s = p.sin + (size_t)rd.pos * (D / 2);
    const int at = p.rope_half ? (l * 8) % (D / 2) : l * 4;
    const float4 c0 = *reinterpret_cast<const float4*>(c + at), s0 = *reinterpret_cast<const float4*>(s + at);
    cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w;
    sn[0] = s0.x, sn[1] = s0.y, sn[2] = s0.z, sn[3] = s0.w;
    if (p.rope_half) {
      const float4 c1 = *reinterpret_cast<const float4*>(c + at + 4), s1 = *reinterpret_cast<const float4*>(s + at + 4);
      cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
      sn[4] = s1.x, sn[5] = s1.y, sn[6] = s1.z, sn[7] = s1.w;
#pragma unroll
      for (int i = 0; i < 8; ++i) sn[i] = l < TPH / 2 ? -sn[i] : sn[i];
    }
  }
  auto turn = [&](const Raw<T>& r, float (&x)[8]) {
    r.get(x);
    if (!rotate) return;
    if (p.rope_half) {
      float y[8];
      r.other(TPH / 2).get(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(y[i], sn[i]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = __fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(b, sn[i]));
        x[2 * i + 1] = __fadd_rn(__fmul_rn(b, cs[i]), __fmul_rn(a, sn[i]));
      }
    }
  };

  const int end = nq + 2 * nk;
  const long long q_at = rd.src * p.q.row_stride + l * 8, qo_at = row * p.q_out.row_stride + l * 8;
  const long long k_at = rd.src * p.k.row_stride + l * 8, v_at = rd.src * p.v.row_stride + l * 8;
  auto fetch = [&](int chunk, Raw<T>& r) {  // every lane takes part in the shuffles: idle ones read the last head
    if (chunk < nq) r.load(p.q, q_at + min(chunk * SLOTS + slot, p.n_heads - 1) * p.q.head_stride, p.wide_q);
    else if (chunk < nq + nk) r.load(p.k, k_at + min((chunk - nq) * SLOTS + slot, p.n_kv - 1) * p.k.head_stride, p.wide_k);
    else r.load(p.v, v_at + min((chunk - nq - nk) * SLOTS + slot, p.n_kv - 1) * p.v.head_stride, p.wide_v);
  };
  Raw<T> ahead;
  fetch(blockIdx.y, ahead);
#pragma unroll 1
  for (int chunk = blockIdx.y; chunk < end; chunk += gridDim.y) {
    const Raw<T> r = ahead;
    if (chunk + gridDim.y < end) fetch(chunk + gridDim.y, ahead);  // in flight while this chunk is worked on
    float x[8];
    if (chunk < nq) {
      const int head = chunk * SLOTS + slot;
      turn(r, x);
      if (head < p.n_heads) store8(p.q_out, qo_at + head * p.q_out.head_stride, p.wide_qo, x);
      continue;
    }
    const bool value = chunk >= nq + nk;
    const int head = (chunk - nq - (value ? nk : 0)) * SLOTS + slot;
    if (value) r.get(x);
    else turn(r, x);

    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = min_nan(lo, x[i]);
      hi = max_nan(hi, x[i]);
    }
    // Out of range (hardly ever): every value is clamped, not lo and hi alone.
    // o is rounded to 16 near the clamp, so a value past it need not have the
    // least or the largest code.
    if (!(lo >= -kClamp && hi <= kClamp)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -kClamp), kClamp);
      lo = min_nan(max_nan(lo, -kClamp), kClamp);
      hi = min_nan(max_nan(hi, -kClamp), kClamp);
    }
    // A NaN anywhere in the head's row makes the whole stored row NaN, so that
    // the attention can tell from one scale pair.
    const uint32_t nans = __ballot_sync(0xffffffffu, lo != lo);
    const bool nan = (nans >> ((threadIdx.x & 31) / TPH * TPH)) & ((1u << TPH) - 1);
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
    if (nan) lo = hi = __int_as_float(0x7fffffff);
    if (head >= p.n_kv) continue;  // no shuffle below
    const __half hs = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 16.f / 15.f));
    const float s = __half2float(hs);
    const __half ho = __float2half_rn(__fsub_rn(lo, s));
    const float o = __half2float(ho);
    const float inv = s > 0.f ? __fdiv_rn(16.f, s) : 0.f;
    // Rounding by adding 1.5 * 2^23 (nearest even, after the clamp, which
    // gives a NaN code 0); four codes are one exact float sum.
    float c[8], sum[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = __fsub_rn(__fmul_rn(__fsub_rn(x[i], o), inv), 16.f);
      c[i] = __fsub_rn(__fadd_rn(fminf(fmaxf(t, 0.f), 15.f), 12582912.f), 12582912.f);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      sum[i] = fmaf(c[4 * i + 3], 4096.f, fmaf(c[4 * i + 2], 256.f, fmaf(c[4 * i + 1], 16.f, c[4 * i])));
    const uint32_t codes = (uint32_t)sum[0] | ((uint32_t)sum[1] << 16);
    const int D32 = D / 32, j = rd.slot;
    uint8_t* blk = p.pool + ((long long)rd.page * p.n_kv + head) * block_bytes(p.P, D);
    const int at = value ? v_codes_at(p.P, D) + v_piece_at(D, j, l >> 3) + (l & 7) * 4 : j * (D / 2) + l * 4;
    *reinterpret_cast<uint32_t*>(blk + at) = codes;
    if ((l & 3) == 0) {
      const int to = value ? v_scales_at(p.P, D) + (j >> 1) * (D32 * 8) + (l >> 2) * 8 + (j & 1) * 4
                           : k_scales_at(p.P, D) + (j * D32 + (l >> 2)) * 4;
      *reinterpret_cast<__half2*>(blk + to) = __halves2half2(hs, ho);
    }
    const Rows& val = value ? p.v_out : p.k_out;
    if (val.ptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = fmaf(s, fmaf(c[i], 0.0625f, 1.f), o);
      store8(val, row * val.row_stride + head * val.head_stride + l * 8, value ? p.wide_vo : p.wide_ko, c);
    }
  }
}

template <int D>
cudaError_t launch(const AppendParams& p, int parts, cudaStream_t s) {
  const dim3 grid(p.n_rows, parts);
  // One instantiation a type for rows of 16-byte pieces, as projections leave
  // them; mixed types and odd strides take the general one.
  const bool same = (!p.q.ptr || p.q.dtype == p.k.dtype) && p.v.dtype == p.k.dtype && p.wide_q && p.wide_k && p.wide_v;
  if (!same) return launch_overlapping(append_kernel<D, -1>, grid, kThreads, 0, s, p);
  if (p.k.dtype == T_BF16) return launch_overlapping(append_kernel<D, T_BF16>, grid, kThreads, 0, s, p);
  if (p.k.dtype == T_F16) return launch_overlapping(append_kernel<D, T_F16>, grid, kThreads, 0, s, p);
  return launch_overlapping(append_kernel<D, T_F32>, grid, kThreads, 0, s, p);
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, int head_dim, cudaStream_t s) {
  if (p.n_rows <= 0) return cudaSuccess;
  const int slots = kThreads / (head_dim / 8);
  const int most = (p.q.ptr ? (p.n_heads + slots - 1) / slots : 0) + 2 * ((p.n_kv + slots - 1) / slots);
  // Few rows: a block a chunk, so that a row's heads are read at once (64 rows
  // of 48 heads: 2.4 us against 3.4).  Many: a block a row, which loads the
  // rotation once and reads ahead (1024 rows: 6.9 us against 10.2; equal at 256).
  const int parts = p.n_rows >= 256 ? 1 : most;
  return head_dim == 128 ? launch<128>(p, parts, s) : launch<64>(p, parts, s);
}

}  // namespace kv4
}  // namespace specb200
