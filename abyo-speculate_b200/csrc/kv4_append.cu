// Appending rows to the 4-bit paged KV cache, the rotation applied on the way.
//
// Per row and head: x' = R(pos) x (rotate-half or neighbour pairs), then per
// group of 32 channels lo / hi, s = f16((hi - lo) * 16/15), o = f16(lo - s),
// code = clamp(round((x' - o) * (16 / s) - 16), 0, 15).  Every operation is
// rounded by itself (no fused multiply-add), so the stored bytes are a
// function of the inputs that a host restatement reproduces bit for bit.
//
// D/8 threads share a head, 8 channels each: one 16-byte load (two for f32),
// the rotate-half partner D/16 lanes away, a group's 4 lanes for lo / hi, one
// 4-byte store of codes.
#include "common.cuh"
#include "kv4.h"

namespace specb200 {
namespace kv4 {
namespace {

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

constexpr int kThreads = 128;

// Block (row, part): the row's heads part * slots + i * slots * gridDim.y.
// Heads are numbered q (when given), k, v.
template <int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int TPH = D / 8;             // threads of a head
  constexpr int SLOTS = kThreads / TPH;  // heads in flight
  const int l = threadIdx.x % TPH, slot = threadIdx.x / TPH;
  const int row = blockIdx.x;
  const RowDev rd = p.rows[row];
  const int nq = p.q.ptr ? p.n_heads : 0, heads = nq + 2 * p.n_kv;
  const bool rotate = p.cos != nullptr;

  // This thread's 8 channels of the rotation: cos / sin of pair index
  // c mod D/2 (rotate-half) or c / 2 (neighbours, 4 pairs).
  float cs[8], sn[8];
  if (rotate) {
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
    }
  }

  for (int h0 = blockIdx.y * SLOTS; h0 < heads; h0 += gridDim.y * SLOTS) {
    const bool live = h0 + slot < heads;
    const int h = min(h0 + slot, heads - 1);  // every lane takes part in the shuffles
    const int what = h < nq ? 0 : h < nq + p.n_kv ? 1 : 2;
    const int head = what == 0 ? h : h - nq - (what - 1) * p.n_kv;
    const Rows& in = what == 0 ? p.q : what == 1 ? p.k : p.v;
    const bool wide = what == 0 ? p.wide_q : what == 1 ? p.wide_k : p.wide_v;
    float x[8];
    load8(in, rd.src * in.row_stride + head * in.head_stride + l * 8, wide, x);
    if (rotate) {
      float y[8];
      if (p.rope_half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float o = __shfl_xor_sync(0xffffffffu, x[i], TPH / 2);
          const float a = __fmul_rn(x[i], cs[i]), b = __fmul_rn(o, sn[i]);
          y[i] = l < TPH / 2 ? __fsub_rn(a, b) : __fadd_rn(a, b);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[2 * i] = __fsub_rn(__fmul_rn(x[2 * i], cs[i]), __fmul_rn(x[2 * i + 1], sn[i]));
          y[2 * i + 1] = __fadd_rn(__fmul_rn(x[2 * i + 1], cs[i]), __fmul_rn(x[2 * i], sn[i]));
        }
      }
      if (what != 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i];
      }
    }
    if (what == 0 && live) store8(p.q_out, row * p.q_out.row_stride + head * p.q_out.head_stride + l * 8, wide, x);
    if (__all_sync(0xffffffffu, what == 0)) continue;

    // A NaN anywhere in the head's row makes the whole stored row NaN, so that
    // the attention can tell from one scale pair.
    bool nan = false;
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      nan |= x[i] != x[i];
      x[i] = fminf(fmaxf(x[i], -kClamp), kClamp);
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
    const uint32_t nans = __ballot_sync(0xffffffffu, nan);
    nan = (nans >> ((threadIdx.x & 31) / TPH * TPH)) & ((1u << TPH) - 1);
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
    if (nan) lo = hi = __int_as_float(0x7fffffff);
    if (what == 0 || !live) continue;  // no shuffle below
    const __half hs = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 16.f / 15.f));
    const float s = __half2float(hs);
    const __half ho = __float2half_rn(__fsub_rn(lo, s));
    const float o = __half2float(ho);
    const float inv = s > 0.f ? __fdiv_rn(16.f, s) : 0.f;
    uint32_t codes = 0;
    float val[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = rintf(__fsub_rn(__fmul_rn(__fsub_rn(x[i], o), inv), 16.f));
      const float c = fminf(fmaxf(t, 0.f), 15.f);  // a NaN gives code 0
      codes |= (uint32_t)c << (4 * i);
      val[i] = fmaf(s, 1.f + c * 0.0625f, o);
    }
    const int D32 = D / 32, j = rd.slot;
    uint8_t* blk = p.pool + ((long long)rd.page * p.n_kv + head) * block_bytes(p.P, D);
    const __half2 so = __halves2half2(hs, ho);
    if (what == 1) {
      *reinterpret_cast<uint32_t*>(blk + j * (D / 2) + l * 4) = codes;
      if ((l & 3) == 0)
        *reinterpret_cast<__half2*>(blk + k_scales_at(p.P, D) + (j * D32 + (l >> 2)) * 4) = so;
      if (p.k_out.ptr)
        store8(p.k_out, row * p.k_out.row_stride + head * p.k_out.head_stride + l * 8, p.wide_ko, val);
    } else {
      *reinterpret_cast<uint32_t*>(blk + v_codes_at(p.P, D) + v_piece_at(D, j, l >> 3) + (l & 7) * 4) = codes;
      if ((l & 3) == 0)
        *reinterpret_cast<__half2*>(blk + v_scales_at(p.P, D) + (j >> 1) * (D32 * 8) + (l >> 2) * 8 + (j & 1) * 4) = so;
      if (p.v_out.ptr)
        store8(p.v_out, row * p.v_out.row_stride + head * p.v_out.head_stride + l * 8, p.wide_vo, val);
    }
  }
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, int head_dim, cudaStream_t s) {
  if (p.n_rows <= 0) return cudaSuccess;
  const int slots = kThreads / (head_dim / 8);
  const int heads = (p.q.ptr ? p.n_heads : 0) + 2 * p.n_kv;
  const int parts = (heads + slots - 1) / slots;
  const dim3 grid(p.n_rows, parts);
  if (head_dim == 128) append_kernel<128><<<grid, kThreads, 0, s>>>(p);
  else append_kernel<64><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace kv4
}  // namespace specb200
