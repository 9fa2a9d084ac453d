// Softmax attention over the 4-bit paged KV cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e)
//
// in one pass with a running reference m and sum.  The G query heads of a KV
// head and a sequence's new rows are stacked as columns n = i * G + g, at most
// 32 to a unit; both products are taken transposed so that the cache is the
// 16-row operand of mma.sync and few columns cost little:
//   S^T [16 tokens x 8 n] = K [16 x D] Q^T,   O^T [D x 8 n] += V^T [D x 16] P^T
// Codes go to the f16 operand in registers: (w >> shift) & 0x03C003C0 | 0x3C003C00
// is the pair 1 + code / 16, and one packed multiply-add by (s, o) gives the
// values.  Any order of the channels (K) and of the tokens (V) along the
// contracted axis will do, so a lane takes the channels of whole 32-bit words
// and never shuffles nibbles; P^T is S^T's fragment through movmatrix.
//
// A CTA is 8 consumer warps, 16 tokens each of a 128-token stage, and one
// producer warp that copies page blocks (K, V and scales of one head lie
// together) by TMA bulk copies into a ring.  The host cuts the batch's stages
// into equal runs, one a CTA; a (sequence, head, column tile) that several
// CTAs share leaves partial (m, l, O) and the last of them to arrive joins
// them in order, so a plan's results do not depend on timing.
#include "common.cuh"
#include "kv4.h"

namespace specb200 {
namespace kv4 {
namespace {

constexpr int kConsumers = 8;
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr float kNone = -1e30f;  // the reference before any score
constexpr float kSlack = 8.f;    // a score may pass the reference by this many octaves before it moves

SPEC_DEV void bar_consumers() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

SPEC_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
SPEC_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
SPEC_DEV uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
SPEC_DEV uint32_t movmatrix(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
SPEC_DEV uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Values of nibbles n and n + 4 of w.
template <int N>
SPEC_DEV uint32_t dq(uint32_t w, uint32_t s2, uint32_t o2) {
  const uint32_t x = N == 0 ? w << 6 : N == 1 ? w << 2 : N == 2 ? w >> 2 : w >> 6;
  return hfma2(lop3_and_or(x, 0x03C003C0u, 0x3C003C00u), s2, o2);
}
SPEC_DEV void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  mma_f16(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}

template <int D, int NT>
struct Shape {
  static constexpr int KS = D / 16;                    // 16-channel steps of q.k
  static constexpr int MT = D / 16;                    // 16-channel tiles of O^T
  static constexpr int STAGE = kStageTokens * D * 5 / 4;
  static constexpr int STAGES = NT <= 1 ? 81920 / STAGE : 81920 / STAGE;
  static constexpr int FRAG = MT * NT * 4;             // O^T floats a lane
  static constexpr int MERGE = (kConsumers / 2) * FRAG * 128;
  static constexpr int Q_AT = STAGES * STAGE + MERGE;
  static constexpr int META_AT = Q_AT + NT * KS * 256;
  static constexpr int SMEM = META_AT + 2048;
};

struct Meta {
  unsigned long long full[8], empty[8];
  unsigned long long mask[32];
  float c[32];  // scale log2(e) 2^e of a column (q is held as q 2^-e)
  int idx[32];  // row of the sequence; -1: no such column
  float m[kConsumers][32], l[kConsumers / 2][32];
  int last;
};
static_assert(sizeof(Meta) <= 2048 + 1024, "meta");

SPEC_DEV float load1(const Rows& r, long long at) {
  if (r.dtype == T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(r.ptr)[at]);
  return __half2float(static_cast<const __half*>(r.ptr)[at]);
}

// One warp's softmax state: lane (g, t) holds columns 8 nt + 2t + {0, 1}.
template <int D, int NT>
struct State {
  float m[NT][2], l[NT][2];
  float o[Shape<D, NT>::MT][NT][4];  // [channel tile][nt]: (g, col 0), (g, col 1), (g + 8, col 0), (g + 8, col 1)
  SPEC_DEV void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = kNone, l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int a = 0; a < Shape<D, NT>::MT; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) o[a][n][0] = o[a][n][1] = o[a][n][2] = o[a][n][3] = 0.f;
  }
  // Moves column (n, e) to reference mm >= m.
  SPEC_DEV void rescale(int n, int e, float mm) {
    const float a = ex2(m[n][e] - mm);
    m[n][e] = mm;
    l[n][e] *= a;
#pragma unroll
    for (int i = 0; i < Shape<D, NT>::MT; ++i) o[i][n][e] *= a, o[i][n][2 + e] *= a;
  }
};

// Joins the warps' states into warp 0's (a tree over shared memory).  l is
// the whole column's in every lane.
template <int D, int NT>
SPEC_DEV void join_warps(State<D, NT>& s, float* buf, Meta* mt, int warp, int lane) {
  constexpr int F = Shape<D, NT>::FRAG;
  const int t = lane & 3;
#pragma unroll 1
  for (int off = kConsumers / 2; off > 0; off >>= 1) {
    if (warp >= off && warp < 2 * off) {
      float4* p = reinterpret_cast<float4*>(buf + (warp - off) * F * 32);
#pragma unroll
      for (int a = 0; a < Shape<D, NT>::MT; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          p[(a * NT + n) * 32 + lane] = make_float4(s.o[a][n][0], s.o[a][n][1], s.o[a][n][2], s.o[a][n][3]);
      if (lane < 4) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mt->m[warp - off][n * 8 + 2 * t + e] = s.m[n][e];
            mt->l[warp - off][n * 8 + 2 * t + e] = s.l[n][e];
          }
      }
    }
    bar_consumers();
    if (warp < off) {
      const float4* p = reinterpret_cast<const float4*>(buf + warp * F * 32);
      float b[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float om = mt->m[warp][n * 8 + 2 * t + e];
          const float mm = fmaxf(s.m[n][e], om);
          s.rescale(n, e, mm);
          b[n][e] = ex2(om - mm);
          s.l[n][e] += mt->l[warp][n * 8 + 2 * t + e] * b[n][e];
        }
#pragma unroll
      for (int a = 0; a < Shape<D, NT>::MT; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 x = p[(a * NT + n) * 32 + lane];
          s.o[a][n][0] += x.x * b[n][0];
          s.o[a][n][1] += x.y * b[n][1];
          s.o[a][n][2] += x.z * b[n][0];
          s.o[a][n][3] += x.w * b[n][1];
        }
    }
    bar_consumers();
  }
}

// Writes columns of a joined state: lane (g, t) holds D/8 consecutive channels.
template <int D, int NT>
SPEC_DEV void write_out(const State<D, NT>& s, const AttendParams& p, const Unit& u, int lane) {
  constexpr int W = D / 8;
  const int g = lane >> 2, t = lane & 3, G = p.n_heads / p.n_kv;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = n * 8 + 2 * t + e;
      if (col >= u.n_cols) continue;
      const int r = u.col0 + col;
      const float inv = s.l[n][e] == 0.f ? 0.f : 1.f / s.l[n][e];
      const long long at = (u.row0 + r / G) * p.out.row_stride + (u.kvh * G + r % G) * p.out.head_stride + g * W;
      float x[W];
#pragma unroll
      for (int a = 0; a < Shape<D, NT>::MT; ++a) {
        x[2 * a] = s.o[a][n][e] * inv;
        x[2 * a + 1] = s.o[a][n][2 + e] * inv;
      }
      if (p.out.dtype == T_F32) {
        float* q = static_cast<float*>(p.out.ptr) + at;
        if (p.wide_out) {
#pragma unroll
          for (int i = 0; i < W / 4; ++i)
            reinterpret_cast<float4*>(q)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) q[i] = x[i];
        }
      } else {
        uint32_t w[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          if (p.out.dtype == T_BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
          } else {
            w[i] = pack2(x[2 * i], x[2 * i + 1]);
          }
        }
        uint16_t* q = static_cast<uint16_t*>(p.out.ptr) + at;
        if (p.wide_out) {
#pragma unroll
          for (int i = 0; i < W / 8; ++i)
            reinterpret_cast<uint4*>(q)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < W / 2; ++i) q[2 * i] = (uint16_t)w[i], q[2 * i + 1] = (uint16_t)(w[i] >> 16);
        }
      }
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, NT <= 1 ? 2 : 1) attend_kernel(const __grid_constant__ AttendParams p) {
  using Sh = Shape<D, NT>;
  constexpr int KW = D / 32;  // code words of K a lane holds of a token
  constexpr int VW = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + Sh::STAGES * Sh::STAGE);
  uint32_t* qs = reinterpret_cast<uint32_t*>(smem + Sh::Q_AT);  // [nt][kstep][lane][2]
  Meta* mt = reinterpret_cast<Meta*>(smem + Sh::META_AT);
  uint64_t* full = reinterpret_cast<uint64_t*>(mt->full);
  uint64_t* empty = reinterpret_cast<uint64_t*>(mt->empty);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int P = p.P, blk = block_bytes(P, D), per = kStageTokens / P;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < Sh::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers);
    }
    fence_mbar_init();
  }
  __syncthreads();
  const int u0 = p.cta_units[blockIdx.x], u1 = p.cta_units[blockIdx.x + 1];
  int k = 0;  // stages so far
  bool ok = true;

  if (warp == kConsumers) {
    // Producer: one lane a page.
    for (int ui = u0; ui < u1 && ok; ++ui) {
      const Unit u = p.units[ui];
      for (int st = u.st0; st < u.st1; ++st, ++k) {
        const int slot = k % Sh::STAGES;
        const int pages = min(per, (u.kv_end + P - 1) / P - st * per);
        const int page = lane < pages ? p.table[u.table + st * per + lane] : 0;
        if (k >= Sh::STAGES) ok = mbar_wait_bounded(&empty[slot], (k / Sh::STAGES - 1) & 1, p.err);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[slot], pages * blk);
        __syncwarp();
        if (lane < pages)
          tma_bulk_g2s(smem + slot * Sh::STAGE + lane * blk, p.pool + ((long long)page * p.n_kv + u.kvh) * blk, blk,
                       &full[slot]);
      }
    }
    if (!ok) {  // leave no copy of this CTA in flight
      for (int i = max(0, k - Sh::STAGES); i < k; ++i)
        mbar_wait_bounded(&full[i % Sh::STAGES], (i / Sh::STAGES) & 1, p.err);
    }
    return;
  }

  const int g = lane >> 2, t = lane & 3, G = p.n_heads / p.n_kv;
  // Offsets of this lane's pieces from its tile's first token.
  const int k_at = g * (D / 2) + t * (KW * 4);
  const int ks_at = (g * (D / 32) + t * (D / 32) / 4) * 4;
  int v_at[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = 2 * t + (e & 1) + (e >> 1) * 8, byte = g * (VW * 4);
    v_at[e] = v_piece_at(D, j, byte / 32) + byte % 32;
  }
  const int vs_at = t * (D / 32 * 8) + (g * (D / 32) / 8) * 8;

  for (int ui = u0; ui < u1; ++ui) {
    const Unit u = p.units[ui];
    // Columns: q rows as f16 B fragments, scaled by a power of two where bf16
    // could leave f16's range.
    for (int col = warp; col < NT * 8; col += kConsumers) {
      const bool live = col < u.n_cols;
      const int r = u.col0 + (live ? col : 0), row = r / G;
      float x[D / 32], a = 0.f;
      const long long at = (u.row0 + row) * p.q.row_stride + (u.kvh * G + r % G) * p.q.head_stride + lane * (D / 32);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        x[i] = live ? load1(p.q, at + i) : 0.f;
        a = fmaxf(a, fabsf(x[i]));
      }
      int ex = 0;
      if (p.q.dtype == T_BF16) {
        a = warp_max(a);
        if (a > 0.f && a < INFINITY) ex = min(max((__float_as_int(a) >> 23) - 127, -100), 126);
      }
      const float down = __int_as_float((127 - ex) << 23);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int c = lane * (D / 32) + i, tt = c / (D / 4), w = c % (D / 4) / 8, n = c % 4, hi = c % 8 / 4;
        __half* dst = reinterpret_cast<__half*>(
            qs + (((col / 8) * Sh::KS + 2 * w + (n >> 1)) * 32 + (col % 8) * 4 + tt) * 2 + (n & 1));
        dst[hi] = __float2half_rn(x[i] * down);
      }
      if (lane == 0) {
        mt->c[col] = p.scale * 1.4426950408889634f * __int_as_float((min(ex + 127, 254)) << 23);
        mt->idx[col] = live ? row : -1;
        mt->mask[col] = live && p.masks ? p.masks[u.row0 + row] : 0ull;
      }
    }
    bar_consumers();
    State<D, NT> s;
    s.clear();
    float c[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) c[n][0] = mt->c[n * 8 + 2 * t], c[n][1] = mt->c[n * 8 + 2 * t + 1];

    for (int st = u.st0; st < u.st1; ++st, ++k) {
      const int slot = k % Sh::STAGES;
      ok = ok && mbar_wait_bounded(&full[slot], (k / Sh::STAGES) & 1, p.err);
      const int tok = st * kStageTokens + warp * 16;
      if (ok && tok < u.kv_end) {
        const int pi = warp * 16 / P, j0 = warp * 16 % P;
        const uint8_t* b = smem + slot * Sh::STAGE + pi * blk;
        const uint8_t* kc = b + j0 * (D / 2) + k_at;
        const uint8_t* ksc = b + k_scales_at(P, D) + j0 * (D / 8) + ks_at;
        const uint8_t* vc = b + v_codes_at(P, D) + j0 * (D / 2);
        const uint8_t* vsc = b + v_scales_at(P, D) + j0 * (D / 8) + vs_at;
        // S^T
        float sc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
        {
          uint32_t wa[KW], wb[KW];
          if constexpr (KW == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(kc), y = *reinterpret_cast<const uint4*>(kc + 8 * (D / 2));
            wa[0] = x.x, wa[1] = x.y, wa[2] = x.z, wa[3] = x.w;
            wb[0] = y.x, wb[1] = y.y, wb[2] = y.z, wb[3] = y.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(kc), y = *reinterpret_cast<const uint2*>(kc + 8 * (D / 2));
            wa[0] = x.x, wa[1] = x.y;
            wb[0] = y.x, wb[1] = y.y;
          }
          const uint32_t ra = *reinterpret_cast<const uint32_t*>(ksc), rb = *reinterpret_cast<const uint32_t*>(ksc + D);
          const uint32_t sa = prmt(ra, ra, 0x1010), oa = prmt(ra, ra, 0x3232);
          const uint32_t sb = prmt(rb, rb, 0x1010), ob = prmt(rb, rb, 0x3232);
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            {
              const uint32_t a0 = dq<0>(wa[w], sa, oa), a1 = dq<0>(wb[w], sb, ob);
              const uint32_t a2 = dq<1>(wa[w], sa, oa), a3 = dq<1>(wb[w], sb, ob);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint2 q = *reinterpret_cast<const uint2*>(qs + ((n * Sh::KS + 2 * w) * 32 + lane) * 2);
                mma(sc[n], a0, a1, a2, a3, q.x, q.y);
              }
            }
            {
              const uint32_t a0 = dq<2>(wa[w], sa, oa), a1 = dq<2>(wb[w], sb, ob);
              const uint32_t a2 = dq<3>(wa[w], sa, oa), a3 = dq<3>(wb[w], sb, ob);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint2 q = *reinterpret_cast<const uint2*>(qs + ((n * Sh::KS + 2 * w + 1) * 32 + lane) * 2);
                mma(sc[n], a0, a1, a2, a3, q.x, q.y);
              }
            }
          }
        }
        // Scales of V, (s, s') and (o, o') of the token pairs (2t, 2t + 1), (2t + 8, 2t + 9).
        uint32_t vs[2], vo[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 r = *reinterpret_cast<const uint2*>(vsc + h * (4 * (D / 32) * 8));
          vs[h] = prmt(r.x, r.y, 0x5410);
          vo[h] = prmt(r.x, r.y, 0x7632);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[n][i] *= c[n][i & 1];
        if (tok + 16 > u.kv_len) {
          // Tokens of this step, or past the end.  A stored NaN row of V is NaN
          // in every scale; its value is taken as zero and the NaN given to the
          // scores of the columns that see it, so that no other column meets it.
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = tok + 2 * t + 8 * h + e;
              const uint32_t keep = e ? 0x0000ffffu : 0xffff0000u;
              const bool bad = ((vs[h] >> (16 * e)) & 0x7fffu) > 0x7c00u;
              if (j >= u.kv_end || bad) vs[h] &= keep, vo[h] &= keep;
            }
            const int j = tok + g + 8 * h, w = j - u.kv_len;
            const uint8_t* one = b + v_scales_at(P, D) + ((j0 + g + 8 * h) >> 1) * (D / 32 * 8) + (g & 1) * 4;
            const bool bad = (*reinterpret_cast<const uint32_t*>(one) & 0x7fffu) > 0x7c00u;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int col = n * 8 + 2 * t + e;
                const bool sees = w < 0 || (j < u.kv_end && (p.masks ? (mt->mask[col] >> w) & 1 : w <= mt->idx[col]));
                float& x = sc[n][2 * h + e];
                x = !sees ? -INFINITY : bad ? __int_as_float(0x7fffffff) : x;
              }
          }
        }
        // Move the reference where a score passes it by more than kSlack.
        bool over = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) over |= fmaxf(sc[n][e], sc[n][2 + e]) > s.m[n][e] + kSlack;
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaxf(sc[n][e], sc[n][2 + e]);
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              s.rescale(n, e, fmaxf(s.m[n][e], x));
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[n][i] = ex2(sc[n][i] - s.m[n][i & 1]);
          s.l[n][0] += sc[n][0] + sc[n][2];
          s.l[n][1] += sc[n][1] + sc[n][3];
          pb[n][0] = movmatrix(pack2(sc[n][0], sc[n][1]));
          pb[n][1] = movmatrix(pack2(sc[n][2], sc[n][3]));
        }
        // O^T
        uint32_t w[4][VW];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (VW == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(vc + v_at[e]);
            w[e][0] = x.x, w[e][1] = x.y;
          } else {
            w[e][0] = *reinterpret_cast<const uint32_t*>(vc + v_at[e]);
          }
        }
#pragma unroll
        for (int i = 0; i < VW; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t sel = h ? 0x7632 : 0x5410;
            const uint32_t x = prmt(w[0][i], w[1][i], sel), y = prmt(w[2][i], w[3][i], sel);
            {
              const uint32_t a0 = dq<0>(x, vs[0], vo[0]), a1 = dq<1>(x, vs[0], vo[0]);
              const uint32_t a2 = dq<0>(y, vs[1], vo[1]), a3 = dq<1>(y, vs[1], vo[1]);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma(s.o[4 * i + 2 * h][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
            }
            {
              const uint32_t a0 = dq<2>(x, vs[0], vo[0]), a1 = dq<3>(x, vs[0], vo[0]);
              const uint32_t a2 = dq<2>(y, vs[1], vo[1]), a3 = dq<3>(y, vs[1], vo[1]);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma(s.o[4 * i + 2 * h + 1][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
            }
          }
      }
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[slot])) : "memory");
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) s.l[n][e] += __shfl_xor_sync(0xffffffffu, s.l[n][e], o);
    join_warps<D, NT>(s, merge, mt, warp, lane);
    if (u.n_parts == 1) {
      if (warp == 0) write_out<D, NT>(s, p, u, lane);
      continue;
    }
    // Leave a partial state; the last CTA of the group to arrive joins all.
    constexpr int PART = Sh::FRAG * 32 + NT * 16;  // floats
    if (warp == 0) {
      float* dst = p.parts + (long long)(u.part0 + u.part) * PART;
#pragma unroll
      for (int a = 0; a < Sh::MT; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          __stcg(reinterpret_cast<float4*>(dst) + (a * NT + n) * 32 + lane,
                 make_float4(s.o[a][n][0], s.o[a][n][1], s.o[a][n][2], s.o[a][n][3]));
      if (lane < 4) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            __stcg(dst + Sh::FRAG * 32 + n * 8 + 2 * t + e, s.m[n][e]);
            __stcg(dst + Sh::FRAG * 32 + NT * 8 + n * 8 + 2 * t + e, s.l[n][e]);
          }
      }
      __threadfence();
      __syncwarp();
      if (lane == 0) {
        const int before = atomicAdd(p.arrived + u.group, 1);
        mt->last = before == u.n_parts - 1;
        if (mt->last) p.arrived[u.group] = 0;  // ready for the next call
      }
    }
    bar_consumers();
    if (!mt->last) continue;
    __threadfence();
    s.clear();
    for (int i = warp; i < u.n_parts; i += kConsumers) {
      const float* src = p.parts + (long long)(u.part0 + i) * PART;
      float b[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float om = __ldcg(src + Sh::FRAG * 32 + n * 8 + 2 * t + e);
          const float mm = fmaxf(s.m[n][e], om);
          s.rescale(n, e, mm);
          b[n][e] = ex2(om - mm);
          s.l[n][e] += __ldcg(src + Sh::FRAG * 32 + NT * 8 + n * 8 + 2 * t + e) * b[n][e];
        }
#pragma unroll
      for (int a = 0; a < Sh::MT; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(src) + (a * NT + n) * 32 + lane);
          s.o[a][n][0] += x.x * b[n][0];
          s.o[a][n][1] += x.y * b[n][1];
          s.o[a][n][2] += x.z * b[n][0];
          s.o[a][n][3] += x.w * b[n][1];
        }
    }
    join_warps<D, NT>(s, merge, mt, warp, lane);
    if (warp == 0) write_out<D, NT>(s, p, u, lane);
    bar_consumers();  // mt->last is read before the next unit writes it
  }
}

template <int D, int NT>
cudaError_t launch(const AttendParams& p, cudaStream_t s) {
  constexpr int smem = Shape<D, NT>::SMEM + 1024;
  const cudaError_t e =
      cudaFuncSetAttribute(attend_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  attend_kernel<D, NT><<<p.n_ctas, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

size_t attend_part_floats(int head_dim, int nt) { return (size_t)head_dim / 16 * nt * 4 * 32 + nt * 16; }
int attend_ctas_per_sm(int nt) { return nt <= 1 ? 2 : 1; }

cudaError_t launch_attend(const AttendParams& p, int head_dim, int nt, cudaStream_t s) {
  if (p.n_ctas <= 0) return cudaSuccess;
  if (head_dim == 128) {
    if (nt == 1) return launch<128, 1>(p, s);
    if (nt == 2) return launch<128, 2>(p, s);
    if (nt == 3) return launch<128, 3>(p, s);
    return launch<128, 4>(p, s);
  }
  if (nt == 1) return launch<64, 1>(p, s);
  if (nt == 2) return launch<64, 2>(p, s);
  if (nt == 3) return launch<64, 3>(p, s);
  return launch<64, 4>(p, s);
}

}  // namespace kv4
}  // namespace specb200
