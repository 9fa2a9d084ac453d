// Softmax attention over the 4-bit paged KV cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e)
//
// in one pass with a running reference m and sum.  The G query heads of a KV
// head and a sequence's new rows are stacked as columns n = i * G + g, at most
// 32 to a unit; both products are taken transposed so that the cache is the
// 16-row operand of mma.sync and few columns cost little:
//   S^T [16 tokens x 8 n] = K [16 x D] Q^T,   O^T [D x 8 n] += V^T [D x 16] P^T
// K's codes are used as they are: (w & 0x000F000F) is a pair of f16 numbers
// code 2^-24 (tensor cores take subnormals), (w & 0x00F000F0) code 2^-20, and
// q carries the inverse powers.  The products code q are exact; a group's sum
// of 32 of them is f32 and takes its scale there,
//   s_j = sum_groups s / 16 (sum code q) + (s + o) (sum q),
// so no rounding of K enters a score; the second term is one more product,
// with the scale pairs as they are stored.  ldmatrix hands the lanes words of
// one group.  V's codes become values in registers: (w >> shift) & 0x03C003C0 |
// 0x3C003C00 is the pair 1 + code / 16, and one packed multiply-add by (s, o)
// rounds the value to f16; P^T is S^T's fragment through movmatrix.  (V's
// channels per m-tile span groups, so its scales cannot wait for the sum.)  V
// and P are rounded to f16, the widest that this rate of mma.sync takes: each
// moves an output by at most 2^-11 of the weighted mean of |v|, about what
// rounding the output to f16 does and an eighth of rounding it to bf16.
//
// A CTA is 4 warps that run on their own: warp w takes the 32-token tiles w,
// w + 4, ... of the CTA's stages, copies them by TMA bulk copies into a ring
// of its own and refills a slot as soon as it has read it, across unit
// boundaries.  The host cuts the batch's 128-token stages into equal runs, one
// a CTA.  A unit's warps join their (m, l, O) in shared memory; a (sequence,
// head, column tile) that several CTAs share is joined by the last arriver of
// every kFanIn of them, level by level and in order, so a plan's results do
// not depend on timing.
//
// Bound by the integer pipe (55 %) and instruction issue (61 %) together: about
// 630 warp instructions per 32 tokens of a head of 128 and 8 columns, a third of
// them V's unpacking, and 160 more per 8 columns.  One row each of 64 sequences
// of 500 to 16000 tokens, 32 query heads on 8 kv heads: 147 us back to back in a
// graph, 4.5 TB/s of the cache's bytes, and 159 where caches change from call
// to call; one of 131072 tokens 50 us; one of 2048 tokens 9.0 us, of which
// launch and one stage are 3.9 and a round of joins 2 to 4.
#include "common.cuh"
#include "kv4.h"
#include "kv4_rows.cuh"
#include "kv4_mma.cuh"

namespace specb200 {
namespace kv4 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;  // tokens of one ring slot

SPEC_DEV uint32_t movmatrix(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
SPEC_DEV void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  // Not volatile: the compiler interleaves the chains with the unpacking.
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// CTAs an SM holds: O^T alone takes 32 registers a thread and 8 columns.
constexpr int ctas_per_sm(int nt) { return nt == 1 ? 4 : nt == 2 ? 3 : 2; }

template <int D, int NT>
struct Shape {
  static constexpr int KS = D / 16;              // 16-channel steps of q.k
  static constexpr int MT = D / 16;              // 16-channel tiles of O^T
  static constexpr int TILE = kTile * D * 5 / 4;  // bytes of a ring slot
  static constexpr int STAGES = (NT <= 2 ? 2 : 3) * (128 / D);
  static constexpr int FRAG = MT * NT * 4;       // O^T floats a lane
  static constexpr int MERGE_AT = kWarps * STAGES * TILE;
  // Two warps' O^T, or the columns on their way out.
  static constexpr int Q_AT = MERGE_AT + ((kWarps / 2) * FRAG * 128 > NT * 8 * (D + 4) * 4 ? (kWarps / 2) * FRAG * 128
                                                                                            : NT * 8 * (D + 4) * 4);
  static constexpr int META_AT = Q_AT + NT * (KS + 1) * 256;
};

struct Meta {
  unsigned long long full[kWarps][8];
  unsigned long long mask[32];
  float c[32];  // scale log2(e) 2^e of a column (q is held as q 2^-e)
  int idx[32];  // row of the sequence; -1: no such column
  float m[kWarps / 2][32], l[kWarps / 2][32];
  int last;
};

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
  for (int off = kWarps / 2; off > 0; off >>= 1) {
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
    __syncthreads();
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
    __syncthreads();
  }
}

// Writes a joined state's columns: warp 0 lays them out in shared memory
// (lane (g, t) holds D/8 consecutive channels of its columns), then D/8
// threads take a column each.
template <int D, int NT>
SPEC_DEV void write_out(const State<D, NT>& s, const AttendParams& p, const Unit& u, float* buf, int warp, int lane) {
  constexpr int LD = D + 4;
  if (warp == 0) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float inv = s.l[n][e] == 0.f ? 0.f : 1.f / s.l[n][e];
        float2* dst = reinterpret_cast<float2*>(buf + (n * 8 + 2 * t + e) * LD + g * (D / 8));
#pragma unroll
        for (int a = 0; a < Shape<D, NT>::MT; ++a) dst[a] = make_float2(s.o[a][n][e] * inv, s.o[a][n][2 + e] * inv);
      }
  }
  __syncthreads();
  constexpr int TPC = D / 8;
  const int G = p.n_heads / p.n_kv;
#pragma unroll 1
  for (int col = threadIdx.x / TPC; col < u.n_cols; col += kThreads / TPC) {
    const int r = u.col0 + col, c = threadIdx.x % TPC * 8;
    const float4 x = *reinterpret_cast<const float4*>(buf + col * LD + c);
    const float4 y = *reinterpret_cast<const float4*>(buf + col * LD + c + 4);
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    store8(p.out, (u.row0 + r / G) * p.out.row_stride + (u.kvh * G + r % G) * p.out.head_stride + c, p.wide_out, v);
  }
}

// Adds partial state src (weights b = 2^(m' - m)) to s.  Half of its O^T is
// under way before its m and l are used.
template <int D, int NT>
SPEC_DEV void take_part(State<D, NT>& s, const float* src, int lane) {
  using Sh = Shape<D, NT>;
  constexpr int H = Sh::MT / 2;
  const int t = lane & 3;
  const float4* o = reinterpret_cast<const float4*>(src) + lane;
  float2 om[NT], ol[NT];
  float b[NT][2];
  float4 x[H][NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    om[n] = __ldcg(reinterpret_cast<const float2*>(src + Sh::FRAG * 32 + n * 8 + 2 * t));
    ol[n] = __ldcg(reinterpret_cast<const float2*>(src + Sh::FRAG * 32 + NT * 8 + n * 8 + 2 * t));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int a = 0; a < H; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) x[a][n] = __ldcg(o + ((h * H + a) * NT + n) * 32);
    if (h == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s.rescale(n, 0, fmaxf(s.m[n][0], om[n].x));
        s.rescale(n, 1, fmaxf(s.m[n][1], om[n].y));
        b[n][0] = ex2(om[n].x - s.m[n][0]);
        b[n][1] = ex2(om[n].y - s.m[n][1]);
        s.l[n][0] += ol[n].x * b[n][0];
        s.l[n][1] += ol[n].y * b[n][1];
      }
    }
#pragma unroll
    for (int a = 0; a < H; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float(&y)[4] = s.o[h * H + a][n];
        y[0] += x[a][n].x * b[n][0];
        y[1] += x[a][n].y * b[n][1];
        y[2] += x[a][n].z * b[n][0];
        y[3] += x[a][n].w * b[n][1];
      }
  }
}

template <int D, int NT>
SPEC_DEV void leave_part(const State<D, NT>& s, float* dst, int lane) {
  using Sh = Shape<D, NT>;
  const int t = lane & 3;
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
}

// One warp's way through the tiles of its CTA's units, ahead of the one it
// computes.  The page ids of a tile are loaded when the tile before it is
// issued; those of a unit's first stage lie in the unit, so that a copy can
// start one load after the kernel does.
struct Cursor {
  int ui, next, last;  // unit; the CTA's units after it
  int tile, end;       // tiles of 32 tokens
  int kvh, kv_end, table;
  int page[2];
  SPEC_DEV bool more() const { return ui >= 0; }
  SPEC_DEV void at_unit(const AttendParams& p, int warp) {
    while (true) {
      const Unit& u = p.units[ui];
      const int* pg = u.pages + (warp * kTile >> p.P_log2);
      page[0] = pg[0];
      page[1] = p.P < kTile ? pg[1] : 0;
      tile = u.st0 * (kStageTokens / kTile) + warp;
      kv_end = u.kv_end;
      end = min(u.st1 * (kStageTokens / kTile), (kv_end + kTile - 1) / kTile);
      kvh = u.kvh;
      table = u.table;
      if (tile < end) return;
      if (next == last) {
        ui = -1;
        return;
      }
      ui = next++;
    }
  }
  SPEC_DEV void advance(const AttendParams& p, int warp) {
    tile += kWarps;
    if (tile >= end) {
      if (next == last) {
        ui = -1;
        return;
      }
      ui = next++;
      at_unit(p, warp);
    } else {
      const int* t = p.table + table + (tile * kTile >> p.P_log2);
      page[0] = t[0];
      page[1] = p.P < kTile && tile * kTile + p.P < kv_end ? t[1] : 0;
    }
  }
};

// Copies the cursor's tile into `dst` as blocks of min(P, 32) tokens: pages
// of 16 and 32 tokens whole, a quarter of a block's four areas of larger ones.
template <int D>
SPEC_DEV void copy_tile(const AttendParams& p, const Cursor& c, uint8_t* dst, uint64_t* bar) {
  const int P = p.P, blk = block_bytes(P, D);
  const uint8_t* src = p.pool + ((long long)c.page[0] * p.n_kv + c.kvh) * blk;
  if (P <= kTile) {
    const int n = P < kTile && c.tile * kTile + P < c.kv_end ? 2 : 1;
    mbar_arrive_expect_tx(bar, n * blk);
    tma_bulk_g2s(dst, src, blk, bar);
    if (n == 2) tma_bulk_g2s(dst + blk, p.pool + ((long long)c.page[1] * p.n_kv + c.kvh) * blk, blk, bar);
  } else {
    const int j = c.tile * kTile & (P - 1);
    mbar_arrive_expect_tx(bar, block_bytes(kTile, D));
    tma_bulk_g2s(dst, src + j * (D / 2), kTile * D / 2, bar);
    tma_bulk_g2s(dst + k_scales_at(kTile, D), src + k_scales_at(P, D) + j * (D / 8), kTile * D / 8, bar);
    tma_bulk_g2s(dst + v_codes_at(kTile, D), src + v_codes_at(P, D) + j * (D / 2), kTile * D / 2, bar);
    tma_bulk_g2s(dst + v_scales_at(kTile, D), src + v_scales_at(P, D) + j * (D / 8), kTile * D / 8, bar);
  }
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NT)) attend_kernel(const __grid_constant__ AttendParams p) {
  using Sh = Shape<D, NT>;
  constexpr int GR = D / 32;  // groups of a token's channels
  constexpr int VW = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + Sh::MERGE_AT);
  uint32_t* qs = reinterpret_cast<uint32_t*>(smem + Sh::Q_AT);  // [nt][kstep][lane][2]
  uint32_t* qoff = qs + NT * Sh::KS * 64;                       // [nt][lane][2]
  Meta* mt = reinterpret_cast<Meta*>(smem + Sh::META_AT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(mt->full[warp]);
  uint8_t* ring = smem + warp * Sh::STAGES * Sh::TILE;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < Sh::STAGES; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_launch_dependents();
  Unit u = p.units[blockIdx.x];  // the plan is older than any kernel this one may overlap
  Cursor cur;
  cur.ui = blockIdx.x;
  cur.next = u.next;
  cur.last = u.last;
  cur.at_unit(p, warp);
  pdl_wait();
#pragma unroll 1
  for (int i = 0; i < Sh::STAGES && cur.more(); ++i) {
    if (lane == 0) copy_tile<D>(p, cur, ring + i * Sh::TILE, &full[i]);
    cur.advance(p, warp);
  }
  int slot = 0, phase = 0;
  bool ok = true;

  const int g = lane >> 2, t = lane & 3, G = p.n_heads / p.n_kv;
  // The slot holds blocks of Pt tokens; the second 16 tokens are in the same
  // block or the next one.
  const int Pt = min(p.P, kTile);
  const int ks0 = k_scales_at(Pt, D), vc0 = v_codes_at(Pt, D), vs0 = v_scales_at(Pt, D);
  const int code16 = Pt == kTile ? 16 * (D / 2) : block_bytes(16, D);   // from the first 16 tokens to the second
  const int scale16 = Pt == kTile ? 16 * (D / 8) : block_bytes(16, D);
  // Offsets of this lane's pieces from a 16-token half's first token.  K: the
  // row this lane addresses for ldmatrix (tokens 0-7, 8-15 of a group, then of
  // the next group).
  const int k_at = (lane % 16) * (D / 2) + lane / 16 * 16;
  const int ks_at = ks0 + (g * GR + t % GR) * 4;
  int v_at[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = 2 * t + (e & 1) + (e >> 1) * 8, byte = g * (VW * 4);
    v_at[e] = vc0 + v_piece_at(D, j, byte / 32) + byte % 32;
  }
  const int vs_at = vs0 + t * (D / 32 * 8) + (g * (D / 32) / 8) * 8;

  for (int next = u.next;; ++next) {
    // Columns: q rows as f16 B fragments q 2^(13 - e), even pairs, and
    // q 2^(9 - e), odd ones (2^e: about the row's largest magnitude), which
    // undo the codes' places, and the sums of q over the groups, 2^(-7 - e).
    // D/8 threads a column, 8 channels each.  All loads are issued first.
    {
      constexpr int TPC = D / 8, PASS = kThreads / TPC, QC = (NT * 8 + PASS - 1) / PASS;
      const int ch = threadIdx.x % TPC, tt = ch % 4, gr = ch / 4;
      float x[QC][8];
#pragma unroll
      for (int i = 0; i < QC; ++i) {
        const int col = i * PASS + threadIdx.x / TPC, r = u.col0 + (col < u.n_cols ? col : 0);
        load8(p.q, (u.row0 + r / G) * p.q.row_stride + (u.kvh * G + r % G) * p.q.head_stride + ch * 8, p.wide_q, x[i]);
      }
#pragma unroll
      for (int i = 0; i < QC; ++i) {
        const int col = i * PASS + threadIdx.x / TPC;
        const bool live = col < u.n_cols;
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) a = fmaxf(a, fabsf(x[i][k]));
#pragma unroll
        for (int o = 1; o < TPC; o <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        float sum = ((x[i][0] + x[i][1]) + (x[i][2] + x[i][3])) + ((x[i][4] + x[i][5]) + (x[i][6] + x[i][7]));
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);  // of the group's 32 channels
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int ex = row_exponent(T_BF16, a);
        const float down = pow2i(-ex);
        if (col < NT * 8) {
          uint32_t f[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float e = k % 2 ? 512.f * down : 8192.f * down;
            f[k] = live ? pack2(x[i][k] * e, x[i][k + 4] * e) : 0u;
          }
          uint32_t* dst = qs + (((col / 8) * Sh::KS + 2 * gr) * 32 + (col % 8) * 4 + tt) * 2;
          *reinterpret_cast<uint2*>(dst) = make_uint2(f[0], f[1]);
          *reinterpret_cast<uint2*>(dst + 64) = make_uint2(f[2], f[3]);
          if (tt < 4 / GR) {  // groups a head of 64 lacks are zero
            const float v = live && tt == 0 ? sum * (down / 128.f) : 0.f;
            const float hi = __half2float(__float2half_rn(v));
            uint32_t* off = qoff + ((col / 8) * 32 + (col % 8) * 4 + tt * GR + gr) * 2;
            *reinterpret_cast<uint2*>(off) = make_uint2(pack2(hi, hi), pack2(v - hi, v - hi));
          }
          if (ch == 0) {
            const int row = (u.col0 + col) / G;
            mt->c[col] = p.scale * kLog2e * 128.f * pow2i(ex);
            mt->idx[col] = live ? row : -1;
            mt->mask[col] = live && p.masks ? p.masks[u.row0 + row] : 0ull;
          }
        }
      }
    }
    __syncthreads();
    State<D, NT> s;
    s.clear();
    float c[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) c[n][0] = mt->c[n * 8 + 2 * t], c[n][1] = mt->c[n * 8 + 2 * t + 1];

    const int end = min(u.st1 * (kStageTokens / kTile), (u.kv_end + kTile - 1) / kTile);
#pragma unroll 1
    for (int tile = u.st0 * (kStageTokens / kTile) + warp; tile < end; tile += kWarps) {
      ok = ok && mbar_wait_bounded(&full[slot], phase, p.err);
      const int tok = tile * kTile;
      const uint8_t* b = ring + slot * Sh::TILE;
      // What column `lane` sees of the tile's tokens, and the tokens whose V
      // counts.  A stored NaN row of V is NaN in every scale; its value is
      // taken as zero and the NaN given to the scores of the columns that see
      // it, so that no other column meets it.
      const bool tail = tok + kTile > u.sure;
      uint32_t sees = ~0u, live = ~0u, bad = 0u;
      if (tail) {
        const bool col = lane < NT * 8;
        sees = seen32(tok, u.kv_len, p.masks != nullptr, col ? mt->mask[lane] : 0ull, col ? mt->idx[lane] : -1);
        live = first32(u.kv_end - tok);
        const uint32_t one = *reinterpret_cast<const uint32_t*>(b + (lane >> 4) * scale16 + vs0 +
                                                                (lane >> 1 & 7) * (D / 32 * 8) + (lane & 1) * 4);
        bad = __ballot_sync(0xffffffffu, (one & 0x7fffu) > 0x7c00u) & live;
        sees &= live;
        live &= ~bad;
      }
      // Both 16-token halves at once: one at a time fetches half the code but
      // leaves the chains of the few resident warps too short (24 sequences of
      // 9 rows and 7 query heads, on this kernel: 94 us against 130).
      constexpr int H = 2;
#pragma unroll 1
      for (int h0 = 0; h0 < 2; h0 += H) {
        const uint8_t* bc = b + h0 * code16;
        const uint8_t* bs = b + h0 * scale16;
        // S^T
        float sc[H][NT][4];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n) sc[h][n][0] = sc[h][n][1] = sc[h][n][2] = sc[h][n][3] = 0.f;
        {
          // (s + o) sum q: the scale pairs as they are stored against the sums of
          // q over the groups, high and low part.
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const uint32_t ra = *reinterpret_cast<const uint32_t*>(bs + h * scale16 + ks_at);
            const uint32_t rb = *reinterpret_cast<const uint32_t*>(bs + h * scale16 + ks_at + D);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint2 q = *reinterpret_cast<const uint2*>(qoff + (n * 32 + lane) * 2);
              mma(sc[h][n], ra, rb, ra, rb, q.x, q.y);
            }
          }
          float sg[H][2][GR];  // s of tokens g and g + 8
          uint32_t w[H][2][GR];
#pragma unroll
          for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int i = 0; i < GR; i += 2) {
              uint32_t r[4];
              ldsm_x4(r, bc + h * code16 + k_at + i * 16);
              w[h][0][i] = r[0], w[h][1][i] = r[1], w[h][0][i + 1] = r[2], w[h][1][i + 1] = r[3];
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const __half2* so = reinterpret_cast<const __half2*>(bs + h * scale16 + ks0 + (g + 8 * e) * (GR * 4));
              if constexpr (GR == 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(so);
                const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) sg[h][e][i] = __low2float(*reinterpret_cast<const __half2*>(&y[i]));
              } else {
                sg[h][e][0] = __low2float(so[0]);
                sg[h][e][1] = __low2float(so[1]);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < GR; ++i) {
            uint2 q0[NT], q1[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              q0[n] = *reinterpret_cast<const uint2*>(qs + ((n * Sh::KS + 2 * i) * 32 + lane) * 2);
              q1[n] = *reinterpret_cast<const uint2*>(qs + ((n * Sh::KS + 2 * i + 1) * 32 + lane) * 2);
            }
#pragma unroll
            for (int h = 0; h < H; ++h) {
              const uint32_t x = w[h][0][i], y = w[h][1][i], x8 = x >> 8, y8 = y >> 8;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float a[4] = {0.f, 0.f, 0.f, 0.f};
                mma(a, x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q0[n].x, q0[n].y);
                mma(a, x8 & 0x000F000Fu, y8 & 0x000F000Fu, x8 & 0x00F000F0u, y8 & 0x00F000F0u, q1[n].x, q1[n].y);
                sc[h][n][0] = fmaf(sg[h][0][i], a[0], sc[h][n][0]);
                sc[h][n][1] = fmaf(sg[h][0][i], a[1], sc[h][n][1]);
                sc[h][n][2] = fmaf(sg[h][1][i], a[2], sc[h][n][2]);
                sc[h][n][3] = fmaf(sg[h][1][i], a[3], sc[h][n][3]);
              }
            }
          }
        }
        // Scales of V, (s, s') and (o, o') of the token pairs (2t, 2t + 1), (2t + 8, 2t + 9).
        uint32_t vs[H][2], vo[H][2];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint2 r = *reinterpret_cast<const uint2*>(bs + h * scale16 + vs_at + e * (4 * (D / 32) * 8));
            vs[h][e] = prmt(r.x, r.y, 0x5410);
            vo[h][e] = prmt(r.x, r.y, 0x7632);
          }
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[h][n][i] *= c[n][i & 1];
        if (tail) {
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t two = live >> (16 * (h0 + h) + 8 * e + 2 * t);
              const uint32_t keep = ((two & 1) ? 0x0000ffffu : 0u) | ((two & 2) ? 0xffff0000u : 0u);
              vs[h][e] &= keep;
              vo[h][e] &= keep;
            }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const uint32_t of_col = __shfl_sync(0xffffffffu, sees, n * 8 + 2 * t + f) >> (16 * h0 + g);
              const uint32_t nan = (bad >> (16 * h0 + g)) & of_col;
#pragma unroll
              for (int h = 0; h < H; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float& y = sc[h][n][2 * e + f];
                  y = (of_col >> (16 * h + 8 * e)) & 1 ? y : -INFINITY;
                  if ((nan >> (16 * h + 8 * e)) & 1) y = __int_as_float(0x7fffffff);
                }
            }
        }
        // Move the reference where a score passes it by more than kSlack.
        bool over = false;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[n][e] = fmaxf(sc[0][n][e], sc[0][n][2 + e]);
            if (H == 2) top[n][e] = fmaxf(top[n][e], fmaxf(sc[H - 1][n][e], sc[H - 1][n][2 + e]));
            over |= top[n][e] > s.m[n][e] + kSlack;
          }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = top[n][e];
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              s.rescale(n, e, fmaxf(s.m[n][e], x));
            }
        }
        uint32_t pb[H][NT][2];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float(&x)[4] = sc[h][n];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = ex2(x[i] - s.m[n][i & 1]);
            s.l[n][0] += x[0] + x[2];
            s.l[n][1] += x[1] + x[3];
            pb[h][n][0] = movmatrix(pack2(x[0], x[1]));
            pb[h][n][1] = movmatrix(pack2(x[2], x[3]));
          }
        // O^T
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t w[4][VW];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint8_t* vc = bc + h * code16 + v_at[e];
            if constexpr (VW == 2) {
              const uint2 x = *reinterpret_cast<const uint2*>(vc);
              w[e][0] = x.x, w[e][1] = x.y;
            } else {
              w[e][0] = *reinterpret_cast<const uint32_t*>(vc);
            }
          }
#pragma unroll
          for (int i = 0; i < VW; ++i)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const uint32_t sel = f ? 0x7632 : 0x5410;
              const uint32_t x = prmt(w[0][i], w[1][i], sel), y = prmt(w[2][i], w[3][i], sel);
              {
                const uint32_t a0 = dq<0>(x, vs[h][0], vo[h][0]), a1 = dq<1>(x, vs[h][0], vo[h][0]);
                const uint32_t a2 = dq<0>(y, vs[h][1], vo[h][1]), a3 = dq<1>(y, vs[h][1], vo[h][1]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma(s.o[4 * i + 2 * f][n], a0, a1, a2, a3, pb[h][n][0], pb[h][n][1]);
              }
              {
                const uint32_t a0 = dq<2>(x, vs[h][0], vo[h][0]), a1 = dq<3>(x, vs[h][0], vo[h][0]);
                const uint32_t a2 = dq<2>(y, vs[h][1], vo[h][1]), a3 = dq<3>(y, vs[h][1], vo[h][1]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma(s.o[4 * i + 2 * f + 1][n], a0, a1, a2, a3, pb[h][n][0], pb[h][n][1]);
              }
            }
        }
      }
      __syncwarp();  // every lane has read the slot
      if (cur.more() && ok) {
        if (lane == 0) copy_tile<D>(p, cur, ring + slot * Sh::TILE, &full[slot]);
        cur.advance(p, warp);
      }
      if (++slot == Sh::STAGES) slot = 0, phase ^= 1;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) s.l[n][e] += __shfl_xor_sync(0xffffffffu, s.l[n][e], o);
    join_warps<D, NT>(s, merge, mt, warp, lane);
    // Up the tree: leave a partial state, and go on where this CTA is the last
    // of its kFanIn to arrive.
    constexpr int PART = Sh::FRAG * 32 + NT * 16;  // floats
    int n = u.n_parts, at = u.part;
    long long base = u.part0;
    int* arrived = p.arrived + u.group;
    while (n > 1) {
      const int node = at / kFanIn, first = node * kFanIn, count = min(kFanIn, n - first);
      if (warp == 0) {
        leave_part<D, NT>(s, p.parts + (base + at) * PART, lane);
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          const bool last = atomicAdd(arrived + node, 1) == count - 1;
          if (last) arrived[node] = 0;  // ready for the next call
          mt->last = last;
        }
      }
      __syncthreads();
      const bool last = mt->last;
      if (!last) break;
      __threadfence();
      s.clear();
      for (int i = warp; i < count; i += kWarps) take_part<D, NT>(s, p.parts + (base + first + i) * PART, lane);
      join_warps<D, NT>(s, merge, mt, warp, lane);
      base += n;
      n = (n + kFanIn - 1) / kFanIn;
      arrived += n;
      at = node;
    }
    if (n == 1) write_out<D, NT>(s, p, u, merge, warp, lane);
    if (next == u.last) break;
    u = p.units[next];
    __syncthreads();  // mt and qs are free for the next unit
  }
  if (!ok && lane == 0) {  // leave no copy of this warp in flight
    for (int i = 0; i < Sh::STAGES; ++i) mbar_wait_bounded(&full[i], (i < slot ? phase ^ 1 : phase), p.err);
  }
}

template <int D, int NT>
int smem_bytes() {
  return Shape<D, NT>::META_AT + (int)sizeof(Meta);
}

template <int D, int NT>
cudaError_t launch(const AttendParams& p, cudaStream_t s) {
  return launch_overlapping(attend_kernel<D, NT>, dim3(p.n_ctas), kThreads, smem_bytes<D, NT>(), s, p);
}
template <int D, int NT>
cudaError_t allow() {
  return cudaFuncSetAttribute(attend_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<D, NT>());
}

}  // namespace

cudaError_t attend_setup() {
  cudaError_t e = allow<128, 1>();
  if (e == cudaSuccess) e = allow<128, 2>();
  if (e == cudaSuccess) e = allow<128, 3>();
  if (e == cudaSuccess) e = allow<128, 4>();
  if (e == cudaSuccess) e = allow<64, 1>();
  if (e == cudaSuccess) e = allow<64, 2>();
  if (e == cudaSuccess) e = allow<64, 3>();
  if (e == cudaSuccess) e = allow<64, 4>();
  return e;
}
size_t attend_part_floats(int head_dim, int nt) { return (size_t)head_dim / 16 * nt * 4 * 32 + nt * 16; }
int attend_ctas_per_sm(int nt) { return ctas_per_sm(nt); }

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
