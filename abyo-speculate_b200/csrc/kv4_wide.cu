// Softmax attention over the 4-bit paged KV cache for many columns: prompt
// chunks and draft trees, on the 5th-generation tensor cores.
//
// A column is a (row of the step, query head of the KV head's group).  A CTA
// takes up to 256 of them as two tiles of 128 and walks the 128-token stages
// of its run:
//   S [128 columns x 128 tokens] = Q K^T        tcgen05.mma, f16 from shared memory
//   P = 2^(c S - m), rounded to f16 in place of S in tensor memory
//   O [128 x D] += P V                          P from tensor memory, V^T from shared memory
// Roles: warps 0-3 and 4-7 are the softmax of tile 0 and 1, one thread a
// column; warps 8-11 unpack the pages' codes into f16 operand tiles; lane 0 of
// warp 12 issues the products.  While one tile's softmax runs, the other
// tile's products do.  Unpacking is paid once for both tiles (1.5 instructions
// an element and 256 columns).
//
// Channels and tokens along a contracted axis may come in any order that both
// operands share, and O's columns in any order that the output undoes: K's
// channels are stored in the order a word's nibbles unpack (n, n + 4), and
// V^T's row for channel 8 c + n is n * D/8 + c, so that the lanes of a warp
// store neighbouring rows.
//
// O is scaled only when a column's reference moves, by a score more than
// kSlack octaves above it.  Runs, partial states and joins are as in the
// narrow kernel (kv4_attend.cu).
#include "common.cuh"
#include "kv4.h"
#include "kv4_mma.cuh"
#include "kv4_rows.cuh"

namespace specb200 {
namespace kv4 {
namespace {

constexpr int kTileCols = 128;
constexpr int kThreads = 13 * 32;
constexpr int kDequant = 8, kIssuer = 12;  // first warps of the roles

// ---- tensor memory ----------------------------------------------------------
template <int N>
SPEC_DEV void tm_load(uint32_t addr, float* r);
template <>
SPEC_DEV void tm_load<8>(uint32_t a, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "r"(a)
               : "memory");
}
template <>
SPEC_DEV void tm_load<32>(uint32_t a, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(a)
      : "memory");
}
SPEC_DEV void tm_store32(uint32_t a, const float* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
      "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
      "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]),
      "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]),
      "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31])
      : "memory");
}
SPEC_DEV void tm_store16(uint32_t a, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
SPEC_DEV void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// f16 A and B, f32 accumulator.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
// D (+)= A B^T, A and B in shared memory.
SPEC_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  umma_bf16(d, a, b, idesc, accumulate);  // kind::f16; the types are the descriptor's
}
// A in tensor memory: two f16 a column, lane = row.
SPEC_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// ---- packed f32 -------------------------------------------------------------
SPEC_DEV unsigned long long two(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
SPEC_DEV void apart(unsigned long long v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
SPEC_DEV unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
SPEC_DEV unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

SPEC_DEV void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Shared-memory writes of this thread become visible to the tensor core.
SPEC_DEV void publish_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
SPEC_DEV void bar_columns() { asm volatile("bar.sync 2, 256;" ::: "memory"); }

template <int D>
struct Shape {
  static constexpr int KS = D / 16;                 // 16-channel steps of Q K^T
  static constexpr int Q_TILE = kTileCols * D * 2;  // also a K tile and a V^T tile: 128 x D f16
  static constexpr int K_AT = 2 * Q_TILE, V_AT = K_AT + 2 * Q_TILE, META_AT = V_AT + 2 * Q_TILE;
  static constexpr int NC = D / 8;
};

struct Meta {
  unsigned long long q_full[2], k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2], o_full[2], idle;
  uint32_t bad[2][4];  // tokens of a V stage whose row is NaN
  uint32_t tmem;
  int last;
};

// A position in the CTA's run: unit fields and stage.
struct Walk {
  int next, last, st, st1;
  bool more;
  SPEC_DEV Walk(const Unit& u) : next(u.next), last(u.last), st(u.st0), st1(u.st1), more(true) {}
  // Moves one stage on; returns the index of the unit entered, -1 within a unit or at the end.
  SPEC_DEV int step(const AttendParams& p) {
    if (++st < st1) return -1;
    if (next == last) {
      more = false;
      return -1;
    }
    const int ui = next++;
    st = p.units[ui].st0;
    st1 = p.units[ui].st1;
    return ui;
  }
};

// ---- unpacking: 128 threads -------------------------------------------------
template <int D>
struct Raw {
  uint4 kc[D / 32];
  uint32_t ks[D / 32];
  uint32_t vc[D / 64][8];
  uint2 vs[D / 64][4];

  SPEC_DEV void load_k(const AttendParams& p, int kvh, int table, int kv_end, int st, int th) {
    const int tok = min(st * kStageTokens + th, kv_end - 1);
    const int j = tok & (p.P - 1);
    const uint8_t* b =
        p.pool + ((long long)__ldg(p.table + table + (tok >> p.P_log2)) * p.n_kv + kvh) * block_bytes(p.P, D);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) kc[i] = *reinterpret_cast<const uint4*>(b + j * (D / 2) + i * 16);
    const uint8_t* s = b + k_scales_at(p.P, D) + j * (D / 8);
    if constexpr (D == 128) {
      const uint4 x = *reinterpret_cast<const uint4*>(s);
      ks[0] = x.x, ks[1] = x.y, ks[2] = x.z, ks[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(s);
      ks[0] = x.x, ks[1] = x.y;
    }
  }
  // Blocks of 8 tokens x 8 channels; tokens past the end read as the last block's.
  SPEC_DEV void load_v(const AttendParams& p, int kvh, int table, int kv_end, int st, int th) {
    constexpr int NC = D / 8;
    const int c = th % NC;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int tok = min(st * kStageTokens + (th / NC + i * (128 / NC)) * 8, (kv_end - 1) & ~7);
      const int j = tok & (p.P - 1);
      const uint8_t* b =
          p.pool + ((long long)__ldg(p.table + table + (tok >> p.P_log2)) * p.n_kv + kvh) * block_bytes(p.P, D);
      const uint8_t* code = b + v_codes_at(p.P, D) + (c % 8) * 4;
#pragma unroll
      for (int u = 0; u < 8; ++u) vc[i][u] = *reinterpret_cast<const uint32_t*>(code + v_piece_at(D, j + u, c / 8));
      const uint8_t* s = b + v_scales_at(p.P, D) + (j >> 1) * (D / 32 * 8) + (c / 4) * 8;
#pragma unroll
      for (int q = 0; q < 4; ++q) vs[i][q] = *reinterpret_cast<const uint2*>(s + q * (D / 32 * 8));
    }
  }
  // K tile: rows are tokens.
  SPEC_DEV void put_k(uint8_t* dst, int th) const {
    uint8_t* at = dst + (th / 8) * 256 + (th % 8) * 16;
#pragma unroll
    for (int g = 0; g < D / 32; ++g) {
      const uint32_t s = prmt(ks[g], ks[g], 0x1010), o = prmt(ks[g], ks[g], 0x3232);
      const uint32_t w[4] = {kc[g].x, kc[g].y, kc[g].z, kc[g].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(at + (2 * g + i / 2) * 4096 + (i % 2) * 128) =
            make_uint4(dq<0>(w[i], s, o), dq<1>(w[i], s, o), dq<2>(w[i], s, o), dq<3>(w[i], s, o));
    }
  }
  // V^T tile: rows are channels, 16 tokens a step.  `tail`: tokens past kv_end
  // and NaN rows are zero.
  SPEC_DEV void put_v(uint8_t* dst, int th, bool tail, int st, int kv_end) const {
    constexpr int NC = D / 8;
    const int c = th % NC;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int tb = th / NC + i * (128 / NC);
      uint32_t out[8][4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t s = prmt(vs[i][q].x, vs[i][q].y, 0x5410), o = prmt(vs[i][q].x, vs[i][q].y, 0x7632);
        if (tail) {
          const int tok = st * kStageTokens + tb * 8 + 2 * q;
          uint32_t keep = 0;
          if (tok < kv_end && (s & 0x7fffu) <= 0x7c00u) keep |= 0x0000ffffu;
          if (tok + 1 < kv_end && (s >> 16 & 0x7fffu) <= 0x7c00u) keep |= 0xffff0000u;
          s &= keep;
          o &= keep;
        }
        const uint32_t lo = prmt(vc[i][2 * q], vc[i][2 * q + 1], 0x5410), hi = prmt(vc[i][2 * q], vc[i][2 * q + 1], 0x7632);
        out[0][q] = dq<0>(lo, s, o);
        out[1][q] = dq<1>(lo, s, o);
        out[2][q] = dq<2>(lo, s, o);
        out[3][q] = dq<3>(lo, s, o);
        out[4][q] = dq<0>(hi, s, o);
        out[5][q] = dq<1>(hi, s, o);
        out[6][q] = dq<2>(hi, s, o);
        out[7][q] = dq<3>(hi, s, o);
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int r = n * NC + c;
        *reinterpret_cast<uint4*>(dst + (tb / 2) * (D * 32) + (r / 8) * 256 + (tb % 2) * 128 + (r % 8) * 16) =
            make_uint4(out[n][0], out[n][1], out[n][2], out[n][3]);
      }
    }
  }
};

template <int D>
SPEC_DEV void unpack_role(const AttendParams& p, uint8_t* smem, Meta* mt, int th) {
  using Sh = Shape<D>;
  Unit u = p.units[blockIdx.x];
  Walk w(u);
  int kvh = u.kvh, table = u.table, kv_len = u.kv_len, kv_end = u.kv_end;
  Raw<D> raw;
  raw.load_k(p, kvh, table, kv_end, w.st, th);
  raw.load_v(p, kvh, table, kv_end, w.st, th);
  bool ok = true;
  for (int k = 0; w.more; ++k) {
    const int slot = k & 1, st = w.st;
    const int now_len = kv_len, now_end = kv_end, now_table = table, now_kvh = kvh;
    const int entered = w.step(p);
    if (entered >= 0) {
      const Unit& n = p.units[entered];
      kvh = n.kvh, table = n.table, kv_len = n.kv_len, kv_end = n.kv_end;
    }
    if (k >= 2) ok = ok && mbar_wait_bounded(reinterpret_cast<uint64_t*>(&mt->k_free[slot]), (k / 2 - 1) & 1, p.err);
    raw.put_k(smem + Sh::K_AT + slot * Sh::Q_TILE, th);
    publish_smem();
    arrive(reinterpret_cast<uint64_t*>(&mt->k_full[slot]));
    if (w.more) raw.load_k(p, kvh, table, kv_end, w.st, th);
    if (k >= 2) ok = ok && mbar_wait_bounded(reinterpret_cast<uint64_t*>(&mt->v_free[slot]), (k / 2 - 1) & 1, p.err);
    const bool tail = (st + 1) * kStageTokens > now_len;
    if (tail) {
      // A stored NaN row of V is NaN in every scale: it is taken as zero here,
      // and the columns that see it are told.
      const int tok = min(st * kStageTokens + th, now_end - 1), j = tok & (p.P - 1);
      const uint8_t* blk =
          p.pool + ((long long)__ldg(p.table + now_table + (tok >> p.P_log2)) * p.n_kv + now_kvh) * block_bytes(p.P, D);
      const uint32_t one = *reinterpret_cast<const uint32_t*>(blk + v_scales_at(p.P, D) + (j >> 1) * (D / 32 * 8) + (j & 1) * 4);
      const uint32_t nans = __ballot_sync(0xffffffffu, (one & 0x7fffu) > 0x7c00u);
      if ((th & 31) == 0) mt->bad[slot][th >> 5] = nans;
    }
    raw.put_v(smem + Sh::V_AT + slot * Sh::Q_TILE, th, tail, st, now_end);
    publish_smem();
    arrive(reinterpret_cast<uint64_t*>(&mt->v_full[slot]));
    if (w.more) raw.load_v(p, kvh, table, kv_end, w.st, th);
  }
}

// ---- products: one thread ---------------------------------------------------
template <int D>
SPEC_DEV void issue_role(const AttendParams& p, uint8_t* smem, Meta* mt, uint32_t tmem) {
  using Sh = Shape<D>;
  auto bar = [](unsigned long long& b) { return reinterpret_cast<uint64_t*>(&b); };
  constexpr uint32_t kS = idesc_f16(kTileCols, kStageTokens), kO = idesc_f16(kTileCols, D);
  const uint32_t base = smem_u32(smem);
  bool ok = true;
  int k = 0;
  int waits[2] = {0, 0}, units[2] = {0, 0};  // phases of p_full and q_full
  auto scores = [&](int a, int slot) {
#pragma unroll
    for (int i = 0; i < Sh::KS; ++i)
      mma_ss(tmem + a * 128, umma_desc_kmajor(base + a * Sh::Q_TILE + i * 4096, 128, 256),
             umma_desc_kmajor(base + Sh::K_AT + slot * Sh::Q_TILE + i * 4096, 128, 256), kS, i > 0);
    umma_commit(bar(mt->s_full[a]));
  };
  int ui = blockIdx.x;
  Unit u = p.units[ui];
  for (int next = u.next; ok; ++next) {
    const int tiles = u.n_cols > kTileCols ? 2 : 1, n = u.st1 - u.st0;
    ok = ok && mbar_wait_bounded(bar(mt->k_full[k & 1]), (k >> 1) & 1, p.err);
    for (int a = 0; a < tiles; ++a) {
      ok = ok && mbar_wait_bounded(bar(mt->q_full[a]), units[a]++ & 1, p.err);
      if (!ok) break;
      tc_fence_after();
      scores(a, k & 1);
    }
    if (!ok) break;
    umma_commit(bar(mt->k_free[k & 1]));
    for (int i = 0; i < n && ok; ++i, ++k) {
      const int slot = k & 1, ahead = (k + 1) & 1;
      ok = ok && mbar_wait_bounded(bar(mt->v_full[slot]), (k >> 1) & 1, p.err);
      for (int a = 0; a < tiles && ok; ++a) {
        ok = ok && mbar_wait_bounded(bar(mt->p_full[a]), waits[a]++ & 1, p.err);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < kStageTokens / 16; ++j)
          mma_ts(tmem + 256 + a * 128, tmem + a * 128 + j * 8,
                 umma_desc_kmajor(base + Sh::V_AT + slot * Sh::Q_TILE + j * (D * 32), 128, 256), kO, i > 0 || j > 0);
        if (i + 1 == n) {
          umma_commit(bar(mt->o_full[a]));
        } else {
          if (a == 0) ok = ok && mbar_wait_bounded(bar(mt->k_full[ahead]), ((k + 1) >> 1) & 1, p.err);
          if (!ok) break;
          scores(a, ahead);
        }
      }
      if (!ok) break;
      umma_commit(bar(mt->v_free[slot]));
      if (i + 1 < n) umma_commit(bar(mt->k_free[ahead]));
    }
    if (next == u.last) break;
    u = p.units[next];
  }
  // Nothing is left in flight when tensor memory is freed.
  umma_commit(bar(mt->idle));
  mbar_wait_bounded(bar(mt->idle), 0, p.err);
}

// ---- softmax: one thread a column -------------------------------------------
template <int D>
SPEC_DEV void softmax_role(const AttendParams& p, uint8_t* smem, Meta* mt, uint32_t tmem, int a) {
  using Sh = Shape<D>;
  constexpr int NC = Sh::NC;
  auto bar = [](unsigned long long& b) { return reinterpret_cast<uint64_t*>(&b); };
  const int th = threadIdx.x & 127, G = p.n_heads / p.n_kv;
  const uint32_t lane_at = (uint32_t)(th / 32 * 32) << 16;
  const uint32_t s_at = tmem + a * 128 + lane_at, o_at = tmem + 256 + a * 128 + lane_at;
  constexpr int PART = (D + 2) * kWideCols;  // floats: [D][256], m, l
  bool ok = true;
  int k = 0, v = 0, unit = 0;  // stages of this tile, of the run; units of this tile
  Unit u = p.units[blockIdx.x];
  for (int next = u.next;; ++next) {
    const int n = u.st1 - u.st0, col = a * kTileCols + th;
    const bool on = a * kTileCols < u.n_cols, live = col < u.n_cols;
    float m = kNone, l = 0.f;
    const int r = u.col0 + (live ? col : 0), row = r / G, head = u.kvh * G + r % G;
    if (on) {
      // This column's q, in the order K's channels are unpacked.
      const long long at = (u.row0 + row) * p.q.row_stride + head * p.q.head_stride;
      uint8_t* dst = smem + a * Sh::Q_TILE + (th / 8) * 256 + (th % 8) * 16;
      float top = 0.f;
#pragma unroll 4
      for (int i = 0; i < NC; ++i) {
        float x[8];
        load8(p.q, at + i * 8, p.wide_q, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
      }
      const int ex = row_exponent(p.q.dtype, top);
      const float down = pow2i(-ex);
#pragma unroll 4
      for (int i = 0; i < NC; ++i) {
        float x[8];
        load8(p.q, at + i * 8, p.wide_q, x);
        uint4 f = make_uint4(0, 0, 0, 0);
        if (live)
          f = make_uint4(pack2(x[0] * down, x[4] * down), pack2(x[1] * down, x[5] * down),
                         pack2(x[2] * down, x[6] * down), pack2(x[3] * down, x[7] * down));
        *reinterpret_cast<uint4*>(dst + (i / 2) * 4096 + (i % 2) * 128) = f;
      }
      publish_smem();
      arrive(bar(mt->q_full[a]));
      const float c = p.scale * kLog2e * pow2i(ex);
      const unsigned long long mask = live && p.masks ? p.masks[u.row0 + row] : 0ull;
      const int idx = live ? row : -1;

      for (int st = u.st0; st < u.st1; ++st, ++k) {
        ok = ok && mbar_wait_bounded(bar(mt->s_full[a]), k & 1, p.err);
        tc_fence_after();
        const int tok = st * kStageTokens;
        const bool tail = tok + kStageTokens > u.kv_len;
        uint32_t sees[4];
        float x[32];
        if (tail) {
          // The V stage's NaN rows are known once it is unpacked.
          const int slot = (v + st - u.st0) & 1;
          ok = ok && mbar_wait_bounded(bar(mt->v_full[slot]), ((v + st - u.st0) >> 1) & 1, p.err);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            sees[q] = seen32(tok + 32 * q, u.kv_len, p.masks != nullptr, mask, idx) & first32(u.kv_end - tok - 32 * q);
          }
        }
        auto chunk = [&](int q) {  // scaled scores of tokens 32 q ..
          tm_load<32>(s_at + 32 * q, x);
          tmem_wait_ld();
        };
        float top2 = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          chunk(q);
          if (tail) {
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = (sees[q] >> i) & 1 ? x[i] * c : -INFINITY;
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] *= c;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) top2 = fmaxf(top2, x[i]);
        }
        const bool over = top2 > m + kSlack;
        if (__any_sync(0xffffffffu, over)) {
          const float mm = over ? top2 : m, f = ex2(m - mm);
          m = mm;
          l *= f;
          if (st > u.st0) {
#pragma unroll 1
            for (int q = 0; q < D / 32; ++q) {
              tm_load<32>(o_at + 32 * q, x);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] *= f;
              tm_store32(o_at + 32 * q, x);
            }
          }
        }
        const unsigned long long c2 = two(c, c), m2 = two(-m, -m);
        unsigned long long sum = two(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          chunk(q);
          uint32_t f[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float y, z;
            apart(fma2(two(x[2 * i], x[2 * i + 1]), c2, m2), y, z);
            if (tail) {
              y = (sees[q] >> (2 * i)) & 1 ? y : -INFINITY;
              z = (sees[q] >> (2 * i + 1)) & 1 ? z : -INFINITY;
            }
            y = ex2(y);
            z = ex2(z);
            sum = add2(sum, two(y, z));
            f[i] = pack2(y, z);
          }
          tm_store16(s_at + 16 * q, f);
        }
        float y, z;
        apart(sum, y, z);
        l += y + z;
        if (tail) {
          // A column that sees a NaN row of V is NaN.
          const uint32_t* b = mt->bad[(v + st - u.st0) & 1];
          if ((b[0] & sees[0]) | (b[1] & sees[1]) | (b[2] & sees[2]) | (b[3] & sees[3])) l = __int_as_float(0x7fffffff);
        }
        tm_wait_st();
        tc_fence_before();
        arrive(bar(mt->p_full[a]));
      }
      ok = ok && mbar_wait_bounded(bar(mt->o_full[a]), unit++ & 1, p.err);
      tc_fence_after();
    }
    v += n;

    // This column's O, or what is joined from partial states, to the output.
    const long long out_at = (u.row0 + row) * p.out.row_stride + head * p.out.head_stride;
    auto write = [&](int c0, const float (&x)[8][8], float inv) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e][c] * inv;
        if (live) store8(p.out, out_at + (c0 + c) * 8, p.wide_out, y);
      }
    };
    auto inverse = [](float l) { return l == 0.f ? 0.f : 1.f / l; };
    if (u.n_parts == 1) {
      if (on) {
#pragma unroll 1
        for (int c0 = 0; c0 < NC; c0 += 8) {
          float x[8][8];
#pragma unroll
          for (int e = 0; e < 8; ++e) tm_load<8>(o_at + e * NC + c0, x[e]);
          tmem_wait_ld();
          write(c0, x, inverse(l));
        }
        tc_fence_before();
      }
    } else {
      int parts = u.n_parts, at = u.part;
      long long base = u.part0;
      int* arrived = p.arrived + u.group;
      bool from_tmem = true;
      float w[kFanIn];  // weights of the parts of the last join
      long long src = 0;
      int count = 0;
      // x[e][c] of the current state: tensor memory, or the weighted parts.
      auto state = [&](int c0, float (&x)[8][8]) {
        if (from_tmem) {
#pragma unroll
          for (int e = 0; e < 8; ++e) tm_load<8>(o_at + e * NC + c0, x[e]);
          tmem_wait_ld();
          return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int c = 0; c < 8; ++c) x[e][c] = 0.f;
#pragma unroll 1
        for (int i = 0; i < count; ++i) {
          const float* s = p.parts + (src + i) * PART + col;
          float f = 0.f;
#pragma unroll
          for (int q = 0; q < kFanIn; ++q) f = q == i ? w[q] : f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int c = 0; c < 8; ++c) x[e][c] += __ldcg(s + (e * NC + c0 + c) * kWideCols) * f;
        }
      };
      while (parts > 1) {
        const int node = at / kFanIn, first = node * kFanIn;
        if (on) {
          float* dst = p.parts + (base + at) * PART + col;
#pragma unroll 1
          for (int c0 = 0; c0 < NC; c0 += 8) {
            float x[8][8];
            state(c0, x);
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
              for (int c = 0; c < 8; ++c) __stcg(dst + (e * NC + c0 + c) * kWideCols, x[e][c]);
          }
          __stcg(dst + D * kWideCols, m);
          __stcg(dst + (D + 1) * kWideCols, l);
          tc_fence_before();
        }
        __threadfence();
        bar_columns();
        if (a == 0 && th == 0) {
          const int of = min(kFanIn, parts - first);
          const bool last = atomicAdd(arrived + node, 1) == of - 1;
          if (last) arrived[node] = 0;  // ready for the next call
          mt->last = last;
        }
        bar_columns();
        if (!mt->last) break;
        __threadfence();
        count = min(kFanIn, parts - first);
        src = base + first;
        if (on) {
          m = kNone;
          float pm[kFanIn];
#pragma unroll
          for (int i = 0; i < kFanIn; ++i) {
            pm[i] = i < count ? __ldcg(p.parts + (src + i) * PART + D * kWideCols + col) : kNone;
            m = fmaxf(m, pm[i]);
          }
          l = 0.f;
#pragma unroll
          for (int i = 0; i < kFanIn; ++i) {
            w[i] = ex2(pm[i] - m);
            if (i < count) l += __ldcg(p.parts + (src + i) * PART + (D + 1) * kWideCols + col) * w[i];
          }
        }
        from_tmem = false;
        base += parts;
        parts = (parts + kFanIn - 1) / kFanIn;
        arrived += parts;
        at = node;
        bar_columns();  // mt->last is free for the next level
      }
      if (parts == 1 && on) {
#pragma unroll 1
        for (int c0 = 0; c0 < NC; c0 += 8) {
          float x[8][8];
          state(c0, x);
          write(c0, x, inverse(l));
        }
      }
      bar_columns();
    }
    if (next == u.last) break;
    u = p.units[next];
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) wide_kernel(const __grid_constant__ AttendParams p) {
  using Sh = Shape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Meta* mt = reinterpret_cast<Meta*>(smem + Sh::META_AT);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    auto init = [](unsigned long long& b, int n) { mbar_init(reinterpret_cast<uint64_t*>(&b), n); };
    for (int i = 0; i < 2; ++i) {
      init(mt->q_full[i], 128);
      init(mt->k_full[i], 128);
      init(mt->k_free[i], 1);
      init(mt->v_full[i], 128);
      init(mt->v_free[i], 1);
      init(mt->s_full[i], 1);
      init(mt->p_full[i], 128);
      init(mt->o_full[i], 1);
    }
    init(mt->idle, 1);
    fence_mbar_init();
  }
  if (warp == kIssuer) tmem_alloc(&mt->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = mt->tmem;
  if (warp < kDequant) {
    softmax_role<D>(p, smem, mt, tmem, warp / 4);
  } else if (warp < kIssuer) {
    unpack_role<D>(p, smem, mt, threadIdx.x - kDequant * 32);
  } else if ((threadIdx.x & 31) == 0) {
    issue_role<D>(p, smem, mt, tmem);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) tmem_dealloc(tmem, 512);
}

template <int D>
int smem_bytes() {
  return Shape<D>::META_AT + (int)sizeof(Meta);
}

}  // namespace

cudaError_t wide_setup() {
  cudaError_t e = cudaFuncSetAttribute(wide_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<128>());
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(wide_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<64>());
  return e;
}
size_t wide_part_floats(int head_dim) { return (size_t)(head_dim + 2) * kWideCols; }

cudaError_t launch_wide(const AttendParams& p, int head_dim, cudaStream_t s) {
  if (p.n_ctas <= 0) return cudaSuccess;
  if (head_dim == 128) wide_kernel<128><<<p.n_ctas, kThreads, smem_bytes<128>(), s>>>(p);
  else wide_kernel<64><<<p.n_ctas, kThreads, smem_bytes<64>(), s>>>(p);
  return cudaGetLastError();
}

}  // namespace kv4
}  // namespace specb200
