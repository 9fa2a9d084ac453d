// Softmax attention over the 4-bit paged KV cache for many columns: prompt
// chunks and draft trees, on the 5th-generation tensor cores.
//
// A column is a (row of the step, query head of the KV head's group).  A CTA
// walks the 128-token stages of its run, either (PAIR false) for up to 256
// columns, two tiles of 128, or (PAIR) for one tile whose stages go to two
// accumulators in turn, which are added at the end:
//   S [128 columns x 128 tokens] = Q K^T        tcgen05.mma, f16 from shared memory
//   P = 2^(c S - m), rounded to f16 in place of S in tensor memory (of every
//       32 columns of S the first 16)
//   O [128 x D] += P V                          P from tensor memory, V^T from shared memory
// Roles: warps 0-7 and 8-15 are the softmax of tile 0 and 1, two threads a
// column (tokens 0-63 and 64-127 of a stage), or of the accumulators of the one
// tile; warps 16-18 unpack K and 19-22 V, from page blocks that TMA bulk copies
// bring, into f16 operand tiles; warp 23 issues the products.  While the softmax
// of one runs, the products of the other do.  Unpacking a stage is paid once for
// both tiles (1.5 instructions an element and 256 columns), in pairs for one.
//
// What bounds it: a stage is 2048 cycles of tensor core and 2048 of
// exponentials an SM, and 2300 issue slots a scheduler.  The loops are kept
// rolled and small: warps in four roles share an instruction cache that
// unrolled ones overflow (2048 rows over 6144 tokens: 407 us unrolled, 361
// rolled).  One thread a column held 64 scores and left the special function
// unit idle three quarters of the time (272 us against 237).  Now 235 us, 1023
// TFLOP/s, in bursts at 1965 MHz; without a pause the power cap holds the clock
// near 1710 MHz and it takes 269 to 274, 880 TFLOP/s.  The tensor pipe and the
// exponentials are busy half the time each, the rest is the chain of scores,
// exponentials and product of two tiles.  A 60-node tree at 4096 tokens, 32
// query heads on 8 kv heads: 31 us, and 26 in pairs,
// where a CTA has half the columns to write out and twice the stages to overlap.
// In pairs a stage serves one tile, and unpacking it (2300 cycles of K's three
// warps, 1500 of V's four) is the longest part: 32 sequences of 64 columns at
// 4096 tokens 143 -> 130 us, but of 256 columns 180 -> 252, so the planner
// chooses.  V stored by tokens, unpacked like K, took 120 and 232 of these and
// made the second product slower (2048 rows over 6144 tokens 237 -> 250 us).
//
// Channels and tokens along a contracted axis may come in any order that both
// operands share, and O's columns in any order that the output undoes: K's
// channels are stored in the order a word's nibbles unpack (n, n + 4), and
// V^T's row for channel 8 c + n is n * D/8 + c, so that the lanes of a warp
// store neighbouring rows.
//
// K, V and P are rounded to f16, the widest operands of this rate; K's codes
// cannot enter as they are, as they do for few columns, since its scales change
// every 32 channels and one accumulator spans them all.  A rounding of K moves a
// score by 2^-11 of its terms' norm: f16 outputs of 24 sequences of 9 rows are
// off by 0.00022 of their norm, the f32 form by 0.00020.
//
// O is scaled only where a column's largest score passes its reference m by
// more than kSlack octaves; P is made before that is known.  Runs are cut as
// for the narrow kernel (kv4_attend.cu); the partial states of a column tile
// that several CTAs share are joined by a second kernel, whose blocks spread
// over the channels.
#include "common.cuh"
#include "kv4.h"
#include "kv4_mma.cuh"
#include "kv4_rows.cuh"

namespace specb200 {
namespace kv4 {
namespace {

constexpr int kTileCols = kPairCols;
constexpr int kThreads = 24 * 32;
constexpr int kUnpackK = 16, kUnpackV = 19, kIssuer = 23;  // first warps of the roles
constexpr int kThreadsK = (kUnpackV - kUnpackK) * 32;
constexpr float kFar = 1048576.f;  // 2^20: references from which scores are rounded before they are compared

// ---- tensor memory ----------------------------------------------------------
SPEC_DEV float tm_load1(uint32_t a) {
  float r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=f"(r) : "r"(a) : "memory");
  return r;
}
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
SPEC_DEV void tm_load<16>(uint32_t a, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(a)
      : "memory");
}
// Waits for the loads; the registers are used after it, not before.
template <int N>
SPEC_DEV void tm_wait(float (&r)[N]) {
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(r[i])::"memory");
}
SPEC_DEV void tm_store8(uint32_t a, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
SPEC_DEV void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// f16 A and B, f32 accumulator.
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// One lane of a converged warp.  The issuing warp runs its role whole and
// elects a lane for the products only, so that descriptors stay in uniform
// registers: a stage's 32 products must each be issued within 64 cycles, next
// to five busy warps.
SPEC_DEV bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// D (+)= A B^T, A and B in shared memory; FIRST: D is written, not added to.
template <bool FIRST>
SPEC_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "n"(FIRST ? 0 : 1)
      : "memory");
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
SPEC_DEV unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The same and others, volatile: they stay in the order they are written.
SPEC_DEV void pin_fma2(float& a, float& b, unsigned long long m, unsigned long long c) {
  unsigned long long r = two(a, b);
  asm volatile("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(r) : "l"(m), "l"(c));
  apart(r, a, b);
}
SPEC_DEV void pin_add2(unsigned long long& sum, float a, float b) {
  asm volatile("add.rn.f32x2 %0, %0, %1;" : "+l"(sum) : "l"(two(a, b)));
}
SPEC_DEV void pin_ex2(float& x) { asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(x)); }
SPEC_DEV uint32_t pin_pack2(float lo, float hi) {
  uint32_t r;
  asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
SPEC_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

SPEC_DEV void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Shared-memory writes of this thread become visible to the tensor core.
SPEC_DEV void publish_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int D, bool PAIR>
struct Shape {
  static constexpr int KS = D / 16;                 // 16-channel steps of Q K^T
  static constexpr int Q_TILE = kTileCols * D * 2;  // also a K tile and a V^T tile: 128 x D f16
  static constexpr int RAW = kStageTokens * D * 5 / 8;  // a stage's K, or V, as stored
  static constexpr int RING = PAIR ? 2 : 1;             // of those
  static constexpr int K_AT = (PAIR ? 1 : 2) * Q_TILE, V_AT = K_AT + 2 * Q_TILE;
  static constexpr int RAW_K_AT = V_AT + 2 * Q_TILE, RAW_V_AT = RAW_K_AT + RING * RAW;
  static constexpr int META_AT = RAW_V_AT + RING * RAW;
  static constexpr int NC = D / 8;
};

struct Meta {
  unsigned long long q_full[2], k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2], o_full[2], idle;
  unsigned long long raw_k[2], raw_v[2];
  uint32_t bad[2][4];  // tokens of a V stage whose row is NaN
  uint32_t tmem;
  float red[4][2][2][kTileCols];  // between the two threads of a column: largest, sum, and largest of two more turns
  float end[2][2][kTileCols];     // PAIR: the two accumulators' m and l
};

// ---- unpacking: 96 threads for K, 128 for V --------------------------------
// A position in the CTA's run: a stage, its unit's fields and (in the copying
// warp) the page of lane `lane`.
struct Walk {
  int next, last, st, st1;
  int kvh, table, sure, kv_end;
  int pages, page;
  bool more;
  SPEC_DEV void enter(const AttendParams& p, int ui) {
    const Unit& u = p.units[ui];
    st = u.st0, st1 = u.st1;
    kvh = u.kvh, table = u.table, sure = u.sure, kv_end = u.kv_end;
    next = u.next, last = u.last;
  }
  SPEC_DEV void step(const AttendParams& p) {
    if (++st < st1) return;
    const int n = next;
    if (n == last) {
      more = false;
      return;
    }
    enter(p, n);
    next = n + 1;
  }
  SPEC_DEV void look_up(const AttendParams& p, int lane) {
    const int per = kStageTokens >> p.P_log2, first = st * per;
    pages = more ? min(per, ((kv_end + p.P - 1) >> p.P_log2) - first) : 0;
    page = lane < pages ? __ldg(p.table + table + first + lane) : 0;
  }
};

// Copies a stage's K (V) halves of its page blocks; one lane a page.
template <int D>
SPEC_DEV void copy_raw(const AttendParams& p, const Walk& w, uint8_t* dst, uint64_t* bar, bool value, int lane) {
  const int half = p.P * (D / 2 + D / 8);
  if (lane == 0) mbar_arrive_expect_tx(bar, w.pages * half);
  __syncwarp();
  if (lane < w.pages)
    tma_bulk_g2s(dst + lane * half, p.pool + ((long long)w.page * p.n_kv + w.kvh) * (2 * half) + (value ? half : 0), half,
                 bar);
}

// K tile: rows are tokens; a thread takes groups of 32 channels of a token.
template <int D>
SPEC_DEV void put_k(const uint8_t* raw, uint8_t* dst, int P, int P_log2, int th) {
#pragma unroll 1
  for (int i = th; i < kStageTokens * (D / 32); i += kThreadsK) {
    const int tok = i % kStageTokens, g = i / kStageTokens, j = tok & (P - 1);
    const uint8_t* b = raw + (tok >> P_log2) * (P * (D / 2 + D / 8));
    const uint4 c = *reinterpret_cast<const uint4*>(b + j * (D / 2) + g * 16);
    const uint32_t r = *reinterpret_cast<const uint32_t*>(b + P * (D / 2) + j * (D / 8) + g * 4);
    const uint32_t s = prmt(r, r, 0x1010), o = prmt(r, r, 0x3232);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint8_t* at = dst + g * 8192 + (tok / 8) * 256 + (tok % 8) * 16;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      *reinterpret_cast<uint4*>(at + (k / 2) * 4096 + (k % 2) * 128) =
          make_uint4(dq<0>(w[k], s, o), dq<1>(w[k], s, o), dq<2>(w[k], s, o), dq<3>(w[k], s, o));
  }
}

// V^T tile: rows are channels, 16 tokens a step; a thread takes blocks of 8
// tokens x 8 channels.  keep8: the tokens (of the stage, 32 a word) that count.
template <int D>
SPEC_DEV void put_v(const uint8_t* raw, uint8_t* dst, int P, int P_log2, int th, const uint32_t (&live)[4]) {
  constexpr int NC = D / 8;
  const int c = th % NC;
#pragma unroll 1
  for (int tb = th / NC; tb < kStageTokens / 8; tb += 128 / NC) {
    const int j = tb * 8 & (P - 1);
    const uint8_t* b = raw + (tb * 8 >> P_log2) * (P * (D / 2 + D / 8));
    const uint8_t* code = b + (c % 8) * 4;
    const uint8_t* scale = b + P * (D / 2) + (j >> 1) * (D / 32 * 8) + (c / 4) * 8;
    const uint32_t word = tb < 4 ? live[0] : tb < 8 ? live[1] : tb < 12 ? live[2] : live[3];
    const uint32_t keep8 = word >> (tb % 4 * 8);
    uint32_t out[8][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint2 r = *reinterpret_cast<const uint2*>(scale + q * (D / 32 * 8));
      const uint32_t keep = ((keep8 >> (2 * q)) & 1 ? 0x0000ffffu : 0u) | ((keep8 >> (2 * q)) & 2 ? 0xffff0000u : 0u);
      const uint32_t s = prmt(r.x, r.y, 0x5410) & keep, o = prmt(r.x, r.y, 0x7632) & keep;
      const uint32_t x = *reinterpret_cast<const uint32_t*>(code + v_piece_at(D, j + 2 * q, c / 8));
      const uint32_t y = *reinterpret_cast<const uint32_t*>(code + v_piece_at(D, j + 2 * q + 1, c / 8));
      const uint32_t lo = prmt(x, y, 0x5410), hi = prmt(x, y, 0x7632);
      out[0][q] = dq<0>(lo, s, o);
      out[1][q] = dq<1>(lo, s, o);
      out[2][q] = dq<2>(lo, s, o);
      out[3][q] = dq<3>(lo, s, o);
      out[4][q] = dq<0>(hi, s, o);
      out[5][q] = dq<1>(hi, s, o);
      out[6][q] = dq<2>(hi, s, o);
      out[7][q] = dq<3>(hi, s, o);
    }
    uint8_t* at = dst + (tb / 2) * (D * 32) + (tb % 2) * 128;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int r = n * NC + c;
      *reinterpret_cast<uint4*>(at + (r / 8) * 256 + (r % 8) * 16) = make_uint4(out[n][0], out[n][1], out[n][2], out[n][3]);
    }
  }
}

template <int D, bool PAIR, bool VALUE>
SPEC_DEV void unpack_role(const AttendParams& p, uint8_t* smem, Meta* mt, int th) {
  using Sh = Shape<D, PAIR>;
  auto bar = [](unsigned long long& b) { return reinterpret_cast<uint64_t*>(&b); };
  uint8_t* ring = smem + (VALUE ? Sh::RAW_V_AT : Sh::RAW_K_AT);
  unsigned long long* raw_full = VALUE ? mt->raw_v : mt->raw_k;
  unsigned long long* full = VALUE ? mt->v_full : mt->k_full;
  unsigned long long* free_ = VALUE ? mt->v_free : mt->k_free;
  Walk w;  // the next stage to copy
  w.more = true;
  w.enter(p, blockIdx.x);
  int copies = 0;
  int st[2], sure[2], kv_end[2];  // of the stages under way
  auto copy = [&](int at, bool ok) {
    if (th < 32 && ok) copy_raw<D>(p, w, ring + copies % Sh::RING * Sh::RAW, bar(raw_full[copies % Sh::RING]), VALUE, th);
    st[at] = w.st, sure[at] = w.sure, kv_end[at] = w.kv_end;
    ++copies;
    w.step(p);
  };
#pragma unroll
  for (int i = 0; i < Sh::RING; ++i) {
    if (th < 32) w.look_up(p, th);
    if (w.more) copy(i, true);
  }
  bool ok = true;
#pragma unroll 1
  for (int k = 0;; ++k) {
    const int slot = k & 1;
    const uint8_t* raw = ring + k % Sh::RING * Sh::RAW;
    if (th < 32) w.look_up(p, th);
    ok = ok && mbar_wait_bounded(bar(raw_full[k % Sh::RING]), k / Sh::RING & 1, p.err);
    if (k >= 2) ok = ok && mbar_wait_bounded(bar(free_[slot]), (k / 2 - 1) & 1, p.err);
    uint8_t* dst = smem + (VALUE ? Sh::V_AT : Sh::K_AT) + slot * Sh::Q_TILE;
    if constexpr (VALUE) {
      uint32_t live[4] = {~0u, ~0u, ~0u, ~0u};
      if ((st[0] + 1) * kStageTokens > sure[0]) {
        // Past the end V counts nothing.  A stored NaN row is NaN in every
        // scale: it is taken as zero here, and the columns that see it are told.
        const int j = th & (p.P - 1);
        const uint32_t one = *reinterpret_cast<const uint32_t*>(
            raw + (th >> p.P_log2) * (p.P * (D / 2 + D / 8)) + p.P * (D / 2) + (j >> 1) * (D / 32 * 8) + (j & 1) * 4);
        const uint32_t nans = __ballot_sync(0xffffffffu, (one & 0x7fffu) > 0x7c00u);
        if ((th & 31) == 0) mt->bad[slot][th >> 5] = nans;
        asm volatile("bar.sync 4, 128;" ::: "memory");
#pragma unroll
        for (int q = 0; q < 4; ++q) live[q] = first32(kv_end[0] - st[0] * kStageTokens - 32 * q) & ~mt->bad[slot][q];
      }
      put_v<D>(raw, dst, p.P, p.P_log2, th, live);
    } else {
      put_k<D>(raw, dst, p.P, p.P_log2, th);
    }
    publish_smem();
    arrive(bar(full[slot]));
    if (k + 1 == copies && !w.more) break;
    if constexpr (PAIR) st[0] = st[1], sure[0] = sure[1], kv_end[0] = kv_end[1];
    if (w.more) {
      // All its threads have read the raw stage.
      if (VALUE) asm volatile("bar.sync 4, 128;" ::: "memory");
      else asm volatile("bar.sync 3, %0;" ::"n"(kThreadsK) : "memory");
      copy(Sh::RING - 1, th >= 32 || __all_sync(0xffffffffu, ok));
    }
  }
  // Leave no copy in flight.
  if (!ok)
#pragma unroll 1
    for (int i = 1; i <= Sh::RING && i <= copies; ++i)
      mbar_wait_bounded(bar(raw_full[(copies - i) % Sh::RING]), (copies - i) / Sh::RING & 1, p.err);
}

// ---- products: one warp -----------------------------------------------------
template <int D, bool PAIR>
SPEC_DEV void issue_role(const AttendParams& p, uint8_t* smem, Meta* mt, uint32_t tmem) {
  using Sh = Shape<D, PAIR>;
  auto bar = [](unsigned long long& b) { return reinterpret_cast<uint64_t*>(&b); };
  constexpr uint32_t kS = idesc_f16(kTileCols, kStageTokens), kO = idesc_f16(kTileCols, D);
  tmem = __shfl_sync(0xffffffffu, tmem, 0);
  const uint64_t q0 = umma_desc_kmajor(smem_u32(smem), 128, 256);  // Q tile 0; the others lie at multiples of 16 bytes
  constexpr uint64_t kTile16 = Sh::Q_TILE / 16, kK16 = Sh::K_AT / 16, kV16 = Sh::V_AT / 16;
  auto wait = [&](unsigned long long& b, int parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar(b), parity, p.err)) != 0;
  };
  auto scores = [&](int a, int slot, bool free_k) {
    if (elect_one()) {
      const uint64_t qa = PAIR ? q0 : q0 + a * kTile16, kb = q0 + kK16 + slot * kTile16;
      const uint32_t d = tmem + a * 128;
      mma_ss<true>(d, qa, kb, kS);
#pragma unroll
      for (int i = 1; i < Sh::KS; ++i) mma_ss<false>(d, qa + i * 256, kb + i * 256, kS);
      umma_commit(bar(mt->s_full[a]));
      if (free_k) umma_commit(bar(mt->k_free[slot]));
    }
    __syncwarp();
  };
  constexpr int kAhead = PAIR ? 2 : 1;  // stages from one of an accumulator to its next
  int k = 0;
  int waits = 0, units = 0;  // phases of p_full and q_full, a bit a tile
  Unit u = p.units[blockIdx.x];
  bool ok = true;
#pragma unroll 1
  for (int next = __shfl_sync(0xffffffffu, u.next, 0);; ++next) {
    const int n = __shfl_sync(0xffffffffu, u.st1 - u.st0, 0), last = __shfl_sync(0xffffffffu, u.last, 0);
    const int tiles = PAIR ? 1 : __shfl_sync(0xffffffffu, u.n_cols, 0) > kTileCols ? 2 : 1;
    const int first = PAIR ? (n > 1 ? 2 : 1) : tiles;  // accumulators that begin
    ok = true;
#pragma unroll 1
    for (int a = 0; a < first && ok; ++a) {
      const int at = PAIR ? k + a : k;
      ok = wait(mt->k_full[at & 1], (at >> 1) & 1) && wait(mt->q_full[a], units >> a & 1);
      if (!ok) break;
      units ^= 1 << a;
      tc_fence_after();
      scores(a, at & 1, PAIR || a == tiles - 1);
    }
#pragma unroll 1
    for (int i = 0; i < n && ok; ++i, ++k) {
      const int slot = k & 1, ahead = k + kAhead;  // the stage whose scores follow
      const bool more = i + kAhead < n;
      ok = wait(mt->v_full[slot], (k >> 1) & 1);
#pragma unroll 1
      for (int t = 0; t < tiles && ok; ++t) {
        const int a = PAIR ? i & 1 : t;
        ok = wait(mt->p_full[a], waits >> a & 1);
        if (!ok) break;
        waits ^= 1 << a;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vb = q0 + kV16 + slot * kTile16;
          const uint32_t d = tmem + 256 + a * 128, pa = tmem + a * 128;
          mma_ts(d, pa, vb, kO, i >= kAhead);
#pragma unroll
          for (int j = 1; j < kStageTokens / 16; ++j)
            mma_ts(d, pa + j / 2 * 32 + j % 2 * 8, vb + j * (D * 2), kO, 1);
          if (!more) umma_commit(bar(mt->o_full[a]));
          if (t == tiles - 1) umma_commit(bar(mt->v_free[slot]));
        }
        __syncwarp();
        if (more) {
          if (t == 0) ok = wait(mt->k_full[ahead & 1], (ahead >> 1) & 1);
          if (!ok) break;
          scores(a, ahead & 1, t == tiles - 1);
        }
      }
    }
    if (!ok || next == last) break;
    u = p.units[next];
  }
  // Nothing is left in flight when tensor memory is freed.
  if (elect_one()) umma_commit(bar(mt->idle));
  __syncwarp();
  wait(mt->idle, 0);
}

// ---- softmax: two threads a column ------------------------------------------
SPEC_DEV uint4 raw8(const Rows& r, long long at, bool wide) {
  const uint16_t* s = static_cast<const uint16_t*>(r.ptr) + at;
  if (wide) return *reinterpret_cast<const uint4*>(s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = s[2 * i] | (uint32_t)s[2 * i + 1] << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Chunk i of a q row as 8 f16 in the order K's channels are unpacked.
template <int D>
SPEC_DEV void put_q(uint8_t* row, int i, const uint4& w, int dtype, float down, bool live) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[e]));
    x[2 * e] = dtype == T_BF16 ? __uint_as_float(v[e] << 16) : f.x;
    x[2 * e + 1] = dtype == T_BF16 ? __uint_as_float(v[e] & 0xffff0000u) : f.y;
  }
  uint4 f = make_uint4(0, 0, 0, 0);
  if (live)
    f = make_uint4(pack2(x[0] * down, x[4] * down), pack2(x[1] * down, x[5] * down), pack2(x[2] * down, x[6] * down),
                   pack2(x[3] * down, x[7] * down));
  *reinterpret_cast<uint4*>(row + (i / 2) * 4096 + (i % 2) * 128) = f;
}

// Scores that are not seen.
SPEC_DEV void hide(float (&x)[32], uint32_t seen) {
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = (seen >> i) & 1 ? x[i] : -INFINITY;
}

template <int D, bool PAIR>
SPEC_DEV void softmax_role(const AttendParams& p, uint8_t* smem, Meta* mt, uint32_t tmem, int a, int half) {
  using Sh = Shape<D, PAIR>;
  constexpr int NC = Sh::NC;
  auto bar = [](unsigned long long& b) { return reinterpret_cast<uint64_t*>(&b); };
  const int th = threadIdx.x & 127, G = p.n_heads / p.n_kv, col = PAIR ? th : a * kTileCols + th;
  const uint32_t lane_at = (uint32_t)(th / 32 * 32) << 16;
  const uint32_t s_at = tmem + a * 128 + 64 * half + lane_at, o_at = tmem + 256 + a * 128 + lane_at;
  // A value of this thread's for the column's other one, and back.  (Between
  // two uses of a `kind` lies a barrier that both threads reach after reading:
  // q_full or p_full.)
  auto meet = [&](int kind, float mine) {
    mt->red[kind][a][half][th] = mine;
    // Of the two warps that share these 32 columns alone: how often they meet
    // depends on the columns' scores.
    asm volatile("bar.sync %0, 64;" ::"r"(5 + a * 4 + th / 32) : "memory");
    return mt->red[kind][a][half ^ 1][th];
  };
  constexpr int kStep = PAIR ? 2 : 1;
  bool ok = true;
  int k = 0, v = 0, unit = 0;  // stages of this tile, of the run; units of this tile
  Unit u = p.units[blockIdx.x];
#pragma unroll 1
  for (int next = u.next;; ++next) {
    const bool both = PAIR && u.st1 - u.st0 > 1;  // accumulators of this unit
    if (a == 0 || (PAIR ? both : u.n_cols > kTileCols)) {
      const bool live = col < u.n_cols;
      const int r = u.col0 + (live ? col : 0), row = r / G, head = u.kvh * G + r % G;
      // This column's q (half of its channels a thread), in the order K's
      // channels are unpacked.  A negative scale goes to q's sign, so that the
      // largest product is the largest score.  Converted as it is, four 16-byte
      // loads in flight; a row whose largest magnitude (16-bit floats without
      // their sign order as integers) is far from 1 is converted again, scaled
      // by a power of two.
      const long long at = (u.row0 + row) * p.q.row_stride + head * p.q.head_stride;
      uint8_t* dst = smem + (PAIR ? 0 : a * Sh::Q_TILE) + (th / 8) * 256 + (th % 8) * 16;
      const float sign = p.scale < 0.f ? -1.f : 1.f;
      uint32_t top = 0;
#pragma unroll 1
      for (int i0 = half * (NC / 2); i0 < (half + 1) * (NC / 2); i0 += 4) {
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = raw8(p.q, at + (i0 + i) * 8, p.wide_q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top = __vmaxu2(top, __vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu));
          top = __vmaxu2(top, __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
          if (!PAIR || a == 0) put_q<D>(dst, i0 + i, w[i], p.q.dtype, sign, live);
        }
      }
      top = max(top & 0xffffu, top >> 16);
      const float other_top = meet(0, __uint_as_float(top << 16));
      int ex = row_exponent(p.q.dtype, fmaxf(__uint_as_float(top << 16), other_top));
      if (ex >= -4 && ex <= 14) {
        ex = 0;
      } else if (!PAIR || a == 0) {
#pragma unroll 1
        for (int i = half * (NC / 2); i < (half + 1) * (NC / 2); ++i)
          put_q<D>(dst, i, raw8(p.q, at + i * 8, p.wide_q), p.q.dtype, sign * pow2i(-ex), live);
      }
      publish_smem();
      arrive(bar(mt->q_full[a]));
      // Not zero: a score that is not seen is -inf, and stays that when scaled.
      const float c = fmaxf(fabsf(p.scale) * kLog2e * pow2i(ex), 1e-37f);
      const unsigned long long mask = live && p.masks ? p.masks[u.row0 + row] : 0ull;
      const int idx = live ? row : -1;
      float m = kNone, l = 0.f;

#pragma unroll 1
      for (int st = u.st0 + (PAIR ? a : 0); st < u.st1; st += kStep, ++k) {
        const int tok = st * kStageTokens + 64 * half, stage = v + st - u.st0;
        const bool tail = (st + 1) * kStageTokens > u.sure;
        uint32_t sees[2] = {~0u, ~0u};
        if (tail) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            sees[q] = seen32(tok + 32 * q, u.kv_len, p.masks != nullptr, mask, idx) & first32(u.kv_end - tok - 32 * q);
        }
        ok = ok && mbar_wait_bounded(bar(mt->s_full[a]), k & 1, p.err);
        tc_fence_after();
        // P against the column's last reference, kept in registers until the
        // column's largest exponent is known.  Where that passes kSlack, or
        // there is no reference yet, it moves the reference and P is made
        // again; the scores are still there.  Two passes, by construction: the
        // second decides nothing.  Its largest exponent is what rounding took
        // off the reference, an eighth at most below kFar.  Above, that would
        // be octaves (8 from 2^27 on): there the scores are rounded in place
        // first and the reference is the largest of them, so that it is 0.
        uint32_t f[32];
        float added;
        int kind = 0;
#pragma unroll 1
        while (true) {
          const float base = m == kNone ? 0.f : m;
          const float by_c = kind == 3 ? 1.f : c;
          const unsigned long long c2 = two(by_c, by_c), m2 = two(-base, -base);
          unsigned long long sum[2] = {two(0.f, 0.f), two(0.f, 0.f)};
          float best = -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x[32];
            tm_load<16>(s_at + 32 * h, x);
            tm_load<16>(s_at + 32 * h + 16, x + 16);
            tm_wait(x);
            if (tail) hide(x, sees[h]);
            // Two exponentials every 16 cycles is what the special function
            // unit gives a scheduler; the pinned order keeps it fed, the
            // multiply-adds two pairs ahead of it and the sums and roundings
            // four pairs behind (32 scores: 328 cycles alone, 487 in the
            // compiler's order).
#pragma unroll
            for (int j = 0; j < 16 + 6; ++j) {
              if (j < 16) {
                pin_fma2(x[2 * j], x[2 * j + 1], c2, m2);
                best = max3(best, x[2 * j], x[2 * j + 1]);
              }
              if (j >= 2 && j < 18) pin_ex2(x[2 * j - 4]), pin_ex2(x[2 * j - 3]);
              if (j >= 6) {
                const int i = j - 6;
                pin_add2(sum[i % 2], x[2 * i], x[2 * i + 1]);
                f[16 * h + i] = pin_pack2(x[2 * i], x[2 * i + 1]);
              }
            }
          }
          float sum_lo, sum_hi;
          apart(add2(sum[0], sum[1]), sum_lo, sum_hi);
          added = sum_lo + sum_hi;
          best = fmaxf(best, meet(kind, best));
          bool over = m == kNone ? best > -INFINITY : best > kSlack;
          // Both warps of these columns decide alike.
          if (kind || !__any_sync(0xffffffffu, over || fabsf(base) >= kFar)) break;
          kind = 2;
          float mm = over ? base + best : m;
          if (__any_sync(0xffffffffu, fabsf(base) >= kFar || (over && fabsf(mm) >= kFar))) {
            kind = 3;
            float top = -INFINITY;
#pragma unroll 1
            for (int q = 0; q < 64; q += 8) {
              float x[8];
              tm_load<8>(s_at + q, x);
              tm_wait(x);
              const uint32_t seen = (q < 32 ? sees[0] : sees[1]) >> (q & 31);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                x[i] = __fmul_rn(x[i], c);
                if ((seen >> i) & 1) top = fmaxf(top, x[i]);
              }
              tm_store8(s_at + q, reinterpret_cast<const uint32_t*>(x));
            }
            tm_wait_st();
            top = fmaxf(top, meet(2, top));
            over = m == kNone ? top > -INFINITY : top - base > kSlack;
            mm = over ? top : m;
          }
          const float by = ex2(m - mm);
          m = mm;
          l *= by;
          if (st >= u.st0 + kStep) {
#pragma unroll 1
            for (int q = half * (D / 2); q < (half + 1) * (D / 2); q += 8) {
              float o[8];
              tm_load<8>(o_at + q, o);
              tm_wait(o);
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] *= by;
              tm_store8(o_at + q, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        l += added;
#pragma unroll
        for (int b = 0; b < 4; ++b) tm_store8(s_at + b / 2 * 32 + b % 2 * 8, f + 8 * b);
        if (tail) {
          // A column that sees a NaN row of V, known once V is unpacked, is NaN.
          ok = ok && mbar_wait_bounded(bar(mt->v_full[stage & 1]), (stage >> 1) & 1, p.err);
          const uint32_t* b = mt->bad[stage & 1] + 2 * half;
          if ((b[0] & sees[0]) | (b[1] & sees[1])) l = __int_as_float(0x7fffffff);
        }
        tm_wait_st();
        tc_fence_before();
        arrive(bar(mt->p_full[a]));
      }
      ok = ok && mbar_wait_bounded(bar(mt->o_full[a]), unit++ & 1, p.err);
      tc_fence_after();
      l += meet(1, l);
      // PAIR: a thread reads both accumulators, which lie in the same lanes.
      float by[2] = {1.f, 0.f};
      if (both) {
        if (half == 0) mt->end[a][0][th] = m, mt->end[a][1][th] = l;
        tc_fence_before();
        asm volatile("bar.sync 2, 512;" ::: "memory");
        tc_fence_after();
        m = fmaxf(mt->end[0][0][th], mt->end[1][0][th]);
#pragma unroll
        for (int i = 0; i < 2; ++i) by[i] = ex2(mt->end[i][0][th] - m);
        l = mt->end[0][1][th] * by[0] + mt->end[1][1][th] * by[1];
      }
      // O to the output, or as a partial state [D][256], m, l; half (a quarter)
      // of the channels a thread.
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const long long out_at = (u.row0 + row) * p.out.row_stride + head * p.out.head_stride;
      float* part = p.parts + (long long)(u.part0 + u.part) * ((D + 2) * kWideCols) + col;
      const int share = both ? NC / 4 : NC / 2, i0 = (both ? 2 * a + half : half) * share;
#pragma unroll 1
      for (int i = i0; i < i0 + share; ++i) {
        float y[8];  // channels 8 i ..
        if (both) {
          float z[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            y[e] = tm_load1(o_at - a * 128 + e * NC + i);
            z[e] = tm_load1(o_at - a * 128 + 128 + e * NC + i);
          }
          tm_wait(y);
          tm_wait(z);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = y[e] * by[0] + z[e] * by[1];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = tm_load1(o_at + e * NC + i);
          tm_wait(y);
        }
        if (u.n_parts == 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= inv;
          if (live) store8(p.out, out_at + i * 8, p.wide_out, y);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) part[(i * 8 + e) * kWideCols] = y[e];
        }
      }
      if (u.n_parts > 1 && half == 0 && (!PAIR || a == 0)) {
        part[D * kWideCols] = m;
        part[(D + 1) * kWideCols] = l;
      }
      tc_fence_before();
      // Before an accumulator, or the states above, are written again.
      if (both) asm volatile("bar.sync 2, 512;" ::: "memory");
    }
    v += u.st1 - u.st0;
    if (next == u.last) break;
    u = p.units[next];
  }
}

// Joins the partial states of a column tile: a thread a column, 8 channels a
// block.  The states are read once and in order.
template <int D>
__global__ void __launch_bounds__(kWideCols) wide_join_kernel(const __grid_constant__ AttendParams p) {
  constexpr int PART = (D + 2) * kWideCols;
  pdl_launch_dependents();
  pdl_wait();
  const Unit& u = p.joins[blockIdx.x];
  const int col = threadIdx.x, c = blockIdx.y, n = u.n_parts, G = p.n_heads / p.n_kv;
  if (col >= u.n_cols) return;
  const float* s = p.parts + (long long)u.part0 * PART + col;
  float m = kNone;
#pragma unroll 8
  for (int i = 0; i < n; ++i) m = fmaxf(m, s[(long long)i * PART + D * kWideCols]);
  float l = 0.f, x[8] = {};
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float* q = s + (long long)i * PART;
    const float w = ex2(q[D * kWideCols] - m);
    l += q[(D + 1) * kWideCols] * w;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += q[(c * 8 + e) * kWideCols] * w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= inv;
  const int r = u.col0 + col;
  store8(p.out, (u.row0 + r / G) * p.out.row_stride + (u.kvh * G + r % G) * p.out.head_stride + c * 8, p.wide_out, x);
}

template <int D, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) wide_kernel(const __grid_constant__ AttendParams p) {
  using Sh = Shape<D, PAIR>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Meta* mt = reinterpret_cast<Meta*>(smem + Sh::META_AT);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    auto init = [](unsigned long long& b, int n) { mbar_init(reinterpret_cast<uint64_t*>(&b), n); };
    for (int i = 0; i < 2; ++i) {
      init(mt->q_full[i], 256);
      init(mt->k_full[i], kThreadsK);
      init(mt->k_free[i], 1);
      init(mt->v_full[i], 128);
      init(mt->v_free[i], 1);
      init(mt->s_full[i], 1);
      init(mt->p_full[i], 256);
      init(mt->o_full[i], 1);
      init(mt->raw_k[i], 1);
      init(mt->raw_v[i], 1);
    }
    init(mt->idle, 1);
    fence_mbar_init();
  }
  if (warp == kIssuer) tmem_alloc(&mt->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = mt->tmem;
  pdl_wait();
  if (warp < kUnpackK) {
    softmax_role<D, PAIR>(p, smem, mt, tmem, warp / 8, warp / 4 % 2);
  } else if (warp < kUnpackV) {
    unpack_role<D, PAIR, false>(p, smem, mt, threadIdx.x - kUnpackK * 32);
  } else if (warp < kIssuer) {
    unpack_role<D, PAIR, true>(p, smem, mt, threadIdx.x - kUnpackV * 32);
  } else {
    issue_role<D, PAIR>(p, smem, mt, tmem);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) tmem_dealloc(tmem, 512);
}

template <int D, bool PAIR>
int smem_bytes() {
  return Shape<D, PAIR>::META_AT + (int)sizeof(Meta);
}
template <int D, bool PAIR>
cudaError_t allow() {
  return cudaFuncSetAttribute(wide_kernel<D, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<D, PAIR>());
}
template <int D, bool PAIR>
cudaError_t launch(const AttendParams& p, cudaStream_t s) {
  const cudaError_t e =
      launch_overlapping(wide_kernel<D, PAIR>, dim3(p.n_ctas), kThreads, smem_bytes<D, PAIR>(), s, p);
  if (e != cudaSuccess || !p.n_joins) return e;
  return launch_overlapping(wide_join_kernel<D>, dim3(p.n_joins, D / 8), PAIR ? kTileCols : kWideCols, 0, s, p);
}

}  // namespace

cudaError_t wide_setup() {
  cudaError_t e = allow<128, false>();
  if (e == cudaSuccess) e = allow<128, true>();
  if (e == cudaSuccess) e = allow<64, false>();
  if (e == cudaSuccess) e = allow<64, true>();
  return e;
}
size_t wide_part_floats(int head_dim) { return (size_t)(head_dim + 2) * kWideCols; }

cudaError_t launch_wide(const AttendParams& p, int head_dim, bool pair, cudaStream_t s) {
  if (p.n_ctas <= 0) return cudaSuccess;
  if (head_dim == 128) return pair ? launch<128, true>(p, s) : launch<128, false>(p, s);
  return pair ? launch<64, true>(p, s) : launch<64, false>(p, s);
}

}  // namespace kv4
}  // namespace specb200
