// Sampling from rows of logits, and acceptance of drafted tokens against them,
// for many sequences at once.
//
//   p_j = w_j / Z,  w_j = exp((l_j - M) / T),  M = max l,  Z = sum w
//   token(u) = the first j with w_0 + ... + w_j > u Z
//   a draft x drawn from q is kept when q(x) <= 0 or u q(x) Z <= w_x; where it
//   is not, the next token is drawn from the weights max(p - q, 0)
//
// Decisions are those of 64-bit arithmetic.  The sums are taken in f32 with
// a bound on their error, and where a comparison falls inside it the row is
// summed again in 64 bits by the whole cluster.  A weight is 2^(l h - R) with
// h = log2(e) / T and a whole number R next to h times the largest logit, one
// multiply-add, so that sums of different R join exactly.  With u = 2^-24 and
// d = (M - l) / T: h is off by 1.5 u and the multiply-add by u, a weight by
// (2.5 d + 0.5) u, the hardware's 2^x by 4 u more.  Of positive terms a chunk's
// sum is off by 9 u (16 a lane in pairs, 5 rounds of shuffles), a prefix of
// chunks by 12 u more (7 additions, 5 rounds), Z by 15 (8 and, of 8 blocks, 7),
// one inside a chunk by 20 u (15 and 5).  The mean of d under the weights of any
// set of columns is their entropy less the logarithm of their sum S, at most
// ln V - ln S, so that weights of sum S are off by (4.5 + 2.5 (ln V - ln S)) u S
// in all (spread(S) below; it grows with S up to V / e).  For S >= 1 and V <= 2^20
// that makes (4.5 + 24 + 2.5 * 13.9) u < 2^-18 of S (kErr).
//
// A comparison of a prefix with v Z, 0 <= v <= 1, is off by what its two sides
// are, or, as the columns before the chunk of the token are summed once for both,
// by max(v, 1 - v) of what all weights are off by and less than twice what the
// chunk's are: the smaller of the two counts.  Targets up to 2^-33, and rows
// with |M| h of 2^22 and more, are left to 64 bits.
//
// Two kernels.  stats_kernel reads every row once, a warp one chunk of 512
// columns or 8 KB, and leaves each chunk's reference and sum.  The second
// kernel runs a cluster a row (sample) or a sequence (chains, trees); a warp
// joins a row's chunks by a scan over their sums, finds the chunk of the token
// and reads that alone.  A rejected draft's max(p - q, 0) is summed by all warps
// of the cluster, from p and q once more.
//
// Device time: one f32 row of 128256 5.2 us (latency), 64 bf16 rows with
// probabilities 20.6 (49 MB), 64 sequences of 5 bf16 rows 43 (115 MB).  The first
// kernel is bound by memory (98 MB in 18 us, 5.4 TB/s), the second by its chain of
// dependent reads and cluster barriers (5 to 20 us).  A row that needs 64 bits takes
// 13 us more, a rejected draft's 30.  One launch for a single short chain, too, saves
// the host 3 us and takes the device 7 longer.  Three blocks an SM of the chains' kernel leave 80
// registers; with f32 rows 72 bytes a thread spill.
#include "batch.h"
#include "common.cuh"
#include "kv4_rows.cuh"

namespace specb200 {
namespace batch {
namespace {

constexpr float kErr = 1.f / (1 << 18);  // of a sum of weights, relative
constexpr int kBad = -1, kUnsure = -2;
constexpr int kPer = kChunk / 32;  // columns of a lane
constexpr int kThreads = 256;      // of the second kernels
constexpr int kWarps = kThreads / 32;

SPEC_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
SPEC_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
SPEC_DEV int cluster_rank() {
  int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
SPEC_DEV int cluster_size() {
  int r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);  // columns of a vector
};

// A row of logits and its temperature.
template <class T>
struct Row {
  const T* p;
  int shift, V;  // columns between the first chunk's start and column 0
  float t;       // temperature; 0: the largest logit
  float h;       // log2(e) / t
  bool ok;       // the temperature is finite and not negative

  SPEC_DEV Row() {}
  SPEC_DEV void place(const Rows& r, int row) {
    p = static_cast<const T*>(r.logits) + row * r.stride;
    V = r.V;
    shift = (int)(reinterpret_cast<uintptr_t>(p) / sizeof(T) % Vec<T>::N);
  }
  SPEC_DEV Row(const Rows& r, int row) {
    place(r, row);
    t = r.temps ? r.temps[row] : r.temp;
    ok = t >= 0.f && t < INFINITY;
    if (t > 0.f) t = fminf(fmaxf(t, 0x1p-60f), 0x1p60f);
    // 1 / t and log2(e) as sums of two numbers, so that h is their product rounded about once.
    const float d = t > 0.f ? t : 1.f, hi = 1.f / d, lo = fmaf(-hi, d, 1.f) * hi;
    const float L = 1.44269504f, Llo = 1.925963033e-8f;
    h = hi * L;
    h += fmaf(hi, L, -h) + fmaf(hi, Llo, lo * L);
  }
};

// The reference of weights whose largest logit is m.
struct Ref {
  float h, m, R;
  bool whole;  // R is a whole number; otherwise m h is too large for one
  SPEC_DEV Ref() {}
  SPEC_DEV Ref(float m_, float h_) : h(h_), m(m_) {
    const float y = m * h;
    whole = fabsf(y) < 0x1p22f;
    R = whole ? rintf(y) : y;
  }
  SPEC_DEV float weight(float x) const { return ex2(whole ? fmaf(x, h, -R) : (x - m) * h); }
};

template <class T>
struct Fill;  // a vector of -inf
template <>
struct Fill<float> {
  static constexpr uint32_t kWord = 0xff800000u;
};
template <>
struct Fill<__nv_bfloat16> {
  static constexpr uint32_t kWord = 0xff80ff80u;
};
template <>
struct Fill<__half> {
  static constexpr uint32_t kWord = 0xfc00fc00u;
};

// Columns e .. of a row (e from a 16-byte boundary); those outside the row are -inf.
template <class T>
SPEC_DEV uint4 load_vec(const Row<T>& r, int e) {
  constexpr int N = Vec<T>::N;
  if (e >= 0 && e + N <= r.V) return *reinterpret_cast<const uint4*>(r.p + e);
  uint32_t w[4] = {Fill<T>::kWord, Fill<T>::kWord, Fill<T>::kWord, Fill<T>::kWord};
  if (e > -N && e < r.V) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (e + k >= 0 && e + k < r.V) {
        if constexpr (N == 4) {
          w[k] = __float_as_uint(r.p[e + k]);
        } else {
          const uint32_t v = reinterpret_cast<const uint16_t*>(r.p)[e + k];
          w[k / 2] = k % 2 ? (w[k / 2] & 0xffffu) | v << 16 : (w[k / 2] & 0xffff0000u) | v;
        }
      }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
SPEC_DEV void unpack(const uint4& v, float (&x)[4], const float*) {
  x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
SPEC_DEV void unpack(const uint4& v, float (&x)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) x[2 * k] = __uint_as_float(w[k] << 16), x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
}
SPEC_DEV void unpack(const uint4& v, float (&x)[8], const __half*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
}
// Largest element of vectors; a NaN counts only where all are.
template <int NV>
SPEC_DEV float largest(const uint4* v, const float*) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y)),
                       fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w))));
  return m;
}
template <int NV, class H, class H2>
SPEC_DEV float largest_of_pairs(const uint4* v) {
  H2 m;
  *reinterpret_cast<uint32_t*>(&m) = Fill<H>::kWord;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) m = __hmax2(m, *reinterpret_cast<const H2*>(&w[k]));
  }
  return fmaxf((float)m.x, (float)m.y);
}
template <int NV>
SPEC_DEV float largest(const uint4* v, const __nv_bfloat16*) {
  return largest_of_pairs<NV, __nv_bfloat16, __nv_bfloat162>(v);
}
template <int NV>
SPEC_DEV float largest(const uint4* v, const __half*) {
  return largest_of_pairs<NV, __half, __half2>(v);
}
SPEC_DEV float to_float(float x) { return x; }
SPEC_DEV float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
SPEC_DEV float to_float(__half x) { return __half2float(x); }

// Where this lane's i-th vector of a chunk starts: vectors 32 i + lane (read
// along the row by all lanes), or the lane's own 16 columns one after another.
template <class T, bool RUN>
SPEC_DEV int column(const Row<T>& r, int c, int i, int lane) {
  return c * kChunk - r.shift + (RUN ? lane * (kPer / Vec<T>::N) + i : i * 32 + lane) * Vec<T>::N;
}
// Whether all of a chunk's columns are the row's.
template <class T>
SPEC_DEV bool inside(const Row<T>& r, int c) {
  return c * kChunk >= r.shift && (c + 1) * kChunk - r.shift <= r.V;
}
template <class T, bool RUN>
SPEC_DEV void load_raw(const Row<T>& r, int c, int lane, uint4 (&v)[kPer / Vec<T>::N]) {
  constexpr int N = Vec<T>::N, NV = kPer / N;
  const int e = column<T, RUN>(r, c, 0, lane);
  if (inside(r, c)) {
    const uint4* at = reinterpret_cast<const uint4*>(r.p + e);
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = at[RUN ? i : i * 32];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = load_vec(r, e + (RUN ? i : i * 32) * N);
  }
}
template <class T>
SPEC_DEV void unpack_chunk(const uint4* v, float (&x)[kPer], const T* tag) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int i = 0; i < kPer / N; ++i) {
    float y[N];
    unpack(v[i], y, tag);
#pragma unroll
    for (int k = 0; k < N; ++k) x[i * N + k] = y[k];
  }
}
template <class T, bool RUN>
SPEC_DEV void load_chunk(const Row<T>& r, int c, int lane, float (&x)[kPer]) {
  uint4 v[kPer / Vec<T>::N];
  load_raw<T, RUN>(r, c, lane, v);
  unpack_chunk(v, x, r.p);
}

// The same columns of a row of f32 probabilities; zeros outside.
template <class T, bool RUN>
SPEC_DEV void load_probs(const Row<T>& r, const float* q, int c, int lane, float (&x)[kPer]) {
  constexpr int N = Vec<T>::N;
  const bool wide = (reinterpret_cast<uintptr_t>(q) / 4 - r.shift) % 4 == 0;
  const int first = column<T, RUN>(r, c, 0, lane);
  if (wide && inside(r, c)) {
#pragma unroll
    for (int i = 0; i < kPer / N; ++i) {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const float4 v = *reinterpret_cast<const float4*>(q + first + (RUN ? i : i * 32) * N + k);
        x[i * N + k] = v.x, x[i * N + k + 1] = v.y, x[i * N + k + 2] = v.z, x[i * N + k + 3] = v.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer / N; ++i) {
      const int e = first + (RUN ? i : i * 32) * N;
#pragma unroll
      for (int k = 0; k < N; ++k) x[i * N + k] = e + k >= 0 && e + k < r.V ? q[e + k] : 0.f;
    }
  }
}

template <class W>
SPEC_DEV W warp_total(W v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <class W>
SPEC_DEV W warp_scan(W v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const W w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}
template <class W, int N>
SPEC_DEV W tree_sum(const W (&x)[N]) {
  W s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = x[i];
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) s[i] += s[i + o];
  return s[0];
}

SPEC_DEV float redux_max(float x) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
  return m;
}

// A warp takes C chunks.  A NaN or +inf makes
// its chunk's sum NaN.
template <class T, int C>
SPEC_DEV void chunk_stats(const Rows& r, const Row<T>& rr, int row, int c0, int lane) {
  constexpr int N = Vec<T>::N, NV = kPer / N;
  uint4 v[C * NV];
  const int first = c0 * kChunk - rr.shift;
  if (first >= 0 && first + C * kChunk <= rr.V) {
    const uint4* at = reinterpret_cast<const uint4*>(rr.p + first) + lane;
#pragma unroll
    for (int i = 0; i < C * NV; ++i) v[i] = at[i * 32];
  } else {
#pragma unroll
    for (int i = 0; i < C * NV; ++i) v[i] = load_vec(rr, first + (i * 32 + lane) * N);
  }
  const float m = C == 1 || rr.t == 0.f ? redux_max(largest<C * NV>(v, rr.p)) : 0.f;
  if (rr.t == 0.f) {  // only the first largest logit counts: its column stands in the sum's place
    bool nan = false;
    int at_column = 0x7fffffff;
#pragma unroll
    for (int i = C * NV - 1; i >= 0; --i) {
      float y[N];
      unpack(v[i], y, rr.p);
#pragma unroll
      for (int k = N - 1; k >= 0; --k) {
        nan |= y[k] != y[k];
        if (y[k] == m) at_column = first + (i * 32 + lane) * N + k;
      }
    }
    at_column = __reduce_min_sync(0xffffffffu, at_column);
    nan = __any_sync(0xffffffffu, nan);
    if (m == -INFINITY) at_column = 0;  // outside the row as well
    if (lane < C)
      r.stats[(long long)row * r.nch + c0 + lane] =
          lane ? make_float2(-INFINITY, 0.f) : make_float2(m, nan ? NAN : __int_as_float(at_column));
    return;
  }
  float s[C], ms[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    ms[c] = C == 1 ? m : redux_max(largest<NV>(v + c * NV, rr.p));
    const Ref ref(ms[c] == -INFINITY ? 0.f : ms[c], rr.h);
    float x[kPer];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float y[N];
      unpack(v[c * NV + i], y, rr.p);
#pragma unroll
      for (int k = 0; k < N; ++k) x[i * N + k] = y[k];
    }
    if (ref.whole) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = ex2(fmaf(x[i], ref.h, -ref.R));
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = ex2((x[i] - ref.m) * ref.h);
    }
    s[c] = tree_sum(x);
  }
  // The sums over the lanes, C at once: each round halves the sums that a lane holds, until it has one.
  int mine = 0;
#pragma unroll
  for (int n = C, o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      const bool up = lane & o;
      n /= 2;
      mine = mine * 2 + up;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        ms[i] = up ? ms[i + n] : ms[i];
        const float keep = up ? s[i + n] : s[i], give = up ? s[i] : s[i + n];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    } else {
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
    }
  }
  if (lane % (32 / C) == 0) r.stats[(long long)row * r.nch + c0 + mine] = make_float2(ms[0], s[0]);
}

template <class T, int C>
__global__ void __launch_bounds__(256) stats_kernel(const __grid_constant__ Rows r) {
  const int lane = threadIdx.x & 31;
  const unsigned per_row = (unsigned)r.nch / C, at = blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  const int row = (int)(at / per_row), c0 = (int)(at - row * per_row) * C;
  if (row >= r.n_rows) return;
  if (c0 == 0 && lane == 0) {
    if (r.path) r.path[row] = -1;
    if (r.drafts) {  // what the verification asks about the row's draft
      const int x = r.drafts[row];
      const bool judged = x >= 0 && x < r.V;
      r.seen[row] = judged ? make_float2(r.q[row * r.q_stride + x], to_float((static_cast<const T*>(r.logits) + row * r.stride)[x]))
                           : make_float2(0.f, 0.f);
    }
  }
  chunk_stats<T, C>(r, Row<T>(r, row), row, c0, lane);
}

// ---------------------------------------------------------------------------
// Joining a row's chunks (one warp)
// ---------------------------------------------------------------------------
// 8 chunks a lane: of chunks 256 b .. 256 b + 255 those from 8 lane on.
constexpr int kBlock = 256;

// A row's chunk statistics: the first 256 chunks in registers, longer rows'
// others loaded where they are needed.
struct Stats {
  const float2* p;
  int nch, lane;
  float2 first[8];
  SPEC_DEV void load(int b, float2 (&v)[8]) const {
    const int c = b * kBlock + lane * 8;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float4 x = c < nch ? __ldcg(reinterpret_cast<const float4*>(p + c + i)) : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      v[i] = make_float2(x.x, x.y);
      v[i + 1] = make_float2(x.z, x.w);
    }
  }
  SPEC_DEV Stats(const float2* p_, int nch_, int lane_) : p(p_), nch(nch_), lane(lane_) { load(0, first); }
  // f(chunk block, its 8 statistics) -> whether to go on
  template <class F>
  SPEC_DEV void each(F f) const {
    if (!f(0, first)) return;
#pragma unroll 1
    for (int b = 1; b * kBlock < nch; ++b) {
      float2 v[8];
      load(b, v);
      if (!f(b, v)) return;
    }
  }
};
// 2^e for a whole e <= 0.
SPEC_DEV float whole_pow2(float e) { return e < -126.f ? 0.f : __int_as_float((127 + (int)e) << 23); }
// Weight of a chunk's statistics with the row's reference.
SPEC_DEV float chunk_weight(float2 v, const Ref& row) {
  const Ref own(v.x, row.h);
  if (own.whole && row.whole) return v.y * whole_pow2(own.R - row.R);
  return v.y * ex2(row.whole ? fmaf(v.x, row.h, -row.R) : own.whole ? fmaf(-row.m, row.h, own.R) : (v.x - row.m) * row.h);
}

struct Joined {
  Ref ref;
  float Z;  // where the reference is whole
  bool ok;   // the row has a finite largest logit, no NaN and a temperature
};

template <class T>
SPEC_DEV Joined join(const Row<T>& r, const Stats& st) {
  Joined j;
  float m = -INFINITY;
  bool nan = false;
  st.each([&](int, const float2(&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, v[i].x), nan |= v[i].y != v[i].y;
    return true;
  });
  m = redux_max(m);
  j.ref = Ref(m, r.h);
  j.ok = r.ok && m > -INFINITY && m < INFINITY && !__any_sync(0xffffffffu, nan);
  j.Z = 0;
  st.each([&](int, const float2(&v)[8]) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = chunk_weight(v[i], j.ref);
    j.Z += warp_total(tree_sum(w));
    return true;
  });
  return j;
}

// Of N values a lane, one lane's after another: the first whose cumulative
// sum passes `target`, and the sums before and with it (from `base` on).  Where
// rounding leaves the lane's own sum a step below the scanned one, its last of
// some weight.  -1: none; then *with is the sum of all.
template <class W, int N>
SPEC_DEV int find(const W (&w)[N], double base, double target, int lane, double* before, double* with) {
  const W own = tree_sum(w), incl = warp_scan(own, lane);
  W excl = __shfl_up_sync(0xffffffffu, incl, 1);
  if (lane == 0) excl = 0;
  // Of a weight: the lanes' sums are added in different orders, so that one of
  // no weight may stand a step above the lane before it.
  const unsigned hit = __ballot_sync(0xffffffffu, own > 0 && base + (double)incl > target);
  if (!hit) {
    *with = base + (double)__shfl_sync(0xffffffffu, incl, 31);
    return -1;
  }
  const int who = __ffs(hit) - 1;
  // In the lane: sums from its own start, against what is left of the target.
  const W left = (W)(target - (base + (double)excl));
  int at = 0;
  W from = 0, run = 0;
  bool open = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const W next = run + w[i];
    const bool take = open && w[i] > 0;
    at = take ? i : at;
    from = take ? run : from;
    run = open ? next : run;
    open = open && !(next > left);
  }
  *before = base + (double)excl + (double)from;
  *with = base + (double)excl + (double)run;
  *before = __shfl_sync(0xffffffffu, *before, who);
  *with = __shfl_sync(0xffffffffu, *with, who);
  return who * N + __shfl_sync(0xffffffffu, at, who);
}
// The last of some weight, or -1.
template <class W, int N>
SPEC_DEV int find_last(const W (&w)[N], int lane) {
  int at = -1;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (w[i] > 0) at = lane * N + i;
  return __reduce_max_sync(0xffffffffu, at);
}

// The first column with the row's largest logit, at temperature 0.
SPEC_DEV int first_largest(const Stats& st, float M) {
  int e = 0x7fffffff;
  st.each([&](int, const float2(&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v[i].x == M) e = min(e, __float_as_int(v[i].y));
    return true;
  });
  return __reduce_min_sync(0xffffffffu, e);
}

// What weights of sum S are off by in all, in units of 2^-24, of a row of V columns.
SPEC_DEV float spread(float S, int V) {
  const float nats = 0.6932f * (__log2f((float)V) - __log2f(S)) + 0.01f;  // the logarithm is off by less than 0.001
  return (4.5f + 2.5f * fmaxf(nats, 1.f)) * S;
}

SPEC_DEV double unit(float u) { return (double)fminf(fmaxf(u, 0.f), 1.f); }  // NaN: 0

// A token of p, or kBad, or kUnsure where f32 does not decide.
template <class T>
SPEC_DEV int draw(const Row<T>& r, const Stats& st, const Joined& j, float u) {
  if (!j.ok) return kBad;
  if (r.t == 0.f) return first_largest(st, j.ref.m);
  const double v = unit(u), target = v * (double)j.Z;
  if (!j.ref.whole || target <= 0x1p-33) return kUnsure;
  double run = 0, lo, hi;
  int c = -1;
  st.each([&](int b, const float2(&v)[8]) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = chunk_weight(v[i], j.ref);
    c = find(w, run, target, st.lane, &lo, &hi);
    if (c < 0) {
      run = hi;
      return true;
    }
    c += b * kBlock;
    run = lo;
    return false;
  });
  if (c < 0) return kUnsure;
  float x[kPer];
  load_chunk<T, true>(r, c, st.lane, x);
  const float t = (float)target, all = spread(j.Z, r.V), apart = spread(t, r.V) + (float)v * all;
  const float shared = (float)fmax(v, 1 - v) * all + 2 * spread(fmaxf((float)(hi - run), 0x1p-60f), r.V);
  const double slack = 1.01 * 0x1p-24 * (double)(45.f * t + fminf(apart, shared));
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = ex2(fmaf(x[i], j.ref.h, -j.ref.R));
  const int e = find(x, run, target, st.lane, &lo, &hi);
  return e >= 0 && lo + slack <= target && target + slack < hi ? c * kChunk - r.shift + e : kUnsure;
}

// ---------------------------------------------------------------------------
// Sums by a cluster
// ---------------------------------------------------------------------------
// What the columns of a row are weighed by: p in 64 bits (P64), max(p - q, 0)
// in f32 (REST32) or in 64 bits (REST64).
enum : int { P64 = 0, REST32 = 1, REST64 = 2 };

// 2^y for y <= 0 in 64 bits: y = n + i / 256 + f, |f| <= 1 / 512, 2^(i / 256) from
// a table and the Taylor series of 2^f to (f ln 2)^4 / 4! (the next term is below
// 2^-54).  Below 2^-1000: zero.
struct Powers {
  double of[256];
  SPEC_DEV void fill() { of[threadIdx.x] = exp2((double)(int)threadIdx.x / 256); }  // by kThreads threads; the block syncs before its use
  // y in 256ths, above -2^31
  SPEC_DEV double pow(double y) const {
    constexpr double c = 0.693147180559945309 / 256, kWhole = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double t = y + kWhole, f = y - (t - kWhole);
    double s = fma(f, c * c * c * c / 24, c * c * c / 6);
    s = fma(s, f, c * c / 2);
    s = fma(s, f, c);
    s = s * f;
    const int n = __double2loint(t);
    const double b = of[n & 255], w = fma(s, b, b);
    const int e = n >> 8;
    return e < -1000 ? 0.0 : __hiloint2double(__double2hiint(w) + (e << 20), __double2loint(w));
  }
};

template <class T>
struct Weigher {
  const Row<T>& r;
  const Ref& ref;
  const float* q;
  float inv_zf;
  float low;  // logits below it weigh nothing; (x - m) h of the others, low's rounding included, is above -2^31
  double h, inv_z;
  const Powers* powers;
  SPEC_DEV Weigher(const Row<T>& r_, const Ref& ref_, const float* q_, int kind, double Z, const Powers* powers_ = nullptr)
      : r(r_), ref(ref_), q(q_), powers(powers_) {
    if (kind == REST32) {
      inv_zf = 1.f / (float)Z;
    } else {
      h = 256 * 1.44269504088896341 / (double)r.t;
      low = ref.m - 1e5f * r.t;
      inv_z = 1.0 / Z;
    }
  }
  SPEC_DEV double p64(float x) const {
    const double w = powers->pow(((double)fmaxf(x, low) - (double)ref.m) * h);
    return x >= low ? w : 0.0;
  }
  SPEC_DEV void rest32(float (&x)[kPer], const float (&y)[kPer]) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = fmaxf(fmaf(ex2(fmaf(x[i], ref.h, -ref.R)), inv_zf, -y[i]), 0.f);
  }
  template <int N>
  SPEC_DEV void exact(int kind, const float (&x)[N], const float (&y)[N], double (&w)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = p64(x[i]);
    if (kind == REST64) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = fmax(w[i] * inv_z - (double)y[i], 0.0);
    }
  }
  // Chunk sums by all warps of the cluster, a chunk's loads ahead; the caller syncs it.
  SPEC_DEV void sum(int kind, double* sums, int nch, int lane) const {
    constexpr int NV = kPer / Vec<T>::N;
    const int nw = blockDim.x >> 5, step = nw * cluster_size();
    int c = cluster_rank() * nw + (threadIdx.x >> 5);
    uint4 v[NV];
    if (c < nch) load_raw<T, false>(r, c, lane, v);
#pragma unroll 1
    for (; c < nch; c += step) {
      float x[kPer], y[kPer];
      unpack_chunk(v, x, r.p);
      if (kind == REST64) load_probs<T, false>(r, q, c, lane, y);
      if (c + step < nch) load_raw<T, false>(r, c + step, lane, v);
      double s = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const double w = p64(x[i]);
        s += kind == REST64 ? fmax(w * inv_z - (double)y[i], 0.0) : w;
      }
      s = warp_total(s);
      if (lane == 0) __stcg(sums + c, s);
    }
  }
  // The same of REST32, two chunks' loads at a time.
  SPEC_DEV void sum32(float* sums, int nch, int lane) const {
    constexpr int NV = kPer / Vec<T>::N;
    const int nw = blockDim.x >> 5, step = nw * cluster_size();
#pragma unroll 1
    for (int c = cluster_rank() * nw + (threadIdx.x >> 5); c < nch; c += 2 * step) {
      const int d = c + step < nch ? c + step : c;
      uint4 v[NV], w[NV];
      float y[kPer], z[kPer], x[kPer];
      load_raw<T, false>(r, c, lane, v);
      load_probs<T, false>(r, q, c, lane, y);
      load_raw<T, false>(r, d, lane, w);
      load_probs<T, false>(r, q, d, lane, z);
      unpack_chunk(v, x, r.p);
      rest32(x, y);
      const float s = warp_total(tree_sum(x));
      unpack_chunk(w, x, r.p);
      rest32(x, z);
      const float t = warp_total(tree_sum(x));
      if (lane == 0) {
        __stcg(sums + c, s);
        if (d != c) __stcg(sums + d, t);
      }
    }
  }
};

// A row's chunk sums, 8 a lane.
SPEC_DEV void load_sums(const double* p, int b, int nch, int lane, double (&w)[8]) {
  const int c = b * kBlock + lane * 8;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const double2 x = c < nch ? __ldcg(reinterpret_cast<const double2*>(p + c + i)) : make_double2(0, 0);
    w[i] = x.x, w[i + 1] = x.y;
  }
}
SPEC_DEV double total(const double* sums, int nch, int lane) {
  double s = 0;
  for (int b = 0; b * kBlock < nch; ++b) {
    double w[8];
    load_sums(sums, b, nch, lane, w);
    s += warp_total(tree_sum(w));
  }
  return s;
}

// A token of the weights in `sums`, whose sum is Zs, in 64 bits.  One warp runs
// this once, and code that runs once is fetched from L2: a vector of columns a turn
// (8.7 us with the chunk's 16 columns of a lane at once, 7 so).
template <class T>
SPEC_DEV int draw_sums(const Weigher<T>& f, int kind, const double* sums, int nch, double Zs, float u, int lane) {
  constexpr int N = Vec<T>::N;
  const double target = unit(u) * Zs;
  double run = 0, lo, hi;
  int c = -1, last = -1;
#pragma unroll 1
  for (int b = 0; b * kBlock < nch && c < 0; ++b) {
    double w[8];
    load_sums(sums, b, nch, lane, w);
    c = find(w, run, target, lane, &lo, &hi);
    run = c < 0 ? hi : lo;
    if (c >= 0) c += b * kBlock;
    const int some = find_last(w, lane);
    if (some >= 0) last = b * kBlock + some;
  }
  const bool whole = c < 0;  // the target is the sum of all: the last column of some weight
  if (whole) c = last;
  if (c < 0) return kBad;
  int token = -1, tail = kBad;
#pragma unroll 1
  for (int i = 0; i < kPer / N && token < 0; ++i) {
    const int first = c * kChunk - f.r.shift + i * 32 * N, e = first + lane * N;
    float x[N], y[N];
    unpack(load_vec(f.r, e), x, f.r.p);
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] = kind == REST64 && e + k >= 0 && e + k < f.r.V ? f.q[e + k] : 0.f;
    double w[N];
    f.exact(kind, x, y, w);
    const int some = find_last(w, lane);
    if (some >= 0) tail = first + some;
    const int at = whole ? -1 : find(w, run, target, lane, &lo, &hi);
    if (at >= 0) token = first + at;
    run = hi;
  }
  return token < 0 ? tail : token;
}

// A token of max(p - q, 0) from REST32 sums, or kUnsure.
template <class T>
SPEC_DEV int draw_rest(const Weigher<T>& f, const float* sums, int nch, float u, int lane) {
  float w[8];
  auto load = [&](int b) {
    const int c = b * kBlock + lane * 8;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 x = c < nch ? __ldcg(reinterpret_cast<const float4*>(sums + c + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
      w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
    }
  };
  load(0);
  double Zs = (double)warp_total(tree_sum(w));
  for (int b = 1; b * kBlock < nch; ++b) {
    load(b);
    Zs += (double)warp_total(tree_sum(w));
  }
  const double target = unit(u) * Zs;
  double run = 0, lo, hi;
  int c = -1;
  for (int b = 0; b * kBlock < nch && c < 0; ++b) {
    if (nch > kBlock) load(b);
    c = find(w, run, target, lane, &lo, &hi);
    run = c < 0 ? hi : lo;
    if (c >= 0) c += b * kBlock;
  }
  if (c < 0) return kUnsure;
  float x[kPer], y[kPer];
  load_chunk<T, true>(f.r, c, lane, x);
  load_probs<T, true>(f.r, f.q, c, lane, y);
  f.rest32(x, y);
  const int e = find(x, run, target, lane, &lo, &hi);
  // max(p - q, 0) is off by no more than p: by the weights' errors and Z's (24 u for its sum and 1
  // for 1 / Z besides), each at most once, as a prefix and u times the whole share the columns.
  // The sums' own are 21 u each, and 2 for the multiply-add.
  const float Z = 1.f / f.inv_zf;
  const double slack = 1.01 * 0x1p-24 * (2.0 * (double)(spread(Z, f.r.V) / Z) + 25 + 44 * Zs);
  return e >= 0 && lo + slack <= target && target + slack < hi ? c * kChunk - f.r.shift + e : kUnsure;
}

// ---------------------------------------------------------------------------
// A cluster a row
// ---------------------------------------------------------------------------

// Probabilities of this warp's chunks (all warps but the first, which draws), two chunks' loads at a time.
template <class T>
SPEC_DEV void write_probs(const SampleParams& p, const Row<T>& r, const Joined& j, int top, int row, int warp, int lane) {
  constexpr int N = Vec<T>::N, NV = kPer / N;
  const int nch = p.r.nch, step = (kWarps - 1) * cluster_size();
  float* out = p.probs + row * p.probs_stride;
  const float inv = 1.f / j.Z;
  const bool wide = (reinterpret_cast<uintptr_t>(out) / 4 - r.shift) % 4 == 0;
  auto write = [&](int c, const uint4* v) {
    float x[kPer];
    unpack_chunk(v, x, r.p);
    const int first = column<T, false>(r, c, 0, lane);
    if (!j.ok || r.t == 0.f) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = j.ok && first + i / N * 32 * N + i % N == top ? 1.f : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = j.ref.weight(x[i]) * inv;
    }
    const bool all = wide && inside(r, c);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = first + i * 32 * N;
      if (all) {
        if constexpr (N == 8) {
          // Two lanes exchange halves, so that a store is 512 bytes behind one another.
          const bool odd = lane & 1;
          float4 a, b;
          float* p0 = &a.x;
          float* p1 = &b.x;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float lo = x[i * N + k], hi = x[i * N + 4 + k], got = __shfl_xor_sync(0xffffffffu, odd ? lo : hi, 1);
            p0[k] = odd ? got : lo;
            p1[k] = odd ? hi : got;
          }
          float* to = out + e - (odd ? 4 : 0);
          *reinterpret_cast<float4*>(to) = a;
          *reinterpret_cast<float4*>(to + 8) = b;
        } else {
          *reinterpret_cast<float4*>(out + e) = make_float4(x[i * N], x[i * N + 1], x[i * N + 2], x[i * N + 3]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (e + k >= 0 && e + k < r.V) out[e + k] = x[i * N + k];
      }
    }
  };
#pragma unroll 1
  for (int c = cluster_rank() * (kWarps - 1) + warp - 1; c < nch; c += 2 * step) {
    const int d = c + step < nch ? c + step : c;
    uint4 v[NV], w[NV];
    load_raw<T, false>(r, c, lane, v);
    load_raw<T, false>(r, d, lane, w);
    write(c, v);
    if (d != c) write(d, w);
  }
}

// ALONE: without the kernel before it, each cluster sums its own row.
template <class T, bool PROBS, bool ALONE>
__global__ void __launch_bounds__(kThreads, ALONE ? 2 : 4) sample_kernel(const __grid_constant__ SampleParams p) {
  __shared__ int s_tok;
  __shared__ Powers s_powers;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), row = blockIdx.x / cluster_size();
  pdl_launch_dependents();
  s_powers.fill();
  pdl_wait();
  const Row<T> r(p.r, row);
  const int nch = p.r.nch;
  const float u = p.r.u[row];
  double* sums = p.r.sums + (long long)row * nch;
  if constexpr (ALONE) {
#pragma unroll 1
    for (int c = (rank * kWarps + warp) * 4; c < nch; c += cluster_size() * kWarps * 4) chunk_stats<T, 4>(p.r, r, row, c, lane);
    cluster_sync();
  }
  Joined j;
  if (PROBS || warp == 0) {
    const Stats st(p.r.stats + (long long)row * nch, nch, lane);
    j = join(r, st);
    if (PROBS && warp) write_probs(p, r, j, r.t == 0.f && j.ok ? first_largest(st, j.ref.m) : -1, row, warp, lane);
    if (warp == 0) {
      const int tok = draw(r, st, j, u);
      if (lane == 0) s_tok = tok;
    }
  }
  __syncthreads();
  int tok = s_tok;
  if (tok == kUnsure) {
    if (!PROBS && warp) j = join(r, Stats(p.r.stats + (long long)row * nch, nch, lane));
    const Weigher<T> f(r, j.ref, nullptr, P64, 1, &s_powers);
    f.sum(P64, sums, nch, lane);
    cluster_sync();
    if (rank || warp) return;
    tok = draw_sums(f, P64, sums, nch, total(sums, nch, lane), u, lane);
  }
  if (rank == 0 && threadIdx.x == 0) p.tokens[row] = tok;
}

// ---------------------------------------------------------------------------
// A cluster a sequence: chains
// ---------------------------------------------------------------------------
enum : int { A_REJECT = 0, A_ACCEPT = 1, A_UNSURE = 2, A_BAD = 3, A_END = 4 };

// Rows first .. last of sequence b, empty where row_start says nothing sound.
SPEC_DEV int rows_of(const VerifyParams& p, int b, int* first) {
  const int r0 = p.row_start[b], r1 = p.row_start[b + 1];
  *first = r0;
  return r0 >= 0 && r1 >= r0 && r1 <= p.r.n_rows ? r1 - r0 : 0;
}

// What the walk knows of a row.
struct Judged {
  Joined join;
  int verdict, x;    // its draft
  float qx, lx;      // the draft's probability and the row's logit of it
  float u, t, h;
};

template <class T>
__global__ void __launch_bounds__(kThreads, 3) chain_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ Judged s_row[kWarps];
  __shared__ int s_tok;
  __shared__ Powers s_powers;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), b = blockIdx.x / cluster_size(), nch = p.r.nch;
  pdl_launch_dependents();
  s_powers.fill();
  pdl_wait();
  int r0;
  const int n = rows_of(p, b, &r0);
  double* sums = p.r.sums + (long long)(n ? r0 : 0) * nch;
  bool used = false;  // other blocks may still read `sums`
  int at = 0, verdict = n ? A_ACCEPT : A_BAD;  // the row under decision; why the walk stopped
  Judged row;
  double z64 = 0;  // of row `at`, once summed in 64 bits
  // The walk, a row a warp.  Every block of the cluster comes to the same verdicts.
#pragma unroll 1
  for (int base = 0; base < n && verdict == A_ACCEPT; base += kWarps) {
    if (base + warp < n) {
      const int i = base + warp, at_row = r0 + i;
      const Stats st(p.r.stats + (long long)at_row * nch, nch, lane);
      const float2 seen = __ldcg(p.r.seen + at_row);
      const Row<T> r(p.r, at_row);
      Judged w;
      w.x = i + 1 < n ? p.tokens[at_row] : -1;
      w.u = p.r.u[at_row];
      w.t = r.t, w.h = r.h;
      w.qx = seen.x, w.lx = seen.y;
      w.join = join(r, st);
      int v = A_END;
      if (!w.join.ok) {
        v = A_BAD;
      } else if (w.x >= 0 && w.x < p.r.V) {
        const double left = unit(w.u) * (double)w.qx;
        if (w.qx <= 0.f) {
          v = A_ACCEPT;
        } else if (r.t == 0.f) {
          v = left <= (w.x == first_largest(st, w.join.ref.m) ? 1.0 : 0.0);
        } else {
          const double px = (double)w.join.ref.weight(w.lx), lz = left * (double)w.join.Z;
          // w_x alone: off by (4.5 + 2.5 * 23) u where it is above 2^-33.
          const double slack = 3 * kErr * lz + 0x1p-33;
          v = !w.join.ref.whole ? A_UNSURE : lz + slack < px ? A_ACCEPT : lz > px + slack ? A_REJECT : A_UNSURE;
          if (w.qx != w.qx) v = A_REJECT;
        }
      }
      w.verdict = v;
      if (lane == 0) s_row[warp] = w;
    }
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < kWarps && base + w < n; ++w) {
      at = base + w;
      verdict = s_row[w].verdict;
      if (verdict == A_ACCEPT) continue;
      row = s_row[w];
      if (verdict == A_UNSURE) {
        const Row<T> r(p.r, r0 + at);
        const Weigher<T> f(r, row.join.ref, nullptr, P64, 1, &s_powers);
        if (used) cluster_sync();
        f.sum(P64, sums, nch, lane);
        cluster_sync();
        used = true;
        z64 = total(sums, nch, lane);
        verdict = unit(row.u) * (double)row.qx * z64 <= f.p64(row.lx) ? A_ACCEPT : A_REJECT;
        if (verdict == A_ACCEPT) z64 = 0;
      }
      if (verdict != A_ACCEPT) break;
    }
    __syncthreads();
  }
  int tok = kBad;
  if (verdict != A_BAD) {
    const bool rest = verdict == A_REJECT;
    const float* q = rest ? p.q + (r0 + at) * p.q_stride : nullptr;
    const float u = rest ? p.r.u[r0 + at + 1] : row.u;  // a row follows every draft
    Row<T> r;
    r.place(p.r, r0 + at);
    r.t = row.t, r.h = row.h, r.ok = true;
    const Ref ref = row.join.ref;
    tok = kUnsure;
    if (r.t == 0.f || !rest) {
      // Temperature 0, all of p on one token: what q leaves of it is that token.
      if (warp == 0) {
        const Stats st(p.r.stats + (long long)(r0 + at) * nch, nch, lane);
        tok = draw(r, st, row.join, u);
      }
    } else if (ref.whole && z64 == 0) {
      const Weigher<T> f(r, ref, q, REST32, (double)row.join.Z);
      float* sums32 = reinterpret_cast<float*>(sums);
      if (used) cluster_sync();
      f.sum32(sums32, nch, lane);
      cluster_sync();
      used = true;
      if (warp == 0) tok = draw_rest(f, sums32, nch, u, lane);
    }
    if (threadIdx.x == 0) s_tok = tok;
    __syncthreads();
    tok = s_tok;
    if (tok == kUnsure) {
      // The sums of p, then those of max(p - q, 0); where that is 0 everywhere, p's again.
      Weigher<T> f(r, ref, q, P64, 1, &s_powers);
      int kind = P64;
      double zs = z64;
#pragma unroll 1
      for (int turn = z64 == 0 ? 0 : 1; turn < 3; ++turn) {
        if (turn && (!rest || (turn == 2 && zs > 0))) break;
        if (turn == 1) f.inv_z = 1.0 / zs;
        kind = turn == 1 ? REST64 : P64;
        if (used) cluster_sync();
        f.sum(kind, sums, nch, lane);
        cluster_sync();
        used = true;
        zs = total(sums, nch, lane);
      }
      if (rank == 0 && warp == 0) tok = draw_sums(f, kind, sums, nch, zs, u, lane);
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.n_out[b] = at;
    p.next[b] = tok;
  }
}

// ---------------------------------------------------------------------------
// A cluster a sequence: trees
// ---------------------------------------------------------------------------
constexpr int kTreeNodes = 512;  // that the walk finds in shared memory

template <class T>
__global__ void __launch_bounds__(kThreads, 3) tree_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ int s_tok, s_drawn[kTreeNodes];
  __shared__ int2 s_node[kTreeNodes];  // parent, token
  __shared__ Powers s_powers;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), size = cluster_size(), b = blockIdx.x / size, nch = p.r.nch;
  pdl_launch_dependents();
  s_powers.fill();
  pdl_wait();
  int r0;
  const int n = rows_of(p, b, &r0), near = min(n, kTreeNodes);
  for (int i = threadIdx.x; i < near; i += kThreads) s_node[i] = make_int2(p.parents[r0 + i], p.tokens[r0 + i]);
#pragma unroll 1
  for (int i = rank * kWarps + warp; i < n; i += size * kWarps) {
    const Row<T> r(p.r, r0 + i);
    const float u = p.r.u[r0 + i];
    const Stats st(p.r.stats + (long long)(r0 + i) * nch, nch, lane);
    const int tok = draw(r, st, join(r, st), u);
    if (lane == 0) __stcg(p.r.drawn + r0 + i, tok);
  }
  cluster_sync();
  for (int i = threadIdx.x; i < near; i += kThreads) s_drawn[i] = __ldcg(p.r.drawn + r0 + i);
  __syncthreads();
  double* sums = p.r.sums + (long long)(n ? r0 : 0) * nch;
  int cur = 0, len = 0, tok = kBad;
#pragma unroll 1
  while (len < n) {
    if (rank == 0 && threadIdx.x == 0) p.r.path[r0 + len] = cur;
    ++len;
    tok = cur < kTreeNodes ? s_drawn[cur] : __ldcg(p.r.drawn + r0 + cur);
    if (tok == kUnsure) {
      const Row<T> r(p.r, r0 + cur);
      const Joined j = join(r, Stats(p.r.stats + (long long)(r0 + cur) * nch, nch, lane));
      const Weigher<T> f(r, j.ref, nullptr, P64, 1, &s_powers);
      cluster_sync();
      f.sum(P64, sums, nch, lane);
      cluster_sync();
      if (warp == 0) {
        tok = draw_sums(f, P64, sums, nch, total(sums, nch, lane), p.r.u[r0 + cur], lane);
        if (lane == 0) s_tok = tok;
      }
      __syncthreads();
      tok = s_tok;
      __syncthreads();
    }
    // The first child that holds the token; every warp looks for itself.
    int child = -1;
#pragma unroll 1
    for (int i = cur + 1; i < n && tok >= 0; i += 32) {
      int2 node = make_int2(-1, -1);
      if (i + lane < near) node = s_node[i + lane];
      else if (i + lane < n) node = make_int2(p.parents[r0 + i + lane], p.tokens[r0 + i + lane]);
      const bool hit = node.x == cur && node.y == tok;
      const unsigned mask = __ballot_sync(0xffffffffu, hit);
      if (mask) {
        child = i + __ffs(mask) - 1;
        break;
      }
    }
    if (child < 0) break;
    cur = child;
  }
  if (rank == 0 && threadIdx.x == 0) {
    p.n_out[b] = len;
    p.next[b] = tok;
  }
}

// ---------------------------------------------------------------------------
template <class K, class P>
cudaError_t launch_clusters(K* kernel, int n, int size, int threads, cudaStream_t s, const P& p) {
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = size;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n * size);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Blocks a cluster: 8, fewer where all clusters' blocks are more than one and a half times those that are resident at once.
int cluster_for(int n, int per_sm, int sms) {
  int size = 8;
  while (size > 1 && (long long)n * size * 2 > (long long)sms * per_sm * 3) size /= 2;
  return size;
}

// A chunk a warp where that is less than the warps that the device holds, else 8 KB.
template <class T>
cudaError_t stats(const Rows& r, int sms, cudaStream_t s) {
  const long long chunks = (long long)r.n_rows * r.nch;
  if (chunks <= sms * 64LL) return kv4::launch_overlapping(stats_kernel<T, 1>, dim3((unsigned)(chunks / 8)), 256, 0, s, r);
  constexpr int C = sizeof(T) == 4 ? 4 : 8;
  return kv4::launch_overlapping(stats_kernel<T, C>, dim3((unsigned)((chunks / C + 7) / 8)), 256, 0, s, r);
}
template <class T, bool PROBS>
cudaError_t sample(const SampleParams& p, int sms, cudaStream_t s) {
  // One launch where all clusters are resident with a multiprocessor a block
  // (one row of 128256: 4.9 us in two kernels, which cost the host 3 us more).
  if ((long long)p.r.n_rows * 8 <= sms) return launch_clusters(sample_kernel<T, PROBS, true>, p.r.n_rows, 8, kThreads, s, p);
  const cudaError_t e = stats<T>(p.r, sms, s);
  if (e != cudaSuccess) return e;
  return launch_clusters(sample_kernel<T, PROBS, false>, p.r.n_rows, cluster_for(p.r.n_rows, 4, sms), kThreads, s, p);
}
template <class T>
cudaError_t sample(const SampleParams& p, int sms, cudaStream_t s) {
  return p.probs ? sample<T, true>(p, sms, s) : sample<T, false>(p, sms, s);
}
template <class T>
cudaError_t verify(const VerifyParams& p, bool trees, int sms, cudaStream_t s) {
  const cudaError_t e = p.r.n_rows ? stats<T>(p.r, sms, s) : cudaSuccess;
  if (e != cudaSuccess) return e;
  const int size = cluster_for(p.n_seqs, 3, sms);
  return trees ? launch_clusters(tree_kernel<T>, p.n_seqs, size, kThreads, s, p)
               : launch_clusters(chain_kernel<T>, p.n_seqs, size, kThreads, s, p);
}

}  // namespace

cudaError_t launch_sample(const SampleParams& p, int dtype, int sms, cudaStream_t s) {
  if (dtype == T_BF16) return sample<__nv_bfloat16>(p, sms, s);
  if (dtype == T_F16) return sample<__half>(p, sms, s);
  return sample<float>(p, sms, s);
}
cudaError_t launch_verify(const VerifyParams& p, int dtype, bool trees, int sms, cudaStream_t s) {
  if (dtype == T_BF16) return verify<__nv_bfloat16>(p, trees, sms, s);
  if (dtype == T_F16) return verify<__half>(p, trees, sms, s);
  return verify<float>(p, trees, sms, s);
}

}  // namespace batch
}  // namespace specb200

