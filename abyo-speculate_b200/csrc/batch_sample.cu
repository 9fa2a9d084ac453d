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
// (2.5 d + 0.5) u, the hardware's 2^x by 4 u more, a chunk's sum of positive
// terms by 9 u (16 a lane in pairs, 5 rounds of shuffles).  The mean of d under
// the weights of any set of columns is their entropy less the logarithm of their
// sum S, at most ln V - ln S; for S >= 1 and V <= 2^20 that makes
// (13.5 + 2.5 * 13.9) u < 2^-18 of S (kErr), for S > 2^-33 less than twice that.
// Smaller sums, and rows with |M| h of 2^22 and more, are left to 64 bits.
//
// Two kernels.  stats_kernel reads every row once, a warp one chunk of 512
// columns or four, and leaves each chunk's reference and sum.  The second
// kernel runs a cluster a row (sample) or a sequence (chains, trees); a warp
// joins a row's chunks by a scan over their sums, finds the chunk of the token
// and reads that alone.  A rejected draft's max(p - q, 0) is summed by all warps
// of the cluster, from p and q once more.
#include "batch.h"
#include "common.cuh"
#include "kv4_rows.cuh"

namespace specb200 {
namespace batch {
namespace {

constexpr float kErr = 1.f / (1 << 18);  // of a sum of weights, relative
constexpr int kBad = -1, kUnsure = -2;
constexpr int kPer = kChunk / 32;  // columns of a lane

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

  SPEC_DEV Row(const Rows& r, int row) {
    p = static_cast<const T*>(r.logits) + row * r.stride;
    V = r.V;
    shift = (int)(reinterpret_cast<uintptr_t>(p) / sizeof(T) % Vec<T>::N);
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
SPEC_DEV float largest(const uint4 (&v)[NV], const float*) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y)),
                       fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w))));
  return m;
}
template <int NV, class H, class H2>
SPEC_DEV float largest_of_pairs(const uint4 (&v)[NV]) {
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
SPEC_DEV float largest(const uint4 (&v)[NV], const __nv_bfloat16*) {
  return largest_of_pairs<NV, __nv_bfloat16, __nv_bfloat162>(v);
}
template <int NV>
SPEC_DEV float largest(const uint4 (&v)[NV], const __half*) {
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
template <class T, bool RUN>
SPEC_DEV void load_chunk(const Row<T>& r, int c, int lane, float (&x)[kPer]) {
  constexpr int N = Vec<T>::N;
  uint4 v[kPer / N];
#pragma unroll
  for (int i = 0; i < kPer / N; ++i) v[i] = load_vec(r, column<T, RUN>(r, c, i, lane));
#pragma unroll
  for (int i = 0; i < kPer / N; ++i) {
    float y[N];
    unpack(v[i], y, r.p);
#pragma unroll
    for (int k = 0; k < N; ++k) x[i * N + k] = y[k];
  }
}

// The same columns of a row of f32 probabilities; zeros outside.
template <class T, bool RUN>
SPEC_DEV void load_probs(const Row<T>& r, const float* q, int c, int lane, float (&x)[kPer]) {
  constexpr int N = Vec<T>::N;
  const bool wide = (reinterpret_cast<uintptr_t>(q) / 4 - r.shift) % 4 == 0;
#pragma unroll
  for (int i = 0; i < kPer / N; ++i) {
    const int e = column<T, RUN>(r, c, i, lane);
    if (wide && e >= 0 && e + N <= r.V) {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const float4 v = *reinterpret_cast<const float4*>(q + e + k);
        x[i * N + k] = v.x, x[i * N + k + 1] = v.y, x[i * N + k + 2] = v.z, x[i * N + k + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[i * N + k] = e + k >= 0 && e + k < r.V ? q[e + k] : 0.f;
    }
  }
}

SPEC_DEV float pair_sum(const float (&x)[kPer]) {
  float s[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) s[i] = x[i];
#pragma unroll
  for (int o = kPer / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) s[i] += s[i + o];
  return s[0];
}

SPEC_DEV float redux_max(float x) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
  return m;
}

// A warp takes C chunks, whose sums share one reference.  A NaN or +inf makes
// its chunk's sum NaN.
template <class T, int C>
__global__ void __launch_bounds__(256) stats_kernel(const __grid_constant__ Rows r) {
  constexpr int N = Vec<T>::N, NV = kPer / N;
  const int lane = threadIdx.x & 31;
  const unsigned per_row = (unsigned)r.nch / C, at = blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  const int row = (int)(at / per_row), c0 = (int)(at - row * per_row) * C;
  if (row >= r.n_rows) return;
  if (r.path && c0 == 0 && lane == 0) r.path[row] = -1;
  const Row<T> rr(r, row);
  uint4 v[C * NV];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < NV; ++i) v[c * NV + i] = load_vec(rr, column<T, false>(rr, c0 + c, i, lane));
  const float m = redux_max(largest(v, rr.p));
  const Ref ref(m == -INFINITY ? 0.f : m, rr.h);
  float s[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
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
    s[c] = pair_sum(x);
  }
  float2* out = r.stats + (long long)row * r.nch + c0;
  if constexpr (C == 4) {
    // Four sums over the lanes at once: lanes 8 c .. end with chunk c's.
    const bool up = lane & 16, odd = lane & 8;
    float a = up ? s[2] : s[0], b = up ? s[3] : s[1];
    a += __shfl_xor_sync(0xffffffffu, up ? s[0] : s[2], 16);
    b += __shfl_xor_sync(0xffffffffu, up ? s[1] : s[3], 16);
    float t = odd ? b : a;
    t += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
    t += __shfl_xor_sync(0xffffffffu, t, 4);
    t += __shfl_xor_sync(0xffffffffu, t, 2);
    t += __shfl_xor_sync(0xffffffffu, t, 1);
    if (lane % 8 == 0) out[lane / 8] = make_float2(m, t);
  } else {
    const float t = specb200::warp_sum(s[0]);
    if (lane == 0) out[0] = make_float2(m, t);
  }
}

// ---------------------------------------------------------------------------
// Joining a row's chunks (one warp)
// ---------------------------------------------------------------------------
SPEC_DEV double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
SPEC_DEV double warp_scan(double v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

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
SPEC_DEV double chunk_weight(float2 v, const Ref& row) {
  const Ref own(v.x, row.h);
  if (own.whole && row.whole) return (double)(v.y * whole_pow2(own.R - row.R));
  return (double)(v.y * ex2(row.whole ? fmaf(v.x, row.h, -row.R) : own.whole ? fmaf(-row.m, row.h, own.R) : (v.x - row.m) * row.h));
}

struct Joined {
  Ref ref;
  double Z;  // where the reference is whole
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
  double z = 0;
  st.each([&](int, const float2(&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z += chunk_weight(v[i], j.ref);
    return true;
  });
  j.Z = warp_sum(z);
  return j;
}

// Of 8 values a lane in 256 chunks: the first chunk whose cumulative weight
// passes `target` (run: the weight before them, moved past them where none does).
SPEC_DEV int find_in_block(const double (&w)[8], int b, double target, int lane, double* run) {
  double own = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) own += w[i];
  const double incl = warp_scan(own, lane) + *run;
  double at = __shfl_up_sync(0xffffffffu, incl, 1);  // not above the target where incl passes it
  if (lane == 0) at = *run;
  const unsigned hit = __ballot_sync(0xffffffffu, incl > target);
  if (!hit) {
    *run = __shfl_sync(0xffffffffu, incl, 31);
    return -1;
  }
  const int who = __ffs(hit) - 1;
  // Rounding may leave the sum of all a step below the scanned one: then the last chunk of some weight.
  int found = -1;
  double before = at;
  bool open = true;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (open && w[i] > 0) {
      found = b * kBlock + lane * 8 + i;
      before = at;
      at += w[i];
      open = at <= target;
    }
  *run = __shfl_sync(0xffffffffu, before, who);
  return __shfl_sync(0xffffffffu, found, who);
}

// The first of a chunk's columns whose cumulative weight passes `target`;
// w[i]: weights of this lane's 16 columns, one after another.  Where none
// does, the last column of some weight.  [lo, hi): cumulative weights around it.
template <class T, class W>
SPEC_DEV int find_column(const Row<T>& r, int c, const W (&w)[kPer], double before, double target, int lane, double* lo,
                         double* hi) {
  const int e = column<T, true>(r, c, 0, lane);
  double own = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) own += (double)w[i];
  const double incl = warp_scan(own, lane) + before;
  double at = __shfl_up_sync(0xffffffffu, incl, 1);
  if (lane == 0) at = before;
  const unsigned hit = __ballot_sync(0xffffffffu, incl > target), some = __ballot_sync(0xffffffffu, own > 0);
  if (!some) return -1;
  const int who = hit ? __ffs(hit) - 1 : 31 - __clz(some);
  int tok = -1;
  double from = at;
  bool open = true;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (open && w[i] > 0) {
      tok = e + i;
      from = at;
      at += (double)w[i];
      open = !hit || at <= target;
    }
  *lo = __shfl_sync(0xffffffffu, hit ? from : -1.0, who);
  *hi = __shfl_sync(0xffffffffu, at, who);
  return __shfl_sync(0xffffffffu, tok, who);
}

// The first column with the row's largest logit.
template <class T>
SPEC_DEV int first_largest(const Row<T>& r, const Stats& st, float M) {
  int c = 0x7fffffff;
  st.each([&](int b, const float2(&v)[8]) {
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (v[i].x == M) c = b * kBlock + st.lane * 8 + i;
    return !__any_sync(0xffffffffu, c < 0x7fffffff);
  });
  c = __reduce_min_sync(0xffffffffu, c);
  // Chunks with one reference share the largest logit that stands beside their sums.
#pragma unroll 1
  for (; c < st.nch; ++c) {
    float x[kPer];
    load_chunk<T, true>(r, c, st.lane, x);
    int e = 0x7fffffff;
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i)
      if (x[i] == M) e = column<T, true>(r, c, 0, st.lane) + i;
    e = __reduce_min_sync(0xffffffffu, e);
    if (e < 0x7fffffff) return e;
  }
  return kBad;
}

SPEC_DEV double unit(float u) { return (double)fminf(fmaxf(u, 0.f), 1.f); }  // NaN: 0

// A token of p, or kBad, or kUnsure where f32 does not decide.
template <class T>
SPEC_DEV int draw(const Row<T>& r, const Stats& st, const Joined& j, float u) {
  if (!j.ok) return kBad;
  if (r.t == 0.f) return first_largest(r, st, j.ref.m);
  const double target = unit(u) * j.Z, slack = (target < 1 ? 4 : 2) * kErr * target;
  if (!j.ref.whole || target <= 0x1p-33) return kUnsure;
  double run = 0, lo, hi;
  int c = -1;
  st.each([&](int b, const float2(&v)[8]) {
    double w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = chunk_weight(v[i], j.ref);
    c = find_in_block(w, b, target, st.lane, &run);
    return c < 0;
  });
  if (c < 0) return kUnsure;
  float x[kPer];
  load_chunk<T, true>(r, c, st.lane, x);
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = ex2(fmaf(x[i], j.ref.h, -j.ref.R));
  const int tok = find_column(r, c, x, run, target, st.lane, &lo, &hi);
  return tok >= 0 && lo >= 0 && lo + slack <= target && target + slack < hi ? tok : kUnsure;
}

// ---------------------------------------------------------------------------
// Sums by a cluster
// ---------------------------------------------------------------------------
// What the columns of a row are weighed by: p in 64 bits (P64), max(p - q, 0)
// in f32 (REST32) or in 64 bits (REST64).
enum : int { P64 = 0, REST32 = 1, REST64 = 2 };

// 2^y for y <= 0 in 64 bits: the Taylor series of 2^f, |f| <= 1/2, to
// (f ln 2)^13 / 13! (the next term is below 2^-57), times the whole power.
SPEC_DEV double pow2_64(double y) {
  constexpr double kLn2 = 0.693147180559945309;
  const double n = rint(fmax(y, -1100.0)), f = (fmax(y, -1100.0) - n) * kLn2;
  double s = 1.0 / 6227020800;
  s = fma(s, f, 1.0 / 479001600);
  s = fma(s, f, 1.0 / 39916800);
  s = fma(s, f, 1.0 / 3628800);
  s = fma(s, f, 1.0 / 362880);
  s = fma(s, f, 1.0 / 40320);
  s = fma(s, f, 1.0 / 5040);
  s = fma(s, f, 1.0 / 720);
  s = fma(s, f, 1.0 / 120);
  s = fma(s, f, 1.0 / 24);
  s = fma(s, f, 1.0 / 6);
  s = fma(s, f, 0.5);
  s = fma(s, f, 1.0);
  s = fma(s, f, 1.0);
  // In two steps, so that results below 2^-1022 keep what bits they have.
  const int e = (int)n, half = e / 2;
  return s * __hiloint2double((1023 + half) << 20, 0) * __hiloint2double((1023 + e - half) << 20, 0);
}

template <class T>
struct Weigher {
  const Row<T>& r;
  const Ref& ref;
  const float* q;
  double h, inv_z;
  SPEC_DEV Weigher(const Row<T>& r_, const Ref& ref_, const float* q_, double Z) : r(r_), ref(ref_), q(q_) {
    h = 1.44269504088896341 / (double)r.t;
    inv_z = q ? 1.0 / Z : 0.0;
  }
  SPEC_DEV double p64(float x) const { return pow2_64(((double)x - (double)ref.m) * h); }
  template <bool RUN>
  SPEC_DEV void rest32(int c, int lane, float (&w)[kPer]) const {
    float y[kPer];
    load_chunk<T, RUN>(r, c, lane, w);
    load_probs<T, RUN>(r, q, c, lane, y);
    const float z = (float)inv_z;
#pragma unroll
    for (int i = 0; i < kPer; ++i) w[i] = fmaxf(fmaf(ex2(fmaf(w[i], ref.h, -ref.R)), z, -y[i]), 0.f);
  }
  template <bool RUN>
  SPEC_DEV void exact(int kind, int c, int lane, double (&w)[kPer]) const {
    float x[kPer];
    load_chunk<T, RUN>(r, c, lane, x);
#pragma unroll
    for (int i = 0; i < kPer; ++i) w[i] = p64(x[i]);
    if (kind == REST64) {
      load_probs<T, RUN>(r, q, c, lane, x);
#pragma unroll
      for (int i = 0; i < kPer; ++i) w[i] = fmax(w[i] * inv_z - (double)x[i], 0.0);
    }
  }
  // Chunk sums by all warps of the cluster; the caller syncs it.
  SPEC_DEV void sum(int kind, double* sums, int nch, int lane) const {
    const int nw = blockDim.x >> 5, step = nw * cluster_size();
#pragma unroll 1
    for (int c = cluster_rank() * nw + (threadIdx.x >> 5); c < nch; c += step) {
      double s = 0;
      if (kind == REST32) {
        float w[kPer];
        rest32<false>(c, lane, w);
        s = (double)specb200::warp_sum(pair_sum(w));
      } else {
        double w[kPer];
        exact<false>(kind, c, lane, w);
#pragma unroll
        for (int i = 0; i < kPer; ++i) s += w[i];
        s = warp_sum(s);
      }
      if (lane == 0) __stcg(sums + c, s);
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
#pragma unroll
    for (int i = 0; i < 8; ++i) s += w[i];
  }
  return warp_sum(s);
}

// A token of the weights in `sums`, whose sum is Zs: exact for P64 and REST64.
template <class T>
SPEC_DEV int draw_sums(const Weigher<T>& f, int kind, const double* sums, int nch, double Zs, float u, int lane) {
  const double target = unit(u) * Zs;
  double run = 0, lo = -1, hi;
  int c = -1, last = -1;
  for (int b = 0; b * kBlock < nch && c < 0; ++b) {
    double w[8];
    load_sums(sums, b, nch, lane, w);
    c = find_in_block(w, b, target, lane, &run);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (w[i] > 0) last = b * kBlock + lane * 8 + i;
  }
  double goal = target;
  if (c < 0) {  // the target is the whole sum: the last column of some weight
    if (kind == REST32) return kUnsure;
    c = __reduce_max_sync(0xffffffffu, last);
    if (c < 0) return kBad;
    goal = INFINITY;
  }
  if (kind == REST32) {
    float w[kPer];
    f.template rest32<true>(c, lane, w);
    const int tok = find_column(f.r, c, w, run, goal, lane, &lo, &hi);
    // The weights and Z are off by kErr of Z in all, max(p - q, 0) by no more
    // than p; so the prefix by 2 kErr, and u times the sum likewise.
    const double slack = 4.25 * kErr;
    return tok >= 0 && lo >= 0 && lo + slack <= target && target + slack < hi ? tok : kUnsure;
  }
  double w[kPer];
  f.template exact<true>(kind, c, lane, w);
  return find_column(f.r, c, w, run, goal, lane, &lo, &hi);
}

// ---------------------------------------------------------------------------
// A cluster a row
// ---------------------------------------------------------------------------
constexpr int kSampleThreads = 128;

template <class T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleParams p) {
  __shared__ int s_tok;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = kSampleThreads / 32;
  const int rank = cluster_rank(), size = cluster_size(), row = blockIdx.x / size;
  pdl_launch_dependents();
  pdl_wait();
  const Row<T> r(p.r, row);
  const int nch = p.r.nch;
  const float u = p.r.u[row];
  const Stats st(p.r.stats + (long long)row * nch, nch, lane);
  double* sums = p.r.sums + (long long)row * nch;
  const Joined j = join(r, st);
  int tok = kUnsure;
  if (warp == 0) {
    tok = draw(r, st, j, u);
    if (lane == 0) s_tok = tok;
  }
  if (p.probs) {
    float* out = p.probs + row * p.probs_stride;
    const float inv = (float)(1.0 / j.Z);
    const int top = j.ok && r.t == 0.f ? first_largest(r, st, j.ref.m) : -1;
    const bool wide = (reinterpret_cast<uintptr_t>(out) / 4 - r.shift) % 4 == 0;
    constexpr int N = Vec<T>::N;
#pragma unroll 1
    for (int c = rank * nw + warp; c < nch; c += nw * size) {
      float x[kPer];
      load_chunk<T, false>(r, c, lane, x);
#pragma unroll
      for (int i = 0; i < kPer / N; ++i) {
        const int e = column<T, false>(r, c, i, lane);
        float y[N];
#pragma unroll
        for (int k = 0; k < N; ++k) y[k] = !j.ok ? 0.f : r.t == 0.f ? (e + k == top ? 1.f : 0.f) : j.ref.weight(x[i * N + k]) * inv;
        if (wide && e >= 0 && e + N <= r.V) {
#pragma unroll
          for (int k = 0; k < N; k += 4)
            *reinterpret_cast<float4*>(out + e + k) = make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (e + k >= 0 && e + k < r.V) out[e + k] = y[k];
        }
      }
    }
  }
  __syncthreads();
  tok = s_tok;
  if (tok == kUnsure) {
    const Weigher<T> f(r, j.ref, nullptr, 0);
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
constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;

enum : int { A_REJECT = 0, A_ACCEPT = 1, A_UNSURE = 2, A_BAD = 3, A_END = 4 };

// Rows first .. last of sequence b, empty where row_start says nothing sound.
SPEC_DEV int rows_of(const VerifyParams& p, int b, int* first) {
  const int r0 = p.row_start[b], r1 = p.row_start[b + 1];
  *first = r0;
  return r0 >= 0 && r1 >= r0 && r1 <= p.r.n_rows ? r1 - r0 : 0;
}

template <class T>
__global__ void __launch_bounds__(kVerifyThreads) chain_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ int s_verdict[kVerifyWarps], s_tok;
  __shared__ Joined s_join[kVerifyWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), b = blockIdx.x / cluster_size(), nch = p.r.nch;
  pdl_launch_dependents();
  pdl_wait();
  int r0;
  const int n = rows_of(p, b, &r0);
  double* sums = p.r.sums + (long long)(n ? r0 : 0) * nch;
  bool used = false;  // other blocks may still read `sums`
  int at = 0, verdict = n ? A_ACCEPT : A_BAD;  // the row under decision; why the walk stopped
  Joined j;
  double z64 = 0;  // of row `at`, once summed in 64 bits
  // The walk, a row a warp.  Every block of the cluster comes to the same verdicts.
#pragma unroll 1
  for (int base = 0; base < n && verdict == A_ACCEPT; base += kVerifyWarps) {
    if (base + warp < n) {
      const int i = base + warp, row = r0 + i;
      const int x = i + 1 < n ? p.tokens[row] : -1;
      const Row<T> r(p.r, row);
      const Stats st(p.r.stats + (long long)row * nch, nch, lane);
      const bool judged = x >= 0 && x < p.r.V;
      const float u = p.r.u[row], q = judged ? p.q[row * p.q_stride + x] : 0.f, lx = judged ? to_float(r.p[x]) : 0.f;
      const Joined w = join(r, st);
      int v = A_END;
      if (!w.ok) {
        v = A_BAD;
      } else if (judged) {
        const double left = unit(u) * (double)q;
        if (q <= 0.f) {
          v = A_ACCEPT;
        } else if (r.t == 0.f) {
          v = left <= (x == first_largest(r, st, w.ref.m) ? 1.0 : 0.0);
        } else {
          const double px = (double)w.ref.weight(lx), lz = left * w.Z;
          // w_x alone: off by (4.5 + 2.5 * 23) u where it is above 2^-33.
          const double slack = 3 * kErr * lz + 0x1p-33;
          v = !w.ref.whole ? A_UNSURE : lz + slack < px ? A_ACCEPT : lz > px + slack ? A_REJECT : A_UNSURE;
          if (q != q) v = A_REJECT;
        }
      }
      if (lane == 0) s_verdict[warp] = v, s_join[warp] = w;
    }
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < kVerifyWarps && base + w < n; ++w) {
      at = base + w;
      verdict = s_verdict[w];
      j = s_join[w];
      if (verdict == A_UNSURE) {
        const Row<T> r(p.r, r0 + at);
        const Weigher<T> f(r, j.ref, nullptr, 0);
        if (used) cluster_sync();
        f.sum(P64, sums, nch, lane);
        cluster_sync();
        used = true;
        z64 = total(sums, nch, lane);
        const int x = p.tokens[r0 + at];
        const double left = unit(p.r.u[r0 + at]) * (double)p.q[(r0 + at) * p.q_stride + x];
        verdict = left * z64 <= f.p64(to_float(r.p[x])) ? A_ACCEPT : A_REJECT;
        if (verdict == A_ACCEPT) z64 = 0;
      }
      if (verdict != A_ACCEPT) break;
    }
    __syncthreads();
  }
  int tok = kBad;
  if (verdict != A_BAD) {
    const int row = r0 + at;
    const Row<T> r(p.r, row);
    const Stats st(p.r.stats + (long long)row * nch, nch, lane);
    const bool rest = verdict == A_REJECT;
    const float* q = rest ? p.q + row * p.q_stride : nullptr;
    const float u = p.r.u[row + rest];  // a row follows every draft
    tok = kUnsure;
    if (r.t == 0.f) {
      // All of p on one token: what is left of it is that token, unless q holds it all too.
      if (warp == 0) tok = first_largest(r, st, j.ref.m);
    } else if (!rest) {
      if (warp == 0) tok = draw(r, st, j, u);
    } else if (j.ref.whole && z64 == 0) {
      const Weigher<T> f(r, j.ref, q, j.Z);
      if (used) cluster_sync();
      f.sum(REST32, sums, nch, lane);
      cluster_sync();
      used = true;
      if (warp == 0) tok = draw_sums(f, REST32, sums, nch, total(sums, nch, lane), u, lane);
    }
    if (threadIdx.x == 0) s_tok = tok;
    __syncthreads();
    tok = s_tok;
    if (tok == kUnsure) {
      const Weigher<T> f(r, j.ref, nullptr, 0);
      double z = z64;
      if (z == 0) {
        if (used) cluster_sync();
        f.sum(P64, sums, nch, lane);
        cluster_sync();
        z = total(sums, nch, lane);
      }
      int kind = P64;
      double zs = z;
      if (rest) {
        const Weigher<T> g(r, j.ref, q, z);
        cluster_sync();
        g.sum(REST64, sums, nch, lane);
        cluster_sync();
        kind = REST64;
        zs = total(sums, nch, lane);
        if (!(zs > 0)) {  // p is nowhere above q: p itself
          cluster_sync();
          f.sum(P64, sums, nch, lane);
          cluster_sync();
          kind = P64;
          zs = z;
        }
      }
      if (rank == 0 && warp == 0) {
        const Weigher<T> g(r, j.ref, kind == P64 ? nullptr : q, z);
        tok = draw_sums(g, kind, sums, nch, zs, u, lane);
      }
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
template <class T>
__global__ void __launch_bounds__(kVerifyThreads) tree_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ int s_tok;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), size = cluster_size(), b = blockIdx.x / size, nch = p.r.nch;
  pdl_launch_dependents();
  pdl_wait();
  int r0;
  const int n = rows_of(p, b, &r0);
#pragma unroll 1
  for (int i = rank * kVerifyWarps + warp; i < n; i += size * kVerifyWarps) {
    const Row<T> r(p.r, r0 + i);
    const float u = p.r.u[r0 + i];
    const Stats st(p.r.stats + (long long)(r0 + i) * nch, nch, lane);
    const int tok = draw(r, st, join(r, st), u);
    if (lane == 0) __stcg(p.r.drawn + r0 + i, tok);
  }
  cluster_sync();
  double* sums = p.r.sums + (long long)(n ? r0 : 0) * nch;
  int cur = 0, len = 0, tok = kBad;
#pragma unroll 1
  while (len < n) {
    if (rank == 0 && threadIdx.x == 0) p.r.path[r0 + len] = cur;
    ++len;
    tok = __ldcg(p.r.drawn + r0 + cur);
    if (tok == kUnsure) {
      const Row<T> r(p.r, r0 + cur);
      const Joined j = join(r, Stats(p.r.stats + (long long)(r0 + cur) * nch, nch, lane));
      const Weigher<T> f(r, j.ref, nullptr, 0);
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
      const bool hit = i + lane < n && p.parents[r0 + i + lane] == cur && p.tokens[r0 + i + lane] == tok;
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

// Blocks a cluster: 8, fewer where those of all clusters would not be resident at once.
int cluster_for(int n, int threads, int sms) {
  int size = 8;
  while (size > 1 && (long long)n * size > (long long)sms * (2048 / threads)) size /= 2;
  return size;
}

// A chunk a warp where that is less than the warps that the device holds, else four.
template <class T>
cudaError_t stats(const Rows& r, int sms, cudaStream_t s) {
  const long long chunks = (long long)r.n_rows * r.nch;
  if (chunks <= sms * 64LL) return kv4::launch_overlapping(stats_kernel<T, 1>, dim3((unsigned)(chunks / 8)), 256, 0, s, r);
  return kv4::launch_overlapping(stats_kernel<T, 4>, dim3((unsigned)((chunks / 4 + 7) / 8)), 256, 0, s, r);
}
template <class T>
cudaError_t sample(const SampleParams& p, int sms, cudaStream_t s) {
  const cudaError_t e = stats<T>(p.r, sms, s);
  if (e != cudaSuccess) return e;
  return launch_clusters(sample_kernel<T>, p.r.n_rows, cluster_for(p.r.n_rows, kSampleThreads, sms), kSampleThreads, s, p);
}
template <class T>
cudaError_t verify(const VerifyParams& p, bool trees, int sms, cudaStream_t s) {
  const cudaError_t e = p.r.n_rows ? stats<T>(p.r, sms, s) : cudaSuccess;
  if (e != cudaSuccess) return e;
  const int size = cluster_for(p.n_seqs, kVerifyThreads, sms);
  return trees ? launch_clusters(tree_kernel<T>, p.n_seqs, size, kVerifyThreads, s, p)
               : launch_clusters(chain_kernel<T>, p.n_seqs, size, kVerifyThreads, s, p);
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
