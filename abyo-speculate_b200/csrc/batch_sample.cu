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
// summed again in 64 bits by the whole cluster.  With u = 2^-24 and d = (M - l) / T:
// l - M, the scale log2(e) / T and their product are off by u each, so a weight
// e^-d by 3 u d, the hardware's 2^x by 4 u more, a chunk's sum of positive terms
// by 9 u (16 a lane in pairs, 5 rounds of shuffles), a chunk's own scale by
// another 4 u.  The mean of d under the weights of any set of columns is their
// entropy less the logarithm of their sum S, at most ln V - ln S; for S >= 1
// and V <= 2^20 that makes (17 + 3 * 13.9) u < 2^-18 of S (kErr), for S > 2^-33
// twice that.  Smaller sums are left to 64 bits.
//
// Two kernels.  stats_kernel reads every row once, a warp a chunk of 512
// columns, and leaves each chunk's largest logit and sum.  The second kernel
// runs a cluster a row (sample) or a sequence (chains, trees); a warp joins a
// row's chunks by a scan over their sums, finds the chunk of the token and reads
// that alone.  A rejected draft's max(p - q, 0) is summed by all warps of the
// cluster, from p and q once more.
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
  SPEC_DEV int column(int c, int i, int lane) const { return c * kChunk - shift + (i * 32 + lane) * Vec<T>::N; }
};

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
SPEC_DEV float to_float(float x) { return x; }
SPEC_DEV float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
SPEC_DEV float to_float(__half x) { return __half2float(x); }

// This lane's 16 columns of chunk c: vectors lane, 32 + lane, ...; columns
// outside the row are -inf.
template <class T>
SPEC_DEV void load_chunk(const Row<T>& r, int c, int lane, float (&x)[kPer]) {
  constexpr int N = Vec<T>::N;
  uint4 v[kPer / N];
#pragma unroll
  for (int i = 0; i < kPer / N; ++i) {
    const int e = r.column(c, i, lane);
    if (e >= 0 && e + N <= r.V) v[i] = *reinterpret_cast<const uint4*>(r.p + e);
  }
#pragma unroll
  for (int i = 0; i < kPer / N; ++i) {
    const int e = r.column(c, i, lane);
    float y[N];
    if (e >= 0 && e + N <= r.V) {
      unpack(v[i], y, r.p);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) y[k] = e + k >= 0 && e + k < r.V ? to_float(r.p[e + k]) : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) x[i * N + k] = y[k];
  }
}

// The same columns of a row of f32 probabilities; zeros outside.
template <class T>
SPEC_DEV void load_probs(const Row<T>& r, const float* q, int c, int lane, float (&x)[kPer]) {
  constexpr int N = Vec<T>::N;
  const bool wide = (reinterpret_cast<uintptr_t>(q) / 4 - r.shift) % 4 == 0;
#pragma unroll
  for (int i = 0; i < kPer / N; ++i) {
    const int e = r.column(c, i, lane);
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

// A NaN or +inf makes its chunk's sum NaN.
template <class T>
__global__ void __launch_bounds__(256) stats_kernel(const __grid_constant__ Rows r) {
  const int lane = threadIdx.x & 31;
  const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  if (at >= (long long)r.n_rows * r.nch) return;
  const int row = (int)(at / r.nch), c = (int)(at - (long long)row * r.nch);
  if (r.path && c == 0 && lane == 0) r.path[row] = -1;
  const Row<T> rr(r, row);
  float x[kPer];
  load_chunk(rr, c, lane, x);
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) m = fmaxf(m, x[i]);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = ex2((x[i] - ref) * rr.h);
  const float s = warp_sum(pair_sum(x));
  if (lane == 0) r.stats[at] = make_float2(m, s);
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

struct Joined {
  float M;
  double Z;
  bool ok;  // the row has a finite largest logit and no NaN
};
// Weight of chunk statistics (m, s) with the row's largest logit as reference.
SPEC_DEV double chunk_weight(float2 v, float M, float h) { return (double)(v.y * ex2((v.x - M) * h)); }

template <class T>
SPEC_DEV Joined join(const Row<T>& r, const float2* st, int nch, int lane) {
  Joined j;
  j.M = -INFINITY;
  for (int c = lane; c < nch; c += 32) j.M = fmaxf(j.M, __ldcg(st + c).x);
  j.M = specb200::warp_max(j.M);
  double z = 0;
  for (int c = lane; c < nch; c += 32) z += chunk_weight(__ldcg(st + c), j.M, r.h);
  j.Z = warp_sum(z);
  j.ok = r.ok && j.M > -INFINITY && j.M < INFINITY && j.Z > 0 && j.Z < INFINITY;
  return j;
}

// The first chunk whose cumulative weight passes `target`, and the weight
// before it; -1: none does.  weight(c): of chunk c.
template <class F>
SPEC_DEV int find_chunk(F weight, int nch, double target, int lane, double* before) {
  const int per = (nch + 31) / 32, c0 = min(lane * per, nch), c1 = min(c0 + per, nch);
  double own = 0;
  for (int c = c0; c < c1; ++c) own += weight(c);
  const double incl = warp_scan(own, lane);
  double run = __shfl_up_sync(0xffffffffu, incl, 1);  // not above the target where incl passes it
  if (lane == 0) run = 0;
  int found = -1;
  const unsigned hit = __ballot_sync(0xffffffffu, incl > target);
  if (!hit) return -1;
  const int who = __ffs(hit) - 1;
  if (lane == who) {
    for (int c = c0; c < c1; ++c) {
      const double w = weight(c);
      if (w > 0) found = c;
      if (run + w > target) break;
      run += w;
    }
    // Rounding may leave the sum of all a step below the scanned one: the last chunk of some weight.
  }
  found = __shfl_sync(0xffffffffu, found, who);
  *before = __shfl_sync(0xffffffffu, run, who);
  return found;
}

// The first of a chunk's columns whose cumulative weight passes `target`;
// w(i): weight of this lane's i-th column.  Where none does, the last column
// of some weight.  [lo, hi): cumulative weights around the column.
template <class T, class F>
SPEC_DEV int find_column(const Row<T>& r, int c, F w, double before, double target, int lane, double* lo, double* hi) {
  constexpr int N = Vec<T>::N;
  int last = -1;
#pragma unroll 1
  for (int i = 0; i < kPer / N; ++i) {
    double own = 0;
    int mine = -1;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const double x = w(i * N + k);
      own += x;
      if (x > 0) mine = r.column(c, i, lane) + k;
    }
    const double incl = warp_scan(own, lane) + before;
    double run = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) run = before;
    const unsigned hit = __ballot_sync(0xffffffffu, incl > target);
    if (hit) {
      const int who = __ffs(hit) - 1;
      int tok = mine;
      double next = incl;
      if (lane == who) {
        double cum = run;
        bool open = true;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const double x = w(i * N + k);
          if (open && cum + x > target) tok = r.column(c, i, lane) + k, run = cum, next = cum + x, open = false;
          cum += x;
        }
      }
      *lo = __shfl_sync(0xffffffffu, run, who);
      *hi = __shfl_sync(0xffffffffu, next, who);
      return __shfl_sync(0xffffffffu, tok, who);
    }
    before = __shfl_sync(0xffffffffu, incl, 31);
    const unsigned some = __ballot_sync(0xffffffffu, mine >= 0);
    if (some) last = __shfl_sync(0xffffffffu, mine, 31 - __clz(some));
  }
  *lo = *hi = -1;
  return last;
}

// The first column with the row's largest logit.
template <class T>
SPEC_DEV int first_largest(const Row<T>& r, const float2* st, int nch, float M, int lane) {
  int c = 0x7fffffff;
  for (int i = lane; i < nch; i += 32)
    if (__ldcg(st + i).x == M) {
      c = i;
      break;
    }
  c = __reduce_min_sync(0xffffffffu, c);
  float x[kPer];
  load_chunk(r, c, lane, x);
  int e = 0x7fffffff;
#pragma unroll
  for (int i = kPer - 1; i >= 0; --i)
    if (x[i] == M) e = r.column(c, i / Vec<T>::N, lane) + i % Vec<T>::N;
  return __reduce_min_sync(0xffffffffu, e);
}

SPEC_DEV double unit(float u) { return (double)fminf(fmaxf(u, 0.f), 1.f); }  // NaN: 0

// A token of p, or kBad, or kUnsure where f32 does not decide.
template <class T>
SPEC_DEV int draw(const Row<T>& r, const float2* st, int nch, const Joined& j, float u, int lane) {
  if (!j.ok) return kBad;
  if (r.t == 0.f) return first_largest(r, st, nch, j.M, lane);
  const double target = unit(u) * j.Z, slack = (target < 1 ? 4 : 2) * kErr * target;
  if (target <= 0x1p-33) return kUnsure;
  double before, lo, hi;
  const int c = find_chunk([&](int i) { return chunk_weight(__ldcg(st + i), j.M, r.h); }, nch, target, lane, &before);
  if (c < 0) return kUnsure;
  float x[kPer];
  load_chunk(r, c, lane, x);
#pragma unroll
  for (int i = 0; i < kPer; ++i) x[i] = ex2((x[i] - j.M) * r.h);
  const int tok = find_column(r, c, [&](int i) { return (double)x[i]; }, before, target, lane, &lo, &hi);
  return lo >= 0 && lo + slack <= target && target + slack < hi ? tok : kUnsure;
}

// ---------------------------------------------------------------------------
// 64-bit sums by a cluster
// ---------------------------------------------------------------------------
template <class T>
SPEC_DEV double weight64(const Row<T>& r, float x, float M) {
  return exp(((double)x - (double)M) * (1.0 / (double)r.t));
}

// Sums of a row's chunks into `sums`, by all warps of the cluster.
// kind 0: p in 64 bits; 1: max(p - q, 0) in f32; 2: the same in 64 bits.
// The caller syncs the cluster.
template <class T>
SPEC_DEV void sum_chunks(const Row<T>& r, float M, double Z, const float* q, int kind, double* sums, int nch, int lane) {
  const int nw = blockDim.x >> 5, step = nw * cluster_size();
  const double inv_t = 1.0 / (double)r.t, inv_z = kind ? 1.0 / Z : 0;
  const float inv_zf = (float)inv_z;
#pragma unroll 1
  for (int c = cluster_rank() * nw + (threadIdx.x >> 5); c < nch; c += step) {
    float x[kPer], y[kPer];
    load_chunk(r, c, lane, x);
    if (kind) load_probs(r, q, c, lane, y);
    double s;
    if (kind == 1) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = fmaxf(fmaf(ex2((x[i] - M) * r.h), inv_zf, -y[i]), 0.f);
      s = (double)specb200::warp_sum(pair_sum(x));
    } else {
      s = 0;
#pragma unroll 4
      for (int i = 0; i < kPer; ++i) {
        const double w = exp(((double)x[i] - (double)M) * inv_t);
        s += kind ? fmax(w * inv_z - (double)y[i], 0.0) : w;
      }
      s = warp_sum(s);
    }
    if (lane == 0) __stcg(sums + c, s);
  }
}
SPEC_DEV double total(const double* sums, int nch, int lane) {
  double s = 0;
  for (int c = lane; c < nch; c += 32) s += __ldcg(sums + c);
  return warp_sum(s);
}
SPEC_DEV int last_chunk(const double* sums, int nch, int lane) {
  int last = -1;
  for (int c = lane; c < nch; c += 32)
    if (__ldcg(sums + c) > 0) last = c;
  return __reduce_max_sync(0xffffffffu, last);
}

// A token of the weights that sum_chunks(kind) summed: exact for kinds 0 and 2.
template <class T>
SPEC_DEV int draw_sums(const Row<T>& r, float M, double Z, const float* q, int kind, const double* sums, int nch, double Zs,
                       float u, int lane) {
  const double target = unit(u) * Zs;
  double before = 0, lo, hi;
  int c = find_chunk([&](int i) { return __ldcg(sums + i); }, nch, target, lane, &before);
  if (c < 0) {
    if (kind == 1) return kUnsure;
    c = last_chunk(sums, nch, lane);
    if (c < 0) return kBad;
    before = -1;  // its last column of some weight
  }
  float x[kPer], y[kPer];
  load_chunk(r, c, lane, x);
  if (kind) load_probs(r, q, c, lane, y);
  const double inv_z = kind ? 1.0 / Z : 0;
  const float inv_zf = (float)inv_z;
  const double end = before < 0 ? INFINITY : target;
  if (before < 0) before = 0;
  const int tok = find_column(
      r, c,
      [&](int i) -> double {
        if (kind == 1) return (double)fmaxf(fmaf(ex2((x[i] - M) * r.h), inv_zf, -y[i]), 0.f);
        const double w = weight64(r, x[i], M);
        return kind ? fmax(w * inv_z - (double)y[i], 0.0) : w;
      },
      before, end, lane, &lo, &hi);
  if (kind != 1) return tok;
  // The weights and Z are off by kErr of Z in all, max(p - q, 0) by no more
  // than p; so the prefix by 2 kErr, and u times the sum likewise.
  const double slack = 4.25 * kErr;
  return lo >= 0 && lo + slack <= target && target + slack < hi ? tok : kUnsure;
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
  const float2* st = p.r.stats + (long long)row * nch;
  double* sums = p.r.sums + (long long)row * nch;
  const Joined j = join(r, st, nch, lane);
  const float u = p.r.u[row];
  int tok = kUnsure;
  if (warp == 0) {
    tok = draw(r, st, nch, j, u, lane);
    if (lane == 0) s_tok = tok;
  }
  if (p.probs) {
    float* out = p.probs + row * p.probs_stride;
    const float inv = j.ok ? (float)(1.0 / j.Z) : 0.f;
    const int top = j.ok && r.t == 0.f ? first_largest(r, st, nch, j.M, lane) : -1;
    const bool wide = (reinterpret_cast<uintptr_t>(out) / 4 - r.shift) % 4 == 0;
    constexpr int N = Vec<T>::N;
#pragma unroll 1
    for (int c = rank * nw + warp; c < nch; c += nw * size) {
      float x[kPer];
      load_chunk(r, c, lane, x);
#pragma unroll
      for (int i = 0; i < kPer / N; ++i) {
        const int e = r.column(c, i, lane);
        float y[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          y[k] = !j.ok ? 0.f : r.t == 0.f ? (e + k == top ? 1.f : 0.f) : ex2((x[i * N + k] - j.M) * r.h) * inv;
        }
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
    sum_chunks(r, j.M, 0, nullptr, 0, sums, nch, lane);
    cluster_sync();
    if (rank || warp) return;
    tok = draw_sums(r, j.M, 0, nullptr, 0, sums, nch, total(sums, nch, lane), u, lane);
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
  int at = 0, verdict = n ? A_ACCEPT : A_BAD;  // the row under decision; why the walk stopped
  Joined j{0.f, 0, false};
  double z64 = 0;  // of row `at`, once summed in 64 bits
  // The walk, a row a warp.  Every block of the cluster comes to the same verdicts.
#pragma unroll 1
  for (int base = 0; base < n && verdict == A_ACCEPT; base += kVerifyWarps) {
    if (base + warp < n) {
      const int i = base + warp, row = r0 + i;
      const Row<T> r(p.r, row);
      const float2* st = p.r.stats + (long long)row * nch;
      const Joined w = join(r, st, nch, lane);
      const int x = i + 1 < n ? p.tokens[row] : -1;
      int v = A_END;
      if (!w.ok) {
        v = A_BAD;
      } else if (x >= 0 && x < p.r.V) {
        const float q = p.q[row * p.q_stride + x];
        const double left = unit(p.r.u[row]) * (double)q;
        if (q <= 0.f) {
          v = A_ACCEPT;
        } else if (r.t == 0.f) {
          v = left <= (x == first_largest(r, st, nch, w.M, lane) ? 1.0 : 0.0);
        } else {
          const double px = (double)ex2((to_float(r.p[x]) - w.M) * r.h), lz = left * w.Z;
          // w_x alone: off by (4 + 3 * 23) u where it is above 2^-33.
          const double slack = 3 * kErr * lz + 0x1p-33;
          v = lz + slack < px ? A_ACCEPT : lz > px + slack ? A_REJECT : A_UNSURE;
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
        cluster_sync();
        sum_chunks(r, j.M, 0, nullptr, 0, sums, nch, lane);
        cluster_sync();
        z64 = total(sums, nch, lane);
        const int x = p.tokens[r0 + at];
        const double left = unit(p.r.u[r0 + at]) * (double)p.q[(r0 + at) * p.q_stride + x];
        verdict = left * z64 <= weight64(r, to_float(r.p[x]), j.M) ? A_ACCEPT : A_REJECT;
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
    const float2* st = p.r.stats + (long long)row * nch;
    const float* q = nullptr;
    int kind = 0;
    float u = p.r.u[row];
    tok = kUnsure;
    if (verdict == A_REJECT) {
      u = p.r.u[row + 1];  // a row follows every draft
      q = p.q + row * p.q_stride;
      kind = 2;
    }
    if (r.t == 0.f) {
      // All of p on one token: what is left of it is that token, unless q holds it all too.
      if (warp == 0) tok = first_largest(r, st, nch, j.M, lane);
    } else if (verdict == A_END) {
      if (warp == 0) tok = draw(r, st, nch, j, u, lane);
    } else if (z64 == 0) {
      cluster_sync();
      sum_chunks(r, j.M, j.Z, q, 1, sums, nch, lane);
      cluster_sync();
      if (warp == 0) tok = draw_sums(r, j.M, j.Z, q, 1, sums, nch, total(sums, nch, lane), u, lane);
    }
    if (threadIdx.x == 0) s_tok = tok;
    __syncthreads();
    tok = s_tok;
    if (tok == kUnsure) {
      double z = z64;
      if (z == 0) {
        cluster_sync();
        sum_chunks(r, j.M, 0, nullptr, 0, sums, nch, lane);
        cluster_sync();
        z = total(sums, nch, lane);
      }
      double zs = z;
      if (kind == 2) {
        cluster_sync();
        sum_chunks(r, j.M, z, q, 2, sums, nch, lane);
        cluster_sync();
        zs = total(sums, nch, lane);
        if (!(zs > 0)) {  // p is nowhere above q: p itself
          cluster_sync();
          sum_chunks(r, j.M, 0, nullptr, 0, sums, nch, lane);
          cluster_sync();
          kind = 0;
          zs = z;
        }
      }
      if (rank == 0 && warp == 0) tok = draw_sums(r, j.M, z, q, kind, sums, nch, zs, u, lane);
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
    const float2* st = p.r.stats + (long long)(r0 + i) * nch;
    const int tok = draw(r, st, nch, join(r, st, nch, lane), p.r.u[r0 + i], lane);
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
      const Joined j = join(r, p.r.stats + (long long)(r0 + cur) * nch, nch, lane);
      cluster_sync();
      sum_chunks(r, j.M, 0, nullptr, 0, sums, nch, lane);
      cluster_sync();
      if (warp == 0) {
        tok = draw_sums(r, j.M, 0, nullptr, 0, sums, nch, total(sums, nch, lane), p.r.u[r0 + cur], lane);
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

template <class T>
cudaError_t stats(const Rows& r, cudaStream_t s) {
  const long long blocks = ((long long)r.n_rows * r.nch + 7) / 8;
  return kv4::launch_overlapping(stats_kernel<T>, dim3((unsigned)blocks), 256, 0, s, r);
}
template <class T>
cudaError_t sample(const SampleParams& p, int sms, cudaStream_t s) {
  const cudaError_t e = stats<T>(p.r, s);
  if (e != cudaSuccess) return e;
  return launch_clusters(sample_kernel<T>, p.r.n_rows, cluster_for(p.r.n_rows, kSampleThreads, sms), kSampleThreads, s, p);
}
template <class T>
cudaError_t verify(const VerifyParams& p, bool trees, int sms, cudaStream_t s) {
  const cudaError_t e = p.r.n_rows ? stats<T>(p.r, s) : cudaSuccess;
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
