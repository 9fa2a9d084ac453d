// 4-bit paged KV cache: handles, the per-step plan, and the checks of every
// argument that the kernels rely on.  A plan is validated on the host and kept
// in device memory of the library's own, so the kernels need no bounds checks
// on pages and slots.
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <memory>
#include <new>
#include <vector>

#include "../../include/spec_b200.h"
#include "kv4.h"
#include "model.h"

using namespace specb200;
using namespace specb200::kv4;

namespace {

// What a cache handle and its batches share.
struct Cache {
  spec_kv4_desc d{};
  uint8_t* pool = nullptr;
  const float *cos = nullptr, *sin = nullptr;
  int n_positions = 0;
  int64_t layer_bytes() const {
    return (int64_t)d.n_pages * d.n_kv_heads * block_bytes(d.page_tokens, d.head_dim);
  }
};

int fail(int rc, const char* msg) {
  set_thread_error(msg);
  return rc;
}
template <class... A>
int fail(int rc, const char* fmt, A... a) {
  char msg[256];
  snprintf(msg, sizeof msg, fmt, a...);
  set_thread_error(msg);
  return rc;
}
int fail_cuda(cudaError_t e, const char* what) {
  cudaGetLastError();  // reported here: the next launch's check is not to find it
  return fail(e == cudaErrorMemoryAllocation ? SPEC_ERR_OOM : SPEC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int check_desc(const spec_kv4_desc* d) {
  if (!d) return fail(SPEC_ERR_INVALID, "spec_kv4: null description");
  if (d->head_dim != 64 && d->head_dim != 128)
    return fail(SPEC_ERR_UNSUPPORTED, "spec_kv4: head_dim %d (64 or 128 are built)", d->head_dim);
  if (d->page_tokens != 16 && d->page_tokens != 32 && d->page_tokens != 64 && d->page_tokens != 128)
    return fail(SPEC_ERR_UNSUPPORTED, "spec_kv4: page_tokens %d (16, 32, 64 or 128 are built)", d->page_tokens);
  if (d->n_layers < 1 || d->n_pages < 1 || d->n_kv_heads < 1 || d->n_kv_heads > 1024 || d->n_heads < d->n_kv_heads ||
      d->n_heads > 4096 || d->n_heads % d->n_kv_heads)
    return fail(SPEC_ERR_INVALID,
                "spec_kv4: n_layers %d, n_pages %d, n_heads %d, n_kv_heads %d: positive counts, n_heads a multiple of "
                "n_kv_heads, at most 4096 and 1024",
                d->n_layers, d->n_pages, d->n_heads, d->n_kv_heads);
  if (d->device < 0) return fail(SPEC_ERR_INVALID, "spec_kv4: device %d", d->device);
  const int64_t block = block_bytes(d->page_tokens, d->head_dim);
  if ((int64_t)d->n_pages * d->n_kv_heads > INT64_MAX / 2 / block / d->n_layers)
    return fail(SPEC_ERR_INVALID, "spec_kv4: the pool's size passes 63 bits");
  return SPEC_OK;
}

}  // namespace

struct spec_kv4 {
  std::shared_ptr<Cache> c;
};

namespace {

// What one attention kernel does in a step.
struct Schedule {
  std::vector<Unit> order;  // first units of all CTAs, then each CTA's others, then (wide) the joins
  const Unit* units = nullptr;  // the same on the device
  int n_units = 0, n_joins = 0;
  int n_ctas = 0, n_parts = 0, n_groups = 0;
  int nt = 1;                   // 8-column tiles of the largest unit
};

}  // namespace

struct spec_kv4_batch {
  std::shared_ptr<Cache> c;
  // The plan: one device allocation, written from one pinned one.
  uint8_t *dev = nullptr, *host = nullptr;
  size_t cap = 0;
  unsigned* err = nullptr;
  cudaEvent_t tail = nullptr, copied = nullptr;
  unsigned long long last = 0;  // id of the stream of the previous call
  bool planned = false, used = false;
  bool many = false;  // calls on more than one stream were made: `tail` is recorded
  int n_rows = 0, max_src = -1;
  int min_pos = 0, max_pos = -1;
  bool has_src = false;
  const RowDev* rows = nullptr;
  const int* table = nullptr;
  const unsigned long long* masks = nullptr;
  // The attention's schedules (narrow and wide kernel), and their workspace:
  // arrival counters (zero between calls) and partial states.
  Schedule narrow, wide;
  int sms = 0;
  int wide_from = -1;  // columns; -1: by estimate
  int wide_pair = -1;  // units in pairs of stages: 0, 1; -1: by estimate
  bool pair = false;   // and the plan's choice
  int force_cols = -1, narrow_cols = kMaxCols;  // columns of a narrow unit at most, likewise
  int* arrived = nullptr;
  size_t arrived_cap = 0;
  float* parts = nullptr;
  size_t parts_cap = 0;
  std::vector<Unit> tiles, runs, joins;
  std::vector<int> cuts;
  std::vector<uint8_t> seen;  // per page: 1 = read, 2 = written; zero between plans
};

namespace {

bool capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(s, &st) == cudaSuccess) return st != cudaStreamCaptureStatusNone;
  cudaGetLastError();
  return false;
}

// A call on stream `s`: ordered after the batch's previous call where that was
// on another stream.  A batch that has only seen one stream records nothing
// (an event costs a call about 1 us); the first change of stream waits for
// the device once, since the old stream may no longer exist, and from then on
// every call leaves an event for the next.  Under capture nothing is ordered.
struct Turn {
  spec_kv4_batch* b;
  cudaStream_t s;
  unsigned long long id = 0;
  bool recorded = false;
  cudaError_t enter() {
    recorded = capturing(s);
    if (recorded) return cudaSuccess;
    cudaError_t e = cudaStreamGetId(s, &id);
    if (e != cudaSuccess || !b->used || id == b->last) return e;
    if (b->many) return cudaStreamWaitEvent(s, b->tail, 0);
    e = cudaDeviceSynchronize();
    if (e == cudaSuccess) b->many = true;
    return e;
  }
  cudaError_t leave() {
    if (recorded) return cudaSuccess;
    b->last = id;
    b->used = true;
    return b->many ? cudaEventRecord(b->tail, s) : cudaSuccess;
  }
};
// Waits for the batch's calls.
cudaError_t drain(spec_kv4_batch* b) {
  if (!b->used) return cudaSuccess;
  return b->many ? cudaEventSynchronize(b->tail) : cudaDeviceSynchronize();
}

// The batch's device is current during a call; the caller's comes back.
struct Current {
  int prev = -1, device;
  int rc = SPEC_OK;
  explicit Current(int d) : device(d) {
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != d) e = cudaSetDevice(d);
    if (e != cudaSuccess) rc = fail_cuda(e, "spec_kv4: cudaSetDevice");
  }
  ~Current() {
    if (prev >= 0 && prev != device) cudaSetDevice(prev);
  }
  Current(const Current&) = delete;
  Current& operator=(const Current&) = delete;
};

void release(spec_kv4_batch* b) {
  drain(b);
  if (b->dev) cudaFree(b->dev);
  if (b->host) cudaFreeHost(b->host);
  if (b->err) cudaFree(b->err);
  if (b->arrived) cudaFree(b->arrived);
  if (b->parts) cudaFree(b->parts);
  if (b->tail) cudaEventDestroy(b->tail);
  if (b->copied) cudaEventDestroy(b->copied);
}

// A device array of at least n elements; its old contents are dropped once
// the batch's calls are done.
template <class T>
cudaError_t grow(spec_kv4_batch* b, T** p, size_t* cap, size_t n, bool zero) {
  if (n <= *cap) return cudaSuccess;
  cudaError_t e = drain(b);
  if (e != cudaSuccess) return e;
  if (*p) cudaFree(*p);
  *p = nullptr;
  *cap = 0;
  n += n / 2;
  e = cudaMalloc(reinterpret_cast<void**>(p), n * sizeof(T));
  if (e == cudaSuccess && zero) e = cudaMemset(*p, 0, n * sizeof(T));
  if (e == cudaSuccess && zero) e = cudaDeviceSynchronize();
  if (e == cudaSuccess) *cap = n;
  return e;
}

// Whether two of rows x heads runs of D elements meet: rows lie `row` elements
// apart, heads `head`.
bool shares_elements(int64_t rows, int64_t heads, int64_t row, int64_t head, int64_t D) {
  if (heads > 1 && head < D) return true;
  if (rows > 1 && row < D) return true;
  if (rows <= 1 || heads <= 1 || row / heads >= head || head / rows >= row) return false;
  // Neither lies inside a step of the other: a run (dr, 0) against (0, dh), for
  // every dh the two dr around it.
  for (int64_t dh = 1; dh < heads; ++dh) {
    const int64_t at = dh * head, dr = at / row;
    if ((dr < rows && at - dr * row < D) || (dr + 1 < rows && (dr + 1) * row - at < D)) return true;
  }
  return false;
}

int check_rows(const char* what, const spec_kv4_rows* r, int64_t need, int heads, int D, bool written) {
  if (!r->ptr) return fail(SPEC_ERR_INVALID, "spec_kv4: %s has no data", what);
  if (r->dtype < T_BF16 || r->dtype > T_F32) return fail(SPEC_ERR_INVALID, "spec_kv4: %s has type %d", what, r->dtype);
  if (r->n_rows < need)
    return fail(SPEC_ERR_INVALID, "spec_kv4: %s has %lld rows, the plan needs %lld", what, (long long)r->n_rows,
                (long long)need);
  const int64_t lim = INT64_C(1) << 40;
  if (r->row_stride < 0 || r->head_stride < 0 || r->row_stride > lim || r->head_stride > lim)
    return fail(SPEC_ERR_INVALID, "spec_kv4: %s has a stride outside [0, 2^40]", what);
  if (reinterpret_cast<uintptr_t>(r->ptr) % (r->dtype == T_F32 ? 4 : 2))
    return fail(SPEC_ERR_INVALID, "spec_kv4: %s is not aligned to its element size", what);
  if (written && shares_elements(need, heads, r->row_stride, r->head_stride, D))
    return fail(SPEC_ERR_INVALID, "spec_kv4: rows or heads of %s overlap (strides %lld and %lld)", what,
                (long long)r->row_stride, (long long)r->head_stride);
  return SPEC_OK;
}

Rows to_rows(const spec_kv4_rows* r) {
  Rows o;
  if (r) {
    o.ptr = r->ptr;
    o.row_stride = r->row_stride;
    o.head_stride = r->head_stride;
    o.dtype = r->dtype;
  }
  return o;
}

// Whether 8 consecutive channels are one (f32: two) aligned 16-byte access.
bool wide(const spec_kv4_rows* r) {
  if (!r) return true;
  const int64_t sz = r->dtype == T_F32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(r->ptr) % 16 == 0 && r->row_stride * sz % 16 == 0 && r->head_stride * sz % 16 == 0;
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

// A unit's queries in and states out cost about as much as two of its stages
// (64 sequences of 500 to 16000 tokens, one row: 163 us at 0, 149 at 1 and 2,
// 153 at 3, 157 at 6).
constexpr int kUnitCost = 2;

constexpr int kNarrowCols[] = {8, 16, kMaxCols};

// Columns of the narrow kernel's tiles of a sequence: of equal size, a multiple
// of 8, at most `most`.
int narrow_tile(int64_t cols, int most) {
  const int64_t tiles = (cols + most - 1) / most;
  return tiles ? (int)(((cols + tiles - 1) / tiles + 7) / 8 * 8) : 0;
}

// Expected time (us) of the step's attention when sequences of more than
// wide_from columns go to the wide kernel, in the form `pair`, and the others to
// the narrow one in tiles of at most narrow_cols; fitted to all on a B200 at head
// size 128 and 8 kv heads, and used as it is elsewhere.  Of 105 shapes (1 to 64
// rows, one sequence of 500 to 16384 tokens or 8 and 32 of 4096; 4, 7 and 1 query
// heads a kv head) the choice is within 5 % of the best form for 101 at head size
// 128, 1.26 times it at worst (33 rows of 7 heads at 16384 tokens: 48 us, 38 in
// pairs), and for 96 at head size 64, 2.6 times it at worst (the same on 2 kv
// heads: 59 us, 23 in tiles of 16).  Smaller tiles unpack the cache more often,
// by code that is shorter and in more CTAs: measured / expected for 20 columns of
// one sequence of 2048 tokens in tiles of 8, 16, 24 columns 12 / 10, 13 / 14,
// 15 / 16 us, of 32 sequences of 4096 tokens 120 / 145, 109 / 110, 83 / 82.
// Wide, 32 sequences of 4096 tokens: 64 columns 143 / 140, in pairs 130 / 134;
// 256 columns 180 / 182, in pairs 252 / 251; one of 2048: 64 columns 24 / 26, in
// pairs 25 / 28, 256 29 / 27, in pairs 24 / 25.  A round is a 128-token stage in
// every resident CTA.
double attend_us(const spec_kv4_batch* b, const spec_kv4_step* s, int wide_from, bool pair, int narrow_cols) {
  static const double kCall[5] = {0, 8, 12.6, 15, 21}, kRound[5] = {0, 3.2, 2.55, 2.35, 2.86};  // narrow, by 8-column tiles
  const Cache& c = *b->c;
  const int G = c.d.n_heads / c.d.n_kv_heads, wide_cols = pair ? kPairCols : kWideCols;
  double narrow = 0, wide = 0, slowest = 0;
  int64_t tiles = 0;
  int nt = 0;
  for (int q = 0; q < s->n_seqs; ++q) {
    const int64_t cols = (int64_t)s->n_rows[q] * G, st = (s->kv_len[q] + s->n_rows[q] + kStageTokens - 1) / kStageTokens;
    if (!cols) continue;
    if (cols > wide_from) {
      const int64_t n = (cols + wide_cols - 1) / wide_cols;
      const double round = pair ? 2.12 : cols <= kWideCols / 2 ? 2.25 : 3.0;
      wide += (double)(n * st * c.d.n_kv_heads) * round;
      if (pair) slowest = 3.0;  // a stage alone
      else if (round > slowest) slowest = round;
      tiles += n * c.d.n_kv_heads;
    } else {
      const int size = narrow_tile(cols, narrow_cols);
      narrow += (double)((cols + size - 1) / size * st * c.d.n_kv_heads);
      if (size / 8 > nt) nt = size / 8;
    }
  }
  double us = 0;
  if (nt) us += kCall[nt] + kRound[nt] * narrow / ((double)b->sms * attend_ctas_per_sm(nt));
  if (tiles) {
    const double parts = (double)b->sms / (double)tiles;  // a tile's, to be joined
    us += (pair ? 15.5 : 14) + (wide / b->sms > slowest ? wide / b->sms : slowest) +
          0.55 * (parts < 1 ? 0 : parts > 18 ? 18 : parts);
  }
  return us;
}

// From how many columns a sequence goes to the wide kernel, that one's form and
// the narrow one's tiles: the best of a few, or what SPEC_B200_KV4_WIDE_FROM,
// SPEC_B200_KV4_WIDE_PAIR and SPEC_B200_KV4_NARROW_COLS said when the batch was made.
int choose_wide_from(const spec_kv4_batch* b, const spec_kv4_step* s, bool* pair, int* narrow_cols) {
  int best = 0;
  double least = 1e300;
  for (const int from : {INT_MAX, 128, 64, kMaxCols})
    for (const bool form : {false, true}) {
      if (b->wide_pair >= 0 && form != (b->wide_pair > 0)) continue;
      const int limit = b->wide_from >= 0 ? b->wide_from : from;
      for (const int most : kNarrowCols) {
        if (b->force_cols > 0 && most != b->force_cols) continue;
        const double us = attend_us(b, s, limit, form, most);
        if (us < least) least = us, best = limit, *pair = form, *narrow_cols = most;
      }
    }
  return best;
}

// Cuts the step's attention into units: per (sequence, kv head, tile of
// columns) the 128-token stages its rows see, then those stages, laid end to
// end, into runs of equal cost, one a CTA.  Sequences of more than wide_from
// columns go to the wide kernel, which takes kWideCols of them a unit, or in
// pairs of stages kPairCols.
void schedule(spec_kv4_batch* b, const spec_kv4_step* s, bool wide, int wide_from, bool pair) {
  const Cache& c = *b->c;
  Schedule& out = wide ? b->wide : b->narrow;
  const int G = c.d.n_heads / c.d.n_kv_heads, P = c.d.page_tokens;
  b->tiles.clear();
  b->runs.clear();
  b->joins.clear();
  b->cuts.clear();
  out.order.clear();
  out.n_ctas = out.n_parts = out.n_groups = out.n_units = out.n_joins = 0;
  out.nt = 1;
  int64_t stages = 0;
  int row0 = 0, table = 0;
  for (int q = 0; q < s->n_seqs; ++q) {
    const int n = s->kv_len[q], m = s->n_rows[q], cols = m * G;
    const int size = !wide ? narrow_tile(cols, b->narrow_cols) : pair ? kPairCols : kWideCols;
    for (int h = 0; h < c.d.n_kv_heads && (cols > wide_from) == wide; ++h)
      for (int c0 = 0; c0 < cols; c0 += size) {
        Unit u{};
        u.kvh = h;
        u.row0 = row0;
        u.col0 = c0;
        u.n_cols = cols - c0 < size ? cols - c0 : size;
        u.kv_len = n;
        u.kv_end = s->masks ? n + m : n + (c0 + u.n_cols - 1) / G + 1;
        u.sure = s->masks ? n : n + c0 / G + 1;
        u.st1 = (u.kv_end + kStageTokens - 1) / kStageTokens;
        u.table = table;
        stages += u.st1;
        if ((u.n_cols + 7) / 8 > out.nt) out.nt = (u.n_cols + 7) / 8;
        b->tiles.push_back(u);
      }
    row0 += m;
    table += (n + m + P - 1) / P;
  }
  if (b->tiles.empty()) return;
  const int64_t slots = (int64_t)b->sms * (wide ? 1 : attend_ctas_per_sm(out.nt));
  // A unit costs its stages and kUnitCost more (queries in, states joined and
  // out).  Either every CTA gets one unit, each tile cut into equal parts of at
  // most `len` stages; or the tiles are laid end to end and cut where the
  // running cost passes a CTA's share.  The first does no unit twice a CTA, the
  // second wastes no CTA where lengths differ: the smaller largest cost wins.
  int64_t longest = 0;
  for (const Unit& u : b->tiles) longest = u.st1 > longest ? u.st1 : longest;
  int64_t lo = 1, len = longest;
  const auto count = [&](int64_t l) {
    int64_t n = 0;
    for (const Unit& u : b->tiles) n += (u.st1 + l - 1) / l;
    return n;
  };
  const bool fits = (int64_t)b->tiles.size() <= slots;
  while (fits && lo < len) {
    const int64_t mid = (lo + len) / 2;
    if (count(mid) <= slots) len = mid;
    else lo = mid + 1;
  }
  const int64_t cost = stages + kUnitCost * ((int64_t)b->tiles.size() + slots);
  const bool even = fits && (len + kUnitCost - 1) * slots <= cost;
  // Past kFanIn parts a tile's states are joined in two rounds; a longer run of
  // up to two stages costs less.
  const int64_t one_round = (longest + kFanIn - 1) / kFanIn;
  if (!wide && len < one_round && one_round <= len + 2) len = one_round;
  int64_t spent = 0;
  int cta = 0;
  b->cuts.push_back(0);
  const auto close = [&] {
    if (b->cuts.back() != (int)b->runs.size()) b->cuts.push_back((int)b->runs.size());
    ++cta;
  };
  for (Unit u : b->tiles) {
    const int end = u.st1;
    const size_t first = b->runs.size();
    const int64_t n_even = (end + len - 1) / len;
    for (int at = 0, i = 0; at < end; ++i) {
      int64_t take;
      if (even) {
        take = (int64_t)end * (i + 1) / n_even - at;  // stages x parts pass 32 bits
      } else {
        // What is left of this CTA's share; at least a stage.
        const int64_t share = cost * (cta + 1) / slots;
        int64_t left = share - spent - kUnitCost;
        if (left < 1 && b->cuts.back() != (int)b->runs.size() && cta + 1 < slots) {
          close();
          left = cost * (cta + 1) / slots - spent - kUnitCost;
        }
        take = left < 1 ? 1 : left;
        if (cta + 1 >= slots || take > end - at) take = end - at;
      }
      u.st0 = at;
      u.st1 = at + (int)take;
      u.part = (int)(b->runs.size() - first);
      b->runs.push_back(u);
      at += (int)take;
      spent += take + kUnitCost;
      if (even || (spent >= cost * (cta + 1) / slots && cta + 1 < slots)) close();
    }
    const int parts = (int)(b->runs.size() - first);
    for (size_t i = first; i < b->runs.size(); ++i) {
      b->runs[i].n_parts = parts;
      b->runs[i].part0 = out.n_parts;
      b->runs[i].group = out.n_groups;
    }
    if (wide) {
      if (parts > 1) out.n_parts += parts, b->joins.push_back(b->runs.back());
      continue;
    }
    for (int n = parts; n > 1;) {
      out.n_parts += n;
      n = (n + kFanIn - 1) / kFanIn;
      out.n_groups += n;
    }
  }
  close();
  out.n_ctas = (int)b->cuts.size() - 1;
  out.order.resize(b->runs.size());
  int at = out.n_ctas;
  for (int i = 0; i < out.n_ctas; ++i) {
    const int first = b->cuts[i], n = b->cuts[i + 1] - first;
    for (int k = 0; k < n; ++k) {
      Unit& u = k == 0 ? out.order[i] : out.order[at + k - 1];
      u = b->runs[first + k];
      u.next = at;
      u.last = at + n - 1;
    }
    at += n - 1;
  }
  out.n_units = (int)out.order.size();
  out.n_joins = (int)b->joins.size();
  out.order.insert(out.order.end(), b->joins.begin(), b->joins.end());
}

int plan(spec_kv4_batch* b, const spec_kv4_step* s, cudaStream_t stream) {
  const Cache& c = *b->c;
  const int P = c.d.page_tokens;
  if (s->n_seqs < 0 || (s->n_seqs > 0 && (!s->kv_len || !s->n_rows || !s->page_table || s->table_stride < 1)))
    return fail(SPEC_ERR_INVALID, "spec_kv4_plan: null array or negative count");
  // Lengths.
  int64_t rows = 0, pages = 0;
  for (int i = 0; i < s->n_seqs; ++i) {
    const int64_t n = s->kv_len[i], m = s->n_rows[i];
    if (n < 0 || m < 0 || n + m > (int64_t)s->table_stride * P || n + m > INT_MAX - 1024)
      return fail(SPEC_ERR_INVALID, "spec_kv4_plan: sequence %d: %lld tokens and %lld rows do not fit %d pages of %d", i,
                  (long long)n, (long long)m, s->table_stride, P);
    if (s->masks && m > 64)
      return fail(SPEC_ERR_UNSUPPORTED, "spec_kv4_plan: sequence %d: masks cover at most 64 rows, got %lld", i,
                  (long long)m);
    rows += m;
    pages += (n + m + P - 1) / P;
  }
  if (rows > (1 << 24) || rows * (c.d.n_heads / c.d.n_kv_heads) > (1 << 30))
    return fail(SPEC_ERR_INVALID, "spec_kv4_plan: %lld rows (at most 2^24, and 2^30 with the query heads of a kv head)",
                (long long)rows);
  if (pages > (INT64_C(1) << 28)) return fail(SPEC_ERR_INVALID, "spec_kv4_plan: page tables of %lld entries", (long long)pages);
  // Pages: inside the pool, and a page that is written is listed once.
  b->seen.resize(c.d.n_pages, 0);
  int rc = SPEC_OK, done = 0;
  for (; done < s->n_seqs && rc == SPEC_OK; ++done) {
    const int32_t* t = s->page_table + (int64_t)done * s->table_stride;
    const int n = s->kv_len[done], m = s->n_rows[done], np = (n + m + P - 1) / P, w0 = m ? n / P : np;
    for (int i = 0; i < np; ++i) {
      if (t[i] < 0 || t[i] >= c.d.n_pages) {
        rc = fail(SPEC_ERR_INVALID, "spec_kv4_plan: sequence %d lists page %d of a pool of %d", done, t[i], c.d.n_pages);
        break;
      }
      uint8_t& f = b->seen[t[i]];
      if (i >= w0 ? f != 0 : f == 2) {
        rc = fail(SPEC_ERR_INVALID, "spec_kv4_plan: page %d is written by one sequence and listed again", t[i]);
        break;
      }
      f = i >= w0 ? 2 : 1;
    }
  }
  for (int q = 0; q < done; ++q) {
    const int32_t* t = s->page_table + (int64_t)q * s->table_stride;
    const int np = (s->kv_len[q] + s->n_rows[q] + P - 1) / P;
    for (int i = 0; i < np; ++i)
      if (t[i] >= 0 && t[i] < c.d.n_pages) b->seen[t[i]] = 0;
  }
  if (rc != SPEC_OK) return rc;
  int min_pos = INT_MAX, max_pos = -1, max_src = -1;
  for (int64_t r = 0; r < rows; ++r) {
    if (s->src_rows) {
      if (s->src_rows[r] < 0) return fail(SPEC_ERR_INVALID, "spec_kv4_plan: src_rows[%lld] is negative", (long long)r);
      if (s->src_rows[r] > max_src) max_src = s->src_rows[r];
    }
  }
  if (!s->src_rows) max_src = (int)rows - 1;

  b->planned = false;
  const int wide_from = choose_wide_from(b, s, &b->pair, &b->narrow_cols);
  schedule(b, s, false, wide_from, b->pair);
  schedule(b, s, true, wide_from, b->pair);
  // One block: rows, masks, pages, units.
  const size_t at_rows = 0, at_masks = at_rows + up(sizeof(RowDev) * rows), at_table = at_masks + (s->masks ? up(8 * rows) : 0),
               at_narrow = at_table + up(4 * pages), at_wide = at_narrow + up(sizeof(Unit) * b->narrow.order.size()),
               total = at_wide + up(sizeof(Unit) * b->wide.order.size());
  Turn turn{b, stream};
  cudaError_t e = turn.enter();
  if (e != cudaSuccess) return fail_cuda(e, "spec_kv4_plan");
  if (total > b->cap) {
    // The old plan's readers and its upload are done before it goes.
    if ((e = drain(b)) != cudaSuccess) return fail_cuda(e, "spec_kv4_plan");
    if (b->dev) cudaFree(b->dev);
    if (b->host) cudaFreeHost(b->host);
    b->dev = b->host = nullptr;
    b->cap = 0;
    const size_t cap = total + total / 2;
    if ((e = cudaMalloc(reinterpret_cast<void**>(&b->dev), cap)) != cudaSuccess) return fail_cuda(e, "spec_kv4_plan");
    if ((e = cudaMallocHost(reinterpret_cast<void**>(&b->host), cap)) != cudaSuccess) {
      cudaFree(b->dev);
      b->dev = nullptr;
      return fail_cuda(e, "spec_kv4_plan");
    }
    b->cap = cap;
  } else if (b->used && (e = cudaEventSynchronize(b->copied)) != cudaSuccess) {
    return fail_cuda(e, "spec_kv4_plan");  // the staging buffer is still being read
  }
  // The two kernels run one after the other and share the partial states.
  const size_t floats_narrow = b->narrow.n_parts * attend_part_floats(c.d.head_dim, b->narrow.nt),
               floats_wide = b->wide.n_parts * wide_part_floats(c.d.head_dim);
  if ((e = grow(b, &b->arrived, &b->arrived_cap, b->narrow.n_groups, true)) != cudaSuccess ||
      (e = grow(b, &b->parts, &b->parts_cap, floats_narrow > floats_wide ? floats_narrow : floats_wide, false)) != cudaSuccess)
    return fail_cuda(e, "spec_kv4_plan");
  RowDev* hr = reinterpret_cast<RowDev*>(b->host + at_rows);
  int* ht = reinterpret_cast<int*>(b->host + at_table);
  int r = 0, tp = 0;
  for (int q = 0; q < s->n_seqs; ++q) {
    const int32_t* t = s->page_table + (int64_t)q * s->table_stride;
    const int n = s->kv_len[q], m = s->n_rows[q], np = (n + m + P - 1) / P;
    memcpy(ht + tp, t, sizeof(int) * np);
    tp += np;
    for (int i = 0; i < m; ++i, ++r) {
      const int pos = s->positions ? s->positions[r] : n + i;
      if (pos < min_pos) min_pos = pos;
      if (pos > max_pos) max_pos = pos;
      hr[r] = RowDev{t[(n + i) / P], (n + i) % P, pos, s->src_rows ? s->src_rows[r] : r};
    }
  }
  if (s->masks) memcpy(b->host + at_masks, s->masks, 8 * (size_t)rows);
  for (Unit& u : b->narrow.order) {
    const int per = kStageTokens / P, first = u.st0 * per, n = (u.kv_end + P - 1) / P - first;
    for (int i = 0; i < per && i < n; ++i) u.pages[i] = ht[u.table + first + i];
  }
  if (b->narrow.n_ctas) memcpy(b->host + at_narrow, b->narrow.order.data(), sizeof(Unit) * b->narrow.order.size());
  if (b->wide.n_ctas) memcpy(b->host + at_wide, b->wide.order.data(), sizeof(Unit) * b->wide.order.size());
  if (total && (e = cudaMemcpyAsync(b->dev, b->host, total, cudaMemcpyHostToDevice, stream)) != cudaSuccess)
    return fail_cuda(e, "spec_kv4_plan");
  if ((e = cudaEventRecord(b->copied, stream)) != cudaSuccess) return fail_cuda(e, "spec_kv4_plan");
  if ((e = turn.leave()) != cudaSuccess) return fail_cuda(e, "spec_kv4_plan");
  b->n_rows = (int)rows;
  b->max_src = max_src;
  b->min_pos = rows ? min_pos : 0;
  b->max_pos = max_pos;
  b->has_src = s->src_rows != nullptr;
  b->rows = reinterpret_cast<const RowDev*>(b->dev + at_rows);
  b->masks = s->masks ? reinterpret_cast<const unsigned long long*>(b->dev + at_masks) : nullptr;
  b->table = reinterpret_cast<const int*>(b->dev + at_table);
  b->narrow.units = reinterpret_cast<const Unit*>(b->dev + at_narrow);
  b->wide.units = reinterpret_cast<const Unit*>(b->dev + at_wide);
  b->planned = true;
  return SPEC_OK;
}

}  // namespace

extern "C" {

int64_t spec_kv4_pool_bytes(const spec_kv4_desc* d) {
  const int rc = check_desc(d);
  if (rc != SPEC_OK) return -rc;
  return (int64_t)d->n_layers * d->n_pages * d->n_kv_heads * block_bytes(d->page_tokens, d->head_dim);
}

int spec_kv4_create(const spec_kv4_desc* d, void* pool_dev, int64_t pool_bytes, const float* cos_dev,
                    const float* sin_dev, int n_positions, spec_kv4** out) {
  if (!out) return fail(SPEC_ERR_INVALID, "spec_kv4_create: null argument");
  *out = nullptr;
  const int64_t need = spec_kv4_pool_bytes(d);
  if (need < 0) return (int)-need;
  if (!pool_dev || reinterpret_cast<uintptr_t>(pool_dev) % 128)
    return fail(SPEC_ERR_INVALID, "spec_kv4_create: the pool is null or not 128-byte aligned");
  if (pool_bytes < need)
    return fail(SPEC_ERR_INVALID, "spec_kv4_create: the pool has %lld bytes, %lld are needed", (long long)pool_bytes,
                (long long)need);
  if (!cos_dev != !sin_dev || (cos_dev && n_positions < 1))
    return fail(SPEC_ERR_INVALID, "spec_kv4_create: both rotation tables or none, of at least one position");
  if (reinterpret_cast<uintptr_t>(cos_dev) % 16 || reinterpret_cast<uintptr_t>(sin_dev) % 16)
    return fail(SPEC_ERR_INVALID, "spec_kv4_create: the rotation tables are not 16-byte aligned");
  try {
    auto h = std::make_unique<spec_kv4>();
    h->c = std::make_shared<Cache>();
    h->c->d = *d;
    h->c->pool = static_cast<uint8_t*>(pool_dev);
    h->c->cos = cos_dev;
    h->c->sin = sin_dev;
    h->c->n_positions = cos_dev ? n_positions : 0;
    *out = h.release();
  } catch (const std::bad_alloc&) {
    return fail(SPEC_ERR_OOM, "spec_kv4_create: out of host memory");
  }
  return SPEC_OK;
}

void spec_kv4_free(spec_kv4* c) { delete c; }

int spec_kv4_batch_create(spec_kv4* c, spec_kv4_batch** out) {
  if (!c || !out) return fail(SPEC_ERR_INVALID, "spec_kv4_batch_create: null argument");
  *out = nullptr;
  Current cur(c->c->d.device);
  if (cur.rc != SPEC_OK) return cur.rc;
  spec_kv4_batch* b = new (std::nothrow) spec_kv4_batch;
  if (!b) return fail(SPEC_ERR_OOM, "spec_kv4_batch_create: out of host memory");
  b->c = c->c;
  if (const char* v = getenv("SPEC_B200_KV4_WIDE_FROM")) b->wide_from = atoi(v);
  if (const char* v = getenv("SPEC_B200_KV4_WIDE_PAIR")) b->wide_pair = atoi(v);
  if (const char* v = getenv("SPEC_B200_KV4_NARROW_COLS"))
    for (const int most : kNarrowCols)
      if (atoi(v) == most) b->force_cols = most;
  cudaError_t e = cudaEventCreateWithFlags(&b->tail, cudaEventDisableTiming);
  if (e == cudaSuccess) e = cudaEventCreateWithFlags(&b->copied, cudaEventDisableTiming);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&b->sms, cudaDevAttrMultiProcessorCount, c->c->d.device);
  if (e == cudaSuccess) e = attend_setup();
  if (e == cudaSuccess) e = wide_setup();
  if (e == cudaSuccess) e = cudaMalloc(reinterpret_cast<void**>(&b->err), 16);
  if (e == cudaSuccess) e = cudaMemset(b->err, 0, 16);
  if (e != cudaSuccess) {
    release(b);
    delete b;
    return fail_cuda(e, "spec_kv4_batch_create");
  }
  *out = b;
  return SPEC_OK;
}

void spec_kv4_batch_free(spec_kv4_batch* b) {
  if (!b) return;
  Current cur(b->c->d.device);
  release(b);
  delete b;
}

int spec_kv4_plan(spec_kv4_batch* b, const spec_kv4_step* s, void* stream) {
  if (!b || !s) return fail(SPEC_ERR_INVALID, "spec_kv4_plan: null argument");
  Current cur(b->c->d.device);
  if (cur.rc != SPEC_OK) return cur.rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (capturing(st)) return fail(SPEC_ERR_UNSUPPORTED, "spec_kv4_plan: the stream is under capture");
  try {
    return plan(b, s, st);
  } catch (const std::bad_alloc&) {
    return fail(SPEC_ERR_OOM, "spec_kv4_plan: out of host memory");
  }
}

int spec_kv4_append(spec_kv4_batch* b, int layer, const spec_kv4_rows* q, const spec_kv4_rows* q_out,
                    const spec_kv4_rows* k, const spec_kv4_rows* v, const spec_kv4_rows* k_out,
                    const spec_kv4_rows* v_out, void* stream) {
  if (!b || !k || !v || !q != !q_out) return fail(SPEC_ERR_INVALID, "spec_kv4_append: null argument, or q without q_out");
  if (!b->planned) return fail(SPEC_ERR_INVALID, "spec_kv4_append: no plan");
  const Cache& c = *b->c;
  if (layer < 0 || layer >= c.d.n_layers)
    return fail(SPEC_ERR_INVALID, "spec_kv4_append: layer %d of %d", layer, c.d.n_layers);
  if (b->n_rows == 0) return SPEC_OK;
  const int64_t src = (int64_t)b->max_src + 1, n = b->n_rows;
  const int D = c.d.head_dim, hq = c.d.n_heads, hk = c.d.n_kv_heads;
  int rc = check_rows("k", k, src, hk, D, false);
  if (rc == SPEC_OK) rc = check_rows("v", v, src, hk, D, false);
  if (rc == SPEC_OK && q) rc = check_rows("q", q, src, hq, D, false);
  if (rc == SPEC_OK && q_out) rc = check_rows("q_out", q_out, n, hq, D, true);
  if (rc == SPEC_OK && k_out) rc = check_rows("k_out", k_out, n, hk, D, true);
  if (rc == SPEC_OK && v_out) rc = check_rows("v_out", v_out, n, hk, D, true);
  if (rc != SPEC_OK) return rc;
  if ((k_out && k_out->dtype != T_F16) || (v_out && v_out->dtype != T_F16))
    return fail(SPEC_ERR_INVALID, "spec_kv4_append: k_out and v_out are f16");
  if (q && q->ptr == q_out->ptr &&
      (b->has_src || q->dtype != q_out->dtype || q->row_stride != q_out->row_stride || q->head_stride != q_out->head_stride))
    return fail(SPEC_ERR_INVALID, "spec_kv4_append: q in place needs one type, one layout and no src_rows");
  if (c.cos && (b->min_pos < 0 || b->max_pos >= c.n_positions))
    return fail(SPEC_ERR_INVALID, "spec_kv4_append: positions %d to %d, the rotation tables have %d", b->min_pos, b->max_pos,
                c.n_positions);
  Current cur(c.d.device);
  if (cur.rc != SPEC_OK) return cur.rc;
  AppendParams p;
  p.pool = c.pool + layer * c.layer_bytes();
  p.cos = c.cos;
  p.sin = c.sin;
  p.rows = b->rows;
  p.q = to_rows(q);
  p.q_out = to_rows(q_out);
  p.k = to_rows(k);
  p.v = to_rows(v);
  p.k_out = to_rows(k_out);
  p.v_out = to_rows(v_out);
  p.n_rows = b->n_rows;
  p.n_heads = hq;
  p.n_kv = hk;
  p.P = c.d.page_tokens;
  p.rope_half = c.d.rope_half ? 1 : 0;
  p.wide_q = wide(q);
  p.wide_qo = wide(q_out);
  p.wide_k = wide(k);
  p.wide_v = wide(v);
  p.wide_ko = wide(k_out);
  p.wide_vo = wide(v_out);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Turn turn{b, st};
  cudaError_t e = turn.enter();
  if (e == cudaSuccess) e = launch_append(p, D, st);
  if (e == cudaSuccess) e = turn.leave();
  return e == cudaSuccess ? SPEC_OK : fail_cuda(e, "spec_kv4_append");
}

int spec_kv4_attend(spec_kv4_batch* b, int layer, const spec_kv4_rows* q, const spec_kv4_rows* out, float scale,
                    void* stream) {
  if (!b || !q || !out) return fail(SPEC_ERR_INVALID, "spec_kv4_attend: null argument");
  if (!b->planned) return fail(SPEC_ERR_INVALID, "spec_kv4_attend: no plan");
  const Cache& c = *b->c;
  if (layer < 0 || layer >= c.d.n_layers)
    return fail(SPEC_ERR_INVALID, "spec_kv4_attend: layer %d of %d", layer, c.d.n_layers);
  if (b->n_rows == 0) return SPEC_OK;
  const int D = c.d.head_dim;
  int rc = check_rows("q", q, b->n_rows, c.d.n_heads, D, false);
  if (rc == SPEC_OK) rc = check_rows("out", out, b->n_rows, c.d.n_heads, D, true);
  if (rc != SPEC_OK) return rc;
  if (q->dtype == T_F32) return fail(SPEC_ERR_UNSUPPORTED, "spec_kv4_attend: q is bf16 or f16");
  if (!(scale == scale) || scale - scale != 0.f) return fail(SPEC_ERR_INVALID, "spec_kv4_attend: scale is not finite");
  Current cur(c.d.device);
  if (cur.rc != SPEC_OK) return cur.rc;
  AttendParams p;
  p.pool = c.pool + layer * c.layer_bytes();
  p.table = b->table;
  p.masks = b->masks;
  p.parts = b->parts;
  p.err = b->err;
  p.q = to_rows(q);
  p.out = to_rows(out);
  p.scale = scale;
  p.wide_q = wide(q);
  p.wide_out = wide(out);
  p.n_heads = c.d.n_heads;
  p.n_kv = c.d.n_kv_heads;
  p.P = c.d.page_tokens;
  p.P_log2 = p.P == 16 ? 4 : p.P == 32 ? 5 : p.P == 64 ? 6 : 7;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Turn turn{b, st};
  cudaError_t e = turn.enter();
  if (e == cudaSuccess && b->wide.n_ctas) {
    p.units = b->wide.units;
    p.joins = b->wide.units + b->wide.n_units;
    p.n_joins = b->wide.n_joins;
    p.n_ctas = b->wide.n_ctas;
    e = launch_wide(p, D, b->pair, st);
  }
  if (e == cudaSuccess && b->narrow.n_ctas) {
    p.units = b->narrow.units;
    p.n_ctas = b->narrow.n_ctas;
    p.arrived = b->arrived;
    e = launch_attend(p, D, b->narrow.nt, st);
  }
  if (e == cudaSuccess) e = turn.leave();
  return e == cudaSuccess ? SPEC_OK : fail_cuda(e, "spec_kv4_attend");
}

int spec_kv4_status(spec_kv4_batch* b) {
  if (!b) return fail(SPEC_ERR_INVALID, "spec_kv4_status: null argument");
  Current cur(b->c->d.device);
  if (cur.rc != SPEC_OK) return cur.rc;
  const cudaError_t e = drain(b);
  if (e != cudaSuccess) return fail_cuda(e, "spec_kv4_status");
  char msg[256];
  const int rc = take_device_error(b->err, nullptr, msg, sizeof msg);
  if (rc != SPEC_OK) {
    set_thread_error(msg);
    // A call that gave up may have left arrivals behind.
    if (b->arrived) cudaMemset(b->arrived, 0, b->arrived_cap * sizeof(int));
    cudaDeviceSynchronize();
  }
  return rc;
}

}  // extern "C"
