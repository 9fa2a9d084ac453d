// Low-rank adapters of many requests: the plan of a step's rows, the C entry
// points and the checks of their arguments.  No state is kept.
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "host_call.h"
#include "lora.h"

using namespace specb200;
using namespace specb200::lora;

namespace {

constexpr int kPlanRows = 1 << 20;
// Which kernel takes an adapter's rows.  us in units of 8 / of 32 for (a) rank 16, 4096 to
// 4096 channels in bf16, (b) rank 64, 2048 to 8192, f32 rows, (c) rank 16, 4096 to 14336,
// f32 rows:
// - up to kNarrowMost rows in units of 8: 24 adapters of 16 rows 12 / 14, 24 / 41, 23 / 36;
// - more, while all rows make kFewUnits units of 8, likewise: 24 of 32 rows b 37 / 45, c 38 / 45;
//   one of 256 9 / 12, 22 / 26, 21 / 29.  16-bit rows only up to kFew16 (known when the plan is
//   used, as what follows is): 6 of 64 rows a 10.5 / 14, 16 of 32 18 / 15.5.  f32 rows up to kSomeUnits
//   as well those of at most 64 rows, where units of 32 are more than kHalvesMost:
//   24 of 48 b 66 / 74, c 68 / 72.  Not where A and B, read again for every 8 rows, are more than kAgainMost times
//   the rows: 24 of 32, rank 64, 14336 to 4096 in bf16 61 / 32.5.  Others are slower so:
//   16 of 64 rows 30 / 20, 66 / 44, 68 / 60;
// - of more than kTallMin rows, kTallFrom units of 128, where the device's SMs are used
//   well by these (lora_tall.cu), which fewer of them do not.
constexpr int kNarrowMost = 16;
constexpr int kFewUnits = 111;   // four blocks a cluster, three an SM
constexpr int kFew16 = 55;       // eight
constexpr int kSomeUnits = 222;  // two
constexpr int kAgainMost = 4;
constexpr int kHalvesMost = 36;  // as many clusters of 8 blocks as a B200 holds, two an SM
constexpr int kTallFrom = 10;
constexpr int kTallMin = 64;

// Layout of a plan: units (of adapters of very many rows by 128, the same by 32,
// those of other adapters of many rows, those of few, rows without one, rows of the
// second and third kind by 8), then the rows in their order, then the word of the
// device's waits.
int64_t plan_bytes(int64_t n_rows) { return n_rows * (int64_t)(sizeof(Unit) + sizeof(int)) + 16; }

struct Matrix {
  const char* name;
  const void* ptr;
  int64_t outer, row;  // strides
};

// Whether 8 elements from any multiple of 8 on are aligned 16-byte accesses.
bool wide(const void* p, int64_t row, int64_t outer, int size) {
  return !misaligned(p, 16) && row * size % 16 == 0 && outer * size % 16 == 0;
}

// Blocks a cluster of units of 8 rows: 8, fewer where three an SM are not enough.
// Three blocks an SM at once; a single block a unit only for many: 256 units of 8
// rows (c above) 141 us, 116 in clusters of two, a few of which start late.
int narrow_cluster(int n, int sms) {
  int size = 8;
  while (size > 1 && (int64_t)n * size > (int64_t)sms * 3) size /= 2;
  return size == 1 && (int64_t)n * 2 <= (int64_t)sms * 5 ? 2 : size;
}

unsigned* status_of(const spec_lora_plan* plan) {
  const uint8_t* b = static_cast<const uint8_t*>(plan->device_copy);
  return const_cast<unsigned*>(reinterpret_cast<const unsigned*>(b + (size_t)plan->n_rows * (sizeof(Unit) + sizeof(int))));
}

int check_plan_shape(const char* what, int64_t n_rows) {
  if (n_rows < 0 || n_rows > kPlanRows) return fail(SPEC_ERR_INVALID, "%s: %lld rows, 0 to %d are taken", what, (long long)n_rows, kPlanRows);
  return SPEC_OK;
}

int make_plan(const char* what, const int32_t* adapters, int n_rows, int n_adapters, void* buf, spec_lora_plan* out) {
  for (int i = 0; i < n_rows; ++i)
    if (adapters[i] < -1 || adapters[i] >= n_adapters)
      return fail(SPEC_ERR_INVALID, "%s: row %d has adapter %d of %d (-1: none)", what, i, adapters[i], n_adapters);
  std::vector<int> order(n_rows);
  for (int i = 0; i < n_rows; ++i) order[i] = i;
  // By adapter, rows in their order; rows without one last.
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return (unsigned)adapters[x] < (unsigned)adapters[y]; });
  // An adapter's rows in units of equal size; rows without one are copied one by
  // one.  Runs of rows that two kernels can take, by x's type or the bank's size, are
  // cut for both.
  struct Run {
    int adapter, begin, end;
  };
  std::vector<Run> runs;
  int64_t halves = 0, tall = 0, eighths = 0, near = 0;  // units of 32, 128 and 8 rows; of 8 of runs of at most 64
  for (int i = 0; i < n_rows;) {
    int e = i;
    while (e < n_rows && adapters[order[e]] == adapters[order[i]]) ++e;
    runs.push_back(Run{adapters[order[i]], i, e});
    const int64_t n = adapters[order[i]] >= 0 ? (e - i + kNarrowRows - 1) / kNarrowRows : 0;
    eighths += n;
    if (e - i <= kTallMin) near += n;
    if (adapters[order[i]] >= 0 && e - i > kNarrowMost) {
      halves += (e - i + kWideRows - 1) / kWideRows;
      if (e - i > kTallMin) tall += (e - i + kTallRows - 1) / kTallRows;
    }
    i = e;
  }
  const bool few = eighths <= kFewUnits, some = few || (halves > kHalvesMost && near <= kSomeUnits);
  std::vector<Unit> units[5], mid_wide, mid;
  auto cut = [&](std::vector<Unit>& to, const Run& r, int most) {
    const int rows = r.end - r.begin, n = (rows + most - 1) / most;
    for (int k = 0; k < n; ++k) {
      const int at = r.begin + (int)((int64_t)rows * k / n), end = r.begin + (int)((int64_t)rows * (k + 1) / n);
      Unit u{r.adapter, at, end - at, 0, {}};
      for (int j = 0; j < kNarrowRows && at + j < end; ++j) u.row[j] = order[at + j];
      to.push_back(u);
    }
  };
  for (const Run& r : runs) {
    const int rows = r.end - r.begin;
    const bool big = r.adapter >= 0 && rows > kTallMin && tall >= kTallFrom;
    if (big) cut(units[0], r, kTallRows);
    if (r.adapter < 0) cut(units[4], r, 1);
    else if (rows <= kNarrowMost) cut(units[3], r, kNarrowRows);
    else if (few || (some && rows <= kTallMin)) cut(big ? units[1] : mid_wide, r, kWideRows), cut(mid, r, kNarrowRows);
    else cut(units[big ? 1 : 2], r, kWideRows);
  }
  units[2].insert(units[2].end(), mid_wide.begin(), mid_wide.end());
  uint8_t* b = static_cast<uint8_t*>(buf);
  if (n_rows) {
    size_t at = 0;
    for (const auto& v : units) {
      if (!v.empty()) memcpy(b + at, v.data(), v.size() * sizeof(Unit));
      at += v.size() * sizeof(Unit);
    }
    // Behind them, at most a row's worth of units a row in all.
    if (!mid.empty()) memcpy(b + at, mid.data(), mid.size() * sizeof(Unit));
    memcpy(b + (size_t)n_rows * sizeof(Unit), order.data(), (size_t)n_rows * sizeof(int));
  }
  memset(b + (size_t)n_rows * (sizeof(Unit) + sizeof(int)), 0, 16);
  *out = spec_lora_plan{};
  out->n_rows = n_rows;
  out->n_adapters = n_adapters;
  out->n_tall = (int)units[0].size();
  out->n_big = (int)units[1].size();
  out->n_wide = (int)units[2].size();
  out->n_narrow = (int)units[3].size();
  out->n_bare = (int)units[4].size();
  out->n_mid = (int)mid.size();
  out->n_mid_wide = (int)mid_wide.size();
  out->mid_all = few;
  return SPEC_OK;
}

}  // namespace

extern "C" {

int64_t spec_lora_plan_bytes(int64_t n_rows) {
  const int rc = check_plan_shape("spec_lora_plan_bytes", n_rows);
  return rc == SPEC_OK ? plan_bytes(n_rows) : -rc;
}

int spec_lora_plan_make(const int32_t* adapters, int n_rows, int n_adapters, void* buf, int64_t buf_bytes,
                        spec_lora_plan* out) {
  const char* what = "spec_lora_plan_make";
  if (!out || !buf || (n_rows > 0 && !adapters)) return fail(SPEC_ERR_INVALID, "%s: null argument", what);
  const int rc = check_plan_shape(what, n_rows);
  if (rc != SPEC_OK) return rc;
  if (n_adapters < 0) return fail(SPEC_ERR_INVALID, "%s: %d adapters", what, n_adapters);
  if (buf_bytes < plan_bytes(n_rows))
    return fail(SPEC_ERR_INVALID, "%s: a buffer of %lld bytes, %lld are needed", what, (long long)buf_bytes,
                (long long)plan_bytes(n_rows));
  try {
    return make_plan(what, adapters, n_rows, n_adapters, buf, out);
  } catch (const std::bad_alloc&) {
    return fail(SPEC_ERR_OOM, "%s: out of host memory", what);
  }
}

int spec_lora_apply(const spec_lora_bank* b, const spec_lora_plan* plan, const spec_lora_rows* x, const spec_lora_rows* y,
                    const spec_lora_rows* out, void* stream) {
  const char* what = "spec_lora_apply";
  if (!b || !plan || !x || !y || !out) return fail(SPEC_ERR_INVALID, "%s: null argument", what);
  if (b->dtype != T_BF16 && b->dtype != T_F16) return fail(SPEC_ERR_UNSUPPORTED, "%s: adapters of type %d (bf16 and f16 are built)", what, b->dtype);
  if (b->k < 1 || b->n < 1 || b->k > (1 << 24) || b->n > (1 << 24) || b->n_adapters < 0)
    return fail(SPEC_ERR_INVALID, "%s: %d adapters of %d to %d channels", what, b->n_adapters, b->k, b->n);
  if (b->rank < 0 || b->rank > kMaxRank) return fail(SPEC_ERR_UNSUPPORTED, "%s: rank %d (up to %d is built)", what, b->rank, kMaxRank);
  if (b->device < 0) return fail(SPEC_ERR_INVALID, "%s: device %d", what, b->device);
  if (plan->n_rows < 0 || plan->n_rows > kPlanRows || plan->n_wide < 0 || plan->n_narrow < 0 || plan->n_bare < 0 || plan->n_tall < 0 || plan->n_big < 0 ||
      plan->n_mid < 0 || plan->n_mid_wide < 0 || plan->n_mid_wide > plan->n_wide ||
      (int64_t)plan->n_tall + plan->n_big + plan->n_wide + plan->n_narrow + plan->n_bare + plan->n_mid > plan->n_rows)
    return fail(SPEC_ERR_INVALID, "%s: not a plan", what);
  if (plan->n_adapters > b->n_adapters)
    return fail(SPEC_ERR_INVALID, "%s: a plan for %d adapters, the bank has %d", what, plan->n_adapters, b->n_adapters);
  if (plan->n_rows == 0) return SPEC_OK;
  if (!plan->device_copy || misaligned(plan->device_copy, 16))
    return fail(SPEC_ERR_INVALID, "%s: the plan's copy on the device is missing or not aligned to 16 bytes", what);
  for (const spec_lora_rows* r : {x, y, out}) {
    const char* name = r == x ? "x" : r == y ? "y" : "out";
    if (!r->ptr) return fail(SPEC_ERR_INVALID, "%s: %s has no data", what, name);
    if (r->dtype != b->dtype && r->dtype != T_F32)
      return fail(SPEC_ERR_UNSUPPORTED, "%s: %s has type %d (f32 and the adapters' type are built)", what, name, r->dtype);
    if (r->n_rows < plan->n_rows)
      return fail(SPEC_ERR_INVALID, "%s: %s has %lld rows, the plan %d", what, name, (long long)r->n_rows, plan->n_rows);
    if (r->row_stride < 0 || r->row_stride > kMaxStride)
      return fail(SPEC_ERR_INVALID, "%s: %s has rows %lld apart", what, name, (long long)r->row_stride);
    if (misaligned(r->ptr, r->dtype == T_F32 ? 4 : 2))
      return fail(SPEC_ERR_INVALID, "%s: %s is not aligned to its element size", what, name);
  }
  if (y->dtype != out->dtype) return fail(SPEC_ERR_INVALID, "%s: y and out have types %d and %d", what, y->dtype, out->dtype);
  if (plan->n_rows > 1 && out->row_stride < b->n)
    return fail(SPEC_ERR_INVALID, "%s: rows of out overlap (%lld apart, %d wide)", what, (long long)out->row_stride, b->n);
  const bool in_place = y->ptr == out->ptr;
  if (in_place && plan->n_rows > 1 && y->row_stride != out->row_stride)
    return fail(SPEC_ERR_INVALID, "%s: y in place needs one row stride", what);
  const int64_t xs = x->dtype == T_F32 ? 4 : 2, ys = y->dtype == T_F32 ? 4 : 2;
  if (rows_meet(x->ptr, x->row_stride * xs, b->k * xs, out->ptr, out->row_stride * ys, b->n * ys, plan->n_rows) ||
      (!in_place && rows_meet(y->ptr, y->row_stride * ys, b->n * ys, out->ptr, out->row_stride * ys, b->n * ys, plan->n_rows)))
    return fail(SPEC_ERR_INVALID, "%s: out shares memory with x, or with other elements of y", what);
  if (plan->n_big || plan->n_wide || plan->n_narrow) {
    if ((b->rank > 0 && (!b->a || !b->b)) || misaligned(b->a, 2) || misaligned(b->b, 2) || misaligned(b->ranks, 4) || misaligned(b->scales, 4))
      return fail(SPEC_ERR_INVALID, "%s: a pointer of the bank is null or not aligned to its element size", what);
    for (const int64_t s : {b->a_adapter_stride, b->a_row_stride, b->b_adapter_stride, b->b_row_stride})
      if (s < 0 || s > kMaxStride) return fail(SPEC_ERR_INVALID, "%s: a stride of the bank is outside [0, 2^40]", what);
  }
  Current cur(b->device, what);
  if (cur.rc != SPEC_OK) return cur.rc;
  Params p{};
  p.a = b->a;
  p.b = b->b;
  p.a_adapter = b->a_adapter_stride;
  p.a_row = b->a_row_stride;
  p.b_adapter = b->b_adapter_stride;
  p.b_row = b->b_row_stride;
  p.ranks = b->ranks;
  p.scales = b->scales;
  p.x = x->ptr;
  p.y = y->ptr;
  p.out = out->ptr;
  p.x_row = x->row_stride;
  p.y_row = y->row_stride;
  p.out_row = out->row_stride;
  const Unit* units = static_cast<const Unit*>(plan->device_copy);
  p.order = reinterpret_cast<const int*>(units + plan->n_rows);
  p.K = b->k;
  p.N = b->n;
  p.rank = b->rank;
  p.a_wide = wide(b->a, b->a_row_stride, b->a_adapter_stride, 2);
  p.b_wide = wide(b->b, b->b_row_stride, b->b_adapter_stride, 2);
  p.x_wide = wide(x->ptr, x->row_stride, 0, x->dtype == T_F32 ? 4 : 2);
  p.y_wide = wide(y->ptr, y->row_stride, 0, y->dtype == T_F32 ? 4 : 2);
  p.out_wide = wide(out->ptr, out->row_stride, 0, y->dtype == T_F32 ? 4 : 2);
  int sms = 0;
  cudaError_t e = multiprocessors(b->device, &sms);
  const bool x_f32 = x->dtype == T_F32, y_f32 = y->dtype == T_F32;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Rows that units of 8 can take as well: do they?
  const bool few = x_f32 || (plan->mid_all && (int64_t)plan->n_narrow + plan->n_mid <= kFew16);
  const bool mid = plan->n_mid && few && (int64_t)b->rank * (b->k + b->n) * 2 <= (int64_t)kAgainMost * kNarrowRows *
                                      (b->k * (x_f32 ? 4LL : 2LL) + 2 * b->n * (y_f32 ? 4LL : 2LL));
  const bool rest = !(mid && plan->mid_all);  // there are others
  bool taken = false;
  p.units = units;
  if (e == cudaSuccess && rest && plan->n_tall && !x_f32)
    e = launch_tall(p, status_of(plan), b->dtype, y_f32, plan->n_tall, sms, s, &taken);
  p.units = units + plan->n_tall + (taken ? plan->n_big : 0);
  const int wide = rest ? plan->n_wide - (mid ? plan->n_mid_wide : 0) + (taken ? 0 : plan->n_big) : 0;
  if (e == cudaSuccess) e = launch_wide(p, b->dtype, x_f32, y_f32, wide, sms, s);
  p.units = units + plan->n_tall + plan->n_big + plan->n_wide;
  // Units of 8 rows, rows without an adapter and the units behind them: at once, but
  // for rows in place, which have nothing to copy.
  const int bare = plan->n_bare, again = mid ? plan->n_mid : 0;
  const int n = in_place && bare ? plan->n_narrow : plan->n_narrow + bare + again;
  if (e == cudaSuccess) e = launch_narrow(p, b->dtype, x_f32, y_f32, n, narrow_cluster(n, sms), s);
  if (in_place && bare && again && e == cudaSuccess) {
    p.units += plan->n_narrow + bare;
    e = launch_narrow(p, b->dtype, x_f32, y_f32, again, narrow_cluster(again, sms), s);
  }
  return e == cudaSuccess ? SPEC_OK : fail_cuda(e, what);
}

int spec_lora_status(const spec_lora_plan* plan, int device, void* stream) {
  const char* what = "spec_lora_status";
  if (!plan || plan->n_rows < 0 || plan->n_rows > kPlanRows || !plan->device_copy || misaligned(plan->device_copy, 16) || device < 0)
    return fail(SPEC_ERR_INVALID, "%s: not a plan on a device", what);
  Current cur(device, what);
  if (cur.rc != SPEC_OK) return cur.rc;
  char msg[256];
  const int rc = take_device_error(status_of(plan), static_cast<cudaStream_t>(stream), msg, sizeof msg);
  if (rc != SPEC_OK) set_thread_error(msg);
  return rc;
}

}  // extern "C"
