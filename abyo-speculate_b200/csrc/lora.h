// Low-rank adapters of many requests: what the host entry points (lora.cpp)
// and the kernels (lora.cu, lora_wide.cu, lora_tall.cu) share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace specb200 {
namespace lora {

enum : int { T_BF16 = 0, T_F16 = 1, T_F32 = 2 };

constexpr int kMaxRank = 128;
constexpr int kNarrowRows = 8;  // rows of a unit of the kernel for few rows: one n-tile of the products
constexpr int kWideRows = 32;   // of the one for many
constexpr int kTallRows = 128;  // and of the one for very many

// Rows of one adapter (-1: none) that one cluster takes.
struct Unit {
  int adapter, first, n_rows, pad;  // rows order[first ..]
  int row[kNarrowRows];             // the first of them
};

struct Params {
  const void *a, *b;  // of the adapters' type
  long long a_adapter, a_row, b_adapter, b_row;  // strides in elements
  const int* ranks;      // or null: all `rank`
  const float* scales;   // or null: 1
  const void* x;
  const void* y;
  void* out;
  long long x_row, y_row, out_row;
  const Unit* units;
  const int* order;
  int K, N, rank;
  int a_wide, b_wide, x_wide, y_wide, out_wide;  // 8 consecutive elements from a multiple of 8 on are aligned 16-byte accesses
};

// n_units units: of at most kNarrowRows rows (and those without an adapter) on
// clusters of `size` blocks, or of at most kWideRows.
cudaError_t launch_narrow(const Params& p, int type, bool x_f32, bool y_f32, int n_units, int size, cudaStream_t s);
cudaError_t launch_wide(const Params& p, int type, bool x_f32, bool y_f32, int n_units, int sms, cudaStream_t s);
// The same of at most kTallRows rows, x of the adapters' type; *taken: whether they were, or are left to units of
// kWideRows.  A device wait that gives up sets *err.
cudaError_t launch_tall(const Params& p, unsigned* err, int type, bool y_f32, int n_units, int sms, cudaStream_t s, bool* taken);

}  // namespace lora
}  // namespace specb200
