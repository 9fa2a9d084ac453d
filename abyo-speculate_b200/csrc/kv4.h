// 4-bit paged KV cache: what the host planner (kv4.cpp) and the kernels
// (kv4_append.cu, kv4_attend.cu) share.  The byte layout of a page is
// documented at spec_kv4 in include/spec_b200.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace specb200 {
namespace kv4 {

enum : int { T_BF16 = 0, T_F16 = 1, T_F32 = 2 };

constexpr float kClamp = 20000.f;  // s = (hi - lo) * 16/15 and o = lo - s stay in f16 range
constexpr int kGroup = 32;         // channels that share a scale pair

// Byte offsets inside a block of P tokens of one kv head.
__host__ __device__ constexpr int k_scales_at(int P, int D) { return P * D / 2; }
__host__ __device__ constexpr int v_codes_at(int P, int D) { return P * D / 2 + P * D / 8; }
__host__ __device__ constexpr int v_scales_at(int P, int D) { return P * D + P * D / 8; }
__host__ __device__ constexpr int block_bytes(int P, int D) { return P * D + P * D / 4; }

// Offset of 32-byte piece `piece` of token j's V codes inside the V code area.
// A 128-byte line holds 2 (D = 128) or 4 (D = 64) tokens; the turn of its
// quarters spreads tokens 0, 2, 4, 6 over all banks, which is how the
// attention reads them.
__host__ __device__ constexpr int v_piece_at(int D, int j, int piece) {
  const int per = 256 / D;
  const int line = j / per;
  return line * 128 + 32 * (((j % per) * (D / 64) + piece) ^ (line % (D / 32)));
}

struct RowDev {
  int page, slot;  // where the row is stored: page id, token within the page
  int pos, src;    // rotation position, row of the input tensors
};

// Rows of heads (spec_kv4_rows).
struct Rows {
  void* ptr = nullptr;
  long long row_stride = 0, head_stride = 0;
  int dtype = 0;
};

struct AppendParams {
  uint8_t* pool;  // of the layer
  const float *cos, *sin;
  const RowDev* rows;
  Rows q, q_out, k, v, k_out, v_out;
  int n_rows, n_heads, n_kv, P, rope_half;
  int wide_q, wide_k, wide_v;  // 8 channels are aligned 16-byte accesses
  int wide_qo, wide_ko, wide_vo;
};
cudaError_t launch_append(const AppendParams& p, int head_dim, cudaStream_t s);

constexpr int kStageTokens = 128;  // tokens the attention's work is cut by
constexpr int kFanIn = 16;         // partial states joined at once
constexpr int kMaxCols = 32;       // (row, query head) columns of one unit
constexpr int kWideCols = 256;     // of one unit of the wide kernel
constexpr int kPairCols = 128;     // of one whose stages alternate between two accumulators

// A run of stages of one (sequence, kv head, column tile), done by one CTA.
struct alignas(16) Unit {
  int kvh;
  int row0;            // first row of the sequence
  int col0, n_cols;    // stacked columns (row * G + query head of the group)
  int st0, st1;        // 128-token stages
  int kv_len, kv_end;  // cached tokens; tokens any column of the tile sees
  int sure;            // tokens every column of it sees
  int table;           // the sequence's pages
  // Partial states of the tile: n_parts at part0, then ceil(n / kFanIn) more
  // a level; arrival counters likewise from `group` on.  n_parts == 1: none.
  int part0, part, n_parts;
  int group;
  int next, last;      // the CTA's next unit and one past its last
  int pages[8];        // pages of the first stage
};

struct AttendParams {
  const uint8_t* pool;  // of the layer
  const Unit* units;  // [n_ctas] first units of the CTAs, then the others
  const Unit* joins;  // wide kernel: a unit of every column tile that several CTAs share
  int n_joins;
  const int* table;
  const unsigned long long* masks;  // null: causal
  float* parts;
  int* arrived;
  unsigned* err;
  Rows q, out;
  float scale;
  int n_ctas, n_heads, n_kv, P, P_log2, wide_q, wide_out;
};
// nt: 8-column tiles a unit has at most.
cudaError_t launch_attend(const AttendParams& p, int head_dim, int nt, cudaStream_t s);
// Once per device, with it current, before the first launch.
cudaError_t attend_setup();
size_t attend_part_floats(int head_dim, int nt);
int attend_ctas_per_sm(int nt);
// The same for sequences of many columns, one CTA an SM.
// pair: units have at most kPairCols columns, and their stages alternate.
cudaError_t launch_wide(const AttendParams& p, int head_dim, bool pair, cudaStream_t s);
cudaError_t wide_setup();
size_t wide_part_floats(int head_dim);

}  // namespace kv4
}  // namespace specb200
