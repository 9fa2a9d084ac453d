// Sampling and verification over rows of logits of many sequences: what the
// host entry points (batch.cpp) and the kernels (batch_sample.cu) share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace specb200 {
namespace batch {

enum : int { T_BF16 = 0, T_F16 = 1, T_F32 = 2 };

// A row is cut into chunks of kChunk columns that start at multiples of 16
// bytes; the first may hold a few columns less.  Their number is a multiple of
// 8, the last ones may be empty.
constexpr int kChunk = 512;
inline int chunks_of(int vocab, int dtype) {
  const int per_vector = dtype == T_F32 ? 4 : 8;
  return (vocab + per_vector - 1 + 8 * kChunk - 1) / (8 * kChunk) * 8;
}

struct Rows {
  const void* logits;
  long long stride;    // elements
  const float* temps;  // per row, or null: `temp`
  float temp;
  const float* u;
  const int* drafts;   // chains: the tokens that the rows judge, and the draft's rows
  const float* q;
  long long q_stride;
  float2* seen;        // [n_rows]: the draft's probability of it, and the row's logit
  int n_rows, V, nch;
  float2* stats;  // [n_rows][nch]: largest logit, sum of exp((l - largest) / T)
  double* sums;   // [n_rows][nch]: sums of one row that a cluster works on
  int* drawn;     // [n_rows]: trees' drawn tokens
  int* path;      // [n_rows]: trees' paths, which start as -1 everywhere, or null
};

struct SampleParams {
  Rows r;
  float* probs;  // null: none
  long long probs_stride;
  int* tokens;
};

struct VerifyParams {
  Rows r;
  const int* row_start;  // [n_seqs + 1]
  int n_seqs;
  const int* tokens;     // drafts, or the trees' tokens
  const int* parents;    // trees
  const float* q;        // chains: draft probabilities
  long long q_stride;
  int *n_out, *next;
};

// The kernels are queued on `s`; the device is current.
cudaError_t launch_sample(const SampleParams& p, int dtype, int sms, cudaStream_t s);
cudaError_t launch_verify(const VerifyParams& p, int dtype, bool trees, int sms, cudaStream_t s);

}  // namespace batch
}  // namespace specb200
