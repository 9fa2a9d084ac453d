// Sampling and verification of a batch: the C entry points and the checks of
// their arguments.  No state is kept: what a call
// needs beyond its inputs is a workspace of the caller's.
#include "batch.h"
#include "host_call.h"

using namespace specb200;
using namespace specb200::batch;

namespace {

size_t up(size_t n) { return (n + 255) / 256 * 256; }

int check_shape(const char* what, int64_t n_rows, int vocab, int dtype) {
  if (dtype < T_BF16 || dtype > T_F32) return fail(SPEC_ERR_INVALID, "%s: logits have type %d", what, dtype);
  if (vocab < 1 || vocab > SPEC_BATCH_MAX_VOCAB)
    return fail(SPEC_ERR_INVALID, "%s: vocabulary of %d, 1 to %d are taken", what, vocab, SPEC_BATCH_MAX_VOCAB);
  if (n_rows < 0 || n_rows > SPEC_BATCH_MAX_ROWS)
    return fail(SPEC_ERR_INVALID, "%s: %lld rows, 0 to %d are taken", what, (long long)n_rows, SPEC_BATCH_MAX_ROWS);
  return SPEC_OK;
}

int64_t workspace_bytes(int64_t n_rows, int vocab, int dtype) {
  const size_t cells = (size_t)n_rows * chunks_of(vocab, dtype);
  return (int64_t)(up(cells * sizeof(float2)) + up(cells * sizeof(double)) + up((size_t)n_rows * sizeof(float2)));
}

int check_logits(const char* what, const spec_batch_logits* l) {
  if (!l) return fail(SPEC_ERR_INVALID, "%s: null argument", what);
  int rc = check_shape(what, l->n_rows, l->vocab, l->dtype);
  if (rc != SPEC_OK) return rc;
  if (l->device < 0) return fail(SPEC_ERR_INVALID, "%s: device %d", what, l->device);
  if (l->n_rows == 0) return SPEC_OK;
  if (!l->logits || !l->uniforms || !l->workspace) return fail(SPEC_ERR_INVALID, "%s: null logits, uniforms or workspace", what);
  if (misaligned(l->logits, l->dtype == T_F32 ? 4 : 2) || misaligned(l->uniforms, 4) || misaligned(l->temperatures, 4))
    return fail(SPEC_ERR_INVALID, "%s: logits, uniforms or temperatures are not aligned to their element size", what);
  if (l->row_stride < 0 || l->row_stride > kMaxStride)
    return fail(SPEC_ERR_INVALID, "%s: row stride %lld outside [0, 2^40]", what, (long long)l->row_stride);
  if (!l->temperatures && !(l->temperature >= 0.f && l->temperature <= 3.402823466e38f))
    return fail(SPEC_ERR_INVALID, "%s: temperature %g", what, (double)l->temperature);
  if (misaligned(l->workspace, 16)) return fail(SPEC_ERR_INVALID, "%s: the workspace is not aligned to 16 bytes", what);
  const int64_t need = workspace_bytes(l->n_rows, l->vocab, l->dtype);
  if (l->workspace_bytes < need)
    return fail(SPEC_ERR_INVALID, "%s: workspace of %lld bytes, %lld are needed", what, (long long)l->workspace_bytes,
                (long long)need);
  return SPEC_OK;
}

Rows to_rows(const spec_batch_logits* l) {
  Rows r;
  r.logits = l->logits;
  r.stride = l->row_stride;
  r.temps = l->temperatures;
  r.temp = l->temperature;
  r.u = l->uniforms;
  r.n_rows = (int)l->n_rows;
  r.V = l->vocab;
  r.nch = chunks_of(l->vocab, l->dtype);
  const size_t cells = (size_t)l->n_rows * r.nch;
  uint8_t* w = static_cast<uint8_t*>(l->workspace);
  r.stats = reinterpret_cast<float2*>(w);
  r.sums = reinterpret_cast<double*>(w + up(cells * sizeof(float2)));
  r.path = nullptr;
  r.drafts = nullptr;
  r.q = nullptr;
  r.q_stride = 0;
  uint8_t* last = w + up(cells * sizeof(float2)) + up(cells * sizeof(double));  // a chain's or a tree's
  r.seen = reinterpret_cast<float2*>(last);
  r.drawn = reinterpret_cast<int*>(last);
  return r;
}

int verify(const char* what, const spec_batch_logits* l, VerifyParams& p, int32_t* path, bool trees, void* stream) {
  if (p.n_seqs < 0 || p.n_seqs > SPEC_BATCH_MAX_ROWS)
    return fail(SPEC_ERR_INVALID, "%s: %d sequences, 0 to %d are taken", what, p.n_seqs, SPEC_BATCH_MAX_ROWS);
  const bool path_alone = p.n_seqs == 0 && trees && l->n_rows > 0;  // rows of no sequence: their path is -1
  if (p.n_seqs == 0 && !path_alone) return SPEC_OK;
  if (p.n_seqs > 0 && (!p.row_start || !p.n_out || !p.next)) return fail(SPEC_ERR_INVALID, "%s: null argument", what);
  for (const void* q : {(const void*)p.row_start, (const void*)p.tokens, (const void*)p.parents, (const void*)p.q,
                        (const void*)path, (const void*)p.n_out, (const void*)p.next})
    if (misaligned(q, 4)) return fail(SPEC_ERR_INVALID, "%s: a pointer is not aligned to 4 bytes", what);
  Current cur(l->device, what);
  if (cur.rc != SPEC_OK) return cur.rc;
  if (path_alone) {
    const cudaError_t e = cudaMemsetAsync(path, 0xff, (size_t)l->n_rows * sizeof(int32_t), static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPEC_OK : fail_cuda(e, what);
  }
  p.r = to_rows(l);
  p.r.path = path;
  if (!trees) p.r.drafts = p.tokens, p.r.q = p.q, p.r.q_stride = p.q_stride;
  int sms = 0;
  cudaError_t e = multiprocessors(l->device, &sms);
  if (e == cudaSuccess) e = launch_verify(p, l->dtype, trees, sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SPEC_OK : fail_cuda(e, what);
}

}  // namespace

extern "C" {

int64_t spec_batch_workspace_bytes(int64_t n_rows, int vocab, int dtype) {
  const int rc = check_shape("spec_batch_workspace_bytes", n_rows, vocab, dtype);
  return rc == SPEC_OK ? workspace_bytes(n_rows, vocab, dtype) : -rc;
}

int spec_batch_sample(const spec_batch_logits* l, float* probs_out, int64_t probs_stride, int32_t* tokens_out,
                      void* stream) {
  const char* what = "spec_batch_sample";
  const int rc = check_logits(what, l);
  if (rc != SPEC_OK) return rc;
  if (l->n_rows == 0) return SPEC_OK;
  if (!tokens_out) return fail(SPEC_ERR_INVALID, "%s: null tokens_out", what);
  if (misaligned(tokens_out, 4) || misaligned(probs_out, 4))
    return fail(SPEC_ERR_INVALID, "%s: an output is not aligned to 4 bytes", what);
  if (probs_out && (probs_stride > kMaxStride || (l->n_rows > 1 && probs_stride < l->vocab)))
    return fail(SPEC_ERR_INVALID, "%s: probability rows %lld apart, the vocabulary is %d", what, (long long)probs_stride,
                l->vocab);
  const int64_t size = l->dtype == T_F32 ? 4 : 2;
  if (probs_out && rows_meet(l->logits, l->row_stride * size, l->vocab * size, probs_out, probs_stride * 4, l->vocab * INT64_C(4), l->n_rows))
    return fail(SPEC_ERR_INVALID, "%s: probabilities share memory with the logits", what);
  Current cur(l->device, what);
  if (cur.rc != SPEC_OK) return cur.rc;
  SampleParams p;
  p.r = to_rows(l);
  p.probs = probs_out;
  p.probs_stride = probs_stride;
  p.tokens = tokens_out;
  int sms = 0;
  cudaError_t e = multiprocessors(l->device, &sms);
  if (e == cudaSuccess) e = launch_sample(p, l->dtype, sms, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SPEC_OK : fail_cuda(e, what);
}

int spec_batch_verify(const spec_batch_logits* l, int n_seqs, const int32_t* row_start, const int32_t* drafts,
                      const float* draft_probs, int64_t probs_stride, int32_t* n_accepted, int32_t* next_token,
                      void* stream) {
  const char* what = "spec_batch_verify";
  const int rc = check_logits(what, l);
  if (rc != SPEC_OK) return rc;
  if (n_seqs > 0 && l->n_rows > 0 && (!drafts || !draft_probs))
    return fail(SPEC_ERR_INVALID, "%s: null drafts or draft probabilities", what);
  if (probs_stride < 0 || probs_stride > kMaxStride)
    return fail(SPEC_ERR_INVALID, "%s: probability rows %lld apart", what, (long long)probs_stride);
  VerifyParams p{};
  p.row_start = row_start;
  p.n_seqs = n_seqs;
  p.tokens = drafts;
  p.q = draft_probs;
  p.q_stride = probs_stride;
  p.n_out = n_accepted;
  p.next = next_token;
  return verify(what, l, p, nullptr, false, stream);
}

int spec_batch_verify_tree(const spec_batch_logits* l, int n_seqs, const int32_t* row_start, const int32_t* tokens,
                           const int32_t* parents, int32_t* path, int32_t* path_len, int32_t* next_token, void* stream) {
  const char* what = "spec_batch_verify_tree";
  const int rc = check_logits(what, l);
  if (rc != SPEC_OK) return rc;
  if (l->n_rows > 0 && (!path || (n_seqs > 0 && (!tokens || !parents))))
    return fail(SPEC_ERR_INVALID, "%s: null tokens, parents or path", what);
  VerifyParams p{};
  p.row_start = row_start;
  p.n_seqs = n_seqs;
  p.tokens = tokens;
  p.parents = parents;
  p.n_out = path_len;
  p.next = next_token;
  return verify(what, l, p, path, true, stream);
}

}  // extern "C"
