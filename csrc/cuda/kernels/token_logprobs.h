// Host interface of log-probabilities over a vocabulary, their gradient, and the join of vocabulary shards (no torch dependency).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ccl {

constexpr int kMaxTopLogprobs = 32;

// dtype: 0 bf16, 1 f16, 2 fp32.
struct LogprobParams {
  const void* logits;        // [rows, vocab], row stride `stride` elements
  long long stride;
  int dtype;
  int rows, vocab, top;      // top: 0 .. 32 alternatives
  const long long* targets;  // [rows] global ids; negative: no token (log-probability 0, no gradient); not in the vocabulary: NaN
  long long vocab_base;      // global id of column 0
  long long vocab_total;
  // whole vocabulary
  float* logprob;            // [rows]
  float* entropy;
  float* lse;                // [rows, 2]: a reference, and the logarithm of the sum of e^(x - reference)
  float* top_logprobs;       // [rows, top], best first; equal ones by id; a NaN is larger than everything
  long long* top_ids;
  // a shard (the five above are not written): [rows, 4 + 2 * top] words {max, sum, weighted sum, target's logit, values.., ids (int32)..}
  float* partial;
};
cudaError_t token_logprobs(const LogprobParams& p, cudaStream_t stream);

// Joins the partial results of `shards` shards, shard-major.
struct LogprobMergeParams {
  const float* partials;     // [shards, rows, 4 + 2 * top]
  const long long* targets;
  long long vocab_total;
  int shards, rows, top;
  float* logprob;
  float* entropy;
  float* lse;
  float* top_logprobs;
  long long* top_ids;
};
cudaError_t token_logprobs_merge(const LogprobMergeParams& p, cudaStream_t stream);

// grad[r, v] = g_logprob (delta_target - p) - g_entropy p (log p + H) + sum_j g_top[j] (delta_top_j - p). A null gradient counts as zero.
struct LogprobBackwardParams {
  const void* logits;
  long long stride;
  int dtype;
  int rows, vocab, top;
  const long long* targets;
  long long vocab_base, vocab_total;
  const float* lse;          // [rows, 2]
  const float* entropy;
  const long long* top_ids;  // [rows, top]
  const float* g_logprob;    // [rows]
  const float* g_entropy;    // [rows]
  const float* g_top;        // [rows, top]
  void* grad;                // [rows, vocab] of the logits' type, row stride `grad_stride`; each row at the logits' offset modulo 16 bytes
  long long grad_stride;
};
cudaError_t token_logprobs_backward(const LogprobBackwardParams& p, cudaStream_t stream);

}  // namespace ccl
