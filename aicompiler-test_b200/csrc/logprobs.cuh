// Log probabilities of given tokens, with entropy, rank and the top
// alternatives, from rows of logits.
#pragma once

#include "common.cuh"

namespace tmc {

constexpr int kLogprobsMaxTop = 32;

enum : int { kLogitsF16 = 0, kLogitsF32 = 1, kLogitsBF16 = 2 };

struct LogprobsParams {
  const void *logits;  // [rows, row_stride], the first vocab of each row are read
  long long row_stride;
  const int *targets;  // [rows]; -1: the row has no target
  int rows, vocab, top;
  float *logprobs;   // [rows] or null
  float *entropy;    // [rows] or null
  int *ranks;        // [rows] or null
  int *top_ids;      // [rows, top], top_logprobs likewise (top > 0)
  float *top_logprobs;
  TmcDeviceStatus *status;
};

// type: kLogits*. top <= min(vocab, kLogprobsMaxTop). Logits are aligned to
// their element size.
cudaError_t launch_token_logprobs(const LogprobsParams &p, int type, int num_sms, cudaStream_t stream);

}  // namespace tmc
