// Causal attention over the paged cache with a sliding window and first
// positions that stay visible (sinks), for ragged query rows.
//
// A query at position p sees the keys j <= p with p - j < window or j < sinks.
// Sequence s owns the query rows [row_starts[s], row_starts[s + 1]) at the
// consecutive positions first_positions[s], first_positions[s] + 1, ...; its
// keys and values are in the pages of block-table row table_rows[s]
// (pools [page][Hkv][page_size][D], as in attention.cuh). One row per sequence
// is single-token decoding, more are (chunks of) prompts.
#pragma once

#include "common.cuh"

namespace tmc {

struct WindowAttentionParams {
  const void *q;  // [rows, Hq, D], row stride q_stride elements
  long long q_stride;
  void *out;  // [rows, Hq, D], row stride out_stride elements
  long long out_stride;
  const void *k_pool, *v_pool;
  const int *block_table;
  int table_stride;
  const int *table_rows;       // [sequences]
  const int *row_starts;       // [sequences + 1]
  const int *first_positions;  // [sequences]
  int sequences, rows, max_rows;  // rows in q and out; most rows of one sequence
  int hq, hkv, d, page_size, pool_pages, capacity;
  int window, sinks;
  float scale;
  void *workspace;  // partial results of splits that meet in a second kernel
  size_t workspace_bytes;
  TmcDeviceStatus *status;
  int page_shift;  // set by the launch: log2(page_size), or -1
};

// Bytes with which a launch runs as many splits as it can use (0: it needs none).
size_t window_attention_workspace_bytes(int sequences, int max_rows, int hq, int hkv, int d, long long window,
                                        long long sinks, int num_sms);

// Kernels that a launch with that workspace is made of (1 or 2).
int window_attention_launches(int sequences, int max_rows, int hq, int hkv, int d, long long window, long long sinks,
                              long long capacity, int num_sms);

// fp16, or bf16 when `bf16`; d 16, 32, 64 or 128; q_stride and out_stride
// multiples of 8, q, out and the pools 16-byte aligned.
cudaError_t launch_window_attention(const WindowAttentionParams &p, bool bf16, int num_sms, cudaStream_t stream,
                                    bool pdl);

}  // namespace tmc
