// Copies inside the paged KV cache: whole pages (forking a sequence, moving
// pages) and kept rows moved together (dropping part of a sequence).
#pragma once

#include "common.cuh"

namespace tmc {

// Copy page src[i] to page dst[i] of every pool, i < count. pools: device
// array of pool_count addresses, each a pool of pool_pages pages of page_bytes
// bytes (a multiple of 16; pools 16-byte aligned). Targets are distinct and no
// target is a source of the same call.
cudaError_t launch_kv_copy_pages(void *const *pools, int pool_count, int pool_pages, size_t page_bytes,
                                 const int *src, const int *dst, int count, TmcDeviceStatus *status,
                                 cudaStream_t stream);

struct CompactParams {
  void *const *pools;  // device array: K and V pool of layer 0, of layer 1, ...
  int layers, pool_pages, hkv, d, page_size;
  const int *src_pages;  // the sequence's pages, position p in page src_pages[p / page_size]
  int src_count;
  const int *dst_pages;
  int dst_count;
  const int *keep;  // [count] kept positions
  int count, first;  // kept row i becomes position first + i
  const float *cos, *sin;  // [rope_rows, d / 2] or null: keys move unrotated
  int rope_rows;
  TmcDeviceStatus *status;
};

// Elements are fp16, or bf16 when `bf16`. d % 8 == 0. No page of dst_pages is
// a page of src_pages.
cudaError_t launch_kv_compact(const CompactParams &p, bool bf16, cudaStream_t stream);

}  // namespace tmc
