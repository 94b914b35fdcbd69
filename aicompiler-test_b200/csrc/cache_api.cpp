// extern "C" boundary of the serving-cache kernels: window attention, token
// log probabilities, page copies and cache compaction (declarations in
// include/tmc_cuda.h).
#include <cmath>
#include <cstdint>
#include <cstring>
#include <string>

#include "api_util.hpp"
#include "cache_ops.cuh"
#include "logprobs.cuh"
#include "tmc_cuda.h"
#include "window_attention.cuh"

using namespace tmc_api;

namespace {

// Makes the device that holds `memory` current for the call's launches. Host
// memory that no kernel can reach is refused here.
class OnDeviceOf {
 public:
  explicit OnDeviceOf(const void *memory) {
    cudaPointerAttributes a{};
    error_ = cudaPointerGetAttributes(&a, memory);
    if (error_ == cudaSuccess && a.type == cudaMemoryTypeUnregistered) error_ = cudaErrorInvalidDevicePointer;
    if (error_ == cudaSuccess) error_ = cudaGetDevice(&previous_);
    if (error_ != cudaSuccess || a.device == previous_) return;
    error_ = cudaSetDevice(a.device);
    switched_ = error_ == cudaSuccess;
  }
  ~OnDeviceOf() {
    if (switched_) cudaSetDevice(previous_);
  }
  OnDeviceOf(const OnDeviceOf &) = delete;
  OnDeviceOf &operator=(const OnDeviceOf &) = delete;
  cudaError_t error() const { return error_; }

 private:
  cudaError_t error_ = cudaSuccess;
  int previous_ = 0;
  bool switched_ = false;
};

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Arguments in 8-byte slots, in declaration order.
class Slots {
 public:
  explicit Slots(const int64_t *slots) : at_(slots) {}
  template <typename T>
  T *pointer() {
    return reinterpret_cast<T *>(static_cast<uintptr_t>(*at_++));
  }
  int64_t wide() { return *at_++; }
  int whole() {
    const int64_t v = *at_++;
    if (v < INT32_MIN || v > INT32_MAX) fits_ = false;
    return static_cast<int>(v);
  }
  float real() {
    const uint32_t bits = static_cast<uint32_t>(*at_++);
    float v;
    std::memcpy(&v, &bits, sizeof v);
    return v;
  }
  bool fits() const { return fits_; }  // every whole number was a 32-bit one

 private:
  const int64_t *at_;
  bool fits_ = true;
};
const char *const kWide = "an integer argument does not fit 32 bits";

}  // namespace

extern "C" {

size_t tmc_k_window_attention_workspace_bytes(int sequences, int max_rows, int hq, int hkv, int d, int window,
                                              int sinks) {
  return tmc::window_attention_workspace_bytes(sequences, max_rows, hq, hkv, d, window, sinks, num_sms());
}

int tmc_k_window_attention(const void *q, int64_t q_stride, void *out, int64_t out_stride, const void *k_pool,
                           const void *v_pool, int dtype, const int32_t *block_table, int table_stride,
                           const int32_t *table_rows, const int32_t *row_starts, const int32_t *first_positions,
                           int sequences, int rows, int max_rows, int hq, int hkv, int d, int page_size,
                           int pool_pages, int capacity, int window, int sinks, float scale, void *workspace,
                           size_t workspace_bytes, void *status, void *stream) {
  if (!q || !out || !k_pool || !v_pool || !block_table || !table_rows || !row_starts || !first_positions)
    return fail(TMC_ERR_INVALID, "null pointer");
  if (dtype != TMC_F16 && dtype != TMC_BF16)
    return fail(TMC_ERR_UNSUPPORTED, "window attention: dtype must be fp16 or bf16");
  if (sequences < 0 || rows < 0 || max_rows < 1)
    return fail(TMC_ERR_INVALID, "window attention: sequences, rows >= 0 and max_rows >= 1");
  if (hq < 1 || hkv < 1 || hq % hkv != 0)
    return fail(TMC_ERR_INVALID, "window attention: hq must be a positive multiple of hkv");
  if (d != 16 && d != 32 && d != 64 && d != 128)
    return fail(TMC_ERR_UNSUPPORTED, "window attention: head dimension must be 16, 32, 64 or 128");
  if (page_size < 1 || pool_pages < 1 || table_stride < 1 || capacity < 1)
    return fail(TMC_ERR_INVALID, "window attention: page_size, pool_pages, table_stride and capacity must be positive");
  if (window < 1 || sinks < 0) return fail(TMC_ERR_INVALID, "window attention: window >= 1 and sinks >= 0");
  if (!(scale >= 0.0f) || std::isinf(scale))
    return fail(TMC_ERR_INVALID, "window attention: scale must be finite and positive, or 0 for 1/sqrt(d)");
  const int64_t width = (int64_t)hq * d;
  if (q_stride < width || out_stride < width || q_stride % 8 != 0 || out_stride % 8 != 0)
    return fail(TMC_ERR_INVALID, "window attention: row strides must be multiples of 8 and hold hq * d elements");
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(workspace))
    return fail(TMC_ERR_INVALID, "window attention: q, out, pools and workspace must be 16-byte aligned");
  if (sequences == 0 || rows == 0) return ok();
  const OnDeviceOf device(out);
  if (device.error() != cudaSuccess) return cuda_fail(device.error(), "window attention: out");
  tmc::WindowAttentionParams p{};
  p.q = q;
  p.q_stride = q_stride;
  p.out = out;
  p.out_stride = out_stride;
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.table_rows = table_rows;
  p.row_starts = row_starts;
  p.first_positions = first_positions;
  p.sequences = sequences;
  p.rows = rows;
  p.max_rows = max_rows;
  p.hq = hq;
  p.hkv = hkv;
  p.d = d;
  p.page_size = page_size;
  p.pool_pages = pool_pages;
  p.capacity = capacity;
  p.window = window;
  p.sinks = sinks;
  p.scale = scale > 0.0f ? scale : static_cast<float>(1.0 / std::sqrt(static_cast<double>(d)));
  p.workspace = workspace;
  p.workspace_bytes = workspace ? workspace_bytes : 0;
  p.status = static_cast<tmc::TmcDeviceStatus *>(status);
  const cudaError_t e = tmc::launch_window_attention(p, dtype == TMC_BF16, num_sms(),
                                                     static_cast<cudaStream_t>(stream), false);
  if (e == cudaErrorInvalidValue) return fail(TMC_ERR_UNSUPPORTED, "window attention: unsupported shape");
  return e == cudaSuccess ? ok() : cuda_fail(e, "window attention launch");
}

int tmc_k_token_logprobs(const void *logits, int dtype, int64_t row_stride, const int32_t *targets, int rows, int vocab,
                         float *logprobs, float *entropy, int32_t *ranks, int top, int32_t *top_ids,
                         float *top_logprobs, void *status, void *stream) {
  if (!logits || (!logprobs && !entropy && !ranks && top == 0)) return fail(TMC_ERR_INVALID, "null pointer");
  if ((logprobs || ranks) && !targets) return fail(TMC_ERR_INVALID, "token logprobs: logprobs and ranks need targets");
  if (top != 0 && (!top_ids || !top_logprobs)) return fail(TMC_ERR_INVALID, "null pointer");
  int type;
  switch (dtype) {
    case TMC_F16: type = tmc::kLogitsF16; break;
    case TMC_F32: type = tmc::kLogitsF32; break;
    case TMC_BF16: type = tmc::kLogitsBF16; break;
    default: return fail(TMC_ERR_UNSUPPORTED, "token logprobs: dtype must be fp16, bf16 or fp32");
  }
  if (rows < 0 || vocab < 1 || row_stride < vocab)
    return fail(TMC_ERR_INVALID, "token logprobs: rows >= 0, vocab >= 1 and row_stride >= vocab");
  if (top < 0 || top > tmc::kLogprobsMaxTop || top > vocab)
    return fail(TMC_ERR_UNSUPPORTED, "token logprobs: top must be in [0, 32] and at most vocab");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == TMC_F32 ? 4 : 2) != 0)
    return fail(TMC_ERR_INVALID, "token logprobs: logits must be aligned to their element size");
  if (rows == 0) return ok();
  const OnDeviceOf device(logits);
  if (device.error() != cudaSuccess) return cuda_fail(device.error(), "token logprobs: logits");
  tmc::LogprobsParams p{};
  p.logits = logits;
  p.row_stride = row_stride;
  p.targets = targets;
  p.rows = rows;
  p.vocab = vocab;
  p.top = top;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.ranks = ranks;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  p.status = static_cast<tmc::TmcDeviceStatus *>(status);
  const cudaError_t e = tmc::launch_token_logprobs(p, type, num_sms(), static_cast<cudaStream_t>(stream));
  if (e == cudaErrorInvalidValue) return fail(TMC_ERR_UNSUPPORTED, "token logprobs: unsupported shape");
  return e == cudaSuccess ? ok() : cuda_fail(e, "token logprobs launch");
}

int tmc_k_kv_copy_pages(void *const *pools, int pool_count, int pool_pages, size_t page_bytes, const int32_t *src,
                        const int32_t *dst, int count, void *status, void *stream) {
  if (!pools || !src || !dst) return fail(TMC_ERR_INVALID, "null pointer");
  if (pool_count < 1 || pool_pages < 1 || count < 0)
    return fail(TMC_ERR_INVALID, "page copy: pool_count, pool_pages >= 1 and count >= 0");
  if (page_bytes == 0 || page_bytes % 16 != 0)
    return fail(TMC_ERR_INVALID, "page copy: page_bytes must be a positive multiple of 16");
  if (count > pool_pages) return fail(TMC_ERR_INVALID, "page copy: more targets than the pool has pages");
  if (count == 0) return ok();
  const OnDeviceOf device(pools);
  if (device.error() != cudaSuccess) return cuda_fail(device.error(), "page copy: pools");
  const cudaError_t e =
      tmc::launch_kv_copy_pages(pools, pool_count, pool_pages, page_bytes, src, dst, count,
                                static_cast<tmc::TmcDeviceStatus *>(status), static_cast<cudaStream_t>(stream));
  if (e == cudaErrorInvalidValue) return fail(TMC_ERR_UNSUPPORTED, "page copy: unsupported shape");
  return e == cudaSuccess ? ok() : cuda_fail(e, "page copy launch");
}

int tmc_k_kv_compact(void *const *pools, int layers, int dtype, int pool_pages, int hkv, int d, int page_size,
                     const int32_t *src_pages, int src_count, const int32_t *dst_pages, int dst_count,
                     const int32_t *keep, int count, int first, const float *rope_cos, const float *rope_sin,
                     int rope_rows, void *status, void *stream) {
  if (!pools || !src_pages || !dst_pages || !keep) return fail(TMC_ERR_INVALID, "null pointer");
  if (!rope_cos != !rope_sin) return fail(TMC_ERR_INVALID, "compact: give both rope tables or neither");
  if (dtype != TMC_F16 && dtype != TMC_BF16) return fail(TMC_ERR_UNSUPPORTED, "compact: dtype must be fp16 or bf16");
  if (layers < 1 || pool_pages < 1 || hkv < 1 || page_size < 1 || src_count < 1 || dst_count < 1)
    return fail(TMC_ERR_INVALID, "compact: layers, pages, hkv and page_size must be positive");
  if (d < 8 || d % 8 != 0) return fail(TMC_ERR_UNSUPPORTED, "compact: head dimension must be a multiple of 8");
  if (count < 0 || first < 0 || (int64_t)first + count > (int64_t)dst_count * page_size)
    return fail(TMC_ERR_INVALID, "compact: count, first >= 0 and the target pages must hold first + count rows");
  if (rope_cos && rope_rows < 1) return fail(TMC_ERR_INVALID, "compact: rope_rows must be positive");
  if (count == 0) return ok();
  const OnDeviceOf device(pools);
  if (device.error() != cudaSuccess) return cuda_fail(device.error(), "compact: pools");
  tmc::CompactParams p{};
  p.pools = pools;
  p.layers = layers;
  p.pool_pages = pool_pages;
  p.hkv = hkv;
  p.d = d;
  p.page_size = page_size;
  p.src_pages = src_pages;
  p.src_count = src_count;
  p.dst_pages = dst_pages;
  p.dst_count = dst_count;
  p.keep = keep;
  p.count = count;
  p.first = first;
  p.cos = rope_cos;
  p.sin = rope_sin;
  p.rope_rows = rope_rows;
  p.status = static_cast<tmc::TmcDeviceStatus *>(status);
  const cudaError_t e = tmc::launch_kv_compact(p, dtype == TMC_BF16, static_cast<cudaStream_t>(stream));
  if (e == cudaErrorInvalidValue) return fail(TMC_ERR_UNSUPPORTED, "compact: unsupported shape");
  return e == cudaSuccess ? ok() : cuda_fail(e, "compact launch");
}

int tmc_k_window_attention_slots(const int64_t *slots) {
  if (!slots) return fail(TMC_ERR_INVALID, "null pointer");
  Slots a(slots);
  const auto *q = a.pointer<const void>();
  const int64_t q_stride = a.wide();
  auto *out = a.pointer<void>();
  const int64_t out_stride = a.wide();
  const auto *k = a.pointer<const void>();
  const auto *v = a.pointer<const void>();
  const int dtype = a.whole();
  const auto *table = a.pointer<const int32_t>();
  const int table_stride = a.whole();
  const auto *table_rows = a.pointer<const int32_t>();
  const auto *row_starts = a.pointer<const int32_t>();
  const auto *first = a.pointer<const int32_t>();
  int n[11];  // sequences .. sinks
  for (int &x : n) x = a.whole();
  const float scale = a.real();
  auto *workspace = a.pointer<void>();
  const int64_t bytes = a.wide();
  auto *status = a.pointer<void>();
  auto *stream = a.pointer<void>();
  if (!a.fits() || bytes < 0) return fail(TMC_ERR_INVALID, kWide);
  return tmc_k_window_attention(q, q_stride, out, out_stride, k, v, dtype, table, table_stride, table_rows, row_starts,
                                first, n[0], n[1], n[2], n[3], n[4], n[5], n[6], n[7], n[8], n[9], n[10], scale,
                                workspace, static_cast<size_t>(bytes), status, stream);
}

int tmc_k_token_logprobs_slots(const int64_t *slots) {
  if (!slots) return fail(TMC_ERR_INVALID, "null pointer");
  Slots a(slots);
  const auto *logits = a.pointer<const void>();
  const int dtype = a.whole();
  const int64_t stride = a.wide();
  const auto *targets = a.pointer<const int32_t>();
  const int rows = a.whole();
  const int vocab = a.whole();
  auto *logprobs = a.pointer<float>();
  auto *entropy = a.pointer<float>();
  auto *ranks = a.pointer<int32_t>();
  const int top = a.whole();
  auto *ids = a.pointer<int32_t>();
  auto *values = a.pointer<float>();
  auto *status = a.pointer<void>();
  auto *stream = a.pointer<void>();
  if (!a.fits()) return fail(TMC_ERR_INVALID, kWide);
  return tmc_k_token_logprobs(logits, dtype, stride, targets, rows, vocab, logprobs, entropy, ranks, top, ids, values,
                              status, stream);
}

int tmc_k_kv_copy_pages_slots(const int64_t *slots) {
  if (!slots) return fail(TMC_ERR_INVALID, "null pointer");
  Slots a(slots);
  auto *pools = a.pointer<void *const>();
  const int pool_count = a.whole();
  const int pool_pages = a.whole();
  const int64_t page_bytes = a.wide();
  const auto *src = a.pointer<const int32_t>();
  const auto *dst = a.pointer<const int32_t>();
  const int count = a.whole();
  auto *status = a.pointer<void>();
  auto *stream = a.pointer<void>();
  if (!a.fits() || page_bytes < 0) return fail(TMC_ERR_INVALID, kWide);
  return tmc_k_kv_copy_pages(pools, pool_count, pool_pages, static_cast<size_t>(page_bytes), src, dst, count, status,
                             stream);
}

int tmc_k_kv_compact_slots(const int64_t *slots) {
  if (!slots) return fail(TMC_ERR_INVALID, "null pointer");
  Slots a(slots);
  auto *pools = a.pointer<void *const>();
  int n[6];  // layers .. page_size
  for (int &x : n) x = a.whole();
  const auto *src = a.pointer<const int32_t>();
  const int src_count = a.whole();
  const auto *dst = a.pointer<const int32_t>();
  const int dst_count = a.whole();
  const auto *keep = a.pointer<const int32_t>();
  const int count = a.whole();
  const int first = a.whole();
  const auto *cos = a.pointer<const float>();
  const auto *sin = a.pointer<const float>();
  const int rope_rows = a.whole();
  auto *status = a.pointer<void>();
  auto *stream = a.pointer<void>();
  if (!a.fits()) return fail(TMC_ERR_INVALID, kWide);
  return tmc_k_kv_compact(pools, n[0], n[1], n[2], n[3], n[4], n[5], src, src_count, dst, dst_count, keep, count, first,
                          cos, sin, rope_rows, status, stream);
}

}  // extern "C"
