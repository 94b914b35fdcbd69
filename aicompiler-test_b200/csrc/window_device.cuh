// Device code shared by the window attention kernels: element types, fragments,
// what a tile of query rows sees, places in the paged cache, partial states.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "mbarrier.cuh"
#include "window_attention.cuh"

namespace tmc {
namespace window {

constexpr float kLog2e = 1.4426950408889634f;

// ---- element types ------------------------------------------------------------------

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) { return half2_bits_to_float2(v); }
__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ void store1(void *p, long long i, float v, __half) {
  static_cast<__half *>(p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ void store1(void *p, long long i, float v, __nv_bfloat16) {
  static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}
// Whether one of eight elements is infinite or NaN (exponent bits all ones).
__device__ __forceinline__ bool any_special(const uint4 &v, uint32_t exponent) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t hit = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) hit |= __vcmpeq2(w[i] & exponent, exponent);
  return hit != 0;
}
__device__ __forceinline__ uint32_t exponent_mask(__half) { return 0x7c007c00u; }
__device__ __forceinline__ uint32_t exponent_mask(__nv_bfloat16) { return 0x7f807f80u; }

// D = A(16x16, row) B(16x8, col) + D, fp32 accumulate.
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// 16 bytes into shared memory; zeros when `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Byte offset of 16-byte chunk c of row r in a tile of rows of D elements. The
// chunks of eight successive rows fall into different banks for ldmatrix.
template <int D>
__device__ __forceinline__ int tile_offset(int r, int c) {
  constexpr int kChunks = D / 8;  // per row
  if constexpr (kChunks >= 8) return r * (D * 2) + ((c ^ (r & 7)) << 4);
  else if constexpr (kChunks == 4) return r * (D * 2) + ((c ^ ((r >> 1) & 3)) << 4);
  else return r * (D * 2) + ((c ^ ((r >> 2) & 1)) << 4);
}

// ---- what a tile of query rows sees ---------------------------------------------------

struct Sequence {
  int start, rows, first;  // rows 0: nothing to do
  const int *table;
};

// Sequence s, checked; a bad description is reported once and the sequence left out.
__device__ __forceinline__ Sequence load_sequence(const WindowAttentionParams &p, int s, bool report) {
  Sequence q{0, 0, 0, nullptr};
  const int a = p.row_starts[s], b = p.row_starts[s + 1], first = p.first_positions[s], row = p.table_rows[s];
  if (a < 0 || b < a || b > p.rows || b - a > p.max_rows) {
    if (report) report_status(p.status, kStatusShape, kWhereAttention, a, b);
    return q;
  }
  if (a == b) return q;
  if (first < 0 || first > p.capacity - (b - a)) {
    if (report) report_status(p.status, kStatusLengthRange, kWhereAttention, first, s);
    return q;
  }
  if (row < 0) {
    if (report) report_status(p.status, kStatusShape, kWhereAttention, row, s);
    return q;
  }
  q.start = a;
  q.rows = b - a;
  q.first = first;
  q.table = p.block_table + (long long)row * p.table_stride;
  return q;
}

// A prompt CTA's place: grid.x counts KV heads fastest, then sequences, splits
// and, last rows first, tiles. The last rows see the most keys: what takes
// longest starts first, over all heads and sequences. (Heads slower than tiles,
// by the kernels of the time: 4096 rows of 32 heads 189 us instead of 161, which
// take 137 today, 152 back to back; 2048 rows of heads of 32 93 us instead of 65.)
struct PromptPlace {
  int head, seq, split, tile;
  bool first;  // one CTA of each sequence
};
__device__ __forceinline__ PromptPlace prompt_place(const WindowAttentionParams &p, int splits) {
  const unsigned heads = p.hkv, seqs = p.sequences;
  const unsigned u = blockIdx.x / heads, n = u / seqs, last = gridDim.x / (heads * seqs) - 1;
  PromptPlace c;
  c.head = (int)(blockIdx.x - u * heads);
  c.seq = (int)(u - n * seqs);
  c.tile = (int)((last - n) / (unsigned)splits);
  c.split = (int)(last - n) - c.tile * splits;
  c.first = n == 0 && c.head == 0;
  return c;
}

// The keys that the positions [p_lo, p_hi] see between them, numbered
// v = 0 .. count - 1: first `sinks` of them are the keys 0 .. sinks - 1, the
// rest the run from `low`.
struct Visible {
  int low, sinks, count;
  __device__ __forceinline__ int key(int v) const { return v < sinks ? v : v - sinks + low; }
};
__device__ __forceinline__ Visible visible_keys(const WindowAttentionParams &p, int p_lo, int p_hi) {
  Visible v;
  v.low = max(0, p_lo - p.window + 1);
  v.sinks = min(p.sinks, v.low);
  v.count = v.sinks + p_hi + 1 - v.low;
  return v;
}

// Where key j of a sequence is: its table entry (as loaded, unchecked: -1
// beyond the table) and its place in the page.
struct KeyPlace {
  int logical, page, offset;
};
__device__ __forceinline__ KeyPlace find_key(const WindowAttentionParams &p, const int *table, int j) {
  KeyPlace k;
  k.logical = p.page_shift >= 0 ? j >> p.page_shift : j / p.page_size;
  k.offset = j - k.logical * p.page_size;
  k.page = k.logical < p.table_stride ? table[k.logical] : -1;
  return k;
}
// The key's pool row (of D elements) for KV head h; -1, reported, when its page is missing.
__device__ __forceinline__ long long pool_row(const WindowAttentionParams &p, const KeyPlace &k, int h, int s) {
  if (k.page < 0 || k.page >= p.pool_pages) {
    report_status(p.status, k.page < 0 ? kStatusPageMissing : kStatusPageRange, kWhereAttention,
                  k.page < 0 ? k.logical : k.page, s);
    return -1;
  }
  return ((long long)k.page * p.hkv + h) * p.page_size + k.offset;
}

// Partial states: acc [split][slot][D], then (m, l) [split][slot], slot = (s max_rows + row) Hq + head.
__device__ __forceinline__ float *partial_acc(const WindowAttentionParams &p, long long slots, int split,
                                              long long slot) {
  return static_cast<float *>(p.workspace) + (split * slots + slot) * p.d;
}
__device__ __forceinline__ float2 *partial_ml(const WindowAttentionParams &p, long long slots, int splits, int split,
                                              long long slot) {
  return reinterpret_cast<float2 *>(static_cast<float *>(p.workspace) + splits * slots * p.d) + split * slots + slot;
}

// Adds 0 for finite numbers, NaN for others.
__device__ __forceinline__ void note_finite(float2 &sum, float a, float b) {
  sum = __ffma2_rn(make_float2(a, b), make_float2(0.0f, 0.0f), sum);
}

// One tile row by plain loops over its own keys (a warp, lanes along D): used
// when a step's values hold an infinity or NaN that some of the tile's rows do
// not see, which 0 x value products would let through; in prompts also when a
// result is not finite although the row's sum is: an infinite value times a
// weight below the storage type's range is NaN, where the weight in fp32 makes
// it infinite.
template <typename E, int D>
__device__ __noinline__ void slow_row(const WindowAttentionParams &p, const Sequence &seq, int s, int h, int head, int row,
                                      const Visible &vis, int v0, int v1, float &m, float &l, float (&o)[(D + 31) / 32],
                                      int lane) {
  constexpr int N = (D + 31) / 32;
  const E *q = static_cast<const E *>(p.q) + (seq.start + row) * p.q_stride + (long long)head * D;
  const int pos = seq.first + row;
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  for (int v = v0; v < v1; ++v) {
    const int j = vis.key(v);
    if (j > pos || (pos - j >= p.window && j >= p.sinks)) continue;
    const long long at = pool_row(p, find_key(p, seq.table, j), h, s);
    if (at < 0) continue;
    const E *k = static_cast<const E *>(p.k_pool) + at * D, *x = static_cast<const E *>(p.v_pool) + at * D;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < D) dot = fmaf((float)q[lane + 32 * i], (float)k[lane + 32 * i], dot);
    dot = warp_sum(dot) * (p.scale * kLog2e);
    const float m_new = fmaxf(m, dot), m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float f = exp2f(m - m_use), w = exp2f(dot - m_use);
    m = m_new;
    l = fmaf(l, f, w);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < D) o[i] = fmaf(w, (float)x[lane + 32 * i], o[i] * f);
  }
}

// The prompt kernel on the tensor cores (d 64 or 128): `pairs` tile pairs of
// 256 rows x heads per KV head and sequence, each cut into `splits`; all
// together below 2^31.
cudaError_t launch_window_tensor(const WindowAttentionParams &p, bool bf16, int pairs, int splits, cudaStream_t stream,
                                 bool pdl);

}  // namespace window
}  // namespace tmc
