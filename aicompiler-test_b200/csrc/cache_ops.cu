// Page copies and row compaction of the paged KV cache (cache_ops.cuh).
#include "cache_ops.cuh"

#include <cuda_bf16.h>

namespace tmc {
namespace {

// ---- whole pages ------------------------------------------------------------------

// Bound by memory: 400 different pages of 32 KB in 64 pools (839 MB read, 839
// written) 254.5 us, 6.6 TB/s, a plain copy's rate. Pages that are copied more
// than once are read from L2 again: 400 copies of 300 different pages 222 us
// (four and eight vectors in flight a thread 223). One page 2.1 us, a launch
// (eight vectors 2.3).
constexpr int kCopyThreads = 256;
constexpr int kCopyVectors = 2;  // 16-byte vectors a thread has in flight

// kv[p][dst_i] = kv[p][src_i]. Grid (pairs x chunks of a page, pools).
__global__ void __launch_bounds__(kCopyThreads)
    kv_copy_pages_kernel(void *const *pools, int pool_pages, size_t page_vectors, int chunks, const int *src,
                         const int *dst, TmcDeviceStatus *status) {
  const int pair = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int s = src[pair], t = dst[pair];
  const int bad = (s < 0 || s >= pool_pages) ? s : t;
  if (bad < 0 || bad >= pool_pages) {
    if (threadIdx.x == 0) report_status(status, bad < 0 ? kStatusPageMissing : kStatusPageRange, kWhereCache, bad, pair);
    return;
  }
  if (s == t) return;
  const size_t begin = (size_t)chunk * (kCopyThreads * kCopyVectors) + threadIdx.x;
  const uint4 *from = static_cast<const uint4 *>(pools[blockIdx.y]) + (size_t)s * page_vectors;
  uint4 *to = static_cast<uint4 *>(pools[blockIdx.y]) + (size_t)t * page_vectors;
  uint4 v[kCopyVectors];
#pragma unroll
  for (int i = 0; i < kCopyVectors; ++i)
    if (begin + i * kCopyThreads < page_vectors) v[i] = from[begin + i * kCopyThreads];
#pragma unroll
  for (int i = 0; i < kCopyVectors; ++i)
    if (begin + i * kCopyThreads < page_vectors) to[begin + i * kCopyThreads] = v[i];
}

// ---- kept rows ----------------------------------------------------------------------

__device__ __forceinline__ float2 unpack2(uint32_t bits, __half) { return half2_bits_to_float2(bits); }
__device__ __forceinline__ float2 unpack2(uint32_t bits, __nv_bfloat16) {
  return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float2 v, __half) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t *>(&h);
}

constexpr int kCompactThreads = 64;
constexpr int kHeads = 4;  // heads whose key and value a thread has in flight

// Row i of the kept list moves from position p = keep[i] to position
// t = first + i of the target pages. A key was stored rotated by its position,
// (x, y) -> R(p f) (x, y) for each interleaved pair with frequency f; stored at
// t it has to be R(t f) = R(-(p - t) f) R(p f): it is turned back by the
// distance moved, in fp32, and rounded once to storage. Values move unchanged.
// A thread owns 8 elements (four pairs, their cosines and sines read once) of
// one kept row and walks the heads of one layer. Grid (row chunks, layers).
// Bound by memory: 2044 rows of 32 layers, 8 heads of 128 (2 x 268 MB) 85 us,
// 6.3 TB/s, 0.96 of a copy's rate; 60 rows of two layers 2.7 us. (One head in
// flight 91 and 3.3 us, eight 85 and 2.9; 256 threads a CTA 88 and 3.2.)
template <typename E>
__global__ void __launch_bounds__(kCompactThreads) kv_compact_kernel(const CompactParams p) {
  const int vectors = p.d / 8;
  const long long index = (long long)blockIdx.x * kCompactThreads + threadIdx.x;
  const int i = (int)(index / vectors), c = (int)(index % vectors);
  if (i >= p.count) return;
  const int from = p.keep[i], to = p.first + i;
  const int from_page = from < 0 ? -1 : from / p.page_size, to_page = to / p.page_size;
  if (from_page < 0 || from_page >= p.src_count || to_page >= p.dst_count) {
    report_status(p.status, kStatusLengthRange, kWhereCache, from, i);
    return;
  }
  const int s = p.src_pages[from_page], t = p.dst_pages[to_page];
  const int bad = (s < 0 || s >= p.pool_pages) ? s : t;
  if (bad < 0 || bad >= p.pool_pages) {
    report_status(p.status, bad < 0 ? kStatusPageMissing : kStatusPageRange, kWhereCache, bad, i);
    return;
  }
  const int back = from - to, distance = back < 0 ? -back : back;
  const bool turn = p.cos != nullptr && back != 0;
  float cs[4] = {1.0f, 1.0f, 1.0f, 1.0f}, sn[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (turn) {
    if (distance >= p.rope_rows) {
      report_status(p.status, kStatusLengthRange, kWhereCache, distance, i);
      return;
    }
    const size_t at = (size_t)distance * (p.d / 2) + c * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cs[j] = p.cos[at + j];
      sn[j] = back < 0 ? -p.sin[at + j] : p.sin[at + j];
    }
  }
  const size_t head = (size_t)p.page_size * vectors;  // 16-byte vectors from one head to the next
  const size_t a = (size_t)s * p.hkv * head + (size_t)(from % p.page_size) * vectors + c;
  const size_t b = (size_t)t * p.hkv * head + (size_t)(to % p.page_size) * vectors + c;
  uint4 *k = static_cast<uint4 *>(p.pools[2 * blockIdx.y]), *v = static_cast<uint4 *>(p.pools[2 * blockIdx.y + 1]);
  for (int h0 = 0; h0 < p.hkv; h0 += kHeads) {
    uint4 key[kHeads], value[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j)
      if (h0 + j < p.hkv) {
        key[j] = k[a + (h0 + j) * head];
        value[j] = v[a + (h0 + j) * head];
      }
#pragma unroll
    for (int j = 0; j < kHeads; ++j)
      if (h0 + j < p.hkv) {
        if (turn) {
          uint32_t *w = reinterpret_cast<uint32_t *>(&key[j]);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 x = unpack2(w[n], E());
            w[n] = pack2(make_float2(fmaf(x.x, cs[n], x.y * sn[n]), fmaf(x.y, cs[n], -x.x * sn[n])), E());
          }
        }
        k[b + (h0 + j) * head] = key[j];
        v[b + (h0 + j) * head] = value[j];
      }
  }
}

}  // namespace

cudaError_t launch_kv_copy_pages(void *const *pools, int pool_count, int pool_pages, size_t page_bytes,
                                 const int *src, const int *dst, int count, TmcDeviceStatus *status,
                                 cudaStream_t stream) {
  if (pool_count <= 0 || pool_count > 65535 || pool_pages <= 0 || page_bytes == 0 || page_bytes % 16 != 0 || count < 0)
    return cudaErrorInvalidValue;
  if (count == 0) return cudaSuccess;
  const size_t vectors = page_bytes / 16;
  const size_t chunks = (vectors + kCopyThreads * kCopyVectors - 1) / (kCopyThreads * kCopyVectors);
  if (chunks * count > 0x7fffffffull) return cudaErrorInvalidValue;
  kv_copy_pages_kernel<<<dim3((unsigned)(chunks * count), pool_count), kCopyThreads, 0, stream>>>(
      pools, pool_pages, vectors, (int)chunks, src, dst, status);
  return cudaGetLastError();
}

cudaError_t launch_kv_compact(const CompactParams &p, bool bf16, cudaStream_t stream) {
  if (p.layers <= 0 || p.layers > 65535 || p.pool_pages <= 0 || p.hkv <= 0 || p.d <= 0 || p.d % 8 != 0 ||
      p.page_size <= 0 || p.src_count <= 0 || p.dst_count <= 0 || p.count < 0 || p.first < 0 ||
      p.first > 0x7fffffff - p.count)
    return cudaErrorInvalidValue;
  if (p.count == 0) return cudaSuccess;
  const long long items = (long long)p.count * (p.d / 8);
  const long long blocks = (items + kCompactThreads - 1) / kCompactThreads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, p.layers);
  if (bf16)
    kv_compact_kernel<__nv_bfloat16><<<grid, kCompactThreads, 0, stream>>>(p);
  else
    kv_compact_kernel<__half><<<grid, kCompactThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace tmc
