// Window attention with sinks over the paged cache (window_attention.cuh).
//
// Both kernels make one pass over the visible keys with a running maximum and
// sum per query row: S = scale log2(e) Q K^T, p = 2^(S - m), O += P V, and
// O / l at the end, S and O in fp32, products by mma.sync m16n8k16. The G = Hq /
// Hkv query heads of a KV head are rows of the same tile, so a key is read
// once for all of them. The visible keys of a tile are numbered without a gap:
// the sinks before the window, then the window's run.
//
// - decode (one row per sequence): a warp takes 16 keys at a time through a
//   ring of its own, with no barrier between warps; the warps of a CTA, and
//   the CTAs of a cluster, split the keys and join their states in shared and
//   distributed shared memory.
// - prompts: a CTA holds 128 query rows x heads, its warps 16 each, and all
//   share 64-key tiles.
// When a launch has too few CTAs for the GPU its splits write their states to
// the workspace, and a second kernel joins them.
#include "window_attention.cuh"

#include <cuda_bf16.h>

#include <mutex>
#include <unordered_map>

#include "mbarrier.cuh"

namespace tmc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxCluster = 16;  // CTAs of a decode cluster (8 where 16 are not available)
constexpr int kMaxOuter = 32;    // splits that meet through the workspace

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

// The pool row (of D elements) of key j for KV head h; -1 when its page is missing.
__device__ __forceinline__ long long pool_row(const WindowAttentionParams &p, const int *table, int j, int h, int s) {
  const int logical = j / p.page_size;
  const int page = logical < p.table_stride ? table[logical] : -1;
  if (page < 0 || page >= p.pool_pages) {
    report_status(p.status, page < 0 ? kStatusPageMissing : kStatusPageRange, kWhereAttention,
                  page < 0 ? logical : page, s);
    return -1;
  }
  return ((long long)page * p.hkv + h) * p.page_size + (j - logical * p.page_size);
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

// ---- decode: one row per sequence --------------------------------------------------------

template <int D>
struct DecodeCfg {
  static constexpr int kWarps = 4;
  static constexpr int kStages = 4;                    // 16-key stages of a warp's ring
  static constexpr int kStageBytes = 16 * D * 2;       // one of K or V
  static constexpr int kRing = kWarps * kStages * 2 * kStageBytes;
  static constexpr int kMerge = kWarps * (16 * D + 32) * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

// Grid (splits, Hkv x head tiles, sequences), clusters of `cluster` CTAs along
// the splits; outer = splits / cluster of them meet in the workspace.
template <typename E, int D>
__global__ void __launch_bounds__(128) window_decode_kernel(const WindowAttentionParams p, int head_tiles, int cluster) {
  using C = DecodeCfg<D>;
  constexpr int S = C::kStages;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int bad_keys[C::kWarps][S];        // a stage's keys whose page is missing
  __shared__ float2 cta_ml[16];                 // this CTA's (m, l) per tile row
  __shared__ float weights[kMaxCluster * 16];   // of the cluster's CTAs
  __shared__ float total_l[16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  pdl_wait();
  const int s = blockIdx.z, h = blockIdx.y / head_tiles, tile = blockIdx.y % head_tiles;
  const int split = blockIdx.x, splits = gridDim.x;
  const Sequence seq = load_sequence(p, s, blockIdx.x == 0 && blockIdx.y == 0 && tid == 0);
  if (seq.rows == 0) return;  // the same for every CTA of the cluster
  const int g = p.hq / p.hkv, head0 = h * g + tile * 16, heads = min(16, g - tile * 16);
  const Visible vis = visible_keys(p, seq.first, seq.first);
  // Whole 64-key steps per split, so that the four warps share each evenly.
  const int chunk = ((vis.count + splits - 1) / splits + 63) / 64 * 64;
  const int v0 = min(vis.count, split * chunk), v1 = min(vis.count, v0 + chunk);
  const int groups = (v1 - v0 + 15) / 16;
  const int mine = groups > warp ? (groups - warp + C::kWarps - 1) / C::kWarps : 0;

  unsigned char *ring = smem + warp * (S * 2 * C::kStageBytes);
  const uint32_t ring_addr = smem_u32(ring);
  // The pool row of this lane's key (lane & 15) of stage i; -1: none.
  auto lookup = [&](int i) -> long long {
    const int v = v0 + (warp + C::kWarps * i) * 16 + (lane & 15);
    return i < mine && v < v1 ? pool_row(p, seq.table, vis.key(v), h, s) : -1;
  };
  constexpr int kChunks = D / 8;               // 16-byte chunks of a row
  constexpr int kLoads = 16 * kChunks / 32;    // of K (and of V) per lane and stage
  long long next_row = lookup(0);
  auto issue = [&](int i) {
    const int v = v0 + (warp + C::kWarps * i) * 16 + (lane & 15);
    const unsigned bad = __ballot_sync(0xffffffffu, next_row < 0 && i < mine && v < v1) & 0xffffu;
    if (lane == 0) bad_keys[warp][i % S] = (int)bad;
    const uint32_t dst = ring_addr + (i % S) * 2 * C::kStageBytes;
#pragma unroll
    for (int e = 0; e < kLoads; ++e) {
      const int at = lane + 32 * e, r = at / kChunks, c = at % kChunks;
      const long long row = __shfl_sync(0xffffffffu, next_row, r);
      const long long off = row < 0 ? 0 : row * D + c * 8;
      const int bytes = row < 0 ? 0 : 16;
      const int to = tile_offset<D>(r, c);
      cp_async16(dst + to, static_cast<const E *>(p.k_pool) + off, bytes);
      cp_async16(dst + C::kStageBytes + to, static_cast<const E *>(p.v_pool) + off, bytes);
    }
    next_row = lookup(i + 1);
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < mine) issue(i);
    cp_async_commit();
  }

  // Query fragments: tile rows gq and gq + 8 are heads head0 + gq and head0 + gq + 8.
  uint32_t qa[D / 16][4];
  {
    const E *q = static_cast<const E *>(p.q) + seq.start * p.q_stride + (long long)head0 * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = gq + 8 * (i & 1), c = kk * 16 + 2 * tq + 8 * (i >> 1);
        qa[kk][i] = r < heads ? *reinterpret_cast<const uint32_t *>(q + (long long)r * D + c) : 0u;
      }
  }
  const float scale = p.scale * kLog2e;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;

  for (int i = 0; i < mine; ++i) {
    if (i + S - 1 < mine) issue(i + S - 1);
    cp_async_commit();
    cp_async_wait<S - 1>();
    __syncwarp();
    const uint32_t sk = ring_addr + (i % S) * 2 * C::kStageBytes, sv = sk + C::kStageBytes;
    const int left = v1 - (v0 + (warp + C::kWarps * i) * 16);  // keys of this stage
    const int bad = bad_keys[warp][i % S];
    float sc[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t b[4];
      ldmatrix4(b, sk + tile_offset<D>((lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
      mma(sc[0], qa[kk], b[0], b[1], E());
      mma(sc[1], qa[kk], b[2], b[3], E());
    }
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[nt][j] *= scale;
    if (left < 16 || bad) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = nt * 8 + 2 * tq + (j & 1);
          if (key >= left || ((bad >> key) & 1)) sc[nt][j] = -INFINITY;
        }
    }
    float rescale[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m_run[r], mx), m_use = m_new == -INFINITY ? 0.0f : m_new;
      rescale[r] = exp2f(m_run[r] - m_use);
      m_run[r] = m_new;
      float sum = 0.0f;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int j = 2 * r; j < 2 * r + 2; ++j) {
          sc[nt][j] = exp2f(sc[nt][j] - m_use);
          sum += sc[nt][j];
        }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      l_run[r] = fmaf(l_run[r], rescale[r], sum);
    }
    // P as the A operand in two parts of the storage type, hi + lo, which keep
    // 22 bits of it (fp16; 16 in bf16): the products are not what bounds this
    // kernel, and the result is then rounded only once, at the end.
    uint32_t pa[4], pl[4];
#pragma unroll
    for (int i2 = 0; i2 < 4; ++i2) {
      const int nt = i2 >> 1, j = 2 * (i2 & 1);
      pa[i2] = pack2(sc[nt][j], sc[nt][j + 1], E());
      const float2 f = unpack2(pa[i2], E());
      pl[i2] = pack2(sc[nt][j] - f.x, sc[nt][j + 1] - f.y, E());
    }
    if (__any_sync(0xffffffffu, rescale[0] != 1.0f || rescale[1] != 1.0f)) {
#pragma unroll
      for (int dt = 0; dt < D / 8; ++dt) {
        acc[dt][0] *= rescale[0];
        acc[dt][1] *= rescale[0];
        acc[dt][2] *= rescale[1];
        acc[dt][3] *= rescale[1];
      }
    }
#pragma unroll
    for (int dt = 0; dt < D / 8; dt += 2) {
      uint32_t b[4];
      ldmatrix4_trans(b, sv + tile_offset<D>(lane & 15, dt + (lane >> 4)));
      mma(acc[dt], pl, b[0], b[1], E());
      mma(acc[dt], pa, b[0], b[1], E());
      mma(acc[dt + 1], pl, b[2], b[3], E());
      mma(acc[dt + 1], pa, b[2], b[3], E());
    }
    __syncwarp();  // the stage is free for issue(i + S)
  }
  pdl_launch_dependents();
  cp_async_wait<0>();
  __syncthreads();

  // Join the warps: their states in shared memory, over the rings.
  float *w_acc = reinterpret_cast<float *>(smem);                                  // [warp][16][D]
  float2 *w_ml = reinterpret_cast<float2 *>(smem + C::kWarps * 16 * D * 4);        // [warp][16]
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = gq + 8 * half;
#pragma unroll
    for (int dt = 0; dt < D / 8; ++dt)
      *reinterpret_cast<float2 *>(w_acc + (warp * 16 + r) * D + dt * 8 + 2 * tq) =
          make_float2(acc[dt][2 * half], acc[dt][2 * half + 1]);
    if (tq == 0) w_ml[warp * 16 + r] = make_float2(m_run[half], l_run[half]);
  }
  __syncthreads();
  for (int i = tid; i < heads * D; i += 128) {
    const int r = i / D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) m = fmaxf(m, w_ml[w * 16 + r].x);
    float l = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) {
      const float2 ml = w_ml[w * 16 + r];
      const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m);
      l = fmaf(ml.y, f, l);
      o = fmaf(w_acc[w * 16 * D + i], f, o);
    }
    w_acc[i] = o;  // only this thread reads element i of warp 0's state
    if (i % D == 0) cta_ml[r] = make_float2(m, l);
  }
  __syncthreads();

  // Join the CTAs of the cluster: each takes a share of the elements and reads
  // them from every CTA.
  const int crank = split % cluster, outer = split / cluster, outers = splits / cluster;
  if (cluster > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  for (int i = tid; i < cluster * 16; i += 128) {
    float2 ml;
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(&cta_ml[i % 16])), "r"(i / 16));
    if (i % 16 < heads)
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(a) : "memory");
    else
      ml = make_float2(-INFINITY, 0.0f);
    weights[i] = ml.x;
    reinterpret_cast<float2 *>(w_ml)[i] = ml;  // cluster * 16 pairs: within the merge area (asserted at launch)
  }
  __syncthreads();
  if (tid < 16) {
    float m = -INFINITY;
    for (int c = 0; c < cluster; ++c) m = fmaxf(m, weights[c * 16 + tid]);
    float l = 0.0f;
    for (int c = 0; c < cluster; ++c) {
      const float2 ml = w_ml[c * 16 + tid];
      const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m);
      weights[c * 16 + tid] = f;
      l = fmaf(ml.y, f, l);
    }
    total_l[tid] = l;
    const long long slots = (long long)p.sequences * p.max_rows * p.hq;
    if (outers > 1 && crank == 0 && tid < heads)
      *partial_ml(p, slots, outers, outer, (long long)s * p.max_rows * p.hq + head0 + tid) = make_float2(m, l);
  }
  __syncthreads();
  const int share = (heads * D + cluster - 1) / cluster;
  const int e1 = min(heads * D, (crank + 1) * share);
  for (int i = crank * share + tid; i < e1; i += 128) {
    const int r = i / D;
    float o = 0.0f;
    for (int c = 0; c < cluster; ++c) {
      uint32_t a;
      float x;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(w_acc + i)), "r"(c));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
      o = fmaf(x, weights[c * 16 + r], o);
    }
    if (outers > 1) {
      const long long slots = (long long)p.sequences * p.max_rows * p.hq;
      partial_acc(p, slots, outer, (long long)s * p.max_rows * p.hq + head0 + r)[i % D] = o;
    } else {
      const float l = total_l[r];
      store1(p.out, seq.start * p.out_stride + (long long)head0 * D + i, l > 0.0f || l != l ? o / l : 0.0f, E());
    }
  }
  if (cluster > 1) {
    // No CTA's memory goes away while another reads it.
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// ---- prompts -------------------------------------------------------------------------------

template <int D>
struct PromptCfg {
  static constexpr int kWarps = 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int BM = kWarps * 16;  // rows x heads of a tile
  static constexpr int BN = 64;           // keys of a step
  static constexpr int kStages = 2;
  static constexpr int kStageBytes = BN * D * 2;
  static constexpr int kSmem = kStages * 2 * kStageBytes;
};

// One tile row by plain loops over its own keys (a warp, lanes along D): used
// when a step's values hold an infinity or NaN that some of the tile's rows do
// not see, which 0 x value products would let through.
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
    const long long at = pool_row(p, seq.table, j, h, s);
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

// Grid (splits x tiles, Hkv, sequences). Tile t holds the tile rows
// t BM .. t BM + BM - 1 of the sequence's (row, head of the KV head) pairs,
// heads fastest.
template <typename E, int D>
__global__ void __launch_bounds__(PromptCfg<D>::kThreads)
    window_prompt_kernel(const WindowAttentionParams p, int splits) {
  using C = PromptCfg<D>;
  constexpr int BN = C::BN;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) unsigned char bad_keys[C::kStages][BN];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  pdl_wait();
  const int s = blockIdx.z, h = blockIdx.y, split = blockIdx.x % splits;
  const Sequence seq = load_sequence(p, s, blockIdx.x == 0 && blockIdx.y == 0 && tid == 0);
  const int g = p.hq / p.hkv;
  const int m0 = (int)(blockIdx.x / splits) * C::BM, total = seq.rows * g;
  if (m0 >= total) return;
  const int r_lo = m0 / g, r_hi = min(m0 + C::BM - 1, total - 1) / g;
  const int p_lo = seq.first + r_lo, p_hi = seq.first + r_hi;
  const Visible vis = visible_keys(p, p_lo, p_hi);
  const int chunk = ((vis.count + splits - 1) / splits + BN - 1) / BN * BN;
  const int v0 = min(vis.count, split * chunk), v1 = min(vis.count, v0 + chunk);
  const int steps = (v1 - v0 + BN - 1) / BN;

  constexpr int kChunks = D / 8;
  constexpr int kLoads = (BN * kChunks + C::kThreads - 1) / C::kThreads;
  auto issue = [&](int i) {
    const uint32_t dst = smem_u32(smem) + (i % C::kStages) * 2 * C::kStageBytes;
#pragma unroll
    for (int e = 0; e < kLoads; ++e) {
      const int at = tid + C::kThreads * e, r = at / kChunks, c = at % kChunks;
      if (BN * kChunks % C::kThreads != 0 && r >= BN) break;
      const int v = v0 + i * BN + r;
      const long long row = v < v1 ? pool_row(p, seq.table, vis.key(v), h, s) : -1;
      if (c == 0) bad_keys[i % C::kStages][r] = row < 0;
      const long long off = row < 0 ? 0 : row * D + c * 8;
      const int to = tile_offset<D>(r, c);
      cp_async16(dst + to, static_cast<const E *>(p.k_pool) + off, row < 0 ? 0 : 16);
      cp_async16(dst + C::kStageBytes + to, static_cast<const E *>(p.v_pool) + off, row < 0 ? 0 : 16);
    }
  };
  if (steps > 0) issue(0);
  cp_async_commit();

  // This thread's two tile rows.
  int pos[2], head[2], row[2];
  bool used[2];
  uint32_t qa[D / 16][4];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int m = m0 + warp * 16 + gq + 8 * half;
    used[half] = m < total;
    row[half] = used[half] ? m / g : r_hi;
    head[half] = h * g + (used[half] ? m % g : 0);
    pos[half] = seq.first + row[half];
    const E *q = static_cast<const E *>(p.q) + (seq.start + row[half]) * p.q_stride + (long long)head[half] * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qa[kk][half + 2 * i] =
            used[half] ? *reinterpret_cast<const uint32_t *>(q + kk * 16 + 2 * tq + 8 * i) : 0u;
  }
  const float scale = p.scale * kLog2e;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
  bool poisoned = false;

  for (int i = 0; i < steps; ++i) {
    if (i + 1 < steps) issue(i + 1);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t sk = smem_u32(smem) + (i % C::kStages) * 2 * C::kStageBytes, sv = sk + C::kStageBytes;
    const int base = v0 + i * BN, last = min(base + BN, v1) - 1;
    // Every row sees every key of the step, or some pairs are masked.
    const int j0 = vis.key(base), j1 = vis.key(last);
    bool whole = base + BN <= v1 && j1 <= p_lo && (j0 > p_hi - p.window || j1 < p.sinks);
    if (!whole) {
      bool special = false;
#pragma unroll
      for (int e = 0; e < kLoads; ++e) {
        const int at = tid + C::kThreads * e;
        if (at < BN * kChunks)
          special |= any_special(*reinterpret_cast<const uint4 *>(smem + (i % C::kStages) * 2 * C::kStageBytes +
                                                                   C::kStageBytes + at * 16),
                                 exponent_mask(E()));
      }
      if (__syncthreads_or(special)) {
        poisoned = true;
        break;
      }
    }
    bool missing = false;
#pragma unroll
    for (int b = 0; b < BN; b += 16) {
      const uint4 w = *reinterpret_cast<const uint4 *>(&bad_keys[i % C::kStages][b]);
      missing |= (w.x | w.y | w.z | w.w) != 0;
    }
    whole = whole && !missing;
    float sc[BN / 8][4];
#pragma unroll
    for (int nt = 0; nt < BN / 8; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int nt = 0; nt < BN / 8; nt += 2) {
        uint32_t b[4];
        ldmatrix4(b, sk + tile_offset<D>(nt * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
        mma(sc[nt], qa[kk], b[0], b[1], E());
        mma(sc[nt + 1], qa[kk], b[2], b[3], E());
      }
#pragma unroll
    for (int nt = 0; nt < BN / 8; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) sc[nt][c] *= scale;
    if (!whole) {
#pragma unroll
      for (int nt = 0; nt < BN / 8; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = nt * 8 + 2 * tq + (c & 1), v = base + r, j = vis.key(v), at = pos[c >> 1];
          const bool see = v < v1 && j <= at && (at - j < p.window || j < p.sinks) && !bad_keys[i % C::kStages][r];
          if (!see) sc[nt][c] = -INFINITY;
        }
    }
    float rescale[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < BN / 8; ++nt) mx = fmaxf(mx, fmaxf(sc[nt][2 * r], sc[nt][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m_run[r], mx), m_use = m_new == -INFINITY ? 0.0f : m_new;
      rescale[r] = exp2f(m_run[r] - m_use);
      m_run[r] = m_new;
      float sum = 0.0f;
#pragma unroll
      for (int nt = 0; nt < BN / 8; ++nt)
#pragma unroll
        for (int c = 2 * r; c < 2 * r + 2; ++c) {
          sc[nt][c] = exp2f(sc[nt][c] - m_use);
          sum += sc[nt][c];
        }
      l_run[r] = fmaf(l_run[r], rescale[r], sum);  // this thread's columns only, joined at the end
    }
#pragma unroll
    for (int dt = 0; dt < D / 8; ++dt) {
      acc[dt][0] *= rescale[0];
      acc[dt][1] *= rescale[0];
      acc[dt][2] *= rescale[1];
      acc[dt][3] *= rescale[1];
    }
    // P is rounded once to the storage type (its largest entry is at most 1;
    // the sum l is taken before the rounding): each output then carries
    // independent errors of half a step per key, which together stay below
    // the rounding of the output itself.
#pragma unroll
    for (int kk = 0; kk < BN / 16; ++kk) {
      uint32_t pa[4];
      pa[0] = pack2(sc[2 * kk][0], sc[2 * kk][1], E());
      pa[1] = pack2(sc[2 * kk][2], sc[2 * kk][3], E());
      pa[2] = pack2(sc[2 * kk + 1][0], sc[2 * kk + 1][1], E());
      pa[3] = pack2(sc[2 * kk + 1][2], sc[2 * kk + 1][3], E());
#pragma unroll
      for (int dt = 0; dt < D / 8; dt += 2) {
        uint32_t b[4];
        ldmatrix4_trans(b, sv + tile_offset<D>(kk * 16 + (lane & 15), dt + (lane >> 4)));
        mma(acc[dt], pa, b[0], b[1], E());
        mma(acc[dt + 1], pa, b[2], b[3], E());
      }
    }
    __syncthreads();  // the stage is free
  }
  pdl_launch_dependents();
  cp_async_wait<0>();

  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  if (poisoned) {
    for (int r = 0; r < 16; ++r) {
      const int m = m0 + warp * 16 + r;
      if (m >= total) break;
      const int q_row = m / g, q_head = h * g + m % g;
      float mm, ll, o[(D + 31) / 32];
      slow_row<E, D>(p, seq, s, h, q_head, q_row, vis, v0, v1, mm, ll, o, lane);
      const long long slot = ((long long)s * p.max_rows + q_row) * p.hq + q_head;
#pragma unroll
      for (int i = 0; i < (D + 31) / 32; ++i) {
        const int d = lane + 32 * i;
        if (d >= D) break;
        if (splits > 1)
          partial_acc(p, slots, split, slot)[d] = o[i];
        else
          store1(p.out, (seq.start + q_row) * p.out_stride + (long long)q_head * D + d,
                 ll > 0.0f || ll != ll ? o[i] / ll : 0.0f, E());
      }
      if (splits > 1 && lane == 0) *partial_ml(p, slots, splits, split, slot) = make_float2(mm, ll);
    }
    return;
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    l_run[half] += __shfl_xor_sync(0xffffffffu, l_run[half], 1);
    l_run[half] += __shfl_xor_sync(0xffffffffu, l_run[half], 2);
    if (!used[half]) continue;
    const float l = l_run[half];
    if (splits > 1) {
      const long long slot = ((long long)s * p.max_rows + row[half]) * p.hq + head[half];
      float *o = partial_acc(p, slots, split, slot);
#pragma unroll
      for (int dt = 0; dt < D / 8; ++dt)
        *reinterpret_cast<float2 *>(o + dt * 8 + 2 * tq) = make_float2(acc[dt][2 * half], acc[dt][2 * half + 1]);
      if (tq == 0) *partial_ml(p, slots, splits, split, slot) = make_float2(m_run[half], l);
    } else {
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // no visible key: zeros
      E *o = static_cast<E *>(p.out) + (seq.start + row[half]) * p.out_stride + (long long)head[half] * D;
#pragma unroll
      for (int dt = 0; dt < D / 8; ++dt)
        *reinterpret_cast<uint32_t *>(o + dt * 8 + 2 * tq) =
            pack2(acc[dt][2 * half] * inv, acc[dt][2 * half + 1] * inv, E());
    }
  }
}

// ---- joining splits ----------------------------------------------------------------------

// One warp per (sequence, row, head): out = sum_i w_i acc_i / sum_i w_i l_i,
// w_i = 2^(m_i - max m).
template <typename E>
__global__ void __launch_bounds__(128) window_join_kernel(const WindowAttentionParams p, int splits) {
  const int lane = threadIdx.x & 31;
  pdl_wait();
  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  const long long slot = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  if (slot >= slots) return;
  const int head = (int)(slot % p.hq), row = (int)(slot / p.hq % p.max_rows), s = (int)(slot / p.hq / p.max_rows);
  const Sequence seq = load_sequence(p, s, false);
  if (row >= seq.rows) return;
  const float2 ml = lane < splits ? __ldcg(partial_ml(p, slots, splits, lane, slot)) : make_float2(-INFINITY, 0.0f);
  const float m = warp_max(ml.x);
  const float w = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m);
  // A state without weight is skipped whatever its sum (a NaN sum stays NaN).
  const float l = warp_sum(ml.x == -INFINITY ? ml.y : ml.y * w);
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  for (int d0 = 0; d0 < p.d; d0 += 32) {
    const int d = d0 + lane;
    float o = 0.0f;
    for (int i = 0; i < splits; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      if (wi != 0.0f && d < p.d) o = fmaf(__ldcg(partial_acc(p, slots, i, slot) + d), wi, o);
    }
    if (d < p.d) store1(p.out, (seq.start + row) * p.out_stride + (long long)head * p.d + d, o * inv, E());
  }
}

// ---- launches ----------------------------------------------------------------------------

struct Plan {
  bool decode;
  int tiles;    // per (sequence, KV head): head tiles (decode) or row tiles
  int cluster;  // decode: CTAs that join in distributed shared memory
  int outer;    // splits that join through the workspace
};

size_t partial_bytes(int sequences, int max_rows, int hq, int d, int outer) {
  return outer <= 1 ? 0 : (size_t)outer * sequences * max_rows * hq * (d + 2) * sizeof(float);
}

// keys: the most keys a row can see. Splits grow while the GPU has room for
// twice as many CTAs and each still has a few steps of keys.
Plan make_plan(int sequences, int max_rows, int hq, int hkv, long long keys, int num_sms, int max_cluster) {
  const int g = hq / hkv;
  Plan plan{max_rows == 1, 1, 1, 1};
  plan.tiles = plan.decode ? (g + 15) / 16 : (int)(((long long)max_rows * g + 127) / 128);
  const long long ctas = (long long)sequences * hkv * plan.tiles;
  const long long room = 2 * num_sms;
  if (plan.decode)
    while (plan.cluster < max_cluster && ctas * plan.cluster < room && keys > 64 * plan.cluster) plan.cluster *= 2;
  const long long steps = plan.decode ? keys / (64 * plan.cluster) : keys / 64;
  while (plan.outer < kMaxOuter && ctas * plan.cluster * plan.outer * 2 <= room && steps > 4 * plan.outer)
    plan.outer *= 2;
  return plan;
}

long long visible_bound(long long window, long long sinks, int max_rows, long long capacity) {
  const long long keys = window + sinks + (max_rows > 1 ? max_rows : 0);
  return keys < capacity ? keys : capacity;
}

// The largest cluster of decode CTAs this device runs (16 is not portable), set up once.
template <typename E, int D>
cudaError_t decode_cluster_limit(int *limit) {
  static std::mutex mu;
  static std::unordered_map<int, int> limits;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  auto it = limits.find(dev);
  if (it == limits.end()) {
    auto kernel = window_decode_kernel<E, D>;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeCfg<D>::kSmem);
    if (e != cudaSuccess) return e;
    int n = 8;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
      cudaLaunchConfig_t probe = {};
      probe.gridDim = dim3(kMaxCluster, 1, 1);
      probe.blockDim = dim3(128);
      probe.dynamicSmemBytes = DecodeCfg<D>::kSmem;
      cudaLaunchAttribute a;
      a.id = cudaLaunchAttributeClusterDimension;
      a.val.clusterDim.x = kMaxCluster;
      a.val.clusterDim.y = a.val.clusterDim.z = 1;
      probe.attrs = &a;
      probe.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &probe) == cudaSuccess && clusters > 0) n = kMaxCluster;
    }
    (void)cudaGetLastError();
    it = limits.emplace(dev, n).first;
  }
  *limit = it->second;
  return cudaSuccess;
}

template <typename E, int D>
cudaError_t prompt_setup() {
  static std::mutex mu;
  static std::unordered_map<int, bool> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  if (done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(window_prompt_kernel<E, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptCfg<D>::kSmem);
  if (e == cudaSuccess) done[dev] = true;
  return e;
}

template <typename E, int D>
cudaError_t launch(const WindowAttentionParams &p, int num_sms, cudaStream_t stream, bool pdl) {
  static_assert(DecodeCfg<D>::kMerge <= DecodeCfg<D>::kSmem, "warp states fit over the rings");
  static_assert(kMaxCluster * 16 * 8 <= DecodeCfg<D>::kSmem - DecodeCfg<D>::kWarps * 16 * D * 4,
                "the cluster's (m, l) pairs fit behind the warp states");
  int limit = 8;
  cudaError_t e;
  if (p.max_rows == 1) {
    if ((e = decode_cluster_limit<E, D>(&limit)) != cudaSuccess) return e;
  } else if ((e = prompt_setup<E, D>()) != cudaSuccess) {
    return e;
  }
  const long long keys = visible_bound(p.window, p.sinks, p.max_rows, p.capacity);
  Plan plan = make_plan(p.sequences, p.max_rows, p.hq, p.hkv, keys, num_sms, limit);
  while (plan.outer > 1 &&
         (p.workspace == nullptr ||
          partial_bytes(p.sequences, p.max_rows, p.hq, D, plan.outer) > p.workspace_bytes))
    plan.outer /= 2;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cfg.attrs = attr;
  auto add_pdl = [&] {
    if (!pdl) return;
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  };
  if (plan.decode) {
    cfg.gridDim = dim3(plan.cluster * plan.outer, p.hkv * plan.tiles, p.sequences);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = DecodeCfg<D>::kSmem;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = plan.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    add_pdl();
    e = cudaLaunchKernelEx(&cfg, window_decode_kernel<E, D>, p, plan.tiles, plan.cluster);
  } else {
    cfg.gridDim = dim3((unsigned)(plan.tiles * plan.outer), p.hkv, p.sequences);
    cfg.blockDim = dim3(PromptCfg<D>::kThreads);
    cfg.dynamicSmemBytes = PromptCfg<D>::kSmem;
    add_pdl();
    e = cudaLaunchKernelEx(&cfg, window_prompt_kernel<E, D>, p, plan.outer);
  }
  if (e != cudaSuccess || plan.outer == 1) return e;
  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  cfg.gridDim = dim3((unsigned)((slots + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 0;
  add_pdl();
  return cudaLaunchKernelEx(&cfg, window_join_kernel<E>, p, plan.outer);
}

template <typename E>
cudaError_t dispatch(const WindowAttentionParams &p, int num_sms, cudaStream_t stream, bool pdl) {
  switch (p.d) {
    case 16: return launch<E, 16>(p, num_sms, stream, pdl);
    case 32: return launch<E, 32>(p, num_sms, stream, pdl);
    case 64: return launch<E, 64>(p, num_sms, stream, pdl);
    case 128: return launch<E, 128>(p, num_sms, stream, pdl);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

size_t window_attention_workspace_bytes(int sequences, int max_rows, int hq, int hkv, int d, long long window,
                                        long long sinks, int num_sms) {
  if (sequences <= 0 || max_rows <= 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || d <= 0 || window <= 0 || sinks < 0)
    return 0;
  const long long keys = visible_bound(window, sinks, max_rows, 0x7fffffffll);
  size_t most = 0;
  for (int cluster = 8; cluster <= kMaxCluster; cluster *= 2) {
    const Plan plan = make_plan(sequences, max_rows, hq, hkv, keys, num_sms, cluster);
    const size_t bytes = partial_bytes(sequences, max_rows, hq, d, plan.outer);
    most = bytes > most ? bytes : most;
  }
  return most;
}

cudaError_t launch_window_attention(const WindowAttentionParams &p, bool bf16, int num_sms, cudaStream_t stream,
                                    bool pdl) {
  if (p.sequences <= 0 || p.sequences > 65535 || p.rows < 0 || p.max_rows <= 0 || p.hkv <= 0 || p.hq <= 0 ||
      p.hq % p.hkv != 0 || p.page_size <= 0 || p.pool_pages <= 0 || p.table_stride <= 0 || p.capacity <= 0 ||
      p.window <= 0 || p.sinks < 0 || p.q_stride % 8 != 0 || p.out_stride % 8 != 0)
    return cudaErrorInvalidValue;
  const long long g = p.hq / p.hkv;
  if ((long long)p.hkv * ((g + 15) / 16) > 65535 || (long long)p.max_rows * g > (1ll << 30) / kMaxOuter ||
      (long long)p.sequences * p.max_rows > (1ll << 32) / p.hq)
    return cudaErrorInvalidValue;
  return bf16 ? dispatch<__nv_bfloat16>(p, num_sms, stream, pdl) : dispatch<__half>(p, num_sms, stream, pdl);
}

}  // namespace tmc
