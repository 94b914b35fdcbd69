// Window attention with sinks over the paged cache (window_attention.cuh).
//
// One pass over the visible keys with a running maximum and sum per query row:
// S = scale log2(e) Q K^T, p = 2^(S - m), O += P V, and O / l at the end, S and
// O in fp32. The G = Hq / Hkv query heads of a KV head are rows of the same
// tile, so a key is read once for all of them. The visible keys of a tile are
// numbered without a gap: the sinks before the window, then the window's run.
//
// - decode (one row per sequence, or few): bound by the reads of K and V, G products a
//   key, so mma.sync m16n8k16 keeps up. A warp takes 16 keys at a time through
//   a ring of its own, with no barrier between warps; the warps of a CTA, and
//   the CTAs of a cluster, split the keys and join their states in shared and
//   distributed shared memory. Heads of 128, 8 KV heads: 64 sequences of 700 to
//   8192 positions, window 4096, 146 us (5.9 TB/s, 0.91 of a copy's rate); one
//   sequence, window 1024, 7.0 us, which is launch, three dependent reads
//   (sequence, table, keys) and the joins.
//   Prompts of a few rows run the same way, each row with its own mask.
// - prompts with heads of 64 and 128 run in window_tensor.cu. Short heads (16,
//   32) have a quarter of the products or less per exponential and stay on
//   mma.sync: a CTA holds 128 query rows x heads, its warps 16 each, and all
//   share 64-key tiles.
// When a launch has too few CTAs for the GPU its splits write their states to
// the workspace, and a second kernel joins them.
#include "window_attention.cuh"

#include <map>
#include <mutex>
#include <utility>

#include "window_device.cuh"
#include "window_plan.hpp"

namespace tmc {
namespace {

using namespace window;

// Add a state's weighted part: ml its (maximum, sum), m the maximum over all.
__device__ __forceinline__ void join_part(const float2 &ml, const float4 &x, float m, float &l, float4 &o) {
  const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m);
  l = fmaf(ml.y, f, l);
  o.x = fmaf(x.x, f, o.x);
  o.y = fmaf(x.y, f, o.y);
  o.z = fmaf(x.z, f, o.z);
  o.w = fmaf(x.w, f, o.w);
}

// Stores to the same variable in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t in_cta(const void *local, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_cluster(const float *local, int rank, const float4 &v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(in_cta(local, rank)), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ void store_cluster(const float2 *local, int rank, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(in_cta(local, rank)), "f"(a), "f"(b) : "memory");
}

// ---- decode: one row per sequence, or a few ------------------------------------------------

template <int D>
struct DecodeCfg {
  static constexpr int kWarps = 4;
  static constexpr int kStages = 2;                    // 16-key stages of a warp's ring
  static constexpr int kStageBytes = 16 * D * 2;       // one of K or V
  static constexpr int kRing = kWarps * kStages * 2 * kStageBytes;
  static constexpr int kMerge = kWarps * (16 * D + 32) * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
  // and the parts that a cluster's CTAs send: a share each of `rows` tile rows
  static constexpr int smem(int rows) { return kSmem + (rows * D + 4 * kMaxCluster) * 4; }
};

// An infinite value times both parts of a weight is NaN where the low part is 0
// or negative. A thread that has written a NaN although the row's sum is none
// puts the sum of the values that are not finite in its place, looked for among
// the keys once more: an infinity, or NaN. It finds its place anew: what the
// kernel would have to keep for it slows its loop down (64 sequences 160 us for
// 146, with the loop below inside the kernel).
template <typename E, int D, bool ROWS>
__device__ __noinline__ void infinite_values(const WindowAttentionParams &p, int tiles, int cluster) {
  const int s = blockIdx.z, h = blockIdx.y / tiles, m0 = blockIdx.y % tiles * 16, splits = gridDim.x;
  const int crank = blockIdx.x % cluster, outer = blockIdx.x / cluster, outers = splits / cluster;
  const Sequence seq = load_sequence(p, s, false);
  const int g = p.hq / p.hkv, used = min(16, seq.rows * g - m0);
  auto row_of = [&](int r) { return ROWS ? (m0 + r) / g : 0; };
  const Visible vis = visible_keys(p, seq.first + row_of(0), seq.first + row_of(used - 1));
  const int chunk = ((vis.count + splits - 1) / splits + 15) / 16 * 16;
  const int v0 = min(vis.count, outer * cluster * chunk), v1 = min(vis.count, v0 + cluster * chunk);
  const int share = ((used * D + cluster - 1) / cluster + 3) & ~3;
  const int e1 = min(used * D, (crank + 1) * share);
  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  for (int i = crank * share + (int)threadIdx.x * 4; i < e1; i += 128 * 4) {
    const int r = i / D, d = i % D, row = row_of(r), head = h * g + m0 + r - row * g, at = seq.first + row;
    float sum[4] = {};
    for (int v = v0; v < v1; ++v) {
      const int j = vis.key(v);
      if (j > at || (at - j >= p.window && j >= p.sinks)) continue;
      const KeyPlace k = find_key(p, seq.table, j);
      if (k.page < 0 || k.page >= p.pool_pages) continue;
      const E *x = static_cast<const E *>(p.v_pool) + (((long long)k.page * p.hkv + h) * p.page_size + k.offset) * D + d;
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] += isfinite((float)x[c]) ? 0.0f : (float)x[c];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (sum[c] == 0.0f) continue;
      if (outers > 1)
        partial_acc(p, slots, outer, ((long long)s * p.max_rows + row) * p.hq + head)[d + c] = sum[c];
      else
        store1(p.out, (seq.start + row) * p.out_stride + (long long)head * D + d + c, sum[c], E());
    }
  }
}

// Grid (splits, Hkv x tiles, sequences), clusters of `cluster` CTAs along the
// splits; outer = splits / cluster of them meet in the workspace. A tile is 16
// of the (row, head of the KV head) pairs, heads fastest. ROWS: sequences may
// have several rows, whose masks differ.
template <typename E, int D, bool ROWS>
__global__ void __launch_bounds__(128, kDecodePerSm)
    window_decode_kernel(const __grid_constant__ WindowAttentionParams p, int tiles, int cluster) {
  using C = DecodeCfg<D>;
  constexpr int S = C::kStages;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int bad_keys[C::kWarps][S];        // a stage's keys whose page is missing
  __shared__ float2 recv_ml[kMaxCluster][16];   // (m, l) per tile row, from the cluster's CTAs
  float *recv = reinterpret_cast<float *>(smem + C::kSmem);  // their parts of this CTA's share of the results
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3;
  if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  const int s = blockIdx.z, h = blockIdx.y / tiles, m0 = blockIdx.y % tiles * 16;
  const int split = blockIdx.x, splits = gridDim.x;
  const Sequence seq = load_sequence(p, s, blockIdx.x == 0 && blockIdx.y == 0 && tid == 0);
  const int g = p.hq / p.hkv, used = min(16, seq.rows * g - m0);  // tile rows
  if (used <= 0) {  // the same for every CTA of the cluster
    if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }
  auto row_of = [&](int r) { return ROWS ? (m0 + r) / g : 0; };  // of tile row r
  auto head_of = [&](int r) { return h * g + m0 + r - row_of(r) * g; };
  const int p_lo = seq.first + row_of(0), p_hi = seq.first + row_of(used - 1);
  const Visible vis = visible_keys(p, p_lo, p_hi);
  const int chunk = ((vis.count + splits - 1) / splits + 15) / 16 * 16;
  const int v0 = min(vis.count, split * chunk), v1 = min(vis.count, v0 + chunk);
  const int groups = (v1 - v0 + 15) / 16;
  const int mine = groups > warp ? (groups - warp + C::kWarps - 1) / C::kWarps : 0;

  unsigned char *ring = smem + warp * (S * 2 * C::kStageBytes);
  const uint32_t ring_addr = smem_u32(ring);
  // The place of this lane's key (lane & 15) of stage i, looked up one stage
  // ahead: nothing waits for the table entry until the stage is issued.
  auto lookup = [&](int i) {
    const int v = v0 + (warp + C::kWarps * i) * 16 + (lane & 15);
    return i < mine && v < v1 ? find_key(p, seq.table, vis.key(v)) : KeyPlace{0, -1, 0};
  };
  constexpr int kChunks = D / 8;               // 16-byte chunks of a row
  constexpr int kLoads = 16 * kChunks / 32;    // of K (and of V) per lane and stage
  KeyPlace next = lookup(0);
  auto issue = [&](int i) {
    const int v = v0 + (warp + C::kWarps * i) * 16 + (lane & 15);
    const long long next_row = v < v1 ? pool_row(p, next, h, s) : -1;
    const unsigned bad = __ballot_sync(0xffffffffu, next_row < 0 && v < v1) & 0xffffu;
    next = lookup(i + 1);
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
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < mine) issue(i);
    cp_async_commit();
  }

  // Query fragments and positions of the tile rows gq and gq + 8.
  uint32_t qa[D / 16][4];
  int pos[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = min(gq + 8 * half, used - 1);
    const bool there = gq + 8 * half < used;
    pos[half] = seq.first + row_of(r);
    const E *q = static_cast<const E *>(p.q) + (seq.start + row_of(r)) * p.q_stride + (long long)head_of(r) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qa[kk][half + 2 * i] = there ? *reinterpret_cast<const uint32_t *>(q + kk * 16 + 2 * tq + 8 * i) : 0u;
  }
  bool poisoned = false;  // an infinity or NaN beside masked pairs
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
    if (ROWS) {
      const int v = v1 - left, j0 = vis.key(v), j1 = vis.key(v + min(left, 16) - 1);
      if (j1 > p_lo || (j0 <= p_hi - p.window && j1 >= p.sinks)) {  // not every row sees every key
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = vis.key(v + nt * 8 + 2 * tq + (j & 1)), at = pos[j >> 1];
            if (k > at || (at - k >= p.window && k >= p.sinks)) sc[nt][j] = -INFINITY;
          }
#pragma unroll
        for (int e = 0; e < kLoads; ++e)
          poisoned |= any_special(*reinterpret_cast<const uint4 *>(ring + (i % S) * 2 * C::kStageBytes +
                                                                   C::kStageBytes + (lane + 32 * e) * 16),
                                  exponent_mask(E()));
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

  // Join the warps: their states in shared memory, over the rings.
  float *w_acc = reinterpret_cast<float *>(smem);                                  // [warp][16][D]
  float2 *w_ml = reinterpret_cast<float2 *>(smem + C::kWarps * 16 * D * 4);        // [warp][16]
  if (ROWS && __syncthreads_or(poisoned)) {  // the rows again, by plain loops; one state each
    for (int r = warp; r < used; r += C::kWarps) {
      float mm, ll, o[(D + 31) / 32];
      slow_row<E, D>(p, seq, s, h, head_of(r), row_of(r), vis, v0, v1, mm, ll, o, lane);
      for (int w = 0; w < C::kWarps; ++w) {
#pragma unroll
        for (int n = 0; n < (D + 31) / 32; ++n)
          if (lane + 32 * n < D) w_acc[(w * 16 + r) * D + lane + 32 * n] = w == 0 ? o[n] : 0.0f;
        if (lane == 0) w_ml[w * 16 + r] = w == 0 ? make_float2(mm, ll) : make_float2(-INFINITY, 0.0f);
      }
    }
  } else {
    if (!ROWS) __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = gq + 8 * half;
      if (r >= used) break;
#pragma unroll
      for (int dt = 0; dt < D / 8; ++dt)
        *reinterpret_cast<float2 *>(w_acc + (warp * 16 + r) * D + dt * 8 + 2 * tq) =
            make_float2(acc[dt][2 * half], acc[dt][2 * half + 1]);
      if (tq == 0) w_ml[warp * 16 + r] = make_float2(m_run[half], l_run[half]);
    }
  }
  __syncthreads();
  // Join the warps' states, then the CTAs': CTA c of the cluster owns the
  // elements [c share, (c + 1) share) of the tile's results; every CTA
  // stores its part of them, and its (m, l), in the owner's shared memory, and
  // after one barrier each owner joins what it was sent.
  const int crank = split % cluster, outer = split / cluster, outers = splits / cluster;
  const int share = ((used * D + cluster - 1) / cluster + 3) & ~3;
  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  bool lost = false;  // a NaN of this thread's
  auto finish = [&](int i, const float4 &o, float m, float l) {  // elements i .. i + 3, of one row
    const int row = row_of(i / D), head = head_of(i / D);
    const float all = (o.x + o.y) + (o.z + o.w);
    lost |= all != all && l == l;
    if (outers > 1) {
      const long long slot = ((long long)s * p.max_rows + row) * p.hq + head;
      *reinterpret_cast<float4 *>(partial_acc(p, slots, outer, slot) + i % D) = o;
      if (i % D == 0) *partial_ml(p, slots, outers, outer, slot) = make_float2(m, l);
    } else {
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // no visible key: zeros
      *reinterpret_cast<uint2 *>(static_cast<E *>(p.out) + (seq.start + row) * p.out_stride + (long long)head * D +
                                 i % D) = make_uint2(pack2(o.x * inv, o.y * inv, E()), pack2(o.z * inv, o.w * inv, E()));
    }
  };
  if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA has started
  for (int i = tid * 4; i < used * D; i += 128 * 4) {
    const int r = i / D;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) m = fmaxf(m, w_ml[w * 16 + r].x);
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) join_part(w_ml[w * 16 + r], *reinterpret_cast<const float4 *>(w_acc + w * 16 * D + i), m, l, o);
    if (cluster == 1) {
      finish(i, o, m, l);
      continue;
    }
    const int owner = i / share;
    store_cluster(recv + crank * share + (i - owner * share), owner, o);
    if (i % D / 4 < cluster) store_cluster(&recv_ml[crank][r], i % D / 4, m, l);
    if (D / 4 < cluster && i % D == 0)
      for (int c = D / 4; c < cluster; ++c) store_cluster(&recv_ml[crank][r], c, m, l);
  }
  if (cluster == 1) {
    if (lost) infinite_values<E, D, ROWS>(p, tiles, cluster);
    return;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int e0 = crank * share, e1 = min(used * D, e0 + share);
  for (int i = e0 + tid * 4; i < e1; i += 128 * 4) {
    const int r = i / D;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c)
      if (c < cluster) m = fmaxf(m, recv_ml[c][r].x);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c)
      if (c < cluster) join_part(recv_ml[c][r], *reinterpret_cast<const float4 *>(recv + c * share + i - e0), m, l, o);
    finish(i, o, m, l);
  }
  if (lost) infinite_values<E, D, ROWS>(p, tiles, cluster);
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

// Grid as prompt_place counts it. Tile t holds the tile rows t BM .. t BM + BM - 1
// of the sequence's (row, head of the KV head) pairs, heads fastest.
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
  const PromptPlace place = prompt_place(p, splits);
  const int s = place.seq, h = place.head, split = place.split;
  const Sequence seq = load_sequence(p, s, place.first && tid == 0);
  const int g = p.hq / p.hkv;
  const int m0 = place.tile * C::BM, total = seq.rows * g;
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
      const long long row = v < v1 ? pool_row(p, find_key(p, seq.table, vis.key(v)), h, s) : -1;
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
    // the sum l is taken before the rounding), as in window_tensor.cu: an output
    // is off by 2^-11 (fp16) or 2^-8 (bf16) of sum p |v| at most, beside its own
    // rounding.
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

  bool lost = false;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float2 sum{};
#pragma unroll
    for (int dt = 0; dt < D / 8; ++dt) note_finite(sum, acc[dt][2 * half], acc[dt][2 * half + 1]);
    const float all = sum.x + sum.y;
    lost |= all != all && l_run[half] == l_run[half];
  }

  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  if (poisoned || __any_sync(0xffffffffu, lost)) {
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

// out = sum_i w_i acc_i / sum_i w_i l_i with w_i = 2^(m_i - max m). Grid (rows
// of a sequence, sequences, head groups); a thread owns four elements of one
// head. Empty splits hold no sums: their weight is 0 and they are left out.
// (A thread per element that found its place by divisions took 33 us where
// this takes 5: 256 rows of 32 heads, three splits.)
constexpr int kJoinThreads = 128;
template <typename E, int D>
__global__ void __launch_bounds__(kJoinThreads) window_join_kernel(const WindowAttentionParams p, int splits) {
  constexpr int kHeads = kJoinThreads * 4 / D;  // of a group
  __shared__ float2 parts[kHeads][kMaxOuter];   // (m, l)
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x, s = blockIdx.y, h0 = blockIdx.z * kHeads, tid = threadIdx.x;
  const int heads = min(kHeads, p.hq - h0);
  const Sequence seq = load_sequence(p, s, false);
  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  const long long slot0 = ((long long)s * p.max_rows + row) * p.hq + h0;
  if (row >= seq.rows) return;
  for (int i = tid; i < heads * kMaxOuter; i += kJoinThreads) {
    const int h = i / kMaxOuter, n = i % kMaxOuter;
    if (n < splits) parts[h][n] = __ldcg(partial_ml(p, slots, splits, n, slot0 + h));
  }
  const int h = tid / (D / 4), d = tid % (D / 4) * 4;
  const bool own = h < heads;
  const float *acc = partial_acc(p, slots, 0, slot0 + (own ? h : 0)) + d;
  constexpr int kBatch = 8;
  float4 x[kBatch];
  auto load = [&](int n0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (n0 + i < splits) x[i] = __ldcg(reinterpret_cast<const float4 *>(acc + (n0 + i) * slots * D));
  };
  load(0);
  __syncthreads();
  if (!own) return;
  float m = -INFINITY, l = 0.0f;
  for (int n = 0; n < splits; ++n) m = fmaxf(m, parts[h][n].x);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int n0 = 0; n0 < splits; n0 += kBatch) {
    if (n0 > 0) load(n0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (n0 + i >= splits) break;
      const float2 ml = parts[h][n0 + i];
      if (ml.x == -INFINITY)
        l += ml.y;  // nothing but its sum counts: 0, or NaN
      else
        join_part(ml, x[i], m, l, o);
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  *reinterpret_cast<uint2 *>(static_cast<E *>(p.out) + (seq.start + row) * p.out_stride + (long long)(h0 + h) * D + d) =
      make_uint2(pack2(o.x * inv, o.y * inv, E()), pack2(o.z * inv, o.w * inv, E()));
}

// ---- launches ----------------------------------------------------------------------------

// Allows a kernel its dynamic shared memory, once per device.
cudaError_t allow_smem(const void *kernel, int bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, const void *>, bool> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  bool &set = done[{dev, kernel}];
  if (!set && (e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) == cudaSuccess)
    set = true;
  return e;
}

template <typename E, int D>
cudaError_t launch(const WindowAttentionParams &p, int num_sms, cudaStream_t stream, bool pdl) {
  using C = DecodeCfg<D>;
  static_assert(C::kMerge <= C::kSmem, "warp states fit over the rings");
  static_assert(kDecodePerSm * (C::smem(16) + 1024 + 1280) <= 228 * 1024, "CTAs that an SM holds");
  const long long keys = visible_bound(p.window, p.sinks, p.max_rows, p.capacity);
  Plan plan = make_plan(p.sequences, p.max_rows, p.hq, p.hkv, D, keys, num_sms);
  while (plan.outer > 1 &&
         (p.workspace == nullptr ||
          partial_bytes(p.sequences, p.max_rows, p.hq, D, plan.outer) > p.workspace_bytes))
    plan.outer /= 2;
  if (!plan.decode && (long long)plan.tiles * plan.outer * p.hkv > 0x7fffffffll / p.sequences)
    return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cfg.attrs = attr;
  auto add_pdl = [&] {
    if (!pdl) return;
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  };
  cudaError_t e;
  if (plan.decode) {
    const auto kernel = p.max_rows == 1 ? window_decode_kernel<E, D, false> : window_decode_kernel<E, D, true>;
    if ((e = allow_smem(reinterpret_cast<const void *>(kernel), C::smem(16))) != cudaSuccess) return e;
    const long long rows = (long long)p.max_rows * (p.hq / p.hkv);
    cfg.gridDim = dim3(plan.cluster * plan.outer, p.hkv * plan.tiles, p.sequences);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = C::smem(rows < 16 ? (int)rows : 16);
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = plan.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    add_pdl();
    e = cudaLaunchKernelEx(&cfg, kernel, p, plan.tiles, plan.cluster);
  } else if constexpr (D == 64 || D == 128) {
    e = launch_window_tensor(p, std::is_same<E, __nv_bfloat16>::value, plan.tiles, plan.outer, stream, pdl);
  } else {
    const auto kernel = window_prompt_kernel<E, D>;
    if ((e = allow_smem(reinterpret_cast<const void *>(kernel), PromptCfg<D>::kSmem)) != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned)((long long)plan.tiles * plan.outer * p.hkv * p.sequences));
    cfg.blockDim = dim3(PromptCfg<D>::kThreads);
    cfg.dynamicSmemBytes = PromptCfg<D>::kSmem;
    add_pdl();
    e = cudaLaunchKernelEx(&cfg, kernel, p, plan.outer);
  }
  if (e != cudaSuccess || plan.outer == 1) return e;
  constexpr int kHeads = kJoinThreads * 4 / D;
  cfg.gridDim = dim3(p.max_rows, p.sequences, (p.hq + kHeads - 1) / kHeads);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 0;
  pdl = true;  // its launch overlaps the splits' end, which it waits for
  add_pdl();
  return cudaLaunchKernelEx(&cfg, window_join_kernel<E, D>, p, plan.outer);
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
  if (!can_plan(sequences, max_rows, hq, hkv) || d <= 0 || window <= 0 || sinks < 0) return 0;
  return partial_bytes(sequences, max_rows, hq, d,
                       most_splits(sequences, max_rows, hq, hkv, d,
                                   visible_bound(window, sinks, max_rows, 0x7fffffffll), num_sms));
}

int window_attention_launches(int sequences, int max_rows, int hq, int hkv, int d, long long window, long long sinks,
                              long long capacity, int num_sms) {
  if (!can_plan(sequences, max_rows, hq, hkv)) return 1;
  const long long keys = visible_bound(window, sinks, max_rows, capacity);
  return make_plan(sequences, max_rows, hq, hkv, d, keys, num_sms).outer > 1 ? 2 : 1;
}

cudaError_t launch_window_attention(const WindowAttentionParams &p, bool bf16, int num_sms, cudaStream_t stream,
                                    bool pdl) {
  if (!can_plan(p.sequences, p.max_rows, p.hq, p.hkv) || p.rows < 0 || p.page_size <= 0 || p.pool_pages <= 0 || p.table_stride <= 0 || p.capacity <= 0 ||
      p.window <= 0 || p.sinks < 0 || p.q_stride % 8 != 0 || p.out_stride % 8 != 0)
    return cudaErrorInvalidValue;
  if ((long long)p.pool_pages * p.hkv > (1ll << 32) / p.page_size - 1)  // pool rows are counted in 32 bits
    return cudaErrorInvalidValue;
  WindowAttentionParams q = p;
  q.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p.page_size == 1 << i) q.page_shift = i;
  return bf16 ? dispatch<__nv_bfloat16>(q, num_sms, stream, pdl) : dispatch<__half>(q, num_sms, stream, pdl);
}

}  // namespace tmc
