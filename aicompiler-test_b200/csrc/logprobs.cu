// Token log probabilities, entropy, rank and top alternatives (logprobs.cuh).
//
// For a row x of V logits and a number m near its maximum, with
//   s = sum e^(x - m),  u = sum e^(x - m) (x - m)
// the log normaliser is m + log s, the target's log probability
// (x_t - m) - log s and the entropy log s - u / s. One pass over the row keeps
// (m, s, u) per thread, rescaled when the running maximum rises, and counts
// the logits that come before the target (larger, or equal at a lower index).
// u is summed about (nearly) the maximum so that a peaked row's small entropy
// does not come out as a difference of two large numbers.
//
// The top alternatives come from the same read. Every thread keeps its largest
// logit; the top-th largest of each warp's four best of these is reached by at
// least `top` logits, so it bounds the CTA's top-th logit from below. The few
// threads whose own largest reaches it are read again (from L2), what reaches
// the bound is collected, and each of these candidates finds its place by
// counting the larger ones. Rows with too many candidates (long runs of equal
// logits) or too few threads with a logit above -inf are read again as a whole,
// every warp keeping a sorted list.
//
// A row is shared by a thread-block cluster when there are few rows; its CTAs
// hand their (m, s, u), counts and top lists to the cluster's first CTA
// through distributed shared memory.
//
// Bound: many rows by issue slots (11.5 instructions a logit of 16 bits, of
// which two for the exponential; 1500 rows of 50021 bf16 38 us, 3.9 TB/s, with
// the last of two and a half rounds of CTAs part empty); one row of 128256 fp32
// 8.1 us, by the chain of launch, reads, candidates and the cluster's joins.
#include "logprobs.cuh"

#include <cuda_bf16.h>

#include "mbarrier.cuh"

namespace tmc {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
static_assert(kMaxCluster <= kWarps, "a warp for each CTA's list");
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

using Key = unsigned long long;

// kVec logits of a 16-byte vector: unpacked to fp32, their maximum (NaN only
// if all are), and how many exceed (or reach) a threshold.
template <typename T>
struct Logit;
template <>
struct Logit<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float get(const float *p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint4 &v, float *x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float largest(const uint4 &v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  template <bool REACH>
  static __device__ __forceinline__ float above(const uint4 &v, float t) {
    float x[4];
    unpack(v, x);
    float n = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += (REACH ? x[i] >= t : x[i] > t) ? 1.0f : 0.0f;
    return n;
  }
};
// Two logits to a register: the maximum and the comparisons take them in pairs.
template <typename H, typename H2>
struct PairLogit {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ H2 pair(uint32_t w) { return *reinterpret_cast<const H2 *>(&w); }
  static __device__ __forceinline__ float2 both(const H2 &h);
  static __device__ __forceinline__ void unpack(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = both(pair(w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float largest(const uint4 &v) {
    const float2 f = both(__hmax2(__hmax2(pair(v.x), pair(v.y)), __hmax2(pair(v.z), pair(v.w))));
    return fmaxf(f.x, f.y);
  }
  // t is a logit of this type: exact in it. The counts of a pair add up in the
  // type itself, where they are whole numbers up to 4.
  template <bool REACH>
  static __device__ __forceinline__ float above(const uint4 &v, const H2 &t) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    H2 n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = REACH ? __hge2(pair(w[i]), t) : __hgt2(pair(w[i]), t);
    const float2 f = both(__hadd2(__hadd2(n[0], n[1]), __hadd2(n[2], n[3])));
    return f.x + f.y;
  }
};
template <>
__device__ __forceinline__ float2 PairLogit<__half, __half2>::both(const __half2 &h) {
  return __half22float2(h);
}
template <>
__device__ __forceinline__ float2 PairLogit<__nv_bfloat16, __nv_bfloat162>::both(const __nv_bfloat162 &h) {
  const uint32_t w = *reinterpret_cast<const uint32_t *>(&h);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
struct Logit<__half> : PairLogit<__half, __half2> {
  static __device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
  template <bool REACH>
  static __device__ __forceinline__ float above(const uint4 &v, float t) {
    return PairLogit::above<REACH>(v, __float2half2_rn(t));
  }
};
template <>
struct Logit<__nv_bfloat16> : PairLogit<__nv_bfloat16, __nv_bfloat162> {
  static __device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
  template <bool REACH>
  static __device__ __forceinline__ float above(const uint4 &v, float t) {
    return PairLogit::above<REACH>(v, __float2bfloat162_rn(t));
  }
};

// Running (maximum, sum e^(x-m), sum e^(x-m) (x-m)) of a softmax.
struct Stats {
  float m, s, u;
};
__device__ __forceinline__ Stats empty_stats() { return {-INFINITY, 0.0f, 0.0f}; }

// The statistics about another maximum m >= a.m. A part without finite weight
// (a.m = -inf: nothing but masked logits) has s = u = 0, or NaN.
__device__ __forceinline__ void move_to(Stats &a, float m) {
  if (m == a.m) return;
  const float d = fmaxf(a.m - m, -1e30f), f = exp2f(d * kLog2e);
  a.u = fmaf(a.s, d, a.u) * f;
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ Stats warp_join(Stats a) {
  move_to(a, warp_max(a.m));
  return {a.m, warp_sum(a.s), warp_sum(a.u)};
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2^x, 0 below the normal range
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// A thread's pass over its logits. Four partial sums, so that successive
// logits do not wait for one another.
template <typename T>
struct Pass {
  using L = Logit<T>;
  static constexpr int N = L::kVec;
  float m = -INFINITY;
  float2 s[2] = {}, u[2] = {};
  float before = 0.0f;     // logits before the target: a whole number below 2^24
  float best = -INFINITY;  // the largest logit, and the first index of the vector that holds it
  int best_at = -1;

  // The sums are about m, which follows the maximum only when it has risen by
  // more than kSlack (weights of up to e^kSlack lose no precision): rescaling
  // at every rise of any of a warp's 32 maxima cost a third of the time.
  static constexpr float kSlack = 8.0f;
  __device__ __forceinline__ void raise(float mx, int at) {
    if (mx > best) {
      best = mx;
      best_at = at;
    }
    if (mx > m + kSlack) {
      if (m != -INFINITY) {
        const float d = fmaxf(m - mx, -1e30f), f = exp2f(d * kLog2e);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u[i] = make_float2(fmaf(s[i].x, d, u[i].x) * f, fmaf(s[i].y, d, u[i].y) * f);
          s[i] = make_float2(s[i].x * f, s[i].y * f);
        }
      }
      m = mx;
    }
  }
  // Two logits at once (packed fp32 arithmetic) into partial sums i.
  __device__ __forceinline__ void weigh(float x0, float x1, float about, int i) {
    // A masked logit (-inf) or one far below the maximum: 0 times a finite number.
    float2 d = __fadd2_rn(make_float2(x0, x1), make_float2(-about, -about));
    d = make_float2(max_or_nan(d.x, -1e4f), max_or_nan(d.y, -1e4f));
    const float2 t = __fmul2_rn(d, make_float2(kLog2e, kLog2e));
    const float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
    s[i & 1] = __fadd2_rn(s[i & 1], e);
    u[i & 1] = __ffma2_rn(e, d, u[i & 1]);
  }
  // Before the target come the larger logits behind it and those below it that
  // reach `reach`: its logit, or NaN (none) for a target at -inf, which all
  // lower indices come before.
  static __device__ __forceinline__ bool comes_before(float x, int at, float xt, float reach, int target) {
    return (at > target && x > xt) || (at < target && x >= reach);
  }
  // One logit.
  __device__ __forceinline__ void take(float x, int at, float xt, float reach, int target) {
    raise(x, at);
    weigh(x, -INFINITY, m == -INFINITY ? 0.0f : m, 0);  // -inf weighs nothing
    before += comes_before(x, at, xt, reach, target) ? 1.0f : 0.0f;
  }
  // V vectors, `step` vectors apart, the first at index `at`.
  template <int V>
  __device__ __forceinline__ void take(const uint4 *raw, int at, int step, float xt, float reach, int target) {
    float mx[V];
#pragma unroll
    for (int v = 0; v < V; ++v) mx[v] = L::largest(raw[v]);
#pragma unroll
    for (int v = 0; v < V; ++v) raise(mx[v], at + v * step * N);
    const float about = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float x[N];
      L::unpack(raw[v], x);
#pragma unroll
      for (int i = 0; i < N; i += 2) weigh(x[i], x[i + 1], about, i / 2);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int first = at + v * step * N;
      if (first > target) {
        before += L::template above<false>(raw[v], xt);
      } else if (first + N <= target) {
        before += L::template above<true>(raw[v], reach);
      } else {
        float x[N];
        L::unpack(raw[v], x);
#pragma unroll
        for (int i = 0; i < N; ++i) before += comes_before(x[i], first + i, xt, reach, target) ? 1.0f : 0.0f;
      }
    }
  }
  __device__ __forceinline__ Stats stats() const {
    return {m, (s[0].x + s[0].y) + (s[1].x + s[1].y), (u[0].x + u[0].y) + (u[1].x + u[1].y)};
  }
};

// Larger logits first, then lower indices; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ Key order_key(float x, int index) { return argmax_key(__fadd_rn(x, 0.0f), index); }
__device__ __forceinline__ uint32_t order_value(float x) { return (uint32_t)(order_key(x, 0) >> 32); }

__device__ __forceinline__ Key shfl_key(Key k, int lane) { return __shfl_sync(0xffffffffu, k, lane); }
// The 32 largest of two descending lists of 32 (one key of each per lane), descending.
__device__ __forceinline__ Key warp_merge(Key a, Key b, int lane) {
  const Key r = shfl_key(b, 31 - lane);
  Key k = a > r ? a : r;
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) {
    const Key o = __shfl_xor_sync(0xffffffffu, k, step);
    k = (lane & step) == 0 ? (k > o ? k : o) : (k < o ? k : o);
  }
  return k;
}

// Warp 0 merges `lists` descending lists of 32 keys in shared memory; every
// warp's list has been written.
__device__ __forceinline__ Key merge_lists(const Key *lists, int n, int lane) {
  Key k = lists[lane];
  for (int i = 1; i < n; ++i) k = warp_merge(k, lists[i * 32 + lane], lane);
  return k;
}

// What a CTA hands to the cluster's first CTA.
struct Part {
  Stats st;
  int before;
  Key top[32];
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of a shared variable in the cluster's first CTA, and stores to it.
__device__ __forceinline__ uint32_t in_first_cta(const void *local) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(local)));
  return r;
}
__device__ __forceinline__ void store_cluster(uint32_t at, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t at, Key v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}

constexpr int kWarpBest = 4;           // largest logits per warp that make the bound
constexpr int kMaxCandidates = kThreads;

// Grid (rows x cluster); the CTAs of a cluster share one row.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const LogprobsParams p) {
  using L = Logit<T>;
  constexpr int N = L::kVec;
  static_assert(kWarps * kWarpBest == 32, "a warp ranks the CTA's best, one per lane");
  __shared__ Stats warp_stats[kWarps];
  __shared__ int warp_before[kWarps];
  __shared__ uint32_t warp_best[32];
  __shared__ int flagged[kThreads];
  __shared__ int flagged_count, candidate_count;
  __shared__ __align__(16) Key keys[kMaxCandidates];  // candidates, or the warps' lists
  __shared__ Key sorted[32];                          // the CTA's largest
  __shared__ Part parts[kMaxCluster];
  __shared__ Stats row_stats;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int csize = (int)cluster_size(), crank = (int)cluster_rank(), row = blockIdx.x / csize;
  if (csize > 1) cluster_arrive_relaxed();  // waited for before the first store to another CTA's memory
  const T *x = static_cast<const T *>(p.logits) + (long long)row * p.row_stride;

  const int target = p.targets != nullptr ? p.targets[row] : -1;
  // This CTA's logits: whole vectors [v0, v1) but for the row's ends. The
  // first `head` logits of the row come before its first 16-byte boundary.
  const int misaligned = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(misaligned ? N - misaligned : 0, p.vocab);
  const int vectors = (p.vocab - head) / N, tail = (p.vocab - head) % N;
  const int per = (vectors + csize - 1) / csize;
  const int v0 = min(vectors, crank * per), v1 = min(vectors, v0 + per);
  const uint4 *body = reinterpret_cast<const uint4 *>(x + head);
  // The element at either end that this thread takes besides its vectors (-1: none).
  const int at_head = crank == 0 && tid < head ? tid : -1;
  const int at_tail = crank == csize - 1 && tid < tail ? head + vectors * N + tid : -1;

  // The first vectors are on their way before the target's logit is waited for.
  constexpr int kBatch = 2;
  const int stride = kThreads * kBatch;
  int v = v0 + tid;
  uint4 raw[kBatch];
  auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) raw[i] = __ldg(body + from + i * kThreads);
  };
  const int full = v1 - (kBatch - 1) * kThreads;  // a whole batch starts below
  if (v < full) load(v);
  const bool given = target >= 0 && target < p.vocab;
  float xt = given ? L::get(x + target) : INFINITY;
  if (xt != xt) xt = -INFINITY;  // NaN ranks as -inf (the row's sums, and with them its results, are NaN then)
  const float reach = xt == -INFINITY ? NAN : xt;

  Pass<T> pass;
  if (at_head >= 0) pass.take(L::get(x + at_head), at_head, xt, reach, target);
  while (v < full) {
    uint4 now[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) now[i] = raw[i];
    const int at = head + v * N;
    v += stride;
    if (v < full) load(v);
    pass.template take<kBatch>(now, at, kThreads, xt, reach, target);
  }
  for (; v < v1; v += kThreads) {
    const uint4 one = __ldg(body + v);
    pass.template take<1>(&one, head + v * N, 0, xt, reach, target);
  }
  if (at_tail >= 0) pass.take(L::get(x + at_tail), at_tail, xt, reach, target);

  Stats st = pass.stats();
  int before = (int)pass.before;
  const uint32_t mine = TOP && pass.best_at >= 0 ? order_value(pass.best) : 0u;  // 0: nothing above -inf
  {
    const Stats w = warp_join(st);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) {
      warp_stats[warp] = w;
      warp_before[warp] = before;
    }
  }
  if (TOP) {
    uint32_t left = mine;
#pragma unroll
    for (int i = 0; i < kWarpBest; ++i) {
      const uint32_t best = __reduce_max_sync(0xffffffffu, left);
      const unsigned holders = __ballot_sync(0xffffffffu, left == best);
      if (lane == __ffs(holders) - 1) left = 0;
      if (lane == 0) warp_best[warp * kWarpBest + i] = best;
    }
    if (tid == 0) flagged_count = candidate_count = 0;
    if (tid < 32) sorted[tid] = 0;
  }
  __syncthreads();
  if (TOP) {
    uint32_t bound;
    {
      const uint32_t v = warp_best[lane];
      int larger = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const uint32_t o = warp_best[j];
        larger += (o > v || (o == v && j < lane)) ? 1 : 0;
      }
      const unsigned at = __ballot_sync(0xffffffffu, larger == p.top - 1);
      bound = __shfl_sync(0xffffffffu, v, __ffs(at) - 1);
    }
    if (bound != 0 && mine >= bound) flagged[atomicAdd(&flagged_count, 1)] = tid;
    __syncthreads();
    const int rounds = (v1 - v0 + kThreads - 1) / kThreads;  // vectors of a thread, at most
    const int n = flagged_count;
    auto offer_candidate = [&](float value, int at) {
      if (order_value(value) < bound) return;
      const int slot = atomicAdd(&candidate_count, 1);
      if (slot < kMaxCandidates) keys[slot] = order_key(value, at);
    };
    if (bound != 0) {
      for (int item = tid; item < n * rounds; item += 2 * kThreads) {
        int at[2];
        uint4 again[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = item + j * kThreads;
          at[j] = k < n * rounds ? v0 + flagged[k / rounds] + k % rounds * kThreads : v1;
          if (at[j] < v1) again[j] = __ldg(body + at[j]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (at[j] >= v1 || order_value(L::largest(again[j])) < bound) continue;
          float f[N];
          L::unpack(again[j], f);
#pragma unroll
          for (int i = 0; i < N; ++i) offer_candidate(f[i], head + at[j] * N + i);
        }
      }
      if (at_head >= 0) offer_candidate(L::get(x + at_head), at_head);
      if (at_tail >= 0) offer_candidate(L::get(x + at_tail), at_tail);
    }
    __syncthreads();
    const int found = candidate_count;
    if (bound != 0 && found <= kMaxCandidates) {
      if (tid < found) {
        const Key k = keys[tid];
        int larger = 0;
        for (int j = 0; j < found; ++j) larger += keys[j] > k ? 1 : 0;
        if (larger < p.top) sorted[larger] = k;
      }
    } else {
      // Every element once more; each warp keeps a descending list, one key per lane.
      Key list = 0;
      auto offer = [&](Key k) {
        const Key last = shfl_key(list, 31);
        unsigned want = __ballot_sync(0xffffffffu, k > last && (uint32_t)(k >> 32) >= bound);
        while (want) {
          const Key c = shfl_key(k, __ffs(want) - 1);
          want &= want - 1;
          const int at = __popc(__ballot_sync(0xffffffffu, list > c));
          const Key up = __shfl_up_sync(0xffffffffu, list, 1);
          list = lane < at ? list : (lane == at ? c : up);
        }
      };
      for (int v = v0 + warp * 32; v < v1; v += kThreads) {
        float f[N];
        if (v + lane < v1) L::unpack(__ldg(body + v + lane), f);
#pragma unroll
        for (int i = 0; i < N; ++i) offer(v + lane < v1 ? order_key(f[i], head + (v + lane) * N + i) : 0ull);
      }
      offer(at_head >= 0 ? order_key(L::get(x + at_head), at_head) : 0ull);
      offer(at_tail >= 0 ? order_key(L::get(x + at_tail), at_tail) : 0ull);
      keys[warp * 32 + lane] = list;
      __syncthreads();
      if (warp == 0) sorted[lane] = merge_lists(keys, kWarps, lane);
    }
  }
  if (warp == 1) {
    Stats all = lane < kWarps ? warp_stats[lane] : empty_stats();
    all = warp_join(all);
    int sum = lane < kWarps ? warp_before[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    st = all;
    before = sum;
    if (csize == 1 && lane == 0) row_stats = st;
  }
  __syncthreads();
  if (csize > 1) {
    cluster_wait();
    Part *part = parts + crank;
    if (tid == 32) {
      store_cluster(in_first_cta(&part->st.m), __float_as_uint(st.m));
      store_cluster(in_first_cta(&part->st.s), __float_as_uint(st.s));
      store_cluster(in_first_cta(&part->st.u), __float_as_uint(st.u));
      store_cluster(in_first_cta(&part->before), (uint32_t)before);
    }
    if (TOP && tid < 32) store_cluster(in_first_cta(&part->top[tid]), sorted[tid]);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (crank != 0) return;
    if (warp == 1) {
      st = lane < csize ? parts[lane].st : empty_stats();
      st = warp_join(st);
      before = lane < csize ? parts[lane].before : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
      if (lane == 0) row_stats = st;
    }
    __syncthreads();
  }
  // With nothing but masked logits no token has any probability: every log
  // probability is -inf, the entropy 0. +inf or NaN among the logits make s,
  // and with it every result, NaN.
  const Stats r = row_stats;
  const bool none = r.m == -INFINITY && r.s == 0.0f;
  const float log_s = none ? 0.0f : log2f(r.s) * kLn2;
  auto log_p = [&](float v) { return none ? -INFINITY : (v - r.m) - log_s; };
  if (tid == 32) {
    const bool bad_target = !given && target != -1;
    if (bad_target) report_status(p.status, kStatusTokenRange, kWhereScore, target, row);
    if (p.logprobs) p.logprobs[row] = bad_target ? NAN : (given ? log_p(xt) : 0.0f);
    if (p.entropy) p.entropy[row] = none ? 0.0f : log_s - r.u / r.s;
    if (p.ranks) p.ranks[row] = !given ? -1 : xt == -INFINITY ? before + target : before;
  }
  if (TOP) {
    // A key's place in the row: its place in its own list and the larger keys of the others.
    const int list = warp, i = lane;  // kMaxCluster lists at most, one per warp
    Key k = 0;
    int place = i;
    if (csize == 1) {
      if (list == 0) k = sorted[i];
    } else if (list < csize) {
      k = parts[list].top[i];
      // Binary searches in all lists (padded with 0) side by side.
      int n[kMaxCluster] = {};
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c)
          if (c < csize && parts[c].top[n[c] + step - 1] > k) n[c] += step;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < csize && c != list) place += n[c] + (parts[c].top[n[c]] > k ? 1 : 0);
    }
    if (k != 0 && place < p.top) {
      p.top_ids[(size_t)row * p.top + place] = argmax_key_index(k);
      p.top_logprobs[(size_t)row * p.top + place] = log_p(argmax_key_value(k));
    }
  }
}

template <typename T>
cudaError_t launch(const LogprobsParams &p, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster * p.rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return p.top > 0 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, true>, p)
                   : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, false>, p);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobsParams &p, int type, int num_sms, cudaStream_t stream) {
  if (p.rows < 0 || p.rows > 0x7fffffff / kMaxCluster || p.vocab <= 0 || p.top < 0 || p.top > kLogprobsMaxTop || p.top > p.vocab ||
      p.row_stride < p.vocab)
    return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  // CTAs per row: two rounds of SMs' worth, each with some thousand logits (150
  // rows of 128256: 29 us with two rounds, 45 with one, 35 with four; 100 rows
  // of 32000: 5.7, 6.2, 8.2).
  int cluster = 1;
  while (cluster < kMaxCluster && p.rows * cluster < 2 * num_sms && p.vocab / cluster > 4096) cluster *= 2;
  switch (type) {
    case kLogitsF16: return launch<__half>(p, cluster, stream);
    case kLogitsF32: return launch<float>(p, cluster, stream);
    case kLogitsBF16: return launch<__nv_bfloat16>(p, cluster, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace tmc
