// Window attention of prompts on the tcgen05 tensor cores (head dimensions 64
// and 128; see window_attention.cu for the other shapes and for decoding).
//
// A CTA holds two tiles of 128 tile rows (query row x head of one KV head) and
// walks the visible keys 128 at a time: S = Q_t K^T and O_t += P_t V by
// tcgen05.mma, S, P and O in tensor memory. The tiles take turns in one S (128
// columns): a tile's softmax reads it whole into registers, and the other's
// scores are computed while it takes its exponentials, so that each finds its
// next scores waiting. P (the storage type, 64 columns) and O have places of
// their own. Four warps per tile are its softmax, one thread per tile row; one
// warp per tile issues its products, so that the waits of one pass under the
// products of the other. K and V come in through the block table by two warps:
// pages of whole groups of 16 or 8 positions as TMA boxes (the key numbering
// starts on a group then, and what no row sees of a group is zeroed in V), other
// page sizes as 16-byte copies.
//
// Weights are 2^(s - m) about a number m per row that moves to the maximum only
// when that has passed it by more than kSlack: sums in fp32 and P's
// floating-point numbers lose nothing below that, and O is not rescaled in most
// steps.
//
// P is rounded once to the storage type; the row sum l is taken before that. An
// output is then off by 2^-11 (fp16) or 2^-8 (bf16) of sum p |v| at most: in the
// mean about as much again as its own rounding (four bf16 prompts: 0.0023 of the results' size against
// 64 bits, 0.0016 with weights in fp32; a chunk in fp16 0.00028 and 0.00021).
// A second part of P, as in decoding, is half as many products again, where
// products are the bound, and for heads of 128 has no place: one S, two P and two
// O fill tensor memory.
//
// Values that are infinite or NaN in a step that some row does not wholly see
// would reach that row as 0 x inf: such a step marks the tile, and the tile's
// rows are computed again by plain loops. So are a warp's rows when one of
// their results is not finite although its sum is (slow_row).
//
// Bound: the tensor pipe, at 81 to 90 cycles per product of 128 x 128 x 16 (88
// would be 1675 TFLOP/s, a library product's, at 1.9 GHz), 32 of them per 128 keys of both tiles, beside a
// softmax of 2200 to 2700 cycles: 8192 rows x 32 heads of 128 causally 520 us,
// 1057 TFLOP/s, 0.63 of the library product's short-run rate and 0.77 of its
// rate under the power limit. With P over its own S, scores waited for the
// products before them (592 us); one warp for both tiles' products (606); P in
// shared memory (644: both operands from there); an S of its own for each tile
// where heads of 64 leave room (2 x 4096 rows 258 us against 234: the tiles then
// take their exponentials at the same time). Before that, measured and left
// out: two threads a row, P handed over in halves, an eighth to a half of the
// exponentials as polynomials, steps of 64 keys (a product with N = 64 takes as
// long as with 128), the splits joined in clusters (512 rows over 8k keys 84 us
// against 88, but 57 against 33 where clusters of six leave SMs idle). Short
// calls are set-up and hand-over: 256 rows x 32 heads, window 512, 21 us, of
// which reading the first keys 4, a step 2, the results 2 to 3 and the joining
// kernel 4.
#include <map>
#include <mutex>
#include <utility>

#include "gemm.cuh"
#include "window_device.cuh"

namespace tmc {
namespace window {
namespace {

constexpr int kTileRows = 128;
constexpr int kKeys = 128;  // of a step
constexpr int kSoftmaxWarps = 8;
constexpr int kLoadWarps = 2;  // with boxes one for K, one for V
constexpr int kMmaWarp = kSoftmaxWarps + kLoadWarps;  // and the next: one for each tile's products
constexpr int kThreads = (kMmaWarp + 2) * 32;
constexpr int kFlagRing = 8;  // steps whose missing-key flags are kept
constexpr float kSlack = 8.0f;  // powers of two by which the maximum may pass m
constexpr uint32_t kTmemColumns = 512;

template <int D>
struct TensorCfg {
  static constexpr int kHalf = kKeys * 128;             // bytes of 64 columns of a 128-row tile
  static constexpr int kTile = D / 64 * kHalf;          // one of K, V or a Q tile
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kSmem = 1024 + 2 * kTile + kStages * 2 * kTile;
  static_assert(kStages + 1 < kFlagRing, "keys load a stage ahead of the products, those a step ahead of the softmax");
};

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Consecutive 32-bit columns of this warp's lanes (one row per thread), there
// when the call returns.
__device__ __forceinline__ void tmem_load128(uint32_t at, float *v) {
  uint32_t r[128];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%128];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]), "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]), "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(at));
#pragma unroll
  for (int i = 0; i < 128; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load32(uint32_t at, float *v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load16(uint32_t at, float *v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_store64(uint32_t at, const uint32_t (&r)[64]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x64.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,%64};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
      "r"(r[32]), "r"(r[33]), "r"(r[34]), "r"(r[35]), "r"(r[36]), "r"(r[37]), "r"(r[38]), "r"(r[39]),
      "r"(r[40]), "r"(r[41]), "r"(r[42]), "r"(r[43]), "r"(r[44]), "r"(r[45]), "r"(r[46]), "r"(r[47]),
      "r"(r[48]), "r"(r[49]), "r"(r[50]), "r"(r[51]), "r"(r[52]), "r"(r[53]), "r"(r[54]), "r"(r[55]),
      "r"(r[56]), "r"(r[57]), "r"(r[58]), "r"(r[59]), "r"(r[60]), "r"(r[61]), "r"(r[62]), "r"(r[63])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Shared-memory matrix descriptors of tiles of 128-byte rows with 128-byte
// swizzle (start address, strides in 16 bytes, version 1, layout 2).
// K-major (Q, K: a row is an M or N index): 1024 bytes between groups of 8
// rows; 32 bytes further is 16 elements further along K.
__device__ __forceinline__ uint64_t k_major(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | (uint64_t)1u << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 |
         (uint64_t)2u << 61;
}
// N-major (V: a row is a K index, 64 N indices long): `half` bytes between
// blocks of 64 N indices, 1024 bytes between groups of 8 K indices.
__device__ __forceinline__ uint64_t n_major(uint32_t addr, uint32_t half) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | (uint64_t)(half >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
// kind::f16 instruction: D fp32, M 128, N columns, A and B both fp16 or both bf16.
template <typename E>
__device__ __forceinline__ constexpr uint32_t instruction(int n, bool b_n_major) {
  constexpr uint32_t type = sizeof(E) == 2 && std::is_same<E, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTileRows >> 4) << 24);
}
// One thread (`lead`) issues; the whole warp runs these, so that descriptors
// stay in uniform registers.
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, bool lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u), "r"(lead ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add, bool lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u), "r"(lead ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {  // 2^x, 0 below the normal range
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// mbar_wait, which reads the clock, only where the barrier is not through yet.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done || mbar_wait(bar, parity);
}
__device__ __forceinline__ bool through(uint64_t *bar, uint32_t parity) {  // at this moment
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done;
}
// Bits [a, b) of 32.
__device__ __forceinline__ uint32_t bits_between(int a, int b) {
  a = max(a, 0);
  b = min(b, 32);
  return a < b ? (0xffffffffu >> (32 - (b - a))) << a : 0u;
}

// Byte offset of 16-byte chunk c of row r in a tile of 128 rows.
__device__ __forceinline__ int swizzled(int r, int c) {
  return (c >> 3) * (kKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// Grid as prompt_place counts it, over tile pairs. BOX: positions of the TMA
// boxes that bring K and V, 0 without.
template <typename E, int D, int BOX>
__global__ void __launch_bounds__(kThreads, 1)
    window_tensor_kernel(const WindowAttentionParams p, int splits, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map) {
  constexpr bool BOXES = BOX > 0;
  constexpr int kBox = BOXES ? BOX : 16;
  using C = TensorCfg<D>;
  constexpr int S = C::kStages;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *base = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sQ = base, *sK = base + 2 * C::kTile, *sV = sK + S * C::kTile;
  __shared__ __align__(8) uint64_t q_full, k_full[S], k_empty[S], v_full[S], v_empty[S], s_full[2], s_free[2],
      p_full[2], p_done[2], o_full[2], drained[2], v_landed;
  __shared__ uint32_t tmem_base;
  __shared__ __align__(16) unsigned char bad_keys[kFlagRing][kKeys];  // keys of a step whose page is missing
  __shared__ int bad_any[kFlagRing][2];
  __shared__ int marked[2];  // the tile met an infinity or NaN beside masked pairs

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (BOXES && tid < 2)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tid ? &v_map : &k_map)) : "memory");
  pdl_wait();
  const PromptPlace place = prompt_place(p, splits);
  const int s = place.seq, h = place.head, split = place.split;
  const Sequence seq = load_sequence(p, s, place.first && tid == 0);
  const int g = p.hq / p.hkv;
  const int m0 = place.tile * 2 * kTileRows, total = seq.rows * g;
  if (m0 >= total) return;
  const int tiles = m0 + kTileRows < total ? 2 : 1;
  const int m_end = min(m0 + 2 * kTileRows, total);
  const int p_last = seq.first + (m_end - 1) / g;
  Visible vis = visible_keys(p, seq.first + m0 / g, p_last);
  const int low = vis.low;  // keys below, but for the sinks, are seen by no row
  if (BOXES) {  // both parts start and the first ends on a group
    vis.low = low / kBox * kBox;
    vis.sinks = min((min(p.sinks, vis.low) + kBox - 1) / kBox * kBox, vis.low);
    vis.count = vis.sinks + p_last + 1 - vis.low;
  }
  const int chunk = ((vis.count + splits - 1) / splits + kKeys - 1) / kKeys * kKeys;
  const int v0 = min(vis.count, split * chunk), v1 = min(vis.count, v0 + chunk);
  const int steps = (v1 - v0 + kKeys - 1) / kKeys;
  const long long slots = (long long)p.sequences * p.max_rows * p.hq;
  if (steps == 0) {  // a split beyond the keys
    const int m = m0 + tid;
    if (m < m_end)
      *partial_ml(p, slots, splits, split, ((long long)s * p.max_rows + m / g) * p.hq + h * g + m % g) =
          make_float2(-INFINITY, 0.0f);
    return;
  }

  auto find_box = [&](int j) {  // lane i < 8: group i of step j
    const int v = v0 + j * kKeys + lane * kBox;
    return lane < kKeys / kBox && j < steps && v < v1 ? find_key(p, seq.table, vis.key(v)) : KeyPlace{0, -1, 0};
  };
  auto find_half = [&](int job, int i) {  // lane: key 32 i + lane of a half step; jobs K 0, K 1, V 0, V 1 of each step
    const int v = v0 + (job >> 2) * kKeys + (job & 1) * 64 + i * 32 + lane;
    return job < 4 * steps && v < v1 ? find_key(p, seq.table, vis.key(v)) : KeyPlace{0, -1, 0};
  };
  // The first table entries are on their way over the barrier.
  KeyPlace first_box{0, -1, 0}, first_half[2] = {{0, -1, 0}, {0, -1, 0}};
  if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    if (BOXES) {
      first_box = find_box(0);
    } else {
      first_half[0] = find_half(warp - kSoftmaxWarps, 0);
      first_half[1] = find_half(warp - kSoftmaxWarps, 1);
    }
  }

  if (warp == kMmaWarp) {
    if (lane == 0) {
      mbar_init(&q_full, kSoftmaxWarps);
      mbar_init(&v_landed, 1);
      for (int i = 0; i < S; ++i) {
        mbar_init(&k_full[i], BOXES ? 1 : 2);
        mbar_init(&v_full[i], BOXES ? 1 : 2);
        mbar_init(&k_empty[i], tiles);
        mbar_init(&v_empty[i], tiles);
      }
      for (int t = 0; t < 2; ++t) {
        mbar_init(&s_full[t], 1);
        mbar_init(&s_free[t], 4);
        mbar_init(&p_full[t], 4);
        mbar_init(&p_done[t], 1);
        mbar_init(&o_full[t], 1);
        mbar_init(&drained[t], 1);
        marked[t] = 0;
      }
      fence_barrier_init();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base;
  auto gave_up = [&](int step) {
    report_status(p.status, kStatusWaitTimeout, kWhereAttention, step, s);
  };

  if (warp < kSoftmaxWarps) {
    // ---- softmax: one thread per tile row ----
    const int t = warp >> 2, r = (warp & 3) * 32 + lane, m = m0 + t * kTileRows + r;
    const bool used = m < total;
    const int row = used ? m / g : 0, head = h * g + (used ? m % g : 0), pos = seq.first + row;
    // Rows go to and from shared memory by whole warps, a few rows at a time
    // (each thread its own row: Q 3100 to 9000 cycles instead of 1300 to 4700,
    // the results 4500 instead of 3700).
    constexpr int kChunks = D / 8, kRows = 32 / kChunks;  // 16-byte chunks of a row; rows at a time
    unsigned char *own_rows = sQ + t * C::kTile;
    const int r0 = (warp & 3) * 32;
    {
      const long long at = used ? (seq.start + row) * p.q_stride + (long long)head * D : -1;
#pragma unroll 8
      for (int n = 0; n < 32; n += kRows) {
        const int i = n + lane / kChunks, c = lane % kChunks;
        const long long from = __shfl_sync(0xffffffffu, at, i);
        cp_async16(smem_u32(own_rows + swizzled(r0 + i, c)), static_cast<const E *>(p.q) + (from < 0 ? 0 : from + c * 8),
                   from < 0 ? 0 : 16);
      }
      cp_async_commit();
      cp_async_wait<0>();
      fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    const int t0 = min(m0 + t * kTileRows, total - 1), t1 = min(m0 + (t + 1) * kTileRows, total) - 1;
    const int p_lo = seq.first + t0 / g, p_hi = seq.first + t1 / g;  // of the tile's rows
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes, p_at = s_at + kKeys + t * (kKeys / 2), o_at = s_at + 2 * kKeys + t * D;
    const float scale = p.scale * kLog2e;
    float m_run = -INFINITY;
    float2 l_run[2] = {};
    // What this row sees, as numbers of keys: all below `always` (the sinks,
    // and keys of the run that are sinks), and [from, to) of the run.
    const int always = p.sinks < vis.low ? p.sinks : vis.sinks + max(0, min(p.sinks, pos + 1) - vis.low);
    const int from = vis.sinks + max(0, pos - p.window + 1 - vis.low);
    const int to = min(vis.sinks + pos + 1 - vis.low, v1);
    // Steps that all of the tile's rows see as a whole: those below
    // `always_all`, and those in [from_all, to_all).
    const int always_all = min(p.sinks < vis.low ? p.sinks : vis.sinks + max(0, min(p.sinks, p_lo + 1) - vis.low), v1);
    const int from_all = vis.sinks + max(0, p_hi - p.window + 1 - vis.low);
    const int to_all = min(vis.sinks + p_lo + 1 - vis.low, v1);
    bool failed = false;
    if (t < tiles) {
      for (int j = 0; j < steps; ++j) {
        if (!__all_sync(0xffffffffu, wait(&s_full[t], j & 1))) {
          if (lane == 0) gave_up(j);
          failed = true;
          break;
        }
        fence_after();
        const int first = v0 + j * kKeys;
        const bool whole = first + kKeys <= always_all || (first >= from_all && first + kKeys <= to_all);
        if (!whole) {
          const int st = j % S;
          if (!__all_sync(0xffffffffu, wait(&v_full[st], (j / S) & 1))) {
            if (lane == 0) gave_up(j);
            failed = true;
            break;
          }
          bool special = false;
          const uint4 *v = reinterpret_cast<const uint4 *>(sV + st * C::kTile);
#pragma unroll 4
          for (int i = 0; i < C::kTile / 16 / 128; ++i) special |= any_special(v[r + 128 * i], exponent_mask(E()));
          if (special) marked[t] = 1;
        }
        const bool missing = (bad_any[j % kFlagRing][0] | bad_any[j % kFlagRing][1]) != 0;
        const bool masked = !whole || missing;
        float x[kKeys];
        tmem_load128(s_at, x);
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t]);  // the next step's scores may come
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int v = first + c * 32;
            uint32_t bits = bits_between(0 - v, min(always, v1) - v) | bits_between(from - v, to - v);
            if (missing)
              for (int i = 0; i < 32; ++i)
                if (bad_keys[j % kFlagRing][c * 32 + i]) bits &= ~(1u << i);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[c * 32 + i] = (bits >> i) & 1 ? x[c * 32 + i] : -INFINITY;
          }
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i];
#pragma unroll
        for (int i = 8; i < kKeys; i += 16)
#pragma unroll
          for (int n = 0; n < 8; ++n)
            y[n] = i + 8 + n < kKeys ? fmaxf(fmaxf(y[n], x[i + n]), x[i + 8 + n]) : fmaxf(y[n], x[i + n]);
        const float mx =
            fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7]))) * scale;
        const bool rise = mx > m_run + kSlack || (m_run == -INFINITY && mx > m_run);
        // After the products of the step before, O is complete and P's place free.
        auto products_done = [&] { return j == 0 || __all_sync(0xffffffffu, wait(&p_done[t], (j - 1) & 1)); };
        if (__any_sync(0xffffffffu, rise)) {
          if (!products_done()) {
            if (lane == 0) gave_up(j);
            failed = true;
            break;
          }
          const float f = rise ? exp2_fast(m_run - mx) : 1.0f;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            l_run[i].x *= f;
            l_run[i].y *= f;
          }
          if (rise) m_run = mx;
          if (j > 0) {
            fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_load16(o_at + c, o);
              uint32_t scaled[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) scaled[i] = __float_as_uint(o[i] * f);
              tmem_store16(o_at + c, scaled);
            }
            wait_st();
          }
        }
        // A masked score (-inf) has weight 0; a row that has seen nothing yet has m = -inf.
        const float about = m_run == -INFINITY ? 0.0f : -m_run;
        uint32_t w[kKeys / 2];  // P, two weights to a register
#pragma unroll
        for (int i = 0; i < kKeys / 2; ++i) {
          const float2 z = __ffma2_rn(make_float2(x[2 * i], x[2 * i + 1]), make_float2(scale, scale),
                                      make_float2(about, about));
          const float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
          l_run[i & 1] = __fadd2_rn(l_run[i & 1], e);
          w[i] = pack2(e.x, e.y, E());
        }
        if (!products_done()) {
          if (lane == 0) gave_up(j);
          failed = true;
          break;
        }
        fence_after();
        tmem_store64(p_at, w);
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!failed && !__all_sync(0xffffffffu, mbar_wait(&o_full[t], 0))) {
        if (lane == 0) gave_up(steps);
        failed = true;
      }
      fence_after();
      // The tile's four warps agree on whether it was marked.
      if (t == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
      else asm volatile("bar.sync 2, 128;" ::: "memory");
      const long long slot = ((long long)s * p.max_rows + row) * p.hq + head;
      bool again = marked[t] != 0;  // by plain loops
      if (!failed && !again) {
        const float l = (l_run[0].x + l_run[0].y) + (l_run[1].x + l_run[1].y);
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // no visible key: zeros
        // Q has been read: its place takes the results, 256-byte (D 64: 128-byte) pieces of each row.
        const long long row_at = !used        ? -1
                                 : splits > 1 ? (split * slots + slot) * D
                                              : (seq.start + row) * p.out_stride + (long long)head * D;
        auto hand_out = [&](char *to, int size, int bytes_before) {  // the warp's 32 rows, chunks in order
          __syncwarp();
#pragma unroll 4
          for (int n = 0; n < 32; n += kRows) {
            const int i = n + lane / kChunks, c = lane % kChunks;
            const long long dst = __shfl_sync(0xffffffffu, row_at, i);
            if (dst >= 0)
              *reinterpret_cast<uint4 *>(to + dst * size + bytes_before + c * 16) =
                  *reinterpret_cast<const uint4 *>(own_rows + swizzled(r0 + i, c));
          }
          __syncwarp();
        };
        float2 finite{};
        auto lost = [&] {
          const float all = finite.x + finite.y;
          return __any_sync(0xffffffffu, used && all != all && l == l) != 0;
        };
        if (splits > 1) {
#pragma unroll 1
          for (int part = 0; part < 2; ++part) {  // D / 2 fp32 columns fill a row's place
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 32) {
              float x[32];
              tmem_load32(o_at + part * (D / 2) + c, x);
#pragma unroll
              for (int i = 0; i < 32; i += 2) note_finite(finite, x[i], x[i + 1]);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float4 *>(own_rows + swizzled(r, c / 4 + i)) =
                    make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
            hand_out(static_cast<char *>(p.workspace), 4, part * D * 2);
          }
          again = lost();
        } else {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            float x[32];
            tmem_load32(o_at + c, x);
#pragma unroll
            for (int i = 0; i < 32; i += 2) note_finite(finite, x[i], x[i + 1]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4 *>(own_rows + swizzled(r, c / 8 + i)) =
                  make_uint4(pack2(x[8 * i] * inv, x[8 * i + 1] * inv, E()),
                             pack2(x[8 * i + 2] * inv, x[8 * i + 3] * inv, E()),
                             pack2(x[8 * i + 4] * inv, x[8 * i + 5] * inv, E()),
                             pack2(x[8 * i + 6] * inv, x[8 * i + 7] * inv, E()));
          }
          again = lost();
          if (!again) hand_out(static_cast<char *>(p.out), 2, 0);  // the queries may lie there
        }
        if (used && splits > 1) *partial_ml(p, slots, splits, split, slot) = make_float2(m_run, l);
      }
      if (!failed && again) {
        __syncwarp();
        for (int i = 0; i < 32; ++i) {
          const int mi = m0 + t * kTileRows + (warp & 3) * 32 + i;
          if (mi >= total) break;
          const int q_row = mi / g, q_head = h * g + mi % g;
          float mm, ll, o[(D + 31) / 32];
          slow_row<E, D>(p, seq, s, h, q_head, q_row, vis, v0, v1, mm, ll, o, lane);
          const long long q_slot = ((long long)s * p.max_rows + q_row) * p.hq + q_head;
#pragma unroll
          for (int n = 0; n < D / 32; ++n) {
            const int d = lane + 32 * n;
            if (splits > 1)
              partial_acc(p, slots, split, q_slot)[d] = o[n];
            else
              store1(p.out, (seq.start + q_row) * p.out_stride + (long long)q_head * D + d,
                     ll > 0.0f || ll != ll ? o[n] / ll : 0.0f, E());
          }
          if (splits > 1 && lane == 0) *partial_ml(p, slots, splits, split, q_slot) = make_float2(mm, ll);
        }
      }
    }
  } else if (BOXES && warp < kMmaWarp) {
    // ---- loads by boxes: a warp for K, a warp for V, lane i < 8 takes group i of a step ----
    const int load = warp - kSoftmaxWarps;
    const bool value = load == 1;
    KeyPlace next = first_box;
    uint32_t edges = 0;  // steps whose V rows were cleaned: the phase of v_landed
    for (int j = 0; j < steps && load < 2; ++j) {
      const int st = j % S, first = v0 + j * kKeys;
      const bool here = lane < kKeys / kBox && first + lane * kBox < v1;
      const long long row = here ? pool_row(p, next, h, s) : -1;
      const unsigned bad = __ballot_sync(0xffffffffu, here && row < 0);
      const int boxes = __popc(__ballot_sync(0xffffffffu, row >= 0));
      next = find_box(j + 1);
      uint64_t *full = value ? v_full : k_full, *empty = value ? v_empty : k_empty;
      if (j >= S && !__all_sync(0xffffffffu, wait(&empty[st], ((j / S) - 1) & 1))) {
        if (lane == 0) gave_up(j);
        break;
      }
      // V rows that no row of the tiles sees (outside the window's union, or
      // of a missing page) hold anything: zeros in their place.
      bool hide[kKeys / 32];
      bool any = false;
#pragma unroll
      for (int i = 0; i < kKeys / 32; ++i) {
        const int v = first + i * 32 + lane, k = vis.key(v);
        hide[i] = v >= v1 || (k < low && k >= p.sinks) || ((bad >> ((i * 32 + lane) / kBox)) & 1);
        any |= hide[i];
      }
      const bool edge = __any_sync(0xffffffffu, any) && value;
      if (!value) {
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i)
          bad_keys[j % kFlagRing][i * 32 + lane] = (bad >> ((i * 32 + lane) / kBox)) & 1;
        if (lane < 2) bad_any[j % kFlagRing][lane] = bad != 0;
        __syncwarp();
      }
      uint64_t *bar = edge ? &v_landed : &full[st];
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)boxes * kBox * D * 2);
      __syncwarp();
      unsigned char *dst = (value ? sV : sK) + st * C::kTile;
      if (row >= 0) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_2d(dst + c * C::kHalf + lane * kBox * 128, value ? &v_map : &k_map, c * 64, (int)row, bar);
      }
      if (edge) {
        if (!__all_sync(0xffffffffu, mbar_wait(&v_landed, edges & 1))) {
          if (lane == 0) gave_up(j);
          break;
        }
        ++edges;
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i)
          if (hide[i])
            for (int c = 0; c < D / 8; ++c)
              *reinterpret_cast<uint4 *>(dst + swizzled(i * 32 + lane, c)) = make_uint4(0u, 0u, 0u, 0u);
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
    }
  } else if (!BOXES && warp < kMmaWarp) {
    // ---- loads: the halves (64 keys) of K and of V of every step are dealt out
    // to the warps in the order in which they are needed ----
    const int load = warp - kSoftmaxWarps;
    KeyPlace next[2] = {first_half[0], first_half[1]};
    uint64_t *late = nullptr;  // of the job whose copies may be in flight beside this one's
    auto landed = [&] {
      fence_async();  // what the copies wrote, before the products read it
      __syncwarp();
      if (lane == 0) mbar_arrive(late);
    };
    for (int job = load; job < 4 * steps; job += kLoadWarps) {
      const int j = job >> 2, st = j % S, half = job & 1;
      const bool value = (job & 2) != 0;
      uint32_t at[2];  // pool rows: below 2^32 for 128-byte rows of one GPU's memory; 0xffffffff: none
      bool bad[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int v = v0 + j * kKeys + half * 64 + i * 32 + lane;
        at[i] = v < v1 ? (uint32_t)pool_row(p, next[i], h, s) : 0xffffffffu;
        bad[i] = v < v1 && at[i] == 0xffffffffu;
        next[i] = find_half(job + kLoadWarps, i);
      }
      uint64_t *full = value ? v_full : k_full, *empty = value ? v_empty : k_empty;
      if (j >= S) {
        const uint32_t phase = ((j / S) - 1) & 1;
        if (late && !__all_sync(0xffffffffu, through(&empty[st], phase))) {  // its place may wait for those copies
          cp_async_wait<0>();
          landed();
          late = nullptr;
        }
        if (!__all_sync(0xffffffffu, wait(&empty[st], phase))) {
          if (lane == 0) gave_up(j);
          break;
        }
      }
      if (!value) {
        bad_keys[j % kFlagRing][half * 64 + lane] = bad[0];
        bad_keys[j % kFlagRing][half * 64 + 32 + lane] = bad[1];
        const int any = __any_sync(0xffffffffu, bad[0] || bad[1]);
        if (lane == 0) bad_any[j % kFlagRing][half] = any;
      }
      constexpr int kChunks = D / 8, kRows = 32 / kChunks;  // rows that a warp copies at a time
      const char *pool = static_cast<const char *>(value ? p.v_pool : p.k_pool) + (lane % kChunks) * 16;
      const uint32_t dst = smem_u32((value ? sV : sK) + st * C::kTile) + half * 64 * 128;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll 8
        for (int n = 0; n < 32; n += kRows) {
          const int r = n + lane / kChunks, c = lane % kChunks;
          const uint32_t row = __shfl_sync(0xffffffffu, at[i], r);
          const bool there = row != 0xffffffffu;
          cp_async16(dst + swizzled(i * 32 + r, c), pool + (size_t)(there ? row : 0u) * (D * 2), there ? 16 : 0);
        }
      cp_async_commit();
      if (late) {
        cp_async_wait<1>();
        landed();
      }
      late = &full[st];
    }
    if (late) {
      cp_async_wait<0>();
      landed();
    }
  } else {
    // ---- products ----
    constexpr uint32_t kScores = instruction<E>(kKeys, false), kOutputs = instruction<E>(D, true);
    const bool lead = lane == 0;
    const int t = warp - kMmaWarp;
    const uint64_t q = k_major(smem_u32(sQ + t * C::kTile)), k_at = k_major(smem_u32(sK)),
                   v_at = n_major(smem_u32(sV), C::kHalf);
    const uint32_t o = tmem + 2 * kKeys + t * D, weights = tmem + kKeys + t * (kKeys / 2);
    auto here = [&](uint64_t *bar, int phase) { return __all_sync(0xffffffffu, wait(bar, phase & 1)); };
    auto arrive = [&](uint64_t *bar) {  // when the products so far are done
      if (lead) commit(bar);
      __syncwarp();
    };
    bool ok = __all_sync(0xffffffffu, mbar_wait(&q_full, 0));
    // S = Q K^T of step j, once the scores that were there have been read: the
    // tiles take turns.
    auto scores = [&](int j) {
      ok = ok && here(&k_full[j % S], j / S);
      if (tiles == 1 ? j > 0 : t == 1 || j > 0) ok = ok && here(&s_free[tiles == 1 ? 0 : 1 - t], t == 1 ? j : j - 1);
      if (!ok) return;
      fence_after();
      const uint64_t k = k_at + (j % S) * (C::kTile >> 4);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int off = (i / 4) * (C::kHalf >> 4) + (i % 4) * (32 >> 4);
        mma_smem(tmem, q + off, k + off, kScores, i > 0, lead);
      }
      arrive(&s_full[t]);
      arrive(&k_empty[j % S]);
    };
    if (t < tiles) scores(0);
    for (int j = 0; t < tiles && j < steps && ok; ++j) {
      if (j + 1 < steps) scores(j + 1);
      // O += P V of step j.
      ok = ok && here(&v_full[j % S], j / S) && here(&p_full[t], j);
      if (!ok) break;
      fence_after();
      const uint64_t v = v_at + (j % S) * (C::kTile >> 4);
#pragma unroll
      for (int i = 0; i < kKeys / 16; ++i)
        mma_tmem(o, weights + i * 8, v + i * (16 * 128 >> 4), kOutputs, j > 0 || i > 0, lead);
      arrive(&p_done[t]);
      if (j + 1 == steps) arrive(&o_full[t]);
      arrive(&v_empty[j % S]);
    }
    if (!ok) {
      // Something never came: the products in flight end (a bounded wait) before the memory is given back.
      if (lead) gave_up(-1);
      arrive(&drained[t]);
      (void)mbar_wait(&drained[t], 0);
    }
  }
  pdl_launch_dependents();
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
  }
}

template <typename E, int D, int BOX>
cudaError_t launch(const WindowAttentionParams &p, int pairs, int splits, cudaStream_t stream, bool pdl) {
  const auto kernel = window_tensor_kernel<E, D, BOX>;
  CUtensorMap k_map{}, v_map{};
  if (BOX > 0) {  // 16-bit elements of either kind: boxes only move them
    const uint64_t rows = (uint64_t)p.pool_pages * p.hkv * p.page_size;
    cudaError_t e = make_tensor_map_f16(&k_map, p.k_pool, rows, D, BOX);
    if (e == cudaSuccess) e = make_tensor_map_f16(&v_map, p.v_pool, rows, D, BOX);
    if (e != cudaSuccess) return e;
  }
  {
    static std::mutex mu;
    static std::map<int, bool> done;  // by device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TensorCfg<D>::kSmem);
      if (e != cudaSuccess) return e;
      done[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)pairs * splits * p.hkv * p.sequences));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = TensorCfg<D>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p, splits, k_map, v_map);
}

template <typename E, int D>
cudaError_t dispatch(const WindowAttentionParams &p, int pairs, int splits, cudaStream_t stream, bool pdl) {
  // Boxes of 16 positions where pages are whole numbers of them, else of 8. 4096
  // rows of 32 heads of 128: pages of 24 168 us, by copies 209; pages of 16 150, by
  // boxes of 8 165. 2 x 4096 rows of 16 heads of 64, pages of 24: 131, by copies
  // 165. Pool rows are 32-bit coordinates.
  if ((long long)p.pool_pages * p.hkv <= 0x7fffffffll / p.page_size) {
    if (p.page_size % 16 == 0) return launch<E, D, 16>(p, pairs, splits, stream, pdl);
    if (p.page_size % 8 == 0) return launch<E, D, 8>(p, pairs, splits, stream, pdl);
  }
  return launch<E, D, 0>(p, pairs, splits, stream, pdl);
}

}  // namespace

cudaError_t launch_window_tensor(const WindowAttentionParams &p, bool bf16, int pairs, int splits, cudaStream_t stream,
                                 bool pdl) {
  using Bf16 = __nv_bfloat16;
  if (p.d == 64)
    return bf16 ? dispatch<Bf16, 64>(p, pairs, splits, stream, pdl) : dispatch<__half, 64>(p, pairs, splits, stream, pdl);
  if (p.d == 128)
    return bf16 ? dispatch<Bf16, 128>(p, pairs, splits, stream, pdl)
                : dispatch<__half, 128>(p, pairs, splits, stream, pdl);
  return cudaErrorInvalidValue;
}

}  // namespace window
}  // namespace tmc
