// How a window attention call is split over the GPU (host only).
#pragma once

#include <algorithm>
#include <cstddef>

namespace tmc {
namespace window {

constexpr int kMaxCluster = 8;   // CTAs of a decode cluster; 16 find room later and were slower
// Decode CTAs that an SM holds, at 168 registers a thread. Two (with up to 255)
// take one row of 1k keys in 6.5 us instead of 7.0, but keep fewer reads in
// flight: one row of 32k keys 37 us instead of 30, three stages or not.
constexpr int kDecodePerSm = 3;
constexpr int kMaxOuter = 32;  // splits that meet through the workspace
// Prompts of at most 16 tile rows, or so short that all of their 16-row tiles
// together read no more than this (elements of keys), run as decoding does: it
// has less to set up, but reads the keys for every 16 rows. 32 heads, 8 KV heads
// of 128: 2 rows over 1000 keys 7.7 us (as prompts 13.9), 16 rows 10.7 (14.5), 32
// rows (8.2 million) 14.8 (14.7), 64 rows (16 million) 20.0 (17.1); 64 sequences
// of 4 rows over 1000 to 2000 keys 94 us (131), 16 heads of 64 of their own 86 (211).
constexpr long long kFewElements = 12500000;

struct Plan {
  bool decode, tensor;
  int tiles;    // per (sequence, KV head): of 16 (row, head) pairs (decode), of 128, or pairs of those (tensor)
  int cluster;  // decode: CTAs that join in distributed shared memory
  int outer;    // splits that join through the workspace
};

// Whether a call of this size can be launched: grids and tile rows within
// their types.
inline bool can_plan(int sequences, int max_rows, int hq, int hkv) {
  if (sequences <= 0 || sequences > 65535 || max_rows <= 0 || hkv <= 0 || hq <= 0 || hq > 65535 || hq % hkv != 0)
    return false;
  const long long g = hq / hkv;
  return hkv * ((g + 15) / 16) <= 65535 && max_rows * g <= (1ll << 30) / kMaxOuter &&
         (long long)sequences * max_rows <= (1ll << 32) / hq;
}

inline size_t partial_bytes(int sequences, int max_rows, int hq, int d, int outer) {
  return outer <= 1 ? 0 : (size_t)outer * sequences * max_rows * hq * (d + 2) * sizeof(float);
}

// keys: the most keys a row can see. For calls that can_plan accepts.
inline Plan make_plan(int sequences, int max_rows, int hq, int hkv, int d, long long keys, int num_sms) {
  const int g = hq / hkv;
  const long long tile_rows = (long long)max_rows * g, few_tiles = (tile_rows + 15) / 16 * hkv;  // tiles of decoding
  const bool few = max_rows == 1 || (few_tiles <= 65535 && (tile_rows <= 16 || (double)few_tiles * sequences * keys * d <=
                                                                                   kFewElements));
  Plan plan{few, !few && (d == 64 || d == 128), 1, 1, 1};
  const long long height = plan.decode ? 16 : plan.tensor ? 256 : 128;  // tile rows of a CTA
  plan.tiles = (int)((tile_rows + height - 1) / height);
  const long long ctas = (long long)sequences * hkv * plan.tiles;
  const long long slots = (plan.decode ? kDecodePerSm : plan.tensor ? 1 : 2) * num_sms;  // CTAs that run at the same time
  // Tensor-core prompts: one round of CTAs, down to one step of 128 keys each
  // (64 rows x 32 heads over 1000 keys 17.2 us; two steps at least 18.7).
  if (plan.tensor) {
    const long long steps = (keys + 127) / 128;
    long long splits = slots / ctas;
    splits = splits < 1 ? 1 : splits < kMaxOuter ? splits : kMaxOuter;
    if (splits > steps) splits = steps;
    plan.outer = (int)((steps + (steps + splits - 1) / splits - 1) / ((steps + splits - 1) / splits));  // none empty
    return plan;
  }
  if (!plan.decode) {
    while (plan.outer < kMaxOuter && ctas * plan.outer * 2 <= slots && keys > 256 * plan.outer) plan.outer *= 2;
    return plan;
  }
  // Few CTAs: as many splits as run at once, each with one step of keys for
  // its four warps at least. Many: two and a half rounds of CTAs, which evens
  // out sequences of different lengths, each with eight steps at least (64
  // sequences of 700 .. 4100 keys: one round 161 us, two and a half 147, five
  // 146; 128 of 100 .. 1000 keys: 65, 68, 79).
  long long splits;
  if (2 * ctas <= slots) {
    splits = slots / ctas;
    if (splits * 64 > keys) splits = (keys + 63) / 64;
  } else {
    splits = (5 * slots / 2 + ctas - 1) / ctas;
    if (splits * 512 > keys) splits = (keys + 511) / 512;
  }
  // Beyond a cluster the splits' states meet in the workspace, at the cost of
  // a second launch: three clusters or more, of 128 keys a CTA at least, on
  // seven eighths of the CTAs' places (clusters of eight do not fill the rest).
  // 8 KV heads of one row over 4096 keys 9.8 us (in one cluster 13.2), of two
  // rows over 16k 31 (46), over 2048 keys, where it takes one cluster, 8.8 (two
  // 9.4); one KV head of two rows over 64k 24 us (on all places 30), of one row
  // 16.1 (clusters of four 18.6).
  const long long room = splits < 7 * slots / 8 / ctas ? splits : 7 * slots / 8 / ctas;
  const long long wide = room < keys / 128 ? room : keys / 128;
  if (wide < 3 * kMaxCluster) {
    plan.cluster = (int)(splits < kMaxCluster ? splits : kMaxCluster);
  } else {
    plan.cluster = kMaxCluster;
    plan.outer = (int)(wide / kMaxCluster < kMaxOuter ? wide / kMaxCluster : kMaxOuter);
  }
  return plan;
}

inline long long visible_bound(long long window, long long sinks, int max_rows, long long capacity) {
  const long long keys = window + sinks + (max_rows > 1 ? max_rows : 0);
  return keys < capacity ? keys : capacity;
}

// The most splits that a call with at most `keys` keys a row can have. A prompt
// takes splits that leave none empty, which is not the more the more keys there
// are (room for 4: 4 steps take 4, 5 take 3), and runs as decoding does where
// the keys are few.
inline int most_splits(int sequences, int max_rows, int hq, int hkv, int d, long long keys, int num_sms) {
  const Plan plan = make_plan(sequences, max_rows, hq, hkv, d, keys, num_sms);
  if (plan.decode) return plan.outer;
  long long most = plan.outer;
  if (plan.tensor)
    most = std::clamp<long long>(num_sms / ((long long)sequences * hkv * plan.tiles), 1,
                                 std::min<long long>(kMaxOuter, (keys + 127) / 128));
  const long long few_tiles = ((long long)max_rows * (hq / hkv) + 15) / 16 * hkv;
  const long long few = std::min(keys, kFewElements / std::max(1ll, few_tiles * sequences * d));
  if (few > 0) most = std::max<long long>(most, make_plan(sequences, max_rows, hq, hkv, d, few, num_sms).outer);
  return (int)most;
}

}  // namespace window
}  // namespace tmc
