// Test-only C wrapper around the host plan of the window attention
// (window_plan.hpp), for tests/test_window_plan.py.
#include "window_plan.hpp"

extern "C" {

// decode, tensor, tiles, cluster, outer of a call whose rows see `keys` keys at most.
void plan(int sequences, int max_rows, int hq, int hkv, int d, long long keys, int num_sms, int *out) {
  const auto p = tmc::window::make_plan(sequences, max_rows, hq, hkv, d, keys, num_sms);
  out[0] = p.decode;
  out[1] = p.tensor;
  out[2] = p.tiles;
  out[3] = p.cluster;
  out[4] = p.outer;
}
int most_splits(int sequences, int max_rows, int hq, int hkv, int d, long long keys, int num_sms) {
  return tmc::window::most_splits(sequences, max_rows, hq, hkv, d, keys, num_sms);
}
}
