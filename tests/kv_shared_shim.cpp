// Test-only additions to kv_fork_shim.cpp: own pages filled before they take
// the shared ones' places (tests/test_cache_shared_pages.py).
#include "kv_fork_shim.cpp"

extern "C" {

// Own pages for the positions up to `end`, filled by a copier that notes what
// the sequence's row was when it ran, and fails when told to.
int kv_state_unshare_filled(void *s, std::size_t end, int fail_copy, int *out, int *row_then, std::size_t cap) {
  auto &state = *static_cast<State *>(s)->state;
  std::vector<tensor::runtime::KVPageCopy> copies;
  const auto e = state.unshareTail(&copies, end, [&](const std::vector<tensor::runtime::KVPageCopy> &) -> std::string {
    const auto t = state.pageTable();
    std::memcpy(row_then, t.data(), std::min(cap, t.size()) * sizeof(int));
    return fail_copy ? "the copy failed" : "";
  });
  return copies_out(e, copies, out);
}
}
