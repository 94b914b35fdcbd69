// Test-only additions to kv_state_shim.cpp: forks, copies before appends and
// replaced pages of the cache state (tests/test_cache_fork.py).
#include "kv_state_shim.cpp"

extern "C" {

int kv_pool_retain(void *p, int page) {
  try {
    (*static_cast<std::shared_ptr<KVPagePool> *>(p))->retainPage(page);
    return 0;
  } catch (const std::exception &e) {
    return fail(e.what());
  }
}
std::size_t kv_pool_owners(void *p, int page) { return (*static_cast<std::shared_ptr<KVPagePool> *>(p))->owners(page); }

// Copies (from, to) into out; returns their count, -1 on failure.
static int copies_out(const std::string &e, const std::vector<tensor::runtime::KVPageCopy> &copies, int *out) {
  if (!e.empty()) return fail(e);
  for (std::size_t i = 0; i < copies.size(); ++i) {
    out[2 * i] = copies[i].from;
    out[2 * i + 1] = copies[i].to;
  }
  return static_cast<int>(copies.size());
}
int kv_state_fork(void *s, void *source, int *out) {
  std::vector<tensor::runtime::KVPageCopy> copies;
  const auto e = static_cast<State *>(s)->state->fork(*static_cast<State *>(source)->state, &copies);
  return copies_out(e, copies, out);
}
int kv_state_unshare(void *s, int *out) {
  std::vector<tensor::runtime::KVPageCopy> copies;
  const auto e = static_cast<State *>(s)->state->unshareTail(&copies);
  return copies_out(e, copies, out);
}
int kv_state_replace(void *s, std::size_t lead, const int *pages, std::size_t count, std::size_t length) {
  return status(static_cast<State *>(s)->state->replaceTail(lead, {pages, pages + count}, length));
}
}
