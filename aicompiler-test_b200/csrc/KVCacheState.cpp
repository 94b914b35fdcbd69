// KV page pool and per-sequence cache state (see KVCacheState.hpp).
#include "KVCacheState.hpp"

#include <algorithm>
#include <limits>
#include <stdexcept>

namespace tensor::runtime {

KVPagePool::KVPagePool(std::size_t pageSize, std::size_t physicalPageCount)
    : pageSize_(pageSize), owners_(physicalPageCount, 0) {
  if (pageSize == 0 || physicalPageCount == 0 ||
      physicalPageCount > static_cast<std::size_t>(std::numeric_limits<std::int32_t>::max()))
    throw std::invalid_argument("KV page pool dimensions are invalid.");
  // LIFO free list seeded in ascending order: the first allocation returns the
  // highest page id, as the reference pool does (KVCacheState.cpp:36-41,70-78).
  freePages_.reserve(physicalPageCount);
  for (std::size_t page = 0; page < physicalPageCount; ++page)
    freePages_.push_back(static_cast<std::int32_t>(page));
}

bool KVPagePool::isAllocated(std::int32_t page) const noexcept {
  return owners(page) > 0;
}

std::size_t KVPagePool::owners(std::int32_t page) const noexcept {
  return page >= 0 && static_cast<std::size_t>(page) < owners_.size() ? owners_[static_cast<std::size_t>(page)] : 0;
}

void KVPagePool::retainPage(std::int32_t page) {
  if (!isAllocated(page)) throw std::invalid_argument("Paged KV attempted to share an invalid page.");
  ++owners_[static_cast<std::size_t>(page)];
}

std::int32_t KVPagePool::allocatePage() {
  if (injectedFailures_ > 0) {
    --injectedFailures_;
    return -1;
  }
  if (freePages_.empty()) return -1;
  const auto page = freePages_.back();
  freePages_.pop_back();
  owners_[static_cast<std::size_t>(page)] = 1;
  ++allocationCount_;
  peakUsedPages_ = std::max(peakUsedPages_, usedPages());
  return page;
}

void KVPagePool::releasePage(std::int32_t page) {
  if (!isAllocated(page)) throw std::invalid_argument("Paged KV attempted to release an invalid page.");
  if (--owners_[static_cast<std::size_t>(page)] > 0) return;
  freePages_.push_back(page);
  ++releaseCount_;
}

KVCacheState::KVCacheState(std::shared_ptr<KVPagePool> pool, std::size_t capacity, int slot,
                           BlockTableSink sink)
    : pool_(std::move(pool)), capacity_(capacity), slot_(slot), sink_(std::move(sink)) {
  if (!pool_ || capacity_ == 0) throw std::invalid_argument("KV cache state needs a pool and a capacity.");
  const auto pages = (capacity_ + pool_->pageSize() - 1) / pool_->pageSize();
  if (pages > pool_->capacityPages())
    throw std::invalid_argument("Paged KV pool cannot hold one request at full capacity.");
  logicalToPhysical_.assign(pages, -1);
}

KVCacheState::~KVCacheState() {
  for (auto &page : logicalToPhysical_) {
    if (page < 0) continue;
    try {
      pool_->releasePage(page);
    } catch (...) {
    }
    page = -1;
  }
}

std::size_t KVCacheState::allocatedPageCount() const noexcept {
  std::size_t count = 0;
  while (count < logicalToPhysical_.size() && logicalToPhysical_[count] >= 0) ++count;
  return count;
}

std::vector<std::int32_t> KVCacheState::pageTable() const {
  return {logicalToPhysical_.begin(),
          logicalToPhysical_.begin() + static_cast<std::ptrdiff_t>(allocatedPageCount())};
}

std::string KVCacheState::resizePageAllocation(std::size_t pageCount) {
  const auto allocated = allocatedPageCount();
  if (pageCount > allocated) {
    std::size_t logical = allocated;
    for (; logical < pageCount; ++logical) {
      const auto physical = pool_->allocatePage();
      if (physical < 0) break;
      logicalToPhysical_[logical] = physical;
    }
    if (logical != pageCount) {
      while (logical > allocated) {  // unwind: all or nothing
        --logical;
        pool_->releasePage(logicalToPhysical_[logical]);
        logicalToPhysical_[logical] = -1;
      }
      return "Paged KV cache physical page pool is exhausted.";
    }
    return {};
  }
  for (std::size_t logical = allocated; logical > pageCount; --logical) {
    pool_->releasePage(logicalToPhysical_[logical - 1]);
    logicalToPhysical_[logical - 1] = -1;
  }
  return {};
}

std::string KVCacheState::stageLength(std::size_t length) {
  if (length == 0 || length > capacity_) return "KV cache valid length is outside the configured capacity.";
  const auto previous = allocatedPageCount();
  const auto required = (length + pool_->pageSize() - 1) / pool_->pageSize();
  if (required > logicalToPhysical_.size())
    return "Paged KV cache has no block-table capacity for this length.";
  if (required > previous) {
    auto error = resizePageAllocation(required);
    if (!error.empty()) return error;
    if (sink_) {
      error = sink_(slot_, logicalToPhysical_);
      if (!error.empty()) {
        (void)resizePageAllocation(previous);
        (void)sink_(slot_, logicalToPhysical_);
        return error;
      }
    }
  }
  return {};
}

std::string KVCacheState::rollbackLength(std::size_t length) {
  if (length > capacity_) return "Cannot roll back KV cache beyond its configured capacity.";
  const auto required = length == 0 ? 0 : (length + pool_->pageSize() - 1) / pool_->pageSize();
  const auto previous = allocatedPageCount();
  if (required < previous) {
    auto error = resizePageAllocation(required);
    if (!error.empty()) return error;
    if (sink_) {
      error = sink_(slot_, logicalToPhysical_);
      if (!error.empty()) return error;
    }
  }
  if (currentLength_ > length) currentLength_ = length;
  return {};
}

void KVCacheState::commitLength(std::size_t length) {
  if (length == 0 || length > capacity_) throw std::invalid_argument("Cannot commit an invalid KV cache length.");
  currentLength_ = length;
}

std::string KVCacheState::fork(const KVCacheState &source, std::vector<KVPageCopy> *copies) {
  if (currentLength_ != 0 || allocatedPageCount() != 0) return "A fork needs an empty sequence.";
  const auto length = source.currentLength_, size = pool_->pageSize();
  if (pool_ != source.pool_ || length == 0 || length > capacity_) return "A fork needs a sequence of the same pool to fork from.";
  const auto full = length / size, pages = (length + size - 1) / size;
  if (pages > source.allocatedPageCount()) return "A fork needs a page for every committed position.";
  std::int32_t tail = -1;
  if (pages > full) {
    tail = pool_->allocatePage();
    if (tail < 0) return "Paged KV cache physical page pool is exhausted.";
  }
  for (std::size_t i = 0; i < full; ++i) {
    pool_->retainPage(source.logicalToPhysical_[i]);
    logicalToPhysical_[i] = source.logicalToPhysical_[i];
  }
  if (tail >= 0) logicalToPhysical_[full] = tail;
  if (sink_) {
    const auto error = sink_(slot_, logicalToPhysical_);
    if (!error.empty()) {
      (void)resizePageAllocation(0);
      (void)sink_(slot_, logicalToPhysical_);
      return error;
    }
  }
  if (tail >= 0) copies->push_back({source.logicalToPhysical_[full], tail});
  currentLength_ = length;
  return {};
}

std::string KVCacheState::unshareTail(std::vector<KVPageCopy> *copies, std::size_t end, const PageCopier &copy) {
  const auto size = pool_->pageSize();
  const auto pages = std::min(allocatedPageCount(), end / size + (end % size != 0 ? 1 : 0));
  auto row = logicalToPhysical_;
  std::vector<KVPageCopy> taken;
  const auto giveBack = [&] {
    for (const auto &t : taken) pool_->releasePage(t.to);
  };
  for (auto logical = currentLength_ / size; logical < pages; ++logical) {
    if (pool_->owners(row[logical]) < 2) continue;
    const auto page = pool_->allocatePage();
    if (page < 0) {
      giveBack();
      return "Paged KV cache physical page pool is exhausted.";
    }
    taken.push_back({row[logical], page});
    row[logical] = page;
  }
  if (taken.empty()) return {};
  if (copy) {
    const auto error = copy(taken);
    if (!error.empty()) {
      giveBack();
      return error;
    }
  }
  std::swap(row, logicalToPhysical_);
  if (sink_) {
    const auto error = sink_(slot_, logicalToPhysical_);
    if (!error.empty()) {
      std::swap(row, logicalToPhysical_);
      giveBack();
      (void)sink_(slot_, logicalToPhysical_);
      return error;
    }
  }
  for (const auto &t : taken) pool_->releasePage(t.from);
  copies->insert(copies->end(), taken.begin(), taken.end());
  return {};
}

std::string KVCacheState::replaceTail(std::size_t lead, const std::vector<std::int32_t> &pages, std::size_t length) {
  const auto allocated = allocatedPageCount();
  if (length == 0 || length > capacity_ || lead > allocated || lead + pages.size() > logicalToPhysical_.size() ||
      length > (lead + pages.size()) * pool_->pageSize())
    return "KV cache pages do not hold the new length.";
  auto row = logicalToPhysical_;
  for (std::size_t i = lead; i < row.size(); ++i) row[i] = i < lead + pages.size() ? pages[i - lead] : -1;
  std::swap(row, logicalToPhysical_);
  if (sink_) {
    const auto error = sink_(slot_, logicalToPhysical_);
    if (!error.empty()) {
      std::swap(row, logicalToPhysical_);
      (void)sink_(slot_, logicalToPhysical_);
      return error;
    }
  }
  for (std::size_t i = lead; i < allocated; ++i) pool_->releasePage(row[i]);
  currentLength_ = length;
  return {};
}

std::string KVCacheState::reset() {
  auto error = rollbackLength(0);
  currentLength_ = 0;
  return error;
}

}  // namespace tensor::runtime
