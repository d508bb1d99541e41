#include "core/page_pool.h"

#include <algorithm>
#include <limits>
#include <numeric>

#include "core/enforce.h"

namespace turbo_transformers {
namespace core {

PagePool::PagePool(int64_t pages, int64_t page_size) : page_size_(page_size) {
  TT_ENFORCE(pages >= 0 && pages <= std::numeric_limits<int32_t>::max(), "bad number of pages");
  TT_ENFORCE(page_size >= 1 && page_size <= 4096 && (page_size & (page_size - 1)) == 0, "page_size must be a power of two up to 4096");
  references_.assign((size_t)pages, 0);
  free_.resize((size_t)pages);
  for (int64_t i = 0; i < pages; ++i) free_[(size_t)i] = (int32_t)(pages - 1 - i);
}

const PagePool::Sequence& PagePool::Of(int64_t sequence) const {
  const auto it = sequences_.find(sequence);
  TT_ENFORCE(it != sequences_.end(), "there is no sequence %ld", (long)sequence);
  return it->second;
}

int32_t PagePool::References(int64_t page) const {
  TT_ENFORCE(page >= 0 && page < pages(), "there is no page %ld", (long)page);
  return references_[(size_t)page];
}

void PagePool::Release(int32_t page) {
  if (--references_[(size_t)page] == 0) free_.push_back(page);
}

int64_t PagePool::Add() {
  sequences_[next_];
  return next_++;
}

PagePool::Growth PagePool::GrowthOf(const std::vector<int64_t>& sequences, const std::vector<int64_t>& tokens) const {
  TT_ENFORCE_EQ(sequences.size(), tokens.size(), "one number of tokens for each sequence");
  std::vector<int64_t> named(sequences);
  std::sort(named.begin(), named.end());
  TT_ENFORCE(std::adjacent_find(named.begin(), named.end()) == named.end(), "a sequence is named twice");
  // Sequences that share a last page that is not full: each takes a page of its own but for the one that is left with it alone.  Whether that happens
  // depends on the order in which they come, so the pages are counted as they will be taken.
  std::unordered_map<int32_t, int32_t> left;
  int64_t needed = 0;
  Growth growth;
  growth.splits.assign(sequences.size(), false);
  std::vector<std::pair<int32_t, int64_t>> replaced;  // a shared page, and how many pages are taken before that which takes its place
  for (size_t i = 0; i < sequences.size(); ++i) {
    const Sequence& s = Of(sequences[i]);
    TT_ENFORCE(tokens[i] >= 0 && tokens[i] <= std::numeric_limits<int32_t>::max() - s.length, "bad number of tokens");
    if (tokens[i] > 0 && s.length % page_size_ != 0) {
      const int32_t last = s.pages.back();
      const auto it = left.emplace(last, references_[(size_t)last]).first;
      if (it->second > 1) {
        growth.splits[i] = true;
        --it->second;
        replaced.emplace_back(last, needed++);
      }
    }
    needed += PagesFor(s.length + tokens[i]) - (int64_t)s.pages.size();
  }
  TT_ENFORCE(needed <= free_pages(), "%ld pages are needed, %ld are free", (long)needed, (long)free_pages());
  for (const auto& page : replaced) growth.copies.emplace_back(page.first, free_[free_.size() - 1 - (size_t)page.second]);
  return growth;
}

PagePool::Copies PagePool::CopiesOf(const std::vector<int64_t>& sequences, const std::vector<int64_t>& tokens) const {
  return GrowthOf(sequences, tokens).copies;
}

PagePool::Copies PagePool::Extend(const std::vector<int64_t>& sequences, const std::vector<int64_t>& tokens) {
  Growth growth = GrowthOf(sequences, tokens);
  for (size_t i = 0; i < sequences.size(); ++i) {
    Sequence& s = sequences_[sequences[i]];
    auto take = [&] {
      const int32_t page = free_.back();
      free_.pop_back();
      references_[(size_t)page] = 1;
      return page;
    };
    if (growth.splits[i]) {
      --references_[(size_t)s.pages.back()];  // (others still hold it)
      s.pages.back() = take();
    }
    s.length += tokens[i];
    while ((int64_t)s.pages.size() < PagesFor(s.length)) s.pages.push_back(take());
  }
  return std::move(growth.copies);
}

int64_t PagePool::Fork(int64_t sequence) {
  const Sequence copy = Of(sequence);
  for (int32_t page : copy.pages) ++references_[(size_t)page];
  sequences_[next_] = copy;
  return next_++;
}

void PagePool::Truncate(int64_t sequence, int64_t length) {
  const Sequence& held = Of(sequence);
  TT_ENFORCE(length >= 0 && length <= held.length, "sequence %ld has %ld tokens", (long)sequence, (long)held.length);
  Sequence& s = sequences_[sequence];
  s.length = length;
  while ((int64_t)s.pages.size() > PagesFor(length)) {
    Release(s.pages.back());
    s.pages.pop_back();
  }
}

void PagePool::Free(int64_t sequence) {
  for (int32_t page : Of(sequence).pages) Release(page);
  sequences_.erase(sequence);
}

PagePool::Copies PagePool::MovesOf() const {
  int32_t hole = 0, live = 0;
  for (int32_t n : references_) live += n > 0;
  Copies moves;
  // live pages from number `live` on go to the free ones below it, in order: no page is read that another move writes
  for (int32_t page = live; page < (int32_t)pages(); ++page) {
    if (references_[(size_t)page] == 0) continue;
    while (references_[(size_t)hole] != 0) ++hole;
    moves.emplace_back(page, hole++);
  }
  return moves;
}

PagePool::Copies PagePool::Compact() {
  const Copies moves = MovesOf();
  std::vector<int32_t> to((size_t)pages());
  std::iota(to.begin(), to.end(), 0);
  for (const auto& move : moves) {
    to[(size_t)move.first] = move.second;
    std::swap(references_[(size_t)move.first], references_[(size_t)move.second]);
  }
  for (auto& entry : sequences_)
    for (int32_t& page : entry.second.pages) page = to[(size_t)page];
  free_.clear();
  for (int32_t page = (int32_t)pages() - 1; page >= 0 && references_[(size_t)page] == 0; --page) free_.push_back(page);
  return moves;
}

}  // namespace core
}  // namespace turbo_transformers
