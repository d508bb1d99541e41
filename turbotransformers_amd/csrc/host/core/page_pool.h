// The book of a cache in pages: which pages hold the tokens of which sequence, in order, and how many sequences share each.  Host only; what has to
// happen to the memory (copies of pages) is returned as pairs (from, to) for kernels::CopyPages.  No counterpart in the reference, whose layer
// cache is one dense tensor per layer (turbo_transformers/layers/multi_headed_attention.cpp:205-229).
#pragma once

#include <cstdint>
#include <unordered_map>
#include <utility>
#include <vector>

namespace turbo_transformers {
namespace core {

class PagePool {
 public:
  using Copies = std::vector<std::pair<int32_t, int32_t>>;  // (from, to); no page twice as `to`, none as both

  PagePool(int64_t pages, int64_t page_size);

  int64_t Add();  // a new sequence without tokens -> its number
  // Sequence sequences[i] grows by tokens[i] (a sequence may be named once).  A last page that is shared and not full is replaced by a page of its own,
  // whose copy is returned and has to be made before the new tokens are stored.  Without enough free pages nothing changes and the call throws.
  Copies Extend(const std::vector<int64_t>& sequences, const std::vector<int64_t>& tokens);
  // The copies that Extend would return (it throws where that would), with nothing changed: they go to free pages, so whoever makes them first and then calls
  // Extend has lost nothing where a copy fails.
  Copies CopiesOf(const std::vector<int64_t>& sequences, const std::vector<int64_t>& tokens) const;
  int64_t Fork(int64_t sequence);                         // a sequence with the same tokens in the same pages -> its number
  void Truncate(int64_t sequence, int64_t length);        // back to its first `length` tokens
  void Free(int64_t sequence);
  Copies Compact();  // live pages move to the lowest numbers; the moves have to be made before anything else reads or writes the cache
  Copies MovesOf() const;  // what Compact would return, with nothing changed: moves to free pages as well

  // Neighbours among `sequences` that begin with the same pages, full with their first held[i] tokens: rows [sequences][3] of (number of a family's first, number behind its last, tokens they have in
  // common), (own number, next, 0) for a sequence that is on its own.  A link of fewer than `least` tokens is none.
  struct FamilyRows {
    std::vector<int32_t> rows;
    int64_t count = 0, most = 0;  // families; the most tokens of one
  };
  FamilyRows Families(const std::vector<int64_t>& sequences, const std::vector<int64_t>& held, int64_t least) const;

  int64_t Length(int64_t sequence) const { return Of(sequence).length; }
  const std::vector<int32_t>& Pages(int64_t sequence) const { return Of(sequence).pages; }
  int32_t References(int64_t page) const;
  int64_t free_pages() const { return (int64_t)free_.size(); }
  int64_t pages() const { return (int64_t)references_.size(); }
  int64_t page_size() const { return page_size_; }
  int64_t sequences() const { return (int64_t)sequences_.size(); }

 private:
  struct Sequence {
    std::vector<int32_t> pages;
    int64_t length = 0;
  };
  const Sequence& Of(int64_t sequence) const;
  struct Growth {
    std::vector<bool> splits;  // whether a sequence's last page is replaced
    Copies copies;
  };
  Growth GrowthOf(const std::vector<int64_t>& sequences, const std::vector<int64_t>& tokens) const;
  int64_t PagesFor(int64_t tokens) const { return (tokens + page_size_ - 1) / page_size_; }
  void Release(int32_t page);

  int64_t page_size_, next_ = 0;
  std::vector<int32_t> references_;
  std::vector<int32_t> free_;  // lowest last
  std::unordered_map<int64_t, Sequence> sequences_;
};

}  // namespace core
}  // namespace turbo_transformers
