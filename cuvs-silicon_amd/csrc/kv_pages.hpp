// Host bookkeeping of a paged key/value cache: which pages each sequence
// holds, how many sequences hold each page, and which pages sequences have in
// common.  No HIP here: the device work that a call needs (page copies) is
// returned to the caller.
//
// A page holds `page_tokens` consecutive tokens of a sequence.  Sequences
// share pages by reference count, and a page that several hold is never
// written: extending a sequence whose last page is partly filled and shared
// first gives it a copy of that page (copy on write).  Free pages are handed
// out lowest id first, so page ids depend on the calls alone.
#pragma once

#include <algorithm>
#include <cstdint>
#include <functional>
#include <string>
#include <unordered_map>
#include <vector>

namespace cvs {
namespace kv {

struct PageCopy {
  int32_t src, dst;
};

// Thrown for a bad argument (`full` false) or when the pages run out.
struct PageError {
  std::string what;
  bool full;
};

struct Sequence {
  std::vector<int32_t> pages;
  int64_t length = 0;
  uint64_t version = 0;  // changes whenever pages or length do
  uint64_t mark = 0;     // of the last call that visited it (finds repeats)
};

class PageBook {
 public:
  PageBook(int64_t pages, int64_t page_tokens) : page_tokens_(page_tokens), refs_(size_t(pages), 0) {
    free_.resize(size_t(pages));
    for (int64_t i = 0; i < pages; ++i) free_[size_t(i)] = int32_t(i);  // ascending: a heap already
  }

  int64_t page_tokens() const { return page_tokens_; }
  int64_t pages() const { return int64_t(refs_.size()); }
  int64_t free_pages() const { return int64_t(free_.size()); }
  int64_t sequences() const { return int64_t(seqs_.size()); }
  int64_t pages_for(int64_t tokens) const { return (tokens + page_tokens_ - 1) / page_tokens_; }
  int32_t refs(int32_t page) const { return refs_[size_t(page)]; }

  Sequence& at(int64_t id) {
    auto it = seqs_.find(id);
    if (it == seqs_.end()) throw PageError{"no sequence " + std::to_string(id) + " in this cache", false};
    return it->second;
  }

  // The sequences that `n` ids name, none twice.
  std::vector<Sequence*> find(const int64_t* ids, int64_t n) {
    std::vector<Sequence*> found(static_cast<size_t>(n));
    ++mark_;
    for (int64_t i = 0; i < n; ++i) {
      Sequence& s = at(ids[i]);
      if (s.mark == mark_) throw PageError{"sequence " + std::to_string(ids[i]) + " is given twice", false};
      s.mark = mark_;
      found[size_t(i)] = &s;
    }
    return found;
  }

  int64_t create() {
    const int64_t id = next_id_;
    seqs_[id].version = ++version_;
    ++next_id_;
    return id;
  }

  // A new sequence of the parent's first `length` tokens, on the parent's pages.
  int64_t fork(int64_t parent, int64_t length) {
    const Sequence& p = at(parent);
    if (length < 0 || length > p.length)
      throw PageError{"fork at " + std::to_string(length) + " of a sequence of " + std::to_string(p.length) + " tokens",
                      false};
    Sequence child;
    child.pages.assign(p.pages.begin(), p.pages.begin() + pages_for(length));
    child.length = length;
    child.version = ++version_;
    const int64_t id = next_id_;
    const std::vector<int32_t>& held = seqs_.emplace(id, std::move(child)).first->second.pages;
    ++next_id_;
    for (const int32_t pg : held) ++refs_[size_t(pg)];
    return id;
  }

  // Makes room for tokens[i] more tokens in sequence ids[i], in this order; all of it or, when the pages do not
  // suffice, nothing.  Returns the copies that have to be made before the new tokens are written.
  std::vector<PageCopy> extend(const int64_t* ids, const int64_t* tokens, int64_t n) {
    const std::vector<Sequence*> seqs = find(ids, n);
    // What it takes: `dropped` counts the holders that a shared page loses to copies earlier in this call.
    int64_t need = 0;
    std::unordered_map<int32_t, int32_t> dropped;
    for (int64_t i = 0; i < n; ++i) {
      const Sequence& s = *seqs[size_t(i)];
      if (tokens[i] < 0 || tokens[i] > kMaxTokens - s.length)
        throw PageError{"a sequence of " + std::to_string(s.length) + " tokens cannot grow by " +
                            std::to_string(tokens[i]),
                        false};
      if (tokens[i] == 0) continue;
      need += pages_for(s.length + tokens[i]) - int64_t(s.pages.size());
      if (s.length % page_tokens_ != 0 && refs_[size_t(s.pages.back())] > 1) {
        int32_t& d = dropped[s.pages.back()];
        if (refs_[size_t(s.pages.back())] - d > 1) {
          ++d;
          ++need;
        }
      }
    }
    if (need > free_pages())
      throw PageError{"the cache has " + std::to_string(free_pages()) + " free pages, " + std::to_string(need) +
                          " are needed",
                      true};
    // All memory first, so that nothing throws once something has changed.
    std::vector<PageCopy> copies;
    copies.reserve(size_t(n));
    for (int64_t i = 0; i < n; ++i) {
      std::vector<int32_t>& held = seqs[size_t(i)]->pages;
      const size_t room = size_t(pages_for(seqs[size_t(i)]->length + tokens[i]));
      if (room > held.capacity()) held.reserve(std::max(room, 2 * held.capacity()));
    }
    for (int64_t i = 0; i < n; ++i) {
      if (tokens[i] == 0) continue;
      Sequence& s = *seqs[size_t(i)];
      if (s.length % page_tokens_ != 0 && refs_[size_t(s.pages.back())] > 1) {
        const int32_t own = take();
        copies.push_back({s.pages.back(), own});
        drop(s.pages.back());
        s.pages.back() = own;
      }
      s.length += tokens[i];
      while (int64_t(s.pages.size()) < pages_for(s.length)) s.pages.push_back(take());
      s.version = ++version_;
    }
    return copies;
  }

  // Keeps the first `length` tokens.
  void truncate(int64_t id, int64_t length) {
    Sequence& s = at(id);
    if (length < 0 || length > s.length)
      throw PageError{"truncate to " + std::to_string(length) + " of " + std::to_string(s.length) + " tokens", false};
    if (length == s.length) return;
    while (int64_t(s.pages.size()) > pages_for(length)) {
      drop(s.pages.back());
      s.pages.pop_back();
    }
    s.length = length;
    s.version = ++version_;
  }

  void release(const int64_t* ids, int64_t n) {
    const std::vector<Sequence*> seqs = find(ids, n);
    for (int64_t i = 0; i < n; ++i) {
      for (const int32_t pg : seqs[size_t(i)]->pages) drop(pg);
      seqs_.erase(ids[i]);
    }
  }

  // Moves the live pages whose ids are at or past their number, lowest first, into the free ids below it, lowest
  // first.  Sources and destinations are disjoint, so the copies may run in any order.
  std::vector<PageCopy> compact() {
    const int64_t live = pages() - free_pages();
    std::vector<PageCopy> moves;
    std::vector<int32_t> to(refs_.size(), -1);
    size_t hole = 0;
    for (int64_t pg = live; pg < pages(); ++pg) {
      if (refs_[size_t(pg)] == 0) continue;
      while (refs_[hole] != 0) ++hole;
      to[size_t(pg)] = int32_t(hole);
      moves.push_back({int32_t(pg), int32_t(hole)});
      ++hole;
    }
    if (moves.empty()) return moves;
    for (const PageCopy& m : moves) std::swap(refs_[size_t(m.src)], refs_[size_t(m.dst)]);
    for (auto& kv : seqs_) {
      bool moved = false;
      for (int32_t& pg : kv.second.pages)
        if (to[size_t(pg)] >= 0) {
          pg = to[size_t(pg)];
          moved = true;
        }
      if (moved) kv.second.version = ++version_;
    }
    free_.clear();
    for (int64_t pg = live; pg < pages(); ++pg) free_.push_back(int32_t(pg));
    return moves;
  }

  // Tokens of one sequence; lengths and positions stay within 31 bits on the device.
  static constexpr int64_t kMaxTokens = (int64_t(1) << 31) - 4096;

 private:
  int32_t take() {  // the caller has counted
    std::pop_heap(free_.begin(), free_.end(), std::greater<int32_t>());
    const int32_t pg = free_.back();
    free_.pop_back();
    refs_[size_t(pg)] = 1;
    return pg;
  }
  void drop(int32_t pg) {
    if (--refs_[size_t(pg)] > 0) return;
    free_.push_back(pg);  // within the capacity of the first allocation
    std::push_heap(free_.begin(), free_.end(), std::greater<int32_t>());
  }

  int64_t page_tokens_;
  std::vector<int32_t> refs_;
  std::vector<int32_t> free_;  // a heap, lowest id on top
  std::unordered_map<int64_t, Sequence> seqs_;
  int64_t next_id_ = 1;
  uint64_t version_ = 0, mark_ = 0;
};

// A run of pages that the same sequences have in common, for attention: pages [first, first + count) of the list of
// sequence `member` (any of them), and the sequences order[lo, hi).
struct SharedRun {
  int64_t first, count;
  int64_t lo, hi;
  int64_t member;
};

// The tree of common leading pages of `n` page lists: orders the lists so that those below one run are neighbours
// (`order`) and returns the runs, parents before children.  Each list is the concatenation of its runs.  Reads each
// page id a few times: linear in their number.
inline std::vector<SharedRun> shared_runs(const std::vector<const int32_t*>& lists, const std::vector<int64_t>& counts,
                                          std::vector<int64_t>& order) {
  const int64_t n = int64_t(lists.size());
  order.resize(size_t(n));
  for (int64_t i = 0; i < n; ++i) order[size_t(i)] = i;
  std::vector<SharedRun> runs;
  struct Todo {
    int64_t lo, hi, depth;
  };
  std::vector<Todo> todo{{0, n, 0}};
  while (!todo.empty()) {
    Todo t = todo.back();
    todo.pop_back();
    // Lists that end here first, then by the page at this depth; ties by position, so the order is the calls' alone.
    auto key = [&](int64_t i) { return counts[size_t(i)] > t.depth ? int64_t(lists[size_t(i)][t.depth]) : int64_t(-1); };
    if (t.hi - t.lo > 1)
      std::stable_sort(order.begin() + t.lo, order.begin() + t.hi, [&](int64_t a, int64_t b) { return key(a) < key(b); });
    while (t.lo < t.hi && key(order[size_t(t.lo)]) < 0) ++t.lo;
    for (int64_t lo = t.lo; lo < t.hi;) {
      int64_t hi = lo + 1;
      const int64_t m = order[size_t(lo)], page = key(m);
      while (hi < t.hi && key(order[size_t(hi)]) == page) ++hi;
      int64_t end = counts[size_t(m)];
      for (int64_t j = lo + 1; j < hi; ++j) {
        const int64_t o = order[size_t(j)];
        int64_t e = t.depth + 1;
        const int64_t most = std::min(end, counts[size_t(o)]);
        while (e < most && lists[size_t(o)][e] == lists[size_t(m)][e]) ++e;
        end = e;
      }
      runs.push_back({t.depth, end - t.depth, lo, hi, m});
      if (hi - lo > 1) todo.push_back({lo, hi, end});
      lo = hi;
    }
  }
  return runs;
}

}  // namespace kv
}  // namespace cvs
