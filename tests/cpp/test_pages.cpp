// The page bookkeeping of the key/value cache (csrc/kv_pages.hpp), on the CPU: random calls against a plain model of
// its rules, all-or-nothing extension, and the tree of common leading pages.
#include <cstdio>
#include <map>
#include <random>
#include <set>

#include "check.hpp"
#include "kv_pages.hpp"

using namespace cvs::kv;

namespace {

struct Plain {
  int64_t total, page;
  std::map<int64_t, std::pair<std::vector<int32_t>, int64_t>> seqs;

  int refs(int32_t p) const {
    int n = 0;
    for (const auto& s : seqs)
      for (const int32_t q : s.second.first) n += q == p;
    return n;
  }
  std::set<int32_t> free() const {
    std::set<int32_t> f;
    for (int64_t p = 0; p < total; ++p)
      if (refs(int32_t(p)) == 0) f.insert(int32_t(p));
    return f;
  }
  // False, with nothing changed, when the pages run out.
  bool extend(const std::vector<int64_t>& ids, const std::vector<int64_t>& tokens, std::vector<PageCopy>& copies) {
    const auto before = seqs;
    for (size_t i = 0; i < ids.size(); ++i) {
      auto& s = seqs.at(ids[i]);
      if (tokens[i] == 0) continue;
      auto take = [&](int32_t& out) {
        const auto f = free();
        if (f.empty()) return false;
        out = *f.begin();
        return true;
      };
      if (s.second % page != 0 && refs(s.first.back()) > 1) {
        PageCopy c{s.first.back(), 0};
        if (!take(c.dst)) return seqs = before, copies.clear(), false;
        copies.push_back(c);
        s.first.back() = c.dst;
      }
      s.second += tokens[i];
      while (int64_t(s.first.size()) * page < s.second) {
        int32_t p = 0;
        if (!take(p)) return seqs = before, copies.clear(), false;
        s.first.push_back(p);
      }
    }
    return true;
  }
};

void check_same(PageBook& book, const Plain& plain) {
  CHECK(book.sequences() == int64_t(plain.seqs.size()));
  for (const auto& s : plain.seqs) {
    const Sequence& b = book.at(s.first);
    CHECK(b.pages == s.second.first);
    CHECK(b.length == s.second.second);
    for (const int32_t p : b.pages) CHECK(book.refs(p) == plain.refs(p));
  }
  CHECK(book.free_pages() == int64_t(plain.free().size()));
}

template <typename Fn>
bool refused(Fn&& fn, bool full) {
  try {
    fn();
  } catch (const PageError& e) {
    return e.full == full && !e.what.empty();
  }
  return false;
}

void random_calls(unsigned seed) {
  std::mt19937 r(seed);
  const int64_t total = 24, page = 32;
  PageBook book(total, page);
  Plain plain{total, page, {}};
  auto any = [&](int64_t lo, int64_t hi) { return lo + int64_t(r() % uint64_t(hi - lo + 1)); };
  int64_t full = 0;
  for (int step = 0; step < 400; ++step) {
    std::vector<int64_t> ids;
    for (const auto& s : plain.seqs) ids.push_back(s.first);
    std::shuffle(ids.begin(), ids.end(), r);
    const int64_t what = ids.empty() ? 0 : any(0, 9);
    if (what == 0 && ids.size() < 10) {
      plain.seqs[book.create()] = {};
    } else if (what <= 4) {
      ids.resize(size_t(any(1, std::min<int64_t>(4, int64_t(ids.size())))));
      std::vector<int64_t> tokens;
      for (size_t i = 0; i < ids.size(); ++i) tokens.push_back(any(0, 2) ? any(0, 70) : any(0, 1));
      std::map<int64_t, uint64_t> versions;
      for (const auto& s : plain.seqs) versions[s.first] = book.at(s.first).version;
      std::vector<PageCopy> want, got;
      bool ok = true;
      try {
        got = book.extend(ids.data(), tokens.data(), int64_t(ids.size()));
      } catch (const PageError& e) {
        ok = false;
        CHECK(e.full);
        ++full;
      }
      CHECK(plain.extend(ids, tokens, want) == ok);
      CHECK(got.size() == want.size());
      for (size_t i = 0; i < got.size(); ++i) CHECK(got[i].src == want[i].src && got[i].dst == want[i].dst);
      for (const auto& v : versions) {
        bool grown = false;
        for (size_t i = 0; i < ids.size(); ++i) grown |= ok && ids[i] == v.first && tokens[i] > 0;
        CHECK((book.at(v.first).version != v.second) == grown);
      }
    } else if (what <= 6 && ids.size() < 10) {
      const auto& p = plain.seqs.at(ids[0]);
      const int64_t n = any(0, p.second);
      const int64_t id = book.fork(ids[0], n);
      plain.seqs[id] = {std::vector<int32_t>(p.first.begin(), p.first.begin() + (n + page - 1) / page), n};
    } else if (what == 7) {
      auto& s = plain.seqs.at(ids[0]);
      const int64_t n = any(0, s.second);
      book.truncate(ids[0], n);
      s.first.resize(size_t((n + page - 1) / page));
      s.second = n;
    } else if (what == 8) {
      book.release(ids.data(), 1);
      plain.seqs.erase(ids[0]);
    } else {
      const auto f = plain.free();
      const int64_t live = total - int64_t(f.size());
      std::map<int32_t, int32_t> to;
      auto hole = f.begin();
      for (int64_t p = live; p < total; ++p)
        if (!f.count(int32_t(p))) to[int32_t(p)] = *hole++;
      const auto moves = book.compact();
      CHECK(moves.size() == to.size());
      for (const auto& m : moves) CHECK(to.at(m.src) == m.dst);
      for (auto& s : plain.seqs)
        for (int32_t& p : s.second.first)
          if (to.count(p)) p = to.at(p);
    }
    check_same(book, plain);
  }
  CHECK(full > 0);
}

void refusals() {
  PageBook book(4, 32);
  const int64_t a = book.create(), b = book.create();
  const int64_t ab[] = {a, b}, aa[] = {a, a}, none[] = {77};
  const int64_t t[] = {40, 1}, neg[] = {-1, 0}, far[] = {PageBook::kMaxTokens + 1, 0};
  (void)book.extend(ab, t, 2);
  CHECK(refused([&] { (void)book.extend(aa, t, 2); }, false));
  CHECK(refused([&] { (void)book.extend(none, t, 1); }, false));
  CHECK(refused([&] { (void)book.extend(ab, neg, 2); }, false));
  CHECK(refused([&] { (void)book.extend(ab, far, 2); }, false));
  CHECK(refused([&] { (void)book.fork(a, 41); }, false));
  CHECK(refused([&] { (void)book.fork(a, -1); }, false));
  CHECK(refused([&] { (void)book.fork(77, 0); }, false));
  CHECK(refused([&] { book.truncate(a, 41); }, false));
  CHECK(refused([&] { book.release(aa, 2); }, false));
  CHECK(book.at(a).length == 40 && book.free_pages() == 1);
  // Two holders of one partly filled page: one copies it, the last one keeps it.
  const int64_t c = book.fork(b, 1), bc[] = {b, c};
  const int64_t one[] = {1, 1};
  const auto copies = book.extend(bc, one, 2);
  CHECK(copies.size() == 1 && book.free_pages() == 0);
  CHECK(book.at(b).pages[0] == copies[0].dst && book.at(c).pages[0] == copies[0].src);
  const int64_t d = book.fork(b, 1), bd[] = {d};
  CHECK(refused([&] { (void)book.extend(bd, one, 1); }, true));
}

void runs(unsigned seed) {
  std::mt19937 r(seed);
  auto any = [&](int64_t lo, int64_t hi) { return lo + int64_t(r() % uint64_t(hi - lo + 1)); };
  // Lists that grow as forks do: a prefix of an earlier one, then pages of their own.
  std::vector<std::vector<int32_t>> lists;
  int32_t next = 0;
  const int64_t n = any(1, 20);
  for (int64_t i = 0; i < n; ++i) {
    std::vector<int32_t> l;
    if (!lists.empty() && any(0, 3)) {
      const auto& p = lists[size_t(any(0, int64_t(lists.size()) - 1))];
      l.assign(p.begin(), p.begin() + any(1, int64_t(p.size())));
    }
    for (int64_t k = any(l.empty() ? 1 : 0, 6); k > 0; --k) l.push_back(next++);
    lists.push_back(l);
  }
  std::shuffle(lists.begin(), lists.end(), r);
  std::vector<const int32_t*> p;
  std::vector<int64_t> counts, order;
  for (const auto& l : lists) {
    p.push_back(l.data());
    counts.push_back(int64_t(l.size()));
  }
  const auto got = shared_runs(p, counts, order);
  std::vector<std::vector<int32_t>> built(lists.size());
  int64_t read = 0;
  for (const SharedRun& s : got) {
    CHECK(s.lo < s.hi && s.count > 0);
    read += s.count;
    bool member = false;
    for (int64_t i = s.lo; i < s.hi; ++i) {
      auto& b = built[size_t(order[size_t(i)])];
      CHECK(int64_t(b.size()) == s.first);  // parents before children
      b.insert(b.end(), p[size_t(s.member)] + s.first, p[size_t(s.member)] + s.first + s.count);
      member |= order[size_t(i)] == s.member;
    }
    CHECK(member);
  }
  CHECK(built == lists);
  std::set<int32_t> distinct;
  for (const auto& l : lists) distinct.insert(l.begin(), l.end());
  CHECK(read == int64_t(distinct.size()));  // each page once
}

}  // namespace

int main() {
  for (unsigned s = 0; s < 20; ++s) random_calls(s);
  refusals();
  for (unsigned s = 0; s < 400; ++s) runs(s);
  return apitest::finish("test_pages");
}
