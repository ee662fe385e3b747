// The bookkeeping of a KV pool's pages, shared by the host runtime and its CPU
// checks: which pages states map, what a step has to map or copy before it
// writes, and the moves of a compaction.  Plain C++, no CUDA API.
#pragma once

#include <algorithm>
#include <utility>
#include <vector>

namespace l3g {

// Pages of a shared pool.  Under the pool's lock.
struct PageBook {
  std::vector<int> free_pages;  // a stack of free page ids
  std::vector<int> refs;        // states that map each page
  int take() {
    const int id = free_pages.back();
    free_pages.pop_back();
    refs[id] = 1;
    return id;
  }
  void drop(int id) {  // free once no state maps it
    if (--refs[id] == 0) free_pages.push_back(id);
  }
};

// A state's page table: entry [h * pps + j] is page j of (layer, kv head) h.
struct PageTable {
  int pps = 0;               // pages per (layer, kv head)
  std::vector<int> h_pages;  // -1: not mapped
  int mapped = 0;            // pages [0, mapped) of every (layer, kv head) are mapped
  // pages [own_from, mapped) are mapped by this state alone, as far as is known
  // without a look at their counts (a fork of the state raises it)
  mutable int own_from = 0;
  int heads() const { return pps ? (int)(h_pages.size() / pps) : 0; }
};

// One state's part of making positions writable, and what undoes it.
struct PageMapping {
  size_t want = 0;                // pages that it takes
  int mapped0 = 0, own0 = 0;      // the table's `mapped` and `own_from` before
  int first = 0, last = 0;        // the table's columns that changed
  std::vector<size_t> entries;    // entries whose page others map too, and their
  std::vector<int> src, dst;      // page, the state's own copy of it
  std::vector<int> rows;          // and the rows of it that have been written
};

// Whether positions [pos0, n_pos) are writable as they are: what a step of a
// state finds, but for one in KV_PAGE, without the pool's lock or a walk over
// its pages' counts (64 sessions of 32 layers and 8 kv heads: 16384 of them).
inline bool pages_ready(const PageTable& t, int page, int pos0, int n_pos) {
  const int need = std::min(t.pps, (n_pos + page - 1) / page);
  return need <= t.mapped && (pos0 / page >= t.own_from || pos0 / page >= need);
}

// Makes positions [pos0, n_pos) of table t writable: maps pages for positions
// [0, n_pos), and replaces those of [pos0, n_pos) that other states map too by
// pages of its own (whose copies, m.src to m.dst, the caller makes; positions
// [0, high) have been written).  False where the pool has too few free pages:
// then nothing but m.want has changed.
inline bool pages_map(PageBook& book, PageTable& t, int page, int pos0, int n_pos, int high,
                      PageMapping& m) {
  const int heads = t.heads(), need = std::min(t.pps, (n_pos + page - 1) / page);
  m = PageMapping{};
  m.mapped0 = m.first = t.mapped;
  m.own0 = t.own_from;
  m.last = std::max(t.mapped, need);
  for (int j = pos0 / page; j < std::min(need, t.mapped); ++j)
    for (int h = 0; h < heads; ++h)
      if (book.refs[t.h_pages[(size_t)h * t.pps + j]] > 1)
        m.entries.push_back((size_t)h * t.pps + j);
  m.want = m.entries.size() + (size_t)heads * (m.last - t.mapped);
  if (book.free_pages.size() < m.want) return false;
  for (size_t e : m.entries) {
    const int j = (int)(e % t.pps);
    m.src.push_back(t.h_pages[e]);
    m.dst.push_back(book.take());
    m.rows.push_back(std::max(0, std::min(page, high - j * page)));
    m.first = std::min(m.first, j);
    t.h_pages[e] = m.dst.back();
    book.drop(m.src.back());
  }
  for (int j = t.mapped; j < need; ++j)
    for (int h = 0; h < heads; ++h) t.h_pages[(size_t)h * t.pps + j] = book.take();
  if (std::min(need, t.mapped) >= t.own_from) t.own_from = std::min(t.own_from, pos0 / page);
  t.mapped = m.last;
  return true;
}

// Takes a pages_map back.  Several are taken back in the reverse order: then
// pool and tables are what they were, the order of the free pages too.
inline void pages_unmap(PageBook& book, PageTable& t, const PageMapping& m) {
  const int heads = t.heads();
  for (int j = t.mapped - 1; j >= m.mapped0; --j)
    for (int h = heads - 1; h >= 0; --h) {
      int& id = t.h_pages[(size_t)h * t.pps + j];
      book.drop(id);
      id = -1;
    }
  t.mapped = m.mapped0;
  t.own_from = m.own0;
  for (size_t i = m.entries.size(); i-- > 0;) {
    t.h_pages[m.entries[i]] = m.src[i];
    ++book.refs[m.src[i]];
    book.drop(m.dst[i]);
  }
}

// The moves of a pool compaction (l3g_kvpool_compact).
//
// `order` lists the pages in use in the order they shall have: order[t] is the
// page that becomes page t.  Pages move through a scratch of `batch` pages, a
// round at a time: a round fills the targets [a, a + batch) by
//   1. the wanted pages to scratch,
//   2. the pages that sit on those targets and are not wanted there to the
//      places that step 1 emptied (outside the targets),
//   3. scratch to the targets.
// No copy of a step reads what another copy of it writes.
struct CompactRound {
  std::vector<std::pair<int, int>> out;   // page -> scratch page
  std::vector<std::pair<int, int>> away;  // page -> page
  std::vector<std::pair<int, int>> in;    // scratch page -> page
};

inline std::vector<CompactRound> compact_plan(const std::vector<int>& order, int n_pages,
                                              int batch) {
  std::vector<CompactRound> rounds;
  std::vector<int> holds(n_pages, -1), at(n_pages, -1);  // page in a place, place of a page
  for (int p : order) holds[p] = p, at[p] = p;
  const int used = (int)order.size();
  for (int a = 0; a < used; a += batch) {
    const int b = a + batch < used ? a + batch : used;
    CompactRound r;
    std::vector<int> emptied, homeless;
    std::vector<int> targets;
    for (int t = a; t < b; ++t)
      if (at[order[t]] != t) targets.push_back(t);
    for (int t : targets) {
      const int from = at[order[t]];
      r.out.push_back({from, (int)r.out.size()});
      holds[from] = -1;
    }
    for (int t : targets)
      if (holds[t] >= 0) homeless.push_back(t);
    for (const auto& m : r.out)
      if (holds[m.first] < 0 && !(m.first >= a && m.first < b && at[order[m.first]] != m.first))
        emptied.push_back(m.first);
    for (size_t i = 0; i < homeless.size(); ++i) {
      const int t = homeless[i], to = emptied[i];
      r.away.push_back({t, to});
      holds[to] = holds[t];
      at[holds[to]] = to;
    }
    for (size_t i = 0; i < targets.size(); ++i) {
      r.in.push_back({(int)i, targets[i]});
      holds[targets[i]] = order[targets[i]];
    }
    for (int t : targets) at[order[t]] = t;
    if (!r.out.empty()) rounds.push_back(std::move(r));
  }
  return rounds;
}

}  // namespace l3g
