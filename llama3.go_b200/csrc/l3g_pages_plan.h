// The moves of a pool compaction (l3g_kvpool_compact), shared by the host
// runtime and its CPU check.  Plain C++, no CUDA API.
//
// `order` lists the pages in use in the order they shall have: order[t] is the
// page that becomes page t.  Pages move through a scratch of `batch` pages, a
// round at a time: a round fills the targets [a, a + batch) by
//   1. the wanted pages to scratch,
//   2. the pages that sit on those targets and are not wanted there to the
//      places that step 1 emptied (outside the targets),
//   3. scratch to the targets.
// No copy of a step reads what another copy of it writes.
#pragma once

#include <utility>
#include <vector>

namespace l3g {

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
