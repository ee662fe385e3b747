// CPU check of compact_plan: simulates the copies of random and adversarial
// orders, with every step's copies done at once (reads before writes) and
// checked for disjointness.  Prints "ok".
#include "l3g_pages_plan.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>

static int fail(const char* what, int n, int batch) {
  std::fprintf(stderr, "%s (pages %d, batch %d)\n", what, n, batch);
  return 1;
}

static int run(const std::vector<int>& order, int n, int batch) {
  std::vector<int> mem(n), scratch(batch, -1);
  for (int i = 0; i < n; ++i) mem[i] = i;  // page i holds the value i
  for (const auto& r : l3g::compact_plan(order, n, batch)) {
    if ((int)r.out.size() > batch) return fail("round larger than the scratch", n, batch);
    for (const auto& c : r.out) scratch.at(c.second) = mem.at(c.first);
    std::set<int> src, dst;
    std::vector<int> vals;
    for (const auto& c : r.away) {
      src.insert(c.first);
      if (!dst.insert(c.second).second) return fail("two copies to one page", n, batch);
      vals.push_back(mem.at(c.first));
    }
    for (int d : dst)
      if (src.count(d)) return fail("a page read and written in one step", n, batch);
    for (size_t i = 0; i < r.away.size(); ++i) mem[r.away[i].second] = vals[i];
    for (const auto& c : r.in) mem.at(c.second) = scratch.at(c.first);
  }
  for (size_t t = 0; t < order.size(); ++t)
    if (mem[t] != order[t]) return fail("page not in its place", n, batch);
  return 0;
}

int main() {
  std::mt19937 rng(5);
  for (int it = 0; it < 4000; ++it) {
    const int n = 1 + rng() % 60, used = rng() % (n + 1), batch = 1 + rng() % 9;
    std::vector<int> ids(n);
    for (int i = 0; i < n; ++i) ids[i] = i;
    if (it % 3 == 0) std::reverse(ids.begin(), ids.end());
    else if (it % 3 == 1) std::rotate(ids.begin(), ids.begin() + rng() % n, ids.end());
    else std::shuffle(ids.begin(), ids.end(), rng);
    ids.resize(used);
    if (run(ids, n, batch)) return 1;
  }
  std::puts("ok");
  return 0;
}
