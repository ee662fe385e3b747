// CPU check of pages_map and pages_unmap: states of a pool that are forked,
// written, trimmed and closed at random, with a model of what each position
// holds; the books are compared with the tables after every step, and a batch of
// states is mapped whole or not at all.  Prints "ok".
#include "l3g_pages_plan.h"

#include <cstdio>
#include <map>
#include <random>

using namespace l3g;

namespace {
constexpr int PAGE = 4, HEADS = 2, PPS = 5;

struct State : PageTable {
  int pos = 0, high = 0;
  bool alone = true;       // neither a fork nor forked
  std::vector<int> holds;  // what it wrote at each position
};

struct World {
  PageBook book;
  std::vector<std::vector<int>> mem;  // [page][PAGE]: what each row of a page holds
  std::map<int, State> states;
  explicit World(int n) : mem(n, std::vector<int>(PAGE, -1)) {
    book.refs.assign(n, 0);
    for (int i = n; i-- > 0;) book.free_pages.push_back(i);
  }
};

bool same(const PageBook& a, const PageBook& b) {
  return a.free_pages == b.free_pages && a.refs == b.refs;
}
bool same(const PageTable& a, const PageTable& b) {
  return a.h_pages == b.h_pages && a.mapped == b.mapped && a.pps == b.pps && a.own_from == b.own_from;
}

int fail(const char* what) {
  std::fprintf(stderr, "%s\n", what);
  return 1;
}

// every page's count is the number of tables that hold it, and no other is free
int check(const World& w) {
  std::vector<int> refs(w.mem.size(), 0);
  for (const auto& s : w.states) {
    const State& t = s.second;
    for (int h = 0; h < HEADS; ++h)
      for (int j = 0; j < PPS; ++j) {
        const int id = t.h_pages[h * PPS + j];
        if ((id >= 0) != (j < t.mapped)) return fail("a table entry without its page");
        if (id >= 0) ++refs[id];
        if (id >= 0 && j >= t.own_from && w.book.refs[id] != 1)
          return fail("a page taken for the state's own that others map");
      }
    for (int p = 0; p < t.pos; ++p)
      for (int h = 0; h < HEADS; ++h)
        if (w.mem[t.h_pages[h * PPS + p / PAGE]][p % PAGE] != t.holds[p] * HEADS + h)
          return fail("a position does not hold what its state wrote");
  }
  if (refs != w.book.refs) return fail("counts differ from the tables");
  std::vector<int> free(w.mem.size(), 0);
  for (int id : w.book.free_pages) ++free[id];
  for (size_t i = 0; i < free.size(); ++i)
    if (free[i] != (refs[i] == 0)) return fail("free list differs from the counts");
  return 0;
}

// As a batch of states goes about it: all of it, or none.  n: new positions.
int batch(World& w, const std::vector<std::pair<int, int>>& who, int& stamp, bool give_up) {
  const World before = w;
  std::vector<PageMapping> maps(who.size());
  size_t done = 0;
  for (; done < who.size(); ++done) {
    State& s = w.states[who[done].first];
    const bool ready = pages_ready(s, PAGE, s.pos, s.pos + who[done].second);
    if (s.alone && ready != (s.pos + who[done].second <= s.mapped * PAGE))
      return fail("a state that was never forked: ready once its positions are mapped");
    if (!pages_map(w.book, s, PAGE, s.pos, s.pos + who[done].second, s.high, maps[done])) {
      if (ready) return fail("ready, and no pages");
      break;
    }
    if (ready && maps[done].want) return fail("ready, and not writable");
    if (!pages_ready(s, PAGE, s.pos, s.pos + who[done].second) &&
        (s.pos + who[done].second + PAGE - 1) / PAGE >= s.own_from)
      return fail("not ready behind its mapping");
  }
  if (done < who.size() || give_up) {
    while (done-- > 0) pages_unmap(w.book, w.states[who[done].first], maps[done]);
    if (!same(w.book, before.book)) return fail("the pool is not what it was");
    for (const auto& s : before.states)
      if (!same(s.second, w.states[s.first])) return fail("a table is not what it was");
    return check(w);
  }
  for (size_t i = 0; i < who.size(); ++i)  // the copies, before any write
    for (size_t c = 0; c < maps[i].src.size(); ++c)
      for (int r = 0; r < maps[i].rows[c]; ++r)
        w.mem[maps[i].dst[c]][r] = w.mem[maps[i].src[c]][r];
  for (size_t i = 0; i < who.size(); ++i) {
    State& s = w.states[who[i].first];
    for (int k = 0; k < who[i].second; ++k, ++s.pos) {
      ++stamp;
      s.holds.resize(s.pos);
      s.holds.push_back(stamp);
      for (int h = 0; h < HEADS; ++h) {
        const int id = s.h_pages[h * PPS + s.pos / PAGE];
        if (w.book.refs[id] != 1) return fail("a write to a page that others map");
        w.mem[id][s.pos % PAGE] = stamp * HEADS + h;
      }
    }
    s.high = std::max(s.high, s.pos);
  }
  return check(w);
}

int run(unsigned seed) {
  std::mt19937 rng(seed);
  World w(8 + rng() % 40);
  int stamp = 0, next = 0;
  for (int it = 0; it < 300; ++it) {
    const int what = rng() % 10;
    if (w.states.empty() || (what == 0 && w.states.size() < 6)) {
      State s;
      s.pps = PPS;
      s.h_pages.assign(HEADS * PPS, -1);
      w.states[next++] = s;
      continue;
    }
    auto pick = std::next(w.states.begin(), rng() % w.states.size());
    State& s = pick->second;
    if (what == 1 && w.states.size() < 6) {  // fork
      State f = s;
      f.pos = f.high = rng() % (s.pos + 1);
      f.mapped = (f.pos + PAGE - 1) / PAGE;
      f.holds.resize(f.pos);
      for (int h = 0; h < HEADS; ++h)
        for (int j = 0; j < PPS; ++j) {
          int& id = f.h_pages[h * PPS + j];
          if (j < f.mapped) ++w.book.refs[id];
          else id = -1;
        }
      s.own_from = std::max(s.own_from, f.mapped);
      f.own_from = f.mapped;
      s.alone = f.alone = false;
      w.states[next++] = f;
    } else if (what == 2) {  // close
      for (int id : s.h_pages)
        if (id >= 0) w.book.drop(id);
      w.states.erase(pick);
    } else if (what == 3) {  // back, and trim
      s.pos = s.high = rng() % (s.pos + 1);
      const int keep = (s.pos + PAGE - 1) / PAGE;
      for (int h = 0; h < HEADS; ++h)
        for (int j = keep; j < s.mapped; ++j) {
          w.book.drop(s.h_pages[h * PPS + j]);
          s.h_pages[h * PPS + j] = -1;
        }
      s.own_from = std::min(s.own_from, keep);
      s.mapped = keep;
    } else if (what == 4) {  // back
      s.pos = rng() % (s.pos + 1);
    } else {
      std::vector<std::pair<int, int>> who;
      for (auto& x : w.states) {
        const int room = PPS * PAGE - x.second.pos;
        if (room > 0 && rng() % 3) who.push_back({x.first, 1 + (int)(rng() % std::min(room, 7))});
      }
      if (batch(w, who, stamp, rng() % 5 == 0)) return 1;
    }
    if (check(w)) return 1;
  }
  return 0;
}
}  // namespace

int main() {
  for (unsigned seed = 0; seed < 400; ++seed)
    if (run(seed)) return 1;
  std::puts("ok");
  return 0;
}
