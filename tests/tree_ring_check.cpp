// Every interleaving of the producer warps and the consumer of the tile ring of k_tree_tc, on small rings (see
// test_tree_ring_model.py). Barriers are modelled as the hardware has them: a wait names a parity, and a phase that
// completed twice looks like one that did not complete at all.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "ex_tree_ring.h"

struct Slot {
  int arrived = 0, boxes = 0, expected = 0, laps = 0;  // of the phase that is not complete; completed phases
  int used = 0;                                        // completed phases of the slot's "used up" barrier
  int holds = 0;                                       // boxes that lie in the slot
};
struct State {
  std::vector<int> at;  // next tile of every producer
  int use = 0;          // next tile of the consumer
  std::vector<Slot> s;
  std::string key() const {
    std::string k;
    for (int a : at) k += char('a' + a);
    k += char('a' + use);
    for (const Slot& x : s)
      for (int v : {x.arrived, x.boxes, x.expected, x.laps, x.used, x.holds}) k += char('A' + v);
    return k;
  }
};

// groups[n]: boxes of tile n; box i is producer i % F's. all: every producer arrives on every tile (ptc_arrivals), else the
// first, and for codes the last, alone. Returns 0: right, 1: stuck, 2: a tile of wrong boxes.
int run(bool codes, bool all, int slots, const std::vector<int>& groups) {
  const int F = ex::ptc_feeders(codes), N = (int)groups.size();
  auto arrivals = [&](int f) {
    if (!all && f != 0 && !(codes && f == F - 1)) return 0;
    return ex::ptc_arrivals(codes, f) > 1 ? 2 : 1;  // 32 lanes that arrive together: any number above one tells the same
  };
  int count = 0;
  for (int f = 0; f < F; ++f) count += arrivals(f);
  if (all) {  // and the kernel's own count is the sum of what arrives
    int n = 0;
    for (int f = 0; f < F; ++f) n += ex::ptc_arrivals(codes, f);
    if (n != ex::ptc_loaded_count(codes)) return 3;
  }
  State first;
  first.at.assign(F, 0);
  first.s.resize(slots);
  std::vector<State> todo = {first};
  std::set<std::string> seen = {first.key()};
  while (!todo.empty()) {
    const State st = todo.back();
    todo.pop_back();
    bool moved = false, done = st.use == N;
    for (int f = 0; f < F; ++f) done = done && st.at[f] == N;
    auto push = [&](const State& x) {
      moved = true;
      if (seen.insert(x.key()).second) todo.push_back(x);
    };
    for (int f = 0; f < F; ++f) {  // a producer's tile: wait until the slot is used up, its boxes, its arrivals
      const int n = st.at[f];
      if (n == N) continue;
      const int parity = n / slots % 2 ? 0 : 1;  // starts at 1: the first lap passes at once
      if (st.s[n % slots].used % 2 == parity) continue;
      State x = st;
      Slot& s = x.s[n % slots];
      int mine = 0;
      for (int i = 0; i < groups[n]; ++i) mine += i % F == f;
      if (mine > 0 && (s.laps != n / slots || st.use > n || st.use < n - slots + 1)) return 2;  // into another tile's place
      s.boxes += mine;
      s.holds += mine;
      s.arrived += arrivals(f);
      if (f == 0) s.expected = groups[n];
      if (s.arrived > count) return 2;
      if (s.arrived == count && s.boxes == s.expected) s.arrived = s.boxes = s.expected = 0, ++s.laps;
      ++x.at[f];
      push(x);
    }
    if (st.use < N) {
      const int n = st.use;
      if (st.s[n % slots].laps % 2 != n / slots % 2) {
        State x = st;
        Slot& s = x.s[n % slots];
        if (s.holds != groups[n]) return 2;
        s.holds = 0;
        ++s.used;
        ++x.use;
        push(x);
      }
    }
    if (!moved && !done) return 1;
  }
  return 0;
}

int main() {
  // full tiles, tails of one box, tiles none of whose pages exist
  const std::vector<std::vector<int>> loads = {{4, 4, 4, 4, 4, 4, 4}, {1, 1, 1, 1, 1, 1, 1, 4}, {0, 0, 0, 0, 0, 4, 4},
                                               {4, 1, 1, 0, 1, 1, 4, 4}, {2, 0, 0, 1, 1, 0, 0, 3}};
  long runs = 0, planted = 0;
  for (int codes = 0; codes < 2; ++codes)
    for (int slots = 1; slots <= 3; ++slots)
      for (const auto& g : loads) {
        ++runs;
        if (const int rc = run(codes, true, slots, g)) {
          std::printf("codes %d slots %d: fault %d\n", codes, slots, rc);
          return 1;
        }
        planted += run(codes, false, slots, g) != 0;
      }
  // the tiles' order: every block's keys and values once, keys a block ahead
  for (int nblk = 1; nblk < 40; ++nblk) {
    int keys = 0, values = 0;
    for (int n = 0; n < 2 * nblk; ++n) {
      int j;
      const bool v = ex::ptc_tile(n, nblk, j);
      if (j != (v ? values : keys)) return 2;
      (v ? values : keys)++;
      if (v && keys < (values + 1 < nblk ? values + 1 : nblk)) return 3;
    }
    if (keys != nblk || values != nblk) return 4;
  }
  std::printf("OK %ld %ld\n", runs, planted);
  return 0;
}
