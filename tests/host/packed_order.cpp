// The issuing warps of the paired forward on the CPU: no product reads, and no slot of the ring is given back, before the warp has waited for the
// item; every item is given back once by every issuing warp, after the last product that reads it; scores, outputs and their order are whole.
// Prints one line per check that fails.
#include "packed_order.h"

#include <cstdio>
#include <set>
#include <vector>

using namespace attn;

static int failures = 0;
static void check(bool ok, const char* what, int r0, int row_end, int lo, int window) {
  if (ok || failures++ > 20) return;
  printf("failed: %s (rows %d to %d, keys from %d, window %d)\n", what, r0, row_end, lo, window);
}

// what one issuing warp has done
struct Warp {
  std::set<int> waited;
  std::vector<int> given_back;      // by item
  std::vector<int> scores[2], outputs[2];
  bool early = false, late = false;
  explicit Warp(int items) : given_back(items, 0) {}
  void read(int i, bool release) {
    if (waited.count(i) == 0) early = true;
    if (given_back[i] > 0) late = true;
    if (release) ++given_back[i];
  }
};

static void walk(int r0, int row_end, int lo, int begin, int window) {
  const ProductOrder o = pair_order(r0, row_end, lo, window, 128);
  auto expect = [&](bool ok, const char* what) { check(ok, what, r0, row_end, lo, window); };
  // the tiles that hold a key that a row sees belong to its row tile
  for (int i = r0; i < row_end; ++i) {
    const int x = i >= r0 + 128, first = begin > i - window + 1 ? begin : i - window + 1;
    expect(o.on(x, (first - lo) / 128) && o.on(x, (i - lo) / 128), "a visible key is in a tile of its row");
  }
  expect(o.from(0) == 0 && o.to(0) >= 1 && o.to(0) <= o.tiles && o.from(1) <= o.tiles && o.to(1) <= o.tiles, "the tiles are those of the stream");
  for (int j = 0; j < o.tiles; ++j) expect(o.on(0, j) || o.on(1, j), "every tile has a row tile");

  auto run = [&](Warp& w, int which) {      // which: 0, 1 a row tile alone, 2 both
    Arrivals known;
    auto arrived = [&](int i) { return known(i, [&](int n) { w.waited.insert(n); return true; }); };
    auto skip = [&](int i) { const bool here = arrived(i); w.read(i, true); return here; };
    auto free = [&](int x, int j) { expect(!w.scores[x].empty() && w.scores[x].back() == j, "scores are free after they were asked for"); return true; };
    auto scores = [&](int x, int j, bool release) { arrived(2 * j); w.read(2 * j, release); w.scores[x].push_back(j); return true; };
    auto outputs = [&](int x, int j, bool release) {
      arrived(2 * j + 1);
      w.read(2 * j + 1, release);
      expect(!w.scores[x].empty() && w.scores[x].back() >= j, "P follows its scores");
      w.outputs[x].push_back(j);
      return true;
    };
    expect(which < 2 ? issue_one_row_tile(o, which, skip, free, scores, outputs) : issue_both_row_tiles(o, arrived, scores, outputs), "the walk ends");
    expect(!w.early, "a product or a release before the item was waited for");
    expect(!w.late, "a product of an item that was given back");
    for (int n : w.given_back) expect(n == 1, "an item is given back once");
    for (int x = 0; x < 2; ++x) {
      if (which < 2 && x != which) continue;
      std::vector<int> all;
      for (int j = o.from(x); j < o.to(x); ++j) all.push_back(j);
      expect(w.scores[x] == all && w.outputs[x] == all, "every tile once, in order");
    }
  };
  for (int which = 0; which < 3; ++which) {
    Warp w(2 * o.tiles);
    run(w, which);
  }
}

int main() {
  const int rows[] = {1, 2, 100, 127, 128, 129, 130, 200, 255, 256};
  const int windows[] = {1, 2, 3, 100, 127, 128, 129, 130, 255, 256, 257, 300, 500, 1000, 5000, 1 << 30};
  for (int begin : {0, 77})
    for (int at : {0, 256, 512, 2048})
      for (int n : rows)
        for (int window : windows) {
          const int r0 = begin + at, lo = begin > r0 - window + 1 ? begin : r0 - window + 1;
          walk(r0, r0 + n, lo, begin, window);
        }
  return failures != 0;
}
