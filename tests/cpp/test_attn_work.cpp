// test_attn_work.cpp -- the arithmetic by which the 8-bit cache's attention kernels
// turn a batch's lengths into rows and keys (ifx_attn_work.h), run on the host over
// every item that a batch can come to: each row of Q and of the masks that a lane
// reads is one of its request's, and a request without new tokens has no items.
#include <algorithm>
#include <cstdio>
#include <vector>

#include "../../inferflux_amd/csrc/ifx_attn_rows_q8.h"
#include "../../inferflux_amd/csrc/ifx_attn_tile.h"

using namespace ifx;

static int failures = 0;
#define CHECK(cond, ...)                                                          \
  do {                                                                            \
    if (!(cond) && ++failures < 20) std::printf(__VA_ARGS__), std::printf("\n"); \
  } while (0)

constexpr int kFew = 224, kMost = 100000;

struct Batch {
  const char *name;
  std::vector<int> kv, nq;
};

// A lane reads Q and its mask at q0 + tok, head kvh G + row % G.
static void reads(const Batch &t, const AttnArgs &a, const Request &r, int row, const char *what) {
  const int tok = row / a.G, head = row % a.G, at = r.q0 + tok;
  CHECK(row >= 0 && tok < r.nq && head >= 0 && head < a.G && at >= 0 && at < a.T,
        "%s: %s, G %d: row %d of a request of %d at %d of %d", t.name, what, a.G, row, r.nq, at, a.T);
}

static void items(const Batch &t, const AttnArgs &a, const Request &r, int2 units, int stage, int lds_rows,
                  const char *what) {
  CHECK(r.nq > 0 || units.x == 0, "%s: %s: %d tiles for a request without rows", t.name, what, units.x);
  CHECK(units.y >= 1, "%s: %s: no stages", t.name, what);
  for (int chunk : {1, 3, units.y}) {
    const int ns = (units.y + chunk - 1) / chunk;
    for (int i = 0; i < units.x * ns; ++i) {
      Split s{chunk, ns, 0, 0, i, units.x, r};
      RowsWork w{};
      if (!rows_work(a, s, stage, lds_rows, w)) continue;
      CHECK(w.R > 0 && w.ns <= ns && w.zbeg >= 0 && w.zend <= std::max(r.kv, 0), "%s: %s: rows %d, chunks %d of %d, keys %d to %d",
            t.name, what, w.R, w.ns, ns, w.zbeg, w.zend);
      for (int n = 0; n < kRowsMax; ++n) reads(t, a, r, row_of_lane(w, n), what);
    }
  }
}

int main() {
  const Batch batches[] = {
      {"idle first", {500, 40, 7}, {0, 40, 1}},
      {"idle last", {40, 7, 500}, {40, 1, 0}},
      {"idle first and last", {20000, 40, 64, 7, 300}, {0, 40, 33, 1, 0}},
      {"every second idle", {100, 200, 300, 400, 500, 600}, {0, 1, 0, 64, 0, 7}},
      {"a plan that failed", {500, 1, 0, 70000}, {0, 0, 0, 0}},
      {"fewer keys than rows", {3, 0, 64}, {5, 2, 64}},
      {"no idle request", {1, 33, 5000}, {1, 33, 200}},
  };
  for (const Batch &t : batches)
    for (int G : {1, 3, 5, 8, 32})
      for (int window : {0, 1, 100, 1 << 29})
        for (int extra : {0, 3}) {
          AttnArgs a{};
          a.G = G, a.window = window, a.B = static_cast<int>(t.kv.size());
          int total = 0;
          for (int n : t.nq) total += n;
          a.T = total + extra;
          int q0 = 0;
          for (size_t b = 0; b < t.kv.size(); ++b) {
            const Request r{q0, t.nq[b], t.kv[b]};
            q0 += t.nq[b];
            for (int most : {1, 2, 1 << 20}) {
              const int2 units = rows_units(a, r, most);
              CHECK(units.x <= most, "%s: %d blocks where there are %d", t.name, units.x, most);
              items(t, a, r, units, kRowKeys, kRowsMax, "few rows");
              if (r.nq * G <= 16) items(t, a, r, units, kRowKeys, std::max(r.nq * G, 1), "16 rows");
            }
            const int2 mixed = tile_units_q8(a, r, kQueryRows, kFew, kMost);
            const int2 tiles = tile_units_q8(a, r, kQueryRows, kFew, -1);
            if (few_rows(a, r, kMost)) {
              items(t, a, r, mixed, kFew, kRowsMax, "few rows among tiles");
            } else {
              CHECK(mixed.x == tiles.x && mixed.y == tiles.y, "%s: tiles", t.name);
            }
            CHECK(tiles.x == (r.nq * G + kQueryRows - 1) / kQueryRows, "%s: %d tiles of %d rows", t.name, tiles.x, r.nq * G);
            for (int tile = 0; tile < tiles.x; ++tile)
              for (int n = 0; n < kQueryRows; ++n)
                reads(t, a, r, std::min(tile * kQueryRows + n, r.nq * G - 1), "row tiles");
            if (r.nq == 0) {  // and where an item were there all the same, it ends at once
              RowsWork w{};
              CHECK(!rows_work(a, Split{1, 1, 0, 0, 0, 1, r}, kFew, kRowsMax, w), "%s: rows of an idle request", t.name);
            }
          }
        }
  std::printf("attention's work: %d failure(s)\n", failures);
  return failures != 0;
}
