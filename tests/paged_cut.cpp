// Host test of how paged attention cuts a call's rows into pieces (cut_rows and what follows it in
// moe.cc_amd/csrc/paged.h; built and run by test_paged_cut.py): the kernels' walk, block by block, over random and chosen
// batches.  Every unit of every row has to belong to one launched block, every entry of the join's list that a launch
// reads has to be written, each part to have a place of its own and to be joined.  Prints "ok" or the first difference.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../moe.cc_amd/csrc/paged.h"

using namespace moe;

struct Call {
  int T, n_req, positions, n_q, n_kv, hd;
  bool listed;
  std::vector<int> req, pos;
};

struct Join {
  int row, parts, first, place;
};

// One item of the walk: rows row .. row + n - 1, a weight's first unit.
struct Item {
  int row, n, len;
  uint32_t at, weight;
};

static const char* g_what = "";
static void fail(const Call& c, const char* what, long long a, long long b) {
  std::printf("%s: %s: %lld %lld (T %d, n_req %d, positions %d, heads %d/%d of %d)\n", g_what, what, a, b, c.T, c.n_req, c.positions, c.n_q, c.n_kv,
              c.hd);
  std::exit(1);
}

// The items in order.  Runs: as find_runs and run_at see them, neighbours of one request among the same `share` rows.
static std::vector<Item> items_of(const Call& c, int share) {
  std::vector<Item> items;
  auto len = [&](int t) { return row_length(c.listed ? c.req[t] : t, c.pos[t], c.n_req, c.positions); };
  uint32_t at = 0;
  for (int t = 0; t < c.T;) {
    int n = 1, longest = len(t);
    if (share > 1)
      for (; t + n < c.T && (t + n) % share && len(t) >= 0 && len(t + n) >= 0 && c.req[t + n] == c.req[t]; ++n)
        longest = len(t + n) > longest ? len(t + n) : longest;
    const uint32_t w = share > 1 ? weight_of(longest) : units_of(longest);
    items.push_back({t, n, longest, at, w});
    at += w;
    t += n;
  }
  return items;
}

static void check(const Call& c) {
  const AttnCut cut = cut_rows(c.T, c.n_req, c.listed, c.positions, c.n_q, c.n_kv, c.hd);
  const bool runs = cut.share > 1;
  if (cut.most > kMaxParts || cut.by_row != (c.T <= cut.most)) fail(c, "most", cut.most, cut.by_row);
  // rows a thread of the search for runs
  if (runs && cut.pieces && ((c.T + cut.share - 1) / cut.share + 255) / 256 * cut.share > 16) fail(c, "rows a thread", c.T, cut.share);
  const std::vector<Item> items = items_of(c, cut.share);
  uint32_t total = 0;
  for (const Item& i : items) total += i.weight;
  std::vector<std::vector<int>> seen(c.T);
  for (const Item& i : items)
    for (int r = 0; r < i.n; ++r) seen[i.row + r].resize(units_of(i.len));
  const Join none = {0, -1, 0, 0};   // what `work` held
  std::vector<Join> joins(cut.by_row ? c.T : cut.most * cut.share, none);
  std::vector<int> places(2 * (cut.pieces ? cut.most : 1), -1);   // the item whose part lies there
  const Divider each = make_divider((uint32_t)cut.most);
  if (cut.pieces && total + (uint32_t)cut.most > 0x7fffffffu) fail(c, "past 31 bits", total, cut.most);
  for (int b = 0; b < cut.blocks; ++b) {
    uint32_t begin = 0, end = 1u << 30, per = 1u << 30;
    size_t k = 0;
    if (cut.pieces) {
      per = piece_units(total, each), begin = (uint32_t)b * per, end = begin + per < total ? begin + per : total;
      if (cut.by_row && b == 0)
        for (const Item& i : items)
          if (i.len == kPadding) joins[i.row] = {0, 0, 0, 0};
      if (!cut.by_row)
        for (int i = 0; i < cut.share; ++i) joins[b * cut.share + i] = {0, 0, 0, 0};
      while (k < items.size() && !(begin >= items[k].at && begin - items[k].at < items[k].weight)) ++k;
      if (k == items.size()) continue;
    } else {
      while (items[k].row != b * cut.share) ++k;
    }
    for (; k < items.size(); ++k) {
      const Item& i = items[k];
      const int row_end = cut.pieces ? c.T : (b + 1) * cut.share < c.T ? (b + 1) * cut.share : c.T;
      if (i.row >= row_end) break;
      const uint32_t units = units_of(i.len), at = cut.pieces ? i.at : i.at - items[k].at;
      if (!units) continue;
      if (cut.pieces && at >= end) break;
      const UnitRange u = units_in(begin, end, at, units);
      if (u.from < units) {   // (else it starts among what a run takes besides)
        if (u.to > units || u.from >= u.to) fail(c, "range", u.from, u.to);
        for (int r = 0; r < i.n; ++r)
          for (uint32_t x = u.from; x < u.to; ++x) ++seen[i.row + r][x];
        const RowParts p = parts_of(at, units, per);
        const bool parted = cut.pieces && p.count > 1, last = end >= at + units;
        if (!parted && (u.from || u.to != units)) fail(c, "a part of a whole row", u.from, u.to);
        if (parted) {
          const int place = part_place(b - (u.from != 0), u.from != 0);
          if (place < 0 || place >= 2 * cut.most || places[place] >= 0) fail(c, "place", place, i.row);
          places[place] = (int)k;
        }
        for (int r = 0; r < i.n; ++r) {
          const int entry = cut.by_row ? i.row + r : b * cut.share + r;
          if (parted && (cut.by_row ? u.from == 0 : last)) joins[entry] = {i.row + r, p.count, p.first, r};
          if (!parted && cut.by_row && u.from == 0) joins[entry] = {0, 0, 0, 0};
        }
      }
      if (cut.pieces && at + i.weight >= end) break;
    }
  }
  for (int t = 0; t < c.T; ++t)
    for (size_t u = 0; u < seen[t].size(); ++u)
      if (seen[t][u] != 1) fail(c, seen[t][u] ? "computed twice: row, unit" : "lost: row, unit", t, (long long)u);
  if (!cut.pieces) return;
  // the join: what it reads is what was left for it, and all of that
  std::vector<char> row_joined(c.T);
  std::vector<char> used(places.size());
  for (int e = 0; e < (cut.by_row ? c.T : cut.blocks * cut.share); ++e) {
    const Join j = joins[e];
    if (j.parts < 0) fail(c, "an entry that no one wrote", e, 0);
    if (join_ok(j.row, j.parts, j.first, j.place, c.T, cut.pieces, cut.share) != (j.parts > 1)) fail(c, "join_ok", j.row, j.parts);
    if (j.parts <= 1) continue;
    if (j.row < 0 || j.row >= c.T || row_joined[j.row]++) fail(c, "joined twice", e, j.row);
    for (int i = 0; i < j.parts; ++i) {
      const int at = part_place(j.first, i);
      if (at < 0 || at >= (int)places.size() || places[at] < 0) fail(c, "a part that no one left", j.row, i);
      const Item& it = items[places[at]];
      if (j.row != it.row + j.place || j.place >= it.n) fail(c, "another row's part", j.row, it.row);
      used[at] = 1;
    }
  }
  for (size_t i = 0; i < places.size(); ++i)
    if ((places[i] >= 0) != used[i]) fail(c, "a part that is not joined", (long long)i, places[i]);
}

static std::mt19937 g_rng(7);
static int rnd(int lo, int hi) { return lo + (int)(g_rng() % (uint32_t)(hi - lo + 1)); }

// n requests at `at` positions, a row each, then T - n rows of no request
static Call padded(int n, int T, int at, int positions, int n_q, int n_kv, int hd) {
  Call c{T, n, positions, n_q, n_kv, hd, true, {}, {}};
  for (int t = 0; t < T; ++t) c.req.push_back(t < n ? t : -1), c.pos.push_back(t < n ? at - 1 : -1);
  return c;
}

static void chosen() {
  g_what = "padded batch";
  check(padded(16, 17, 100, 256, 32, 4, 128));
  check(padded(32, 40, 60, 256, 32, 4, 128));
  check(padded(16, 18, 700, 768, 32, 4, 128));
  check(padded(16, 17, 2048, 2048, 8, 1, 64));
  check(padded(10, 11, 500, 512, 32, 4, 128));
  check(padded(16, 18, 512, 512, 32, 4, 128));
  for (int tokens : {1, 2, 3, 8})
    for (int n = 1; n <= 64; ++n)
      for (int units = 1; units <= 17; ++units)
        for (int nkv : {1, 2, 4, 8, 32}) {
          check(padded(n, n + tokens, units * 128, units * 128, 32, nkv, 128));
          check(padded(n, n + tokens, units * 128 - 127, units * 128, 32, nkv, 128));
        }
  g_what = "runs split at group borders";
  Call c{4, 3, 256, 32, 4, 128, true, {0, 1, 1, 2}, {250, 250, 251, 130}};
  check(c);
  g_what = "the largest sums";
  for (int T : {1000, 2000, 2047, 2048})
    for (long long units = 0x7fff0000ll / T - 3; units <= 0x7fff0000ll / T + 3; ++units) {
      const AttnCut k = cut_rows(T, T / 2, true, units * 128, 32, 4, 128);
      if (k.pieces && units * T + (long long)kRunUnits * T + k.most > 0x7fffffffll) fail(c, "past 31 bits", T, units);
      if (k.share < 2) fail(c, "share", T, units);
    }
}

static void drawn() {
  g_what = "drawn batch";
  const int heads[][3] = {{32, 4, 128}, {8, 1, 64}, {32, 32, 128}, {4, 4, 64}, {6, 2, 80}, {10, 2, 48}, {15, 3, 80}, {8, 8, 256}, {40, 2, 128},
                          {16, 1, 256}, {9, 3, 16}, {7, 1, 192}, {64, 8, 128}, {600, 600, 64}, {1, 1, 16}, {12, 3, 256}};
  for (int i = 0; i < 40000; ++i) {
    const auto& h = heads[rnd(0, 15)];
    Call c{0, 0, 0, h[0], h[1], h[2], rnd(0, 3) > 0, {}, {}};
    const int size = rnd(0, 9);
    c.T = size < 5 ? rnd(1, 70) : size < 8 ? rnd(1, 400) : rnd(1, 2300);
    c.positions = rnd(0, 2) ? rnd(1, 20) * rnd(1, 128) : rnd(1, 60000);
    const int near = rnd(0, 2);   // requests: about as many as rows, fewer, any
    c.n_req = !c.listed ? c.T + rnd(0, 3) : near == 0 ? (c.T > 4 ? c.T - rnd(0, 4) : 1) : near == 1 ? rnd(1, c.T) : rnd(1, c.T + 10);
    const int lengths = rnd(0, 3), stretch = rnd(0, 2) ? 1 : rnd(1, 40), odd = rnd(0, 3) ? 0 : 10;
    for (int t = 0; t < c.T; ++t) {
      int r = t && rnd(0, stretch - 1) ? c.req.back() : near == 0 ? (t < c.n_req ? t : -1) : rnd(0, c.n_req - 1);
      if (odd && rnd(0, 99) < odd) r = rnd(0, 1) ? -1 : c.n_req + rnd(0, 1);
      int p = lengths == 0 ? c.positions - 1 : lengths == 1 ? rnd(-1, c.positions - 1) : lengths == 2 ? rnd(0, 9) ? rnd(-1, c.positions / 8) : c.positions - 1 : rnd(-1, 200);
      if (p >= c.positions && !odd) p = c.positions - 1;
      c.req.push_back(r), c.pos.push_back(p);
    }
    check(c);
  }
}

// entries that name anything outside a call's rows, pieces or columns
static void entries() {
  const int junk[] = {-0x7fffffff - 1, -0x5a5a5a5b, -1, 0, 1, 2, 3, 7, 8, 9, 127, 128, 129, 768, 0x3c3c3c3c, 0x7f7f7f7f, 0x7fffffff};
  for (int row : junk)
    for (int parts : junk)
      for (int first : junk)
        for (int place : junk) {
          const bool in = row >= 0 && row < 8 && parts >= 2 && first >= 0 && (long long)first + parts <= 128 && place >= 0 && place < 2;
          if (join_ok(row, parts, first, place, 8, 128, 2) != in) std::printf("join_ok: %d %d %d %d\n", row, parts, first, place), std::exit(1);
          if (in && part_place(first, parts - 1) >= 256) std::printf("part_place: %d %d\n", first, parts), std::exit(1);
        }
}

int main() {
  entries();
  chosen();
  drawn();
  std::printf("ok\n");
  return 0;
}
