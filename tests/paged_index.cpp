// Host test of moe.cc_amd/csrc/paged.h (built and run by test_paged_index.py):
// every result against plain 64-bit arithmetic.  Prints "ok" or the first
// difference.
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#include "../moe.cc_amd/csrc/paged.h"

using namespace moe;

static void fail(const char* what, long long a, long long b, long long c) {
  std::printf("%s: %lld %lld %lld\n", what, a, b, c);
  std::exit(1);
}

static void divisions() {
  const uint32_t top = 0x7fffffffu;
  for (uint32_t d = 1; d <= 70000; d = d < 300 ? d + 1 : d + 97) {
    const Divider v = make_divider(d);
    for (uint32_t k = 0; k < 40; ++k)   // around multiples over the whole range
      for (int o = -1; o <= 1; ++o) {
        const long long x = (long long)(top / d / 39 * k) * d + o;
        if (x < 0 || x > top) continue;
        if (divide((uint32_t)x, v) != (uint32_t)x / d) fail("divide", x, d, divide((uint32_t)x, v));
      }
    for (uint32_t x : {0u, 1u, d - 1, d, d + 1, top - 1, top})
      if (divide(x, v) != x / d) fail("divide", x, d, divide(x, v));
  }
  for (uint32_t d : {1u << 30, (1u << 30) + 1, top - 1, top}) {
    const Divider v = make_divider(d);
    for (uint32_t x : {0u, d - 1, d, top})
      if (divide(x, v) != x / d) fail("divide", x, d, divide(x, v));
  }
}

static void rows() {
  // a cache past 2^32 elements: 60000 pages of 16 positions, 8 heads of 256,
  // slot-major and head-major
  for (int order = 0; order < 2; ++order) {
    PageMap m{60000, 16, 8, 256, 16ll * 8 * 256, order ? 16ll * 256 : 256, order ? 256 : 8ll * 256, make_divider(16)};
    for (int page : {0, 1, 32767, 59999})
      for (int head : {0, 7})
        for (int off : {0, 15}) {
          long long at = -1;
          const long long want = (long long)page * 32768 + (order ? head * 4096ll + off * 256ll : off * 2048ll + head * 256ll);
          if (!page_ok(m, page) || !slot_row(m, page * 16 + off, head, &at) || at != want || page_row(m, page, head, off) != want)
            fail("row", page, head, at);
        }
    // what is no page or no slot of the cache is refused
    for (int page : {-1, 60000, 60001, 0x7fffffff, (int)0x80000000})
      if (page_ok(m, page)) fail("page_ok", page, 0, 0);
    long long at = 5;
    for (int slot : {-1, 960000, 960001, 0x7fffffff, (int)0x80000000})
      if (slot_row(m, slot, 0, &at) || at != 5) fail("slot_row", slot, at, 0);
  }
  for (int ps : {1, 7, 16, 24, 100}) {
    const Divider per = make_divider((uint32_t)ps);
    for (int p = 0; p < 500; ++p) {
      if (position_slot(3, p, 10, ps, per) != 3 * ps + p % ps) fail("position_slot", p, ps, 0);
      for (int page : {-1, 10, 11, (int)0x80000000})   // no page: the first slot behind the cache
        if (position_slot(page, p, 10, ps, per) != 10 * ps) fail("position_slot", p, page, 0);
      if (pages_for(p, per) != p / ps + (p % ps != 0)) fail("pages_for", p, ps, 0);
    }
  }
}

static void plans() {
  // bad, long, tokens, need, back, head, count, n_pages, max_tokens
  struct { bool bad, lng; long long t, n, b; int head, count, pages, most, want; } c[] = {
      {false, false, 10, 3, 0, 0, 3, 8, 10, kPlanOk},      {false, false, 10, 4, 0, 0, 3, 8, 10, kPlanNoPages},
      {false, false, 11, 3, 0, 0, 3, 8, 10, kPlanTokens},  {false, true, 11, 9, 0, 0, 3, 8, 10, kPlanLong},
      {true, true, 0, 0, 0, 0, 3, 8, 10, kPlanBad},        {false, false, 0, 0, 5, 7, 3, 8, 10, kPlanOk},
      {false, false, 0, 0, 6, 7, 3, 8, 10, kPlanBad},      {false, false, 0, 0, 0, 8, 3, 8, 10, kPlanBad},
      {false, false, 0, 0, 0, -1, 3, 8, 10, kPlanBad},     {false, false, 0, 0, 0, 0, 9, 8, 10, kPlanBad},
      {false, false, 0, 0, 0, 0, -1, 8, 10, kPlanBad},     {false, false, 0, 0, 0, 0, 0, 1, 0, kPlanOk},
      {false, false, 1ll << 40, 1ll << 40, 0, 0, 8, 8, 0x7fffffff, kPlanTokens}};
  for (auto& x : c) {
    const int got = plan_status(x.bad, x.lng, x.t, x.n, x.b, x.head, x.count, x.pages, x.most);
    if (got != x.want) fail("plan_status", got, x.want, x.n);
  }
  for (int n : {1, 2, 7, 100})
    for (int from = 0; from < n; ++from)
      for (int i = 0; i <= n; ++i)
        if (ring_place(from, i, n) != (from + i) % n) fail("ring_place", from, i, n);
  if (pages_for(0x7fffffff, make_divider(1)) != 0x7fffffff) fail("pages_for", 0, 0, 0);
  if (ring_place(0x7ffffffe, 0x7fffffff, 0x7fffffff) != 0x7ffffffe) fail("ring_place", 0, 0, 0);
}

int main() {
  divisions();
  rows();
  plans();
  std::printf("ok\n");
  return 0;
}
