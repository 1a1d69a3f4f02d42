// paged.h - the index arithmetic of the paged cache, shared by the kernels of
// paged.hip and a host test.  No HIP types: it also compiles as plain C++.
//
// A cache is `n_pages` pages of `page_size` positions.  A slot is one
// position's place in it, page * page_size + offset; a request's position p
// is in page tables[request][p / page_size].  An element's offset from the
// pool's base is 64-bit throughout (a long cache passes 2^32 elements).
#pragma once
#include <stdint.h>

#if defined(__HIP__) || defined(__HIPCC__)
#define MOE_BOTH __host__ __device__ inline
#else
#define MOE_BOTH inline
#endif

namespace moe {

// x / d for 0 <= x < 2^31 and a divisor fixed on the host: a high product, an
// add and a shift (division by invariant integers, Granlund and Montgomery:
// with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// x / d = (hi(m x) + x) >> s; the sum stays under 2^32 for x < 2^31).
struct Divider {
  uint32_t d, m, s;
};

MOE_BOTH Divider make_divider(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return Divider{d, (uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
}

MOE_BOTH uint32_t divide(uint32_t x, const Divider& v) {
  return ((uint32_t)(((uint64_t)x * v.m) >> 32) + x) >> v.s;
}

// One layer's pages: sizes and strides in elements (the same for K and V).
struct PageMap {
  int n_pages, page_size, n_kv, head_dim;
  long long page_stride, head_stride, slot_stride;
  Divider per;   // by page_size
};

// Offset of (page, head, offset in the page); the page must be page_ok.
MOE_BOTH long long page_row(const PageMap& m, int page, int head, int off) {
  return (long long)page * m.page_stride + (long long)head * m.head_stride + (long long)off * m.slot_stride;
}

MOE_BOTH bool page_ok(const PageMap& m, int page) { return (uint32_t)page < (uint32_t)m.n_pages; }

// Offset of a slot's row, false where the slot is none of the cache's.
MOE_BOTH bool slot_row(const PageMap& m, int slot, int head, long long* at) {
  const uint32_t page = divide((uint32_t)slot & 0x7fffffffu, m.per);
  if (slot < 0 || page >= (uint32_t)m.n_pages) return false;
  *at = page_row(m, (int)page, head, slot - (int)page * m.page_size);
  return true;
}

// The slot of position p of a request: its table entry `page`, or, where that
// is no page, the first slot behind the cache, which every reader refuses.
MOE_BOTH int position_slot(int page, int p, int n_pages, int page_size, const Divider& per) {
  if ((uint32_t)page >= (uint32_t)n_pages) return n_pages * page_size;
  return page * page_size + (p - (int)divide((uint32_t)p, per) * page_size);
}

// Pages that n >= 0 positions fill.
MOE_BOTH int pages_for(int n, const Divider& per) { return n ? (int)divide((uint32_t)n - 1, per) + 1 : 0; }

// What a step's plan comes to, from its totals.
enum PlanStatus { kPlanOk = 0, kPlanNoPages = 1, kPlanTokens = 2, kPlanLong = 3, kPlanBad = 4 };

MOE_BOTH int plan_status(bool bad, bool too_long, long long tokens, long long need, long long back, int head, int count,
                         int n_pages, int max_tokens) {
  if (bad || head < 0 || head >= n_pages || count < 0 || count > n_pages || count + back > n_pages) return kPlanBad;
  if (too_long) return kPlanLong;
  if (tokens > max_tokens) return kPlanTokens;
  if (need > count) return kPlanNoPages;
  return kPlanOk;
}

// Place `i` entries past `from` in a ring of n (0 <= from < n, 0 <= i <= n).
MOE_BOTH int ring_place(int from, int i, int n) {
  const uint32_t at = (uint32_t)from + (uint32_t)i;
  return (int)(at >= (uint32_t)n ? at - (uint32_t)n : at);
}

}  // namespace moe
