// paged.h - the index arithmetic of the paged cache, and how attention cuts its
// rows into pieces, shared by the kernels of paged.hip and paged_attn.hip and
// host tests.  No HIP types: it also compiles as plain C++.
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

// What a call of moe_paged_fork_dev comes to.
enum ForkStatus { kForkOk = 0, kForkNoPages = 1, kForkCopies = 2, kForkBad = 4 };

// Place `i` entries past `from` in a ring of n (0 <= from < n, 0 <= i <= n).
MOE_BOTH int ring_place(int from, int i, int n) {
  const uint32_t at = (uint32_t)from + (uint32_t)i;
  return (int)(at >= (uint32_t)n ? at - (uint32_t)n : at);
}

// ---- attention: the rows' positions, laid end to end in units, cut into pieces (paged_attn.hip)

constexpr int kUnit = 128;         // positions of a unit: a step of every wave
// More rows than this are not cut, since every block looks through all of them for its piece: a block a row (or run).  A
// row at position 100000 (42 us alone) beside 2047 of a prompt 241 us, beside 2048 1106.
constexpr int kSplitRows = 2048;
constexpr int kCUs = 256;

// Positions that a row attends; kPadding: no row; kOutside: a request or position outside the tables.
constexpr int kPadding = -1, kOutside = -2, kNone = -3;
MOE_BOTH int row_length(int req, int pos, int n_req, int positions) {
  return req < 0 ? kPadding : req >= n_req || pos >= positions ? kOutside : pos + 1 > 0 ? pos + 1 : 0;
}

MOE_BOTH uint32_t units_of(int len) {
  return len == kPadding || len == kNone ? 0 : len <= kUnit ? 1 : ((uint32_t)len + kUnit - 1) / kUnit;
}

// What a run counts for among the pieces: its units, and kRunUnits for what each takes besides (its first loads, the join
// of the waves); the piece that starts among these has nothing to do for it.  512 / 2048 rows from position 0: none 41.6 /
// 367 us, 2 37.3 / 211, 8 38.0 / 239; a block a run, which leaves a long row to one block, 27.8 / 192.
constexpr uint32_t kRunUnits = 2;
MOE_BOTH uint32_t weight_of(int len) {
  const uint32_t n = units_of(len);
  return n ? n + kRunUnits : 0;
}

// Pieces that the rows are cut into: as many as blocks of all heads are resident at once, by the kernels' registers.
// (Twice as many, heads of 128: 24 rows 19.0 -> 21.5 us, one long row 52.8 -> 56.3, the e4m3 batch 56 -> 64.)
constexpr int kMaxParts = 3 * kCUs;   // of one row: no more than pieces
MOE_BOTH int pieces_for(int n_q, int n_kv, int head_dim) {
  const int blocks = kCUs * (head_dim <= 64 ? 3 : head_dim <= 128 ? 2 : 1), per = n_kv * ((n_q / n_kv + 15) / 16);
  return blocks > per ? blocks / per : 1;
}

// Rows of one request that a tile's columns hold.
MOE_BOTH int rows_shared(int n_q, int n_kv) { return n_q / n_kv <= 8 ? 16 / (n_q / n_kv) : 1; }

// How a call of T rows is cut, each of at most `positions`.
struct AttnCut {
  int share;    // rows that a tile's columns hold: runs are looked for; 1: each row for itself
  int most;     // pieces at most
  int pieces;   // most, or 0: rows are not cut, a block a row (or `share` rows)
  int blocks;   // of a head
  bool by_row;  // joins are listed a row, else a piece (`share` of each)
};

MOE_BOTH AttnCut cut_rows(int T, int n_req, bool listed, long long positions, int n_q, int n_kv, int head_dim) {
  AttnCut c;
  // rows outnumber the requests: some are of one request (or of none), so runs are looked for (where there are none the
  // search costs: 24 rows with 6 of no request 22.3 us, 18.5 without it)
  c.share = listed && T > n_req ? rows_shared(n_q, n_kv) : 1;
  c.most = pieces_for(n_q, n_kv, head_dim);
  // what all rows count for at most: as many pieces where that is less than `most`, a unit each
  const long long row = (positions + kUnit - 1) / kUnit, total = (row + (c.share > 1 ? kRunUnits : 0)) * T;
  // rows that no piece can cut (a unit at most), and more than a block's search takes, get a block each
  c.pieces = row > 1 && total <= 0x7fff0000ll && T <= kSplitRows ? c.most : 0;
  c.blocks = c.pieces ? (int)(total < c.most ? total : c.most) : (T + c.share - 1) / c.share;
  c.by_row = T <= c.most;
  return c;
}

// Units of a piece, from those of all rows (at most 2^31 with the pieces).
MOE_BOTH uint32_t piece_units(uint32_t total, const Divider& pieces) { return divide(total + pieces.d - 1, pieces); }

// Which units of a row (a run) that starts at `at` the piece begin .. end - 1 holds.
struct UnitRange {
  uint32_t from, to;
};
MOE_BOTH UnitRange units_in(uint32_t begin, uint32_t end, uint32_t at, uint32_t units) {
  return {begin > at ? begin - at : 0, end - at < units ? end - at : units};
}

// The pieces of `per` units that a row lies in: the first, and their number.
struct RowParts {
  int first, count;
};
MOE_BOTH RowParts parts_of(uint32_t at, uint32_t units, uint32_t per) {
  const uint32_t first = at / per;
  return {(int)first, units ? (int)((at + units - 1) / per - first + 1) : 0};
}

// A piece holds at most two parts of rows that go on in other pieces: part 0 of one (its start), in 2 piece + 1, and a
// later part of another, in 2 piece.
MOE_BOTH int part_place(int first_piece, int i) { return i == 0 ? 2 * first_piece + 1 : 2 * (first_piece + i); }

// Whether an entry of the join's list names parts to join: a row of the call, more than one part, all of them in its
// pieces.  What the rows' kernel leaves does; the join takes nothing else, so that no content of `work` leads it outside
// the call's buffers.
MOE_BOTH bool join_ok(int row, int parts, int first_piece, int place, int T, int pieces, int share) {
  const uint32_t first = (uint32_t)first_piece, all = (uint32_t)pieces;   // (no branches: one row of 131072 positions 49.7 -> 49.3 us)
  return ((uint32_t)row < (uint32_t)T) & (parts > 1) & (first < all) & ((uint32_t)parts <= all - first) & ((uint32_t)place < (uint32_t)share);
}

}  // namespace moe
