// paged_shared.hip - attention of rows whose requests begin in the same pages
// (moe_paged_share_dev, moe_paged_attn_shared_dev, include/moehip.h).
//
// out_t = softmax(scale q_t . k) v over positions 0 .. pos[t], in two parts that
// a last kernel joins by their maxima and sums: the positions that a group of
// rows shares, with the query heads of all its rows as columns of one product,
// and the rest of each row for itself.  Which positions those are, and how they
// are cut into blocks, is the same in every layer of a step, so
// moe_paged_share_dev writes it down once: a list of items, each some columns
// against some positions of one request's table, a block each.
//
// A column is a (row, query head) of one key-value head: column c of a group
// is head c % G of its row c / G, G = n_q / n_kv.
#include <math.h>

#include <type_traits>

#include "block_scan.h"
#include "moe_device.h"
#include "paged_attn.h"
#include "paged_tile.h"

namespace moe {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMostShared = 1 << 14;   // rows, groups of a call
constexpr int kN = 1024;               // threads of the plan's block
constexpr int kTile = 64;              // columns of a prefix item at most

// ---------------------------------------------------------------- the plan

// Columns `col0` .. of the rows from row0 on, against positions begin .. end - 1 of request req.
struct Item {
  int row0, col0, cols, req;
  int begin, end;
  int part;     // where its sums go
  int direct;   // 1: it is all that its row has
};

// A row's parts: of column c of its group tile c / columns, pieces part0 + tile * pieces ..; of its own own0 + tile * owns ..
struct RowPlan {
  int state, group, row0;
  int part0, pieces;
  int own0, owns, pad;
};
enum RowState { kLeave, kZero, kNan, kDone, kJoin };

struct GroupPlan {
  int row0, rows, req, prefix;   // prefix: positions taken together, 0: none
  int tiles, units, part0, pieces;
};

struct PlanHead {
  int prefix_items, own_items, pad[2];
};

// How a call is cut: the same for moe_paged_share_dev and moe_paged_attn_shared_dev.
struct ShareCut {
  int group;          // query heads of a key-value head
  int columns;        // of a prefix item: 1 << shift
  int shift;
  int own_columns;    // of a row's own
  int own_tiles;      // of a row
  int slots, own_slots;   // items that are resident at once, about
  int prefix_items, own_items;   // at most
};

ShareCut share_cut(int T, int n_groups, int n_q, int n_kv, int head_dim) {
  ShareCut c;
  c.group = n_q / n_kv;
  const long long mean = n_groups ? ((long long)T + n_groups - 1) / n_groups * c.group : 0;
  c.shift = 4;
  while (1 << c.shift < mean && 1 << c.shift < kTile) ++c.shift;
  c.columns = 1 << c.shift;
  c.own_columns = c.group < 16 ? c.group : 16;
  c.own_tiles = (c.group + 15) / 16;
  // Two blocks a CU are resident; as many pieces pay where the products do (bf16, us with two and with one: 64 rows of 8000 41.0,
  // 45.2; 8 groups of 8 rows of 4000 33.6, 32.6), else the parts that a piece more writes and the join reads cost more than
  // they gain (32 groups of 4 rows of 1000 27.7, 23.8; 4 of 4 of 4000 21.9, 17.2; 4 rows of 16000 24.2, 17.6; twice the
  // pieces: 8 of 8 of 4000 43.3, 64 of 8000 48.2).
  const int resident = kCUs * (head_dim <= 128 && c.columns == kTile ? 2 : 1);
  c.slots = resident > n_kv ? resident / n_kv : 1;
  c.prefix_items = c.slots + (int)((long long)T * c.group / c.columns) + n_groups;
  c.own_slots = 2 * kCUs > n_kv ? 2 * kCUs / n_kv : 1;
  c.own_items = c.own_slots + T * c.own_tiles;
  return c;
}

struct PlanParts {
  PlanHead* head;
  int* common;       // [T] leading pages that a row and its group's first share; kNotLive: no row to count
  RowPlan* rows;     // [T]
  GroupPlan* groups; // [n_groups]
  Item* prefix;      // [prefix_items]
  Item* own;         // [own_items]
};
constexpr int kNotLive = 0x7fffffff;

size_t plan_parts(const ShareCut& c, int T, int n_groups, void* base, PlanParts* p) {
  char* at = (char*)base;
  auto take = [&](auto** q, size_t n) {
    *q = (std::remove_reference_t<decltype(*q)>)at;
    at += (n * sizeof(**q) + 15) / 16 * 16;
  };
  take(&p->head, 1);
  take(&p->common, (size_t)T);
  take(&p->rows, (size_t)T);
  take(&p->groups, (size_t)n_groups);
  take(&p->prefix, (size_t)c.prefix_items);
  take(&p->own, (size_t)c.own_items);
  return (size_t)(at - (char*)base);
}

struct ShareArgs {
  moe_paged_share s;
  Divider per;    // by page_size
  ShareCut cut;
  PlanParts p;
};

// A wave a row: the group that holds it, that group's first live row, and how many leading pages the two have in common.
__global__ __launch_bounds__(256) void share_rows_kernel(ShareArgs a) {
  const moe_paged_share& s = a.s;
  const int t = (int)blockIdx.x * 4 + (int)threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (t >= s.T) return;
  const int positions = s.max_pages * s.page_size;
  auto length = [&](int r) { return row_length(s.req ? s.req[r] : r, s.pos[r], s.n_req, positions); };
  const int len = length(t);
  int lo = 0, hi = s.n_groups;   // the last group that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (s.first[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  const int group = lo > 0 && t < s.first[lo] ? lo - 1 : -1;
  if (lane == 0) a.p.rows[t].group = group;
  if (len <= 0) {
    if (lane == 0) a.p.common[t] = kNotLive;
    return;
  }
  int lead = t;
  if (group >= 0) {
    for (int r0 = max(s.first[group], 0); r0 < t; r0 += kWave) {
      const int r = r0 + lane;
      const uint64_t live = __ballot(r < t && length(r) > 0);
      if (live) {
        lead = r0 + __builtin_ctzll(live);
        break;
      }
    }
  }
  int same = (int)divide((uint32_t)len, a.per);
  const int* mine = s.tables + (size_t)(s.req ? s.req[t] : t) * s.max_pages;
  const int* other = s.tables + (size_t)(s.req ? s.req[lead] : lead) * s.max_pages;
  if (mine != other)
    for (int c0 = 0; c0 < same; c0 += kWave) {
      const int c = c0 + lane;
      const uint64_t differ = __ballot(c < same && mine[c] != other[c]);
      if (differ) {
        same = c0 + __builtin_ctzll(differ);
        break;
      }
    }
  if (lane == 0) a.p.common[t] = same;
}

__device__ __forceinline__ int units_in_all(int positions) { return (positions + kUnit - 1) / kUnit; }

// One block: the groups' prefixes, and the items.  Prefix tiles' units (128 positions) and rows' own are each cut so that
// their items are about as many as are resident at once: pieces of ceil(all units / slots), at least one an item, so no
// more items than `slots` and one for each tile or row.  ONE: a thread a group and a row (at most N of each), whose numbers
// stay in its registers and LDS; else they go around through the plan, N at a time.  Latency bounds it (us with both kernels:
// 8 groups of 8 rows 9.9 with 256 threads, 11.3 with 1024, 12.1 around through the plan; 120 groups of 8 16.1 and 27.7).
template <int N>
struct PlanShared {
  int wave[N / kWave];
  unsigned long long units, own;
  int least[N], lead[N], live[N];      // ONE: of the groups
  int part0[N], pieces[N], prefix[N];
  int own0[N];                           // ONE: of the rows
};

// The last of n ascending numbers, the first of which is 0, that is at most i.
__device__ __forceinline__ int owner_of(const int* at, int n, int i) {
  int lo = 0;
  for (int hi = n; hi - lo > 1;) {
    const int mid = (lo + hi) / 2;
    if (at[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ceil(all / slots), at least 1 (whole numbers below 2^53: the quotient is not rounded past one)
__device__ __forceinline__ int piece_of(unsigned long long all, int slots) {
  const double n = floor((double)(all + (unsigned long long)(slots - 1)) / (double)slots);
  return (int)fmin(fmax(n, 1.0), 1073741824.0);
}

// Units before piece j of `pieces` even ones.
__device__ __forceinline__ int units_before(int units, int pieces, int j) {
  const int each = units / pieces;
  return each * j + min(j, units - each * pieces);
}

// A group of rows row0 .. row0 + rows - 1 with `live` to count and `least` leading pages in common.  One row alone reads its
// positions as its own; so do several whose common ones are no more than a unit, which is less than the parts that it takes to
// share them (us of bf16, taken together and not: 64 groups of 4 rows of 100 and up to 100 own 27.8, 22.3, 64 of 16 of 112 and
// 60 71.0, 63.8; fp32 109.9, 121.3; but 8 of 8 of 240 and 30, bf16 14.3, 16.9).
__device__ __forceinline__ GroupPlan group_plan(const ShareArgs& a, int row0, int rows, int req, int live, int least) {
  GroupPlan p = {row0, rows, req, 0, 0, 0, 0, 0};
  if (live > 1 && (long long)least * a.s.page_size > kUnit) {
    p.prefix = least * a.s.page_size;
    p.tiles = (int)(((long long)rows * a.cut.group + a.cut.columns - 1) >> a.cut.shift);
    p.units = units_in_all(p.prefix);
  }
  return p;
}

// Item i of a group's.
__device__ __forceinline__ Item prefix_item(const ShareArgs& a, const GroupPlan& p, int i) {
  const int tile = i / p.pieces, j = i - tile * p.pieces;
  Item x = {p.row0, tile * a.cut.columns, min(a.cut.columns, p.rows * a.cut.group - tile * a.cut.columns), p.req, 0, 0, p.part0 + i, 0};
  x.begin = units_before(p.units, p.pieces, j) * kUnit;
  x.end = min(units_before(p.units, p.pieces, j + 1) * kUnit, p.prefix);
  return x;
}

// Item i of row r's own positions, `own` from `prefix` on, in `owns` pieces.
__device__ __forceinline__ Item own_item(const ShareArgs& a, int r, int req, int prefix, int own, int owns, int own0, int i, bool done) {
  const int tile = i / owns, j = i - tile * owns, units = units_in_all(own);
  Item x = {r, tile * 16, min(16, a.cut.group - tile * 16), req, 0, 0, own0 + i, done};
  x.begin = prefix + units_before(units, owns, j) * kUnit;
  x.end = prefix + min(units_before(units, owns, j + 1) * kUnit, own);
  return x;
}

__device__ __forceinline__ RowPlan row_plan(int len, int group, const GroupPlan& p, int r, int own0, int owns) {
  RowPlan x = {kJoin, group, r, 0, 0, own0, owns, 0};
  if (group >= 0) x.row0 = p.row0, x.part0 = p.part0, x.pieces = p.pieces;
  if (len <= 0) x.state = len == kPadding ? kLeave : len == kOutside ? kNan : kZero;
  else if (group < 0 && owns == 1) x.state = kDone;
  return x;
}

template <int N, bool ONE>
__global__ __launch_bounds__(N) void share_plan_kernel(ShareArgs a) {
  const moe_paged_share& s = a.s;
  const ShareCut& cut = a.cut;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, positions = s.max_pages * s.page_size;
  __shared__ PlanShared<N> sh;
  auto request = [&](int r) { return s.req ? s.req[r] : r; };
  if (tid == 0) sh.units = sh.own = 0;
  if constexpr (ONE) {
    const bool is_group = tid < s.n_groups, is_row = tid < s.T;
    int row0 = 0, row1 = 0, common = kNotLive, group = -1, req = 0, len = 0;
    if (is_group) row0 = s.first[tid], row1 = s.first[tid + 1];
    if (is_row) {
      common = a.p.common[tid];
      group = a.p.rows[tid].group;
      req = request(tid);
      len = row_length(req, s.pos[tid], s.n_req, positions);
    }
    sh.least[tid] = sh.lead[tid] = kNotLive;
    sh.live[tid] = 0;
    const bool bad = __syncthreads_or(is_group && (row0 < 0 || row0 > row1 || row1 > s.T));
    if (bad) group = -1, row1 = row0;
    if (common != kNotLive && group >= 0) {
      atomicMin(&sh.least[group], common);
      atomicMin(&sh.lead[group], tid);
      atomicAdd(&sh.live[group], 1);
    }
    __syncthreads();
    GroupPlan p = {};
    if (is_group) {
      const int least = sh.least[tid];
      s.prefix[tid] = least == kNotLive ? 0 : least * s.page_size;
      p = group_plan(a, row0, row1 - row0, least == kNotLive ? 0 : request(sh.lead[tid]), sh.live[tid], least == kNotLive ? 0 : least);
      if (p.tiles) atomicAdd(&sh.units, (unsigned long long)p.tiles * p.units);
    }
    __syncthreads();
    const int per = piece_of(sh.units, cut.slots);
    p.pieces = (p.units + per - 1) / per;
    int all;
    p.part0 = block_scan<N>(p.tiles * p.pieces, sh.wave, &all);
    sh.part0[tid] = p.part0, sh.pieces[tid] = p.pieces, sh.prefix[tid] = p.prefix;
    if (is_group) a.p.groups[tid] = p;
    __syncthreads();
    // ---- the rows' own
    const int prefix = group >= 0 && len > 0 ? sh.prefix[group] : 0, own = len > 0 ? len - prefix : 0, units = units_in_all(own);
    if (!prefix) group = -1;
    if (units) atomicAdd(&sh.own, (unsigned long long)units * cut.own_tiles);
    for (int i = tid; i < all; i += N) {
      const int g = owner_of(sh.part0, s.n_groups, i);
      a.p.prefix[i] = prefix_item(a, a.p.groups[g], i - sh.part0[g]);
    }
    if (tid == 0) a.p.head->prefix_items = all;
    __syncthreads();
    const int per_own = piece_of(sh.own, cut.own_slots), owns = (units + per_own - 1) / per_own;
    int owned;
    const int own0 = block_scan<N>(owns * cut.own_tiles, sh.wave, &owned);
    if (is_row) {
      GroupPlan of = {};
      if (group >= 0) of = a.p.groups[group];
      const RowPlan x = row_plan(len, group, of, tid, own0, owns);
      a.p.rows[tid] = x;
      for (int i = 0; i < owns * cut.own_tiles; ++i) a.p.own[own0 + i] = own_item(a, tid, req, prefix, own, owns, own0, i, x.state == kDone);
    }
    if (tid == 0) a.p.head->own_items = owned;
    return;
  }
  bool bad = false;
  for (int g = tid; g < s.n_groups; g += N) bad |= s.first[g] < 0 || s.first[g] > s.first[g + 1] || s.first[g + 1] > s.T;
  bad = __syncthreads_or(bad);
  // ---- the groups: a wave each
  for (int g = wave; g < s.n_groups; g += N / kWave) {
    const int r0 = s.first[g], r1 = bad ? r0 : s.first[g + 1];
    int least = kNotLive, live = 0, lead = kNotLive;
    for (int r = r0 + lane; r < r1; r += kWave) {
      const int c = a.p.common[r];
      least = min(least, c);
      if (c != kNotLive) ++live, lead = min(lead, r);
    }
#pragma unroll
    for (int c = 32; c; c /= 2) {
      least = min(least, __shfl_xor(least, c));
      lead = min(lead, __shfl_xor(lead, c));
      live += __shfl_xor(live, c);
    }
    if (lane == 0) {
      s.prefix[g] = least == kNotLive ? 0 : least * s.page_size;
      const GroupPlan p = group_plan(a, r0, r1 - r0, least == kNotLive ? 0 : request(lead), live, least == kNotLive ? 0 : least);
      if (p.tiles) atomicAdd(&sh.units, (unsigned long long)p.tiles * p.units);
      a.p.groups[g] = p;
    }
  }
  __syncthreads();
  const int per = piece_of(sh.units, cut.slots);
  int done = 0;
  for (int g0 = 0; g0 < s.n_groups; g0 += N) {
    const int g = g0 + tid;
    int pieces = 0, tiles = 0;
    if (g < s.n_groups) {
      pieces = (a.p.groups[g].units + per - 1) / per;
      tiles = a.p.groups[g].tiles;
    }
    int all;
    const int at = done + block_scan<N>(tiles * pieces, sh.wave, &all);
    if (g < s.n_groups) a.p.groups[g].part0 = at, a.p.groups[g].pieces = pieces;
    done += all;
  }
  if (tid == 0) a.p.head->prefix_items = done;
  __syncthreads();
  for (int g = wave; g < s.n_groups; g += N / kWave) {
    const GroupPlan p = a.p.groups[g];
    for (int i = lane; i < p.tiles * p.pieces; i += kWave) a.p.prefix[p.part0 + i] = prefix_item(a, p, i);
  }
  // ---- the rows: a thread each
  auto own_of = [&](int r, int* len, int* group) {
    const int g = a.p.rows[r].group;
    *len = row_length(request(r), s.pos[r], s.n_req, positions);
    *group = !bad && g >= 0 && *len > 0 && a.p.groups[g].prefix ? g : -1;
    return *len > 0 ? *len - (*group >= 0 ? a.p.groups[*group].prefix : 0) : 0;
  };
  unsigned long long mine = 0;
  for (int r = tid; r < s.T; r += N) {
    int len, group;
    mine += (unsigned long long)units_in_all(own_of(r, &len, &group)) * cut.own_tiles;
  }
  if (mine) atomicAdd(&sh.own, mine);
  __syncthreads();
  const int per_own = piece_of(sh.own, cut.own_slots);
  done = 0;
  for (int r0 = 0; r0 < s.T; r0 += N) {
    const int r = r0 + tid;
    int len = 0, group = -1, own = 0, owns = 0;
    if (r < s.T) {
      own = own_of(r, &len, &group);
      owns = (units_in_all(own) + per_own - 1) / per_own;
    }
    int all;
    const int at = done + block_scan<N>(owns * cut.own_tiles, sh.wave, &all);
    if (r < s.T) {
      GroupPlan of = {};
      if (group >= 0) of = a.p.groups[group];
      const RowPlan x = row_plan(len, group, of, r, at, owns);
      a.p.rows[r] = x;
      for (int i = 0; i < owns * cut.own_tiles; ++i) a.p.own[at + i] = own_item(a, r, request(r), of.prefix, own, owns, at, i, x.state == kDone);
    }
    done += all;
  }
  if (tid == 0) a.p.head->own_items = done;
}

moe_status check_share(const moe_paged_share* s, const char* who) {
  if (!s) return set_error(MOE_ERR_ARG, "%s: null argument", who);
  if (s->T < 0 || s->n_req < 0 || s->max_pages < 1 || s->page_size < 1 || s->n_groups < 0 ||
      (long long)s->max_pages * s->page_size > kMostPositions)
    return set_error(MOE_ERR_ARG, "%s: %d rows, %d requests of %d pages of %d, %d groups", who, s->T, s->n_req, s->max_pages, s->page_size,
                     s->n_groups);
  if (s->T > kMostShared || s->n_groups > kMostShared)
    return set_error(MOE_ERR_UNSUPPORTED, "%s: %d rows, %d groups (at most %d)", who, s->T, s->n_groups, kMostShared);
  if (s->n_q < 1 || s->n_kv < 1 || s->n_q % s->n_kv || s->n_q > 65535 || s->head_dim < 16 || s->head_dim > 256 || s->head_dim % 16)
    return set_error(MOE_ERR_ARG, "%s: %d query heads over %d of %d", who, s->n_q, s->n_kv, s->head_dim);
  if (!s->req && s->T > s->n_req) return set_error(MOE_ERR_ARG, "%s: %d rows for %d requests", who, s->T, s->n_req);
  if ((s->T && (!s->pos || !s->tables)) || (s->n_groups && (!s->first || !s->prefix)) || !s->plan)
    return set_error(MOE_ERR_ARG, "%s: null pointer", who);
  const size_t need = moe_paged_share_plan_bytes(s->T, s->n_groups, s->n_q, s->n_kv, s->head_dim);
  if (s->plan_bytes < need || (uintptr_t)s->plan % 16)
    return set_error(MOE_ERR_ARG, "%s: %zu bytes of plan at %p, %zu needed, 16-byte aligned", who, s->plan_bytes, s->plan, need);
  return MOE_OK;
}

// ---------------------------------------------------------------- attention

struct SharedLaunch {
  AttnPages g;
  ShareCut cut;
  PlanParts p;
  Divider by_group, by_kv;
  bool tiles;          // prefix items are taken whole, not in sixteens
  int prefix_blocks;   // of a launch; the rest are rows' own
  // work: [n_kv][items][columns] maxima and sums, [n_kv][items][columns][head_dim] values
  float* prefix_ml;
  float* prefix_o;
  float* own_ml;
  float* own_o;
};

size_t shared_work(const ShareCut& c, int n_kv, int head_dim, void* base, SharedLaunch* L) {
  const size_t prefix = (size_t)n_kv * c.prefix_items * c.columns, own = (size_t)n_kv * c.own_items * c.own_columns;
  if (L) {
    L->prefix_o = (float*)base;
    L->own_o = L->prefix_o + prefix * head_dim;
    L->prefix_ml = L->own_o + own * head_dim;
    L->own_ml = L->prefix_ml + 2 * prefix;
  }
  return (prefix + own) * (head_dim + 2) * 4 + 16;
}

// What an item says must lie in the call's rows and tables, whatever the plan holds.
__device__ __forceinline__ bool item_ok(const SharedLaunch& L, const Item& x, int parts, int columns) {
  const moe_paged_attn& a = L.g.a;
  return x.row0 >= 0 && x.col0 >= 0 && x.cols > 0 && x.cols <= columns && x.col0 <= (1 << 29) &&
         x.row0 <= a.T - 1 - (int)divide((uint32_t)(x.col0 + x.cols - 1), L.by_group) && (uint32_t)x.req < (uint32_t)a.n_req &&
         x.begin >= 0 && x.begin < x.end && x.end <= a.max_pages * L.g.map.page_size && (uint32_t)x.part < (uint32_t)parts;
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// 1, which the compiler does not know: a product with it makes x - (float)h one instruction that takes fp16 instead of two.
__device__ __forceinline__ float opaque_one() {
  float one = 1.0f;
  asm("" : "+s"(one));
  return one;
}

// Two fp32 values into the same place of three operands whose sum they are: bf16 parts by truncation, f16 parts each rounded
// to nearest even, which hold all bits but those below 2^-24.
template <bool HALF>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&p)[3]) {
  if constexpr (HALF) {
    const float one = opaque_one();
    const f16x2 h = __builtin_convertvector(f32x2{x, y}, f16x2);
    const float x1 = __builtin_fmaf(-(float)h[0], one, x), y1 = __builtin_fmaf(-(float)h[1], one, y);
    const f16x2 m = __builtin_convertvector(f32x2{x1, y1}, f16x2);
    const f16x2 l = {(_Float16)__builtin_fmaf(-(float)m[0], one, x1), (_Float16)__builtin_fmaf(-(float)m[1], one, y1)};
    p[0] = __builtin_bit_cast(uint32_t, h);
    p[1] = __builtin_bit_cast(uint32_t, m);
    p[2] = __builtin_bit_cast(uint32_t, l);
  } else {
    split2<false>(x, y, &p[0], &p[1], &p[2]);
  }
}

// Row and query head of an item's column.
struct Column {
  int row, head;
};
__device__ __forceinline__ Column column_of(const SharedLaunch& L, const Item& x, int kv, int c) {
  const int at = x.col0 + c, r = (int)divide((uint32_t)at, L.by_group);
  return {x.row0 + r, kv * L.cut.group + at - r * L.cut.group};
}

// ---------------------------------------------------------------- sixteen columns

// A block takes sixteen columns of an item, those from `sub` on; its waves take every fourth step of 32 positions and are
// joined in LDS at the end.  K and V go straight into the registers that the matrix instructions read, 16 bytes a lane, keys and
// values requested a step ahead:
//   scores   16 keys x 16 columns a tile: lane l holds 16-byte pieces of key l % 16 and the matching query values of column l % 16
//   weights  come out as keys 4 (l / 16) + i of column l % 16 and go back in as the second operand from the same lane
//   values   lane l holds the keys 4 (l / 16) + i of both tiles at its 1 / 16 of the dimensions; pairs of keys are put side by
//            side by byte permutes
// 16-bit operands, queries and weights in three parts: f16 for f16 pages, bf16 for bf16 and 8-bit ones (exact in bf16).  fp32
// pages use the fp32 instruction.  A block's own chain of latencies bounds few rows: one group of 4 rows of 550 positions,
// 32 heads over 4 of 128, fp32, takes 14 us with the join, of 1000 shared by 8 groups of 4, bf16, 19 (15 in tiles, below).
template <int HDP>
struct ColumnsShared {   // 128 dimensions at a time
  float o[kWaves][HDP > 128 ? HDP / 2 : HDP][17], m[kWaves][16], l[kWaves][16], div[16];
};

template <int CT, int HDP>
__device__ __forceinline__ void columns_block(const SharedLaunch& L, const Item& it, int kv, int sub, bool own, ColumnsShared<HDP>& sh) {
  constexpr bool HALF = CT == F16;
  constexpr int NP = 3;                            // parts of an fp32 value
  constexpr int S = CT == F32 ? 4 : CT == E4M3 ? 1 : 2;
  constexpr int E = 16 / S;                        // elements of a 16-byte piece
  constexpr int NK = HDP / E / 4;                  // a lane's pieces of a key
  constexpr int VE = HDP / 16;                     // a lane's dimensions of a value
  constexpr int EV = VE < E ? VE : E, NV = VE / EV, VW = EV * S / 4;   // its pieces: elements, number, dwords
  constexpr int KT = CT == F32 && HDP == 256 ? 1 : 2;   // tiles of 16 positions a step
  constexpr int NQ = CT == F32 ? 1 : HDP / 32;     // query operands of 8 values
  constexpr int STEP = 16 * KT;
  constexpr float kLift = HALF ? 14.0f : 0.0f;     // weights are held times 2^14 where their parts are f16

  const AttnPages& g = L.g;
  const moe_paged_attn& a = g.a;
  const int parts = own ? L.cut.own_items : L.cut.prefix_items, columns = own ? L.cut.own_columns : L.cut.columns;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int hd = g.map.head_dim;
  const int heads = min(16, it.cols - sub);
  if (heads <= 0) return;
  const float scale = a.scale * (g.k_scale ? scalar_load(g.k_scale, kv) : 1.0f) * 1.44269504088896340736f;
  const float vs = g.v_scale ? scalar_load(g.v_scale, kv) : 1.0f;
  const long long head_at = (long long)kv * g.map.head_stride;
  const char* kbase = (const char*)g.k + head_at * S;
  const char* vbase = (const char*)g.v + head_at * S;
  const int col = lane % 16, quad = lane / 16;
  const int first = it.begin, end = it.end;

  uint32_t kpiece[NK], vpiece[NV];
#pragma unroll
  for (int j = 0; j < NK; ++j) kpiece[j] = (uint32_t)min((4 * j + quad) * 16, hd * S - 16);
#pragma unroll
  for (int h = 0; h < NV; ++h) vpiece[h] = (uint32_t)min((16 * h + col) * EV * S, hd * S - EV * S);

  const Column mine = column_of(L, it, kv, sub + min(col, heads - 1));
  const float* q = a.q + (size_t)mine.row * a.ldq + (size_t)mine.head * hd;
  constexpr int NX = CT == F32 ? NK : 2 * NQ;
  f32x4 x[NX];
  auto query_dim = [&](int s) {   // of x[s]
    return CT == F32 ? (4 * s + quad) * 4 : CT == E4M3 ? (4 * (s / 4) + quad) * 16 + 4 * (s % 4) : (4 * (s / 2) + quad) * 8 + 4 * (s % 2);
  };
#pragma unroll
  for (int s = 0; s < NX; ++s) x[s] = *(const f32x4u*)(q + min(query_dim(s), hd - 4));

  const int* table = a.tables + (size_t)it.req * a.max_pages;
  bool bad = false;
  auto base_of = [&](int step) { return first + (step * kWaves + wave) * STEP; };
  // of the lane's position of a step (positions past the end take the last one's row): its page, its byte offset
  auto look = [&](int step) { return table[divide((uint32_t)min(base_of(step) + lane, end - 1), g.map.per)]; };
  auto place = [&](int step, int page) {
    const int p = min(base_of(step) + lane, end - 1);
    if (!page_ok(g.map, page)) bad = true, page = 0;
    const int off = p - (int)divide((uint32_t)p, g.map.per) * g.map.page_size;
    return ((long long)page * g.map.page_stride + (long long)off * g.map.slot_stride) * S;
  };
  uint32_t kr[KT][NK][4], vr[4 * KT][NV][VW];
  auto load_k = [&](long long at) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const char* base = kbase + __shfl(at, 16 * t + col);
#pragma unroll
      for (int j = 0; j < NK; ++j) load_piece<16, false>(base + kpiece[j], kr[t][j]);
    }
  };
  auto load_v = [&](long long at) {
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* base = vbase + __shfl(at, 16 * t + 4 * quad + i);
#pragma unroll
        for (int h = 0; h < NV; ++h) load_piece<EV * S, false>(base + vpiece[h], vr[4 * t + i][h]);
      }
  };

  f32x4 o[VE];
#pragma unroll
  for (int c = 0; c < VE; ++c) o[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  f32x4 s[KT];
  u32x4 qp[NP][NQ];
  float unlift = 1.0f;
  auto score = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < KT; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        if constexpr (CT == F32) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[t][j][c]), x[j][c], s[t], 0, 0, 0);
        } else if constexpr (CT == E4M3) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const u32x2 y = widen(kr[t][j][2 * u]), z = widen(kr[t][j][2 * u + 1]);
            const u32x4 k = {y[0], y[1], z[0], z[1]};
#pragma unroll
            for (int n = 0; n < NP; ++n) s[t] = mfma32<HALF>(k, qp[n][2 * j + u], s[t]);
          }
        } else {
          const u32x4 k = {kr[t][j][0], kr[t][j][1], kr[t][j][2], kr[t][j][3]};
#pragma unroll
          for (int n = 0; n < NP; ++n) s[t] = mfma32<HALF>(k, qp[n][j], s[t]);
        }
      }
  };
  auto gather = [&](int base) __attribute__((always_inline)) {
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (HALF) s[t][i] *= unlift;
        if (base + STEP > end && base + 16 * t + 4 * quad + i >= end) s[t][i] = -INFINITY;
        top = fmaxf(top, s[t][i]);
      }
    top = fmaxf(m, head_max(top));
    if (__any(top > m)) {
      const float keep = top == -INFINITY ? 1.0f : exp2_hw(m - top);
      l *= keep;
#pragma unroll
      for (int c = 0; c < VE; ++c) o[c] *= keep;
      m = top;
    }
    const float from = (m == -INFINITY ? 0.0f : m) - kLift;
    float p[KT][4];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[t][i] = exp2_hw(s[t][i] - from);
        l += p[t][i];
      }
    if constexpr (CT == F32) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < VE; ++c)
            o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[4 * t + i][c / EV][c % EV]), p[t][i], o[c], 0, 0, 0);
    } else {
      u32x4 pp[NP];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t u[NP];
        split_pair<HALF>(p[c / 2][2 * (c % 2)], p[c / 2][2 * (c % 2) + 1], u);
#pragma unroll
        for (int n = 0; n < NP; ++n) pp[n][c] = u[n];
      }
#pragma unroll
      for (int h = 0; h < NV; ++h) {
        uint32_t w16[8][EV / 2];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int d = 0; d < VW; ++d) {
            if constexpr (CT == E4M3) {
              const u32x2 y = widen(vr[k][h][d]);
              w16[k][2 * d] = y[0], w16[k][2 * d + 1] = y[1];
            } else {
              w16[k][d] = vr[k][h][d];
            }
          }
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          u32x4 y;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            y[c] = __builtin_amdgcn_perm(w16[2 * c + 1][e / 2], w16[2 * c][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int n = 0; n < NP; ++n) o[h * EV + e] = mfma32<HALF>(y, pp[n], o[h * EV + e]);
        }
      }
    }
  };

  if (base_of(0) < end) {
    long long at = place(0, look(0));
    load_k(at);
    load_v(at);
    int next = look(1);
    // ---- queries times scale and log2(e): scores are powers of two
    float lift = 1.0f;
#pragma unroll
    for (int s = 0; s < NX; ++s) x[s] *= query_dim(s) < hd && col < heads ? scale : 0.0f;
    if constexpr (HALF) {   // the column's largest value to 2^14 .. 2^15, so that f16 parts hold the others against it
      float big = 0.0f;
#pragma unroll
      for (int s = 0; s < NX; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) big = fmaxf(big, fabsf(x[s][c]));
      big = head_max(big);
      if (big > 0.0f && big < INFINITY) {
        const int e = max((int)(__float_as_uint(big) >> 23) - 127, -100);
        lift = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        unlift = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
      }
    }
    if constexpr (CT != F32)
#pragma unroll
      for (int s = 0; s < NQ; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f32x4 y = x[2 * s + c / 2];
          uint32_t u[NP];
          split_pair<HALF>(y[2 * (c % 2)] * lift, y[2 * (c % 2) + 1] * lift, u);
#pragma unroll
          for (int n = 0; n < NP; ++n) qp[n][s][c] = u[n];
        }
    int step = 0;
    for (; base_of(step + 1) < end; ++step) {
      score();
      at = place(step + 1, next);
      load_k(at);
      next = look(step + 2);
      gather(base_of(step));
      load_v(at);
    }
    score();
    gather(base_of(step));
  }
  l = head_sum(l);
  if (__any(bad)) l = NAN;

  // ---- the waves' sums joined, 128 dimensions at a time
  constexpr int PASS = HDP > 128 ? 2 : 1, VP = VE / PASS;
  auto& o_s = sh.o;
  auto& m_s = sh.m;
  auto& l_s = sh.l;
  if (quad == 0) m_s[wave][col] = m, l_s[wave][col] = l;
  __syncthreads();
  float top = m_s[0][col];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_s[w][col]);
  const float from = top == -INFINITY ? 0.0f : top;
  const float by = exp2_hw(m - from);
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += l_s[w][col] * exp2_hw(m_s[w][col] - from);
  auto& div_s = sh.div;
  const size_t part = ((size_t)kv * parts + it.part) * columns + sub;
  float* part_o = own ? L.own_o : L.prefix_o;
  if (wave == 0 && quad == 0) {
    div_s[col] = sum == 0.0f ? 0.0f : vs / sum;
    if (!it.direct && col < heads) {
      float* ml = (own ? L.own_ml : L.prefix_ml) + (part + col) * 2;
      ml[0] = top - kLift;   // what the weights are powers from
      ml[1] = sum;
    }
  }
#pragma unroll
  for (int ps = 0; ps < PASS; ++ps) {
#pragma unroll
    for (int c = 0; c < VP; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) o_s[wave][(4 * quad + i) * VP + c][col] = o[ps * VP + c][i] * by;
    __syncthreads();
    for (int i = tid; i < heads * 16 * VP; i += kThreads) {
      const int h = i / (16 * VP), at = i % (16 * VP), c = ps * VP + at % VP;
      const int d = c / EV * 16 * EV + at / VP * EV + c % EV;
      if (d >= hd) continue;
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) y += o_s[w][at][h];
      if (it.direct) {
        const Column to = column_of(L, it, kv, sub + h);
        a.out[(size_t)to.row * a.ldo + (size_t)to.head * hd + d] = y * div_s[h];
      } else {
        part_o[(part + h) * hd + d] = y;
      }
    }
    if (ps + 1 < PASS) __syncthreads();
  }
}

// ---------------------------------------------------------------- many columns

// A block takes an item of up to 32 or 64 columns: WC waves lie beside each other over the columns, CPW sixteens each, the
// others over the positions, 32 each of a step (fp32 pages: 16).  K and V of a step go through LDS, a
// step ahead, where the waves over the columns share them: rows of 16-bit values in 16-byte pieces, piece p of row r at
// p ^ swizzle(r), so that the reads of both lie evenly over the banks.  Keys are read as rows; a value operand, 8 keys of one
// dimension, is two reads that turn 4 rows x 16 dimensions around on their way.  16-bit pages go straight from memory into
// LDS, 8-bit pages become bf16 in registers.  A wave stages the 8 rows of one (32 positions, quad of lanes that reads them),
// whose addresses lie in its lanes, found once for K and V.  One barrier a step.  A column's largest score is raised only
// when one is more than 2^kSlack above it, so that most steps need no sums across lanes.  fp32 pages lie in LDS as they are and
// use the fp32 instruction: a lane's 16 bytes of a key or a value are four operands.
//
// 32 heads over 4 of 128, us, and of sixteens: bf16, 8 groups of 4 rows of 4000 positions 23, 34; of 8 rows 33, 52; 64 rows of
// 8000 41, 85; 32 heads over 4 of 256, 8 groups of 4 rows of 2000 32, 44, of 8 rows 39, 66.  Matrix instructions bound many
// rows: 64 of 16000 are 16.8 GFLOP, which fp32 does in 158 us (106 TFLOP/s of the 153 that a large product reaches here), bf16
// and 8-bit pages in 60, their three parts at 0.84 PFLOP/s of 1.23, fp16 in 63.  (Two fp16 parts, 22 bits, took 52 to 55: a
// score of 2^17 was then off by up to 2^-6, and weights below 2^-35 of a row's largest were lost.)  What the
// parts' instructions leave is the weights' arithmetic (two waves of a SIMD hardly overlap it with matrix instructions) and
// about 10 us of a block's start and end.  Items of 128 columns gain 4 % where all is large and lose 10 % elsewhere (16 rows
// of 3800 20.6, with 128 22.6).
constexpr int type_size(int type) { return type == F32 ? 4 : type == E4M3 ? 1 : 2; }

template <int CT, int HDP, int WC, int CPW>
struct TileShape {
  static constexpr int S = type_size(CT), WP = kWaves / WC;
  static constexpr int PW = CT == F32 ? 32 / WP : 32;    // positions of a step and a wave
  static constexpr int ROWS = PW * WP;             // of a step
  static constexpr int RB = HDP * (CT == F32 ? 4 : 2);   // bytes of a row in LDS
  static constexpr int STAGE = 2 * ROWS * RB;      // K and V
  static constexpr int JOIN = (WP - 1) * WC * CPW * kWave * (HDP + 8);
  static constexpr int BYTES = 2 * STAGE > JOIN ? 2 * STAGE : JOIN;
};

// Of the 16 lanes of a quad, each at 8 bytes of one of four rows (lane / 4) and 16 columns (lane % 4 * 4 ..): four 16-bit
// values of column lane, one a row.
__device__ __forceinline__ u32x2 read_turned(const uint8_t* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

template <int CT, int HDP, int WC, int CPW>
__device__ __forceinline__ void tile_block(const SharedLaunch& L, const Item& it, int kv, uint8_t* lds) {
  using T = TileShape<CT, HDP, WC, CPW>;
  constexpr bool HALF = CT == F16;
  constexpr int NP = CT == F32 ? 1 : 3, S = T::S, RB = T::RB;
  constexpr int NK = CT == F32 ? HDP / 16 : HDP / 32, VE = HDP / 16, KT = T::PW / 16;
  constexpr int SETS = T::ROWS / 32;                              // (32 positions, q) that a wave stages
  constexpr int NL = (8 * HDP * S + 1023) / 1024;              // 16-byte loads of a lane for their keys
  constexpr int KP = HDP * S / 16;                             // such pieces of a row
  constexpr float kSlack = HALF ? 2.0f : 4.0f, kLift = HALF ? 13.0f : 0.0f;  // weights reach 2^(kSlack + kLift)
  const AttnPages& g = L.g;
  const moe_paged_attn& a = g.a;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wc = wave % WC, wp = wave / WC, hd = g.map.head_dim, col = lane % 16, quad = lane / 16, end = it.end;
  const float scale = a.scale * (g.k_scale ? scalar_load(g.k_scale, kv) : 1.0f) * 1.44269504088896340736f;
  const long long head_at = (long long)kv * g.map.head_stride * S;
  const char* kbase = (const char*)g.k + head_at;
  const char* vbase = (const char*)g.v + head_at;
  const int* table = a.tables + (size_t)it.req * a.max_pages;
  bool bad = false;

  // ---- staging: set n of a wave is quad set % 4 of positions 32 (set / 4) .. of the step, set = wave + 4 n; row k (lane % 8)
  // of it position 16 (k / 4) + 4 q + k % 4, which is row 8 q + k of its 32 in LDS
  auto swizzle = [](int row) {
    return RB == 128 ? (row >> 1 & 1) | (row >> 3 & 3) << 1 : (row & 3) | (row >> 3 & 3) << 2;
  };
  auto position = [&](int step, int n) {
    const int set = wave + n * kWaves, k = lane % 8;
    return min(it.begin + step * T::ROWS + set / 4 * 32 + 16 * (k / 4) + 4 * (set % 4) + k % 4, end - 1);
  };
  struct Look { int p[SETS]; };
  auto look = [&](int step) {
    Look x;
#pragma unroll
    for (int n = 0; n < SETS; ++n) x.p[n] = table[divide((uint32_t)position(step, n), g.map.per)];
    return x;
  };
  u32x4 raw[CT == E4M3 ? SETS : 1][NL][2];
  auto load = [&](int step, const Look& x) {
#pragma unroll
    for (int n = 0; n < SETS; ++n) {
      const int set = wave + n * kWaves, p = position(step, n);
      int page = x.p[n];
      if (!page_ok(g.map, page)) bad = true, page = 0;
      const int off = p - (int)divide((uint32_t)p, g.map.per) * g.map.page_size;
      const long long at = ((long long)page * g.map.page_stride + (long long)off * g.map.slot_stride) * S;
      uint8_t* to = lds + (step & 1) * T::STAGE + set * 8 * RB;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if (KP * 8 < kWave && lane >= KP * 8) break;
        const int k = (lane + i * kWave) / KP, piece = (lane + i * kWave) % KP;
        const long long row = __shfl(at, k);
        if constexpr (CT == E4M3) {
          const int d = min(piece * 16, hd - 16);
          raw[n][i][0] = *(const u32x4*)(kbase + row + d);
          raw[n][i][1] = *(const u32x4*)(vbase + row + d);
        } else {
          const int d = min((piece ^ swizzle(set % 4 * 8 + k)) * 16, hd * S - 16);
          lds_load16(kbase + row + d, to + i * 1024);
          lds_load16(vbase + row + d, to + T::ROWS * RB + i * 1024);
        }
      }
    }
  };
  auto store = [&](int step) {
    if constexpr (CT == E4M3) {
#pragma unroll
      for (int n = 0; n < SETS; ++n) {
        const int set = wave + n * kWaves;
        uint8_t* to = lds + (step & 1) * T::STAGE;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          if (KP * 8 < kWave && lane >= KP * 8) break;
          const int k = (lane + i * kWave) / KP, piece = (lane + i * kWave) % KP * 2, sw = swizzle(set % 4 * 8 + k);
#pragma unroll
          for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const u32x2 y = widen(raw[n][i][side][2 * u]), z = widen(raw[n][i][side][2 * u + 1]);
              *(u32x4*)(to + side * T::ROWS * RB + (set * 8 + k) * RB + ((piece + u) ^ sw) * 16) = u32x4{y[0], y[1], z[0], z[1]};
            }
        }
      }
    }
  };
  const int steps = (end - it.begin + T::ROWS - 1) / T::ROWS;
  Look next = look(0);
  load(0, next);
  next = look(1);

  // ---- queries times scale and log2(e), in parts
  u32x4 qp[CPW][NP][NK];   // (fp32: the values)
  float unlift[CPW];
  constexpr int NX = CT == F32 ? NK : 2 * NK;
#pragma unroll
  for (int ct = 0; ct < CPW; ++ct) {
    const int c = (wc * CPW + ct) * 16 + col;
    const Column mine = column_of(L, it, kv, min(c, it.cols - 1));
    const float* q = a.q + (size_t)mine.row * a.ldq + (size_t)mine.head * hd;
    f32x4 x[NX];
#pragma unroll
    for (int s = 0; s < NX; ++s) {
      const int d = CT == F32 ? (4 * s + quad) * 4 : (4 * (s / 2) + quad) * 8 + 4 * (s % 2);
      x[s] = *(const f32x4u*)(q + min(d, hd - 4));
      x[s] *= d < hd && c < it.cols ? scale : 0.0f;
    }
    float lift = 1.0f;
    unlift[ct] = 1.0f;
    if constexpr (HALF) {
      float big = 0.0f;
#pragma unroll
      for (int s = 0; s < NX; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) big = fmaxf(big, fabsf(x[s][i]));
      big = head_max(big);
      if (big > 0.0f && big < INFINITY) {
        const int e = max((int)(__float_as_uint(big) >> 23) - 127, -100);
        lift = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        unlift[ct] = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
      }
    }
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      if constexpr (CT == F32) {
        qp[ct][0][s] = __builtin_bit_cast(u32x4, x[s]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 y = x[2 * s + i / 2];
          uint32_t u[NP];
          split_pair<HALF>(y[2 * (i % 2)] * lift, y[2 * (i % 2) + 1] * lift, u);
#pragma unroll
          for (int n = 0; n < NP; ++n) qp[ct][n][s][i] = u[n];
        }
      }
    }
  }
  store(0);

  f32x4 o[CPW][VE];
  float m[CPW], l[CPW];
#pragma unroll
  for (int ct = 0; ct < CPW; ++ct) {
    m[ct] = -INFINITY, l[ct] = 0.0f;
#pragma unroll
    for (int c = 0; c < VE; ++c) o[ct][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int step = 0; step < steps; ++step) {
    stage_sync<0>();
    if (step + 1 < steps) {
      load(step + 1, next);
      next = look(step + 2);
    }
    const int base = it.begin + step * T::ROWS + wp * T::PW;
    if (base < end) {
      // (a wave's 16 positions of 32 are rows 8 q + 4 wp .. + 3)
      const uint8_t* ks = lds + (step & 1) * T::STAGE + wp * (KT == 2 ? 32 : 4) * RB;
      const uint8_t* vs = ks + T::ROWS * RB + (quad * 8 + col / 4) * RB + col % 2 * 8;
      // ---- scores
      f32x4 s[CPW][KT];
#pragma unroll
      for (int ct = 0; ct < CPW; ++ct)
#pragma unroll
        for (int t = 0; t < KT; ++t) s[ct][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      // operands in pieces, which leave registers for the rest (bf16, 128 dimensions, 64 rows of 16000 positions 64 us, in halves
      // 60; 256 dimensions, 8 groups of 8 rows of 700 in halves 30.0, in quarters 28.9; 8-bit pages, whose next rows lie in
      // registers, 64 columns, 8 groups of 64 rows of 4000 in halves 126, in quarters 113)
      constexpr int CUT = HDP > 128 || (CT == E4M3 && CPW == 2 && HDP > 64) ? 4 : HDP > 64 ? 2 : 1, KC = NK / CUT, VN = CT == F32 ? KT * VE : VE / CUT;
#pragma unroll
      for (int j0 = 0; j0 < NK; j0 += KC) {
        u32x4 k[KC][KT];
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            const int row = 8 * (col / 4) + 4 * t + col % 4;
            k[j][t] = *(const u32x4*)(ks + row * RB + ((4 * (j0 + j) + quad) ^ swizzle(row)) * 16);
          }
        if constexpr (CT != F32) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int n = 0; n < (CT == F32 ? 4 : NP); ++n)
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
              for (int ct = 0; ct < CPW; ++ct) {
                if constexpr (CT == F32)
                  s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[j][t][n]), __uint_as_float(qp[ct][0][j0 + j][n]), s[ct][t], 0, 0, 0);
                else
                  s[ct][t] = mfma32<HALF>(k[j][t], qp[ct][n][j0 + j], s[ct][t]);
              }
      }
      // the values' first operands are requested before the weights are worked on: of fp32 pages four dimensions of keys
      // 16 t + 4 quad + i in v[(4 t + i) HDP / 64 + h]
      u32x4 v[VN];
      auto load_v = [&](int e0) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          if constexpr (CT == F32) {
            const int row = 8 * quad + e / (VE / 4), piece = 16 * (e % (VE / 4)) + col;
            v[e] = *(const u32x4*)(ks + T::ROWS * RB + row * RB + (piece ^ swizzle(row)) * 16);
          } else {
            const int piece = 2 * (e0 + e) + col % 4 / 2;
            const u32x2 x = read_turned(vs + (piece ^ swizzle(quad * 8 + col / 4)) * 16);
            const u32x2 y = read_turned(vs + 4 * RB + (piece ^ swizzle(quad * 8 + 4 + col / 4)) * 16);
            v[e] = u32x4{x[0], x[1], y[0], y[1]};
          }
        }
      };
      load_v(0);
      __builtin_amdgcn_sched_barrier(0);
      // ---- weights
      u32x4 pp[CPW][NP];
      float p[CPW][4 * KT];
#pragma unroll
      for (int ct = 0; ct < CPW; ++ct) {
        if (base + T::PW > end) {
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (base + 16 * t + 4 * quad + i >= end) s[ct][t][i] = -INFINITY;
        }
        float top = s[ct][0][0];
#pragma unroll
        for (int i = 1; i < 4 * KT; ++i) top = fmaxf(top, s[ct][i / 4][i % 4]);
        if (HALF) top *= unlift[ct];
        if (__any(top > m[ct] + kSlack)) {
          const float now = fmaxf(m[ct], head_max(top)), keep = now == -INFINITY ? 1.0f : exp2_hw(m[ct] - now);
          l[ct] *= keep;
#pragma unroll
          for (int c = 0; c < VE; ++c) o[ct][c] *= keep;
          m[ct] = now;
        }
        const float from = (m[ct] == -INFINITY ? 0.0f : m[ct]) - kLift;
#pragma unroll
        for (int i = 0; i < 4 * KT; ++i) {
          p[ct][i] = exp2_hw(HALF ? fmaf(s[ct][i / 4][i % 4], unlift[ct], -from) : s[ct][i / 4][i % 4] - from);
          l[ct] += p[ct][i];
        }
        if constexpr (CT != F32)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t u[NP];
            split_pair<HALF>(p[ct][2 * c], p[ct][2 * c + 1], u);
#pragma unroll
            for (int n = 0; n < NP; ++n) pp[ct][n][c] = u[n];
          }
      }
      // ---- values
      if constexpr (CT == F32) {
#pragma unroll
        for (int i = 0; i < 4 * KT; ++i)
#pragma unroll
          for (int e = 0; e < VE; ++e)
#pragma unroll
            for (int ct = 0; ct < CPW; ++ct)
              o[ct][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[i * (VE / 4) + e / 4][e % 4]), p[ct][i], o[ct][e], 0, 0, 0);
      } else {
#pragma unroll
        for (int e0 = 0; e0 < VE; e0 += VN) {
          if (e0) load_v(e0);
#pragma unroll
          for (int e = 0; e < VN; ++e)
#pragma unroll
            for (int n = 0; n < NP; ++n)
#pragma unroll
              for (int ct = 0; ct < CPW; ++ct) o[ct][e0 + e] = mfma32<HALF>(v[e], pp[ct][n], o[ct][e0 + e]);
        }
      }
    }
    if (step + 1 < steps) store(step + 1);
  }
  bad = __syncthreads_or(bad);   // (every wave is done with the rows in LDS)
#pragma unroll
  for (int ct = 0; ct < CPW; ++ct) {
    l[ct] = head_sum(l[ct]);
    if (bad) l[ct] = NAN;
  }
  // ---- waves over the positions joined
  if constexpr (T::WP > 1) {
    f32x4* o_s = (f32x4*)lds;
    float2* ml_s = (float2*)(lds + (T::WP - 1) * WC * CPW * kWave * HDP);
    const int at = ((wp - 1) * WC + wc) * CPW;
    if (wp) {
#pragma unroll
      for (int ct = 0; ct < CPW; ++ct) {
        ml_s[(at + ct) * kWave + lane] = float2{m[ct], l[ct]};
#pragma unroll
        for (int c = 0; c < VE; ++c) o_s[((at + ct) * VE + c) * kWave + lane] = o[ct][c];
      }
    }
    __syncthreads();
    if (wp) return;
#pragma unroll 1
    for (int w = 0; w < T::WP - 1; ++w)
#pragma unroll
      for (int ct = 0; ct < CPW; ++ct) {
        const int from = (w * WC + wc) * CPW + ct;
        const float2 ml = ml_s[from * kWave + lane];
        const float top = fmaxf(m[ct], ml.x), least = top == -INFINITY ? 0.0f : top;
        const float x = exp2_hw(m[ct] - least), y = exp2_hw(ml.x - least);
        m[ct] = top;
        l[ct] = l[ct] * x + ml.y * y;
#pragma unroll
        for (int c = 0; c < VE; ++c) o[ct][c] = o[ct][c] * x + o_s[(from * VE + c) * kWave + lane] * y;
      }
  }
#pragma unroll
  for (int ct = 0; ct < CPW; ++ct) {
    const int c = (wc * CPW + ct) * 16 + col;
    if (c >= it.cols) continue;
    const size_t part = ((size_t)kv * L.cut.prefix_items + it.part) * L.cut.columns + c;
    if (quad == 0) L.prefix_ml[part * 2] = m[ct] - kLift, L.prefix_ml[part * 2 + 1] = l[ct];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      // (fp32: o[4 h + c][i] is dimension 64 h + 16 quad + 4 i + c)
      const int d = CT == F32 ? 64 * (e / 4) + 16 * quad + 4 * (e % 4) : 16 * e + 4 * quad;
      f32x4 y = o[ct][e];
      if constexpr (CT == F32)
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] = o[ct][e / 4 * 4 + x][e % 4];
      if (d < hd) *(f32x4*)(L.prefix_o + part * hd + d) = y;
    }
  }
}

// WC: waves over a prefix item's columns, CPW: their sixteens; 0: the item in sixteens.  Prefix items first, of all heads, then the rows' own:
// the long ones start together.
template <int CT, int HDP, int WC, int CPW>
__global__ __launch_bounds__(kThreads, HDP <= 128 ? 2 : 1) void shared_attn_kernel(SharedLaunch L) {
  constexpr int TILE = TileShape<CT, HDP, WC ? WC : 4, 1>::BYTES, COLUMNS = (int)sizeof(ColumnsShared<HDP>);
  constexpr int BYTES = WC && TILE > COLUMNS ? TILE : COLUMNS;
  __shared__ __attribute__((aligned(16))) uint8_t lds[BYTES];
  const int subs = WC ? 1 : L.cut.columns / 16;
  int b = (int)divide(blockIdx.x, L.by_kv);
  const int kv = (int)blockIdx.x - b * L.g.map.n_kv;
  const bool own = b >= L.prefix_blocks;
  const int sub = own ? 0 : b % subs * 16;
  b = own ? b - L.prefix_blocks : b / subs;
  const int parts = own ? L.cut.own_items : L.cut.prefix_items, some = min(own ? L.p.head->own_items : L.p.head->prefix_items, parts);
  if (b >= some) return;
  const Item it = (own ? L.p.own : L.p.prefix)[b];
  if (!item_ok(L, it, parts, own ? L.cut.own_columns : L.cut.columns)) return;
  if constexpr (WC != 0) {
    if (!own) {
      tile_block<CT, HDP, WC, CPW>(L, it, kv, lds);
      return;
    }
  }
  columns_block<CT, HDP>(L, it, kv, sub, own, *(ColumnsShared<HDP>*)lds);
}

// ---------------------------------------------------------------- the join

// Up to this many (row, query head) a block each, whose waves take its parts in turn: few rows of long prefixes have the most
// parts (us with that and a wave each, one group, 32 heads: 4 rows of 16000 positions 23.7, 35.1; 8 of 8000 19.9, 23.4; 32 of
// 3800 28.3, 28.9; 8 groups of 8 rows of 1000 21.7, 20.5).
constexpr int kFewHeads = 1024;

// W waves a (row, query head): its parts joined, four dimensions a lane, so that 64 / (head_dim / 4) parts are read side by
// side.  Latency: the parts' first rows are requested with their maxima.
template <int W>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(SharedLaunch L) {
  constexpr int U = 4;
  __shared__ f32x4 acc_s[W][W > 1 ? kWave : 1];
  const AttnPages& g = L.g;
  const moe_paged_attn& a = g.a;
  const int t = (int)blockIdx.x, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int head = (int)blockIdx.y * (kWaves / W) + wave / W, w = wave % W;   // (W = 1, 4: a block's waves end together)
  const int hd = g.map.head_dim, lane = threadIdx.x % kWave;
  if (head >= a.n_q) return;
  const RowPlan r = L.p.rows[t];
  if (r.state == kLeave || r.state == kDone) return;
  float* out = a.out + (size_t)t * a.ldo + (size_t)head * hd;
  if (r.state != kJoin) {
    for (int d = w * kWave + lane; d < hd; d += W * kWave) out[d] = r.state == kZero ? 0.0f : NAN;
    return;
  }
  const int G = L.cut.group, kv = (int)divide((uint32_t)head, L.by_group), h = head - kv * G;
  const int c = (t - r.row0) * G + h, tile = c >> L.cut.shift;
  const int np = r.pieces, n = np + r.owns;
  // (a plan that is none leads to no place outside the work)
  if (r.row0 < 0 || r.row0 > t || np < 0 || r.owns < 0 || n == 0 || r.part0 < 0 || r.own0 < 0 ||
      (np && r.part0 + (long long)(tile + 1) * np > L.cut.prefix_items) || (r.owns && r.own0 + (long long)(h / 16 + 1) * r.owns > L.cut.own_items))
    return;
  const size_t at0 = ((size_t)kv * L.cut.prefix_items + r.part0 + (size_t)tile * np) * L.cut.columns + (c & (L.cut.columns - 1));
  const size_t at1 = ((size_t)kv * L.cut.own_items + r.own0 + (size_t)(h / 16) * r.owns) * L.cut.own_columns + h % 16;
  // (part i at a base and i steps from it: prefix parts, then the row's own)
  const float2* const ml0 = (const float2*)L.prefix_ml + at0;
  const float2* const ml1 = (const float2*)L.own_ml + at1 - (size_t)np * L.cut.own_columns;
  const float* const o0 = L.prefix_o + at0 * hd;
  const float* const o1 = L.own_o + at1 * hd - (size_t)np * L.cut.own_columns * hd;
  const uint32_t step0 = (uint32_t)L.cut.columns, step1 = (uint32_t)L.cut.own_columns;
  auto ml_of = [&](int i) { return (i < np ? ml0 : ml1)[(uint32_t)i * (i < np ? step0 : step1)]; };
  auto o_of = [&](int i, int d) { return *(const f32x4*)((i < np ? o0 : o1) + (size_t)((uint32_t)i * (i < np ? step0 : step1)) * hd + d); };
  const int width = hd / 4, rows = kWave / width, row = lane / width, d = lane % width * 4;
  f32x4 y[U];
#pragma unroll
  for (int x = 0; x < U; ++x) y[x] = o_of(min(w * U * rows + row + x * rows, n - 1), d);
  const float2 first = ml_of(min(lane, n - 1));
  float top = first.x;
  if (n > kWave)
    for (int i = lane + kWave; i < n; i += kWave) top = fmaxf(top, ml_of(i).x);
#pragma unroll
  for (int x = 32; x; x /= 2) top = fmaxf(top, __shfl_xor(top, x));
  if (top == -INFINITY) top = 0.0f;
  const float by = exp2_hw(first.x - top);   // lane's part, of the first 64
  float sum = lane < n ? first.y * by : 0.0f;
  if (n > kWave)
    for (int i = lane + kWave; i < n; i += kWave) {
      const float2 ml = ml_of(i);
      sum += ml.y * exp2_hw(ml.x - top);
    }
  sum = wave_total(sum);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = w * U * rows; i0 < n; i0 += W * U * rows) {
    if (i0 >= W * U * rows) {
#pragma unroll
      for (int x = 0; x < U; ++x) y[x] = o_of(min(i0 + row + x * rows, n - 1), d);
    }
    if (i0 + U * rows <= kWave) {
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int i = i0 + row + x * rows;
        const float f = __shfl(by, i);   // (with every lane there)
        acc += y[x] * (row < rows && i < n ? f : 0.0f);
      }
    } else {
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int i = i0 + row + x * rows;
        if (row < rows && i < n) acc += y[x] * exp2_hw(ml_of(i).x - top);
      }
    }
  }
  if constexpr (W > 1) {
    acc_s[w][lane] = acc;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int i = 1; i < W; ++i) acc += acc_s[i][lane];
  }
  // the lanes of a dimension: row by row
  f32x4 all = acc;
  for (int x = 1; x < rows; ++x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) all[e] += __shfl(acc[e], lane + x * width);
  }
  if (lane < width) {
    const float vs = g.v_scale ? g.v_scale[kv] : 1.0f;
#pragma unroll
    for (int x = 0; x < 4; ++x) out[d + x] = sum == 0.0f ? 0.0f : all[x] / sum * vs;
  }
}

template <int CT, int HDP, int WC, int CPW>
hipError_t launch(SharedLaunch L, unsigned prefix, unsigned own, hipStream_t s) {
  L.prefix_blocks = (int)prefix;
  hipLaunchKernelGGL((shared_attn_kernel<CT, HDP, WC, CPW>), dim3((prefix + own) * (unsigned)L.g.map.n_kv), dim3(kThreads), 0, s, L);
  return hipGetLastError();
}

template <int CT, int HDP>
hipError_t launch(const SharedLaunch& L, hipStream_t s) {
  const unsigned prefix = (unsigned)L.cut.prefix_items, own = (unsigned)L.cut.own_items;
  if constexpr (HDP <= 128) {
    if (L.tiles) return L.cut.columns == kTile ? launch<CT, HDP, 2, 2>(L, prefix, own, s) : launch<CT, HDP, 2, 1>(L, prefix, own, s);
  } else if (L.tiles) {
    return L.cut.columns == kTile ? launch<CT, HDP, 4, 1>(L, prefix, own, s) : launch<CT, HDP, 2, 1>(L, prefix, own, s);
  }
  return launch<CT, HDP, 0, 0>(L, prefix * (unsigned)(L.cut.columns / 16), own, s);
}

template <int CT>
hipError_t launch(const SharedLaunch& L, hipStream_t s) {
  const int hd = L.g.map.head_dim;
  return hd <= 64 ? launch<CT, 64>(L, s) : hd <= 128 ? launch<CT, 128>(L, s) : launch<CT, 256>(L, s);
}

hipError_t launch_shared(const AttnPages& g, const moe_paged_share& sh, int dtype, hipStream_t s) {
  SharedLaunch L;
  L.g = g;
  L.cut = share_cut(g.a.T, sh.n_groups, g.a.n_q, g.map.n_kv, g.map.head_dim);
  plan_parts(L.cut, g.a.T, sh.n_groups, sh.plan, &L.p);
  shared_work(L.cut, g.map.n_kv, g.map.head_dim, g.a.work, &L);
  L.by_group = make_divider((uint32_t)L.cut.group);
  L.by_kv = make_divider((uint32_t)g.map.n_kv);
  // Items of 32 and 64 columns are taken whole, but where all of them in sixteens, at their longest, would be resident at once
  // (heads past 128, one block a CU: with the rows' own): then only a block's latency counts (us of bf16 pages, 32 heads over 4,
  // whole and in sixteens; of 128: 8 rows of 600 positions 14.9, 12.0; 8 groups of 8 rows of 250 16.8, 14.6, of 600 18.6, 21.1;
  // of 256: 8 rows of 600 18.4, 15.5, of 2200 20.8, 26.7; 8 groups of 4 of 400 18.5, 24.3).
  const long long tiles = ((long long)g.a.T * L.cut.group + L.cut.columns - 1) / L.cut.columns;
  const long long units = ((long long)g.a.max_pages * g.map.page_size + kUnit - 1) / kUnit;
  const long long blocks = (tiles > sh.n_groups ? tiles : sh.n_groups) * units * (L.cut.columns / 16) * g.map.n_kv;
  const long long own = (long long)g.a.T * L.cut.own_tiles * g.map.n_kv;
  L.tiles = L.cut.columns >= kTile / 2 && (g.map.head_dim <= 128 ? blocks > 2 * kCUs : blocks + own > kCUs);
  const hipError_t e = dtype == F32    ? launch<F32>(L, s)
                       : dtype == F16  ? launch<F16>(L, s)
                       : dtype == BF16 ? launch<BF16>(L, s)
                                       : launch<E4M3>(L, s);
  if (e != hipSuccess) return e;
  if ((long long)g.a.T * g.a.n_q <= kFewHeads)
    hipLaunchKernelGGL(shared_join_kernel<kWaves>, dim3((unsigned)g.a.T, (unsigned)g.a.n_q), dim3(kThreads), 0, s, L);
  else
    hipLaunchKernelGGL(shared_join_kernel<1>, dim3((unsigned)g.a.T, (unsigned)(g.a.n_q + kWaves - 1) / kWaves), dim3(kThreads), 0, s, L);
  return hipGetLastError();
}

}  // namespace

int shared_rows_max() { return kMostShared; }

}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_paged_share_plan_bytes(int T, int n_groups, int n_q, int n_kv, int head_dim) {
  if (T < 0 || T > kMostShared || n_groups < 0 || n_groups > kMostShared || n_q < 1 || n_kv < 1 || n_q % n_kv || head_dim < 1) return 0;
  PlanParts p;
  return plan_parts(share_cut(T, n_groups, n_q, n_kv, head_dim), T, n_groups, nullptr, &p);
}

moe_status moe_paged_share_dev(const moe_paged_share* s) {
  moe_status st = check_share(s, "paged_share");
  if (st || (st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  ShareArgs a;
  a.s = *s;
  a.per = make_divider((uint32_t)s->page_size);
  a.cut = share_cut(s->T, s->n_groups, s->n_q, s->n_kv, s->head_dim);
  plan_parts(a.cut, s->T, s->n_groups, s->plan, &a.p);
  if (s->T) {
    hipLaunchKernelGGL(share_rows_kernel, dim3((unsigned)(s->T + 3) / 4), dim3(256), 0, stream(), a);
    if ((st = check_hip(hipGetLastError(), "paged_share launch"))) return st;
  }
  const int most = s->T > s->n_groups ? s->T : s->n_groups;
  if (most <= 256) hipLaunchKernelGGL((share_plan_kernel<256, true>), dim3(1), dim3(256), 0, stream(), a);
  else if (most <= kN) hipLaunchKernelGGL((share_plan_kernel<kN, true>), dim3(1), dim3(kN), 0, stream(), a);
  else hipLaunchKernelGGL((share_plan_kernel<kN, false>), dim3(1), dim3(kN), 0, stream(), a);
  return check_hip(hipGetLastError(), "paged_share launch");
}

size_t moe_paged_attn_shared_work_bytes(int T, int n_groups, int n_q, int n_kv, int head_dim) {
  if (T < 0 || T > kMostShared || n_groups < 0 || n_groups > kMostShared || n_q < 1 || n_kv < 1 || n_q % n_kv || head_dim < 1) return 0;
  return shared_work(share_cut(T, n_groups, n_q, n_kv, head_dim), n_kv, head_dim, nullptr, nullptr);
}

moe_status moe_paged_attn_shared_dev(const moe_paged_attn* a, const moe_pages* g, const moe_paged_share* s) {
  PageMap map;
  moe_status st = check_attn(a, g, "paged_attn_shared", &map);
  if (st || (st = check_share(s, "paged_attn_shared"))) return st;
  if (s->T != a->T || s->n_req != a->n_req || s->max_pages != a->max_pages || s->page_size != map.page_size || s->n_q != a->n_q ||
      s->n_kv != map.n_kv || s->head_dim != map.head_dim || s->req != a->req || s->pos != a->pos || s->tables != a->tables)
    return set_error(MOE_ERR_ARG, "paged_attn_shared: the rows, tables or heads are not the shared plan's");
  if (a->T == 0) return MOE_OK;
  if (!a->work) return set_error(MOE_ERR_ARG, "paged_attn_shared: null pointer");
  const size_t need = moe_paged_attn_shared_work_bytes(a->T, s->n_groups, a->n_q, map.n_kv, map.head_dim);
  if (a->work_bytes < need || (uintptr_t)a->work % 16)
    return set_error(MOE_ERR_ARG, "paged_attn_shared: %zu bytes of work at %p, %zu needed, 16-byte aligned", a->work_bytes, a->work, need);
  const ShareCut cut = share_cut(a->T, s->n_groups, a->n_q, map.n_kv, map.head_dim);
  if (((long long)cut.prefix_items * (cut.columns / 16) + cut.own_items) * map.n_kv >= 1 << 24)   // (a launch holds fewer than 2^32 threads)
    return set_error(MOE_ERR_UNSUPPORTED, "paged_attn_shared: %d rows in %d groups for %d heads over %d", a->T, s->n_groups, a->n_q, map.n_kv);
  if ((st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  return check_hip(launch_shared(AttnPages{*a, map, g->k, g->v, g->k_scale, g->v_scale}, *s, g->dtype, stream()), "paged_attn_shared launch");
}

}  // extern "C"
