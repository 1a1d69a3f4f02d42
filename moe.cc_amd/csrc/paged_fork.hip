// paged_fork.hip - requests of a paged cache that go on as copies of others:
// the block tables (moe_paged_fork_dev) and the pages that are copied
// (moe_paged_copy_dev).  include/moehip.h.
//
// Requests share pages only by being forked, so a shared page lies at the same
// place of all its holders' tables.  Everything about a page is therefore
// found in one column of the tables, and columns are independent of each
// other: a block takes some columns of all requests and finds which of their
// pages no request holds any more by a number a page, in a hash table in LDS
// (at most half full), the largest of
//   n - r          of the requests r that held it: the lowest gives it back, unless
//   kStays         a request holds it now
// Nothing is kept from one call for the next.  Latency bounds it: launch, the
// requests' numbers, the tables: 64 requests of 160 pages 8.4 us, 1024 of 512
// (whose tables are 2 MB each way) 16.9.  (The pages' numbers in memory instead of
// LDS: 2.6 and 12 more.)
#include <initializer_list>

#include "block_scan.h"
#include "moe_device.h"
#include "moe_lib.h"
#include "paged_attn.h"

namespace moe {
namespace {

constexpr int kN = 1024;             // threads of a block
constexpr int kMostRequests = 4096;
constexpr int kStays = 1 << 30;

// How a request goes on.
struct Goes {
  int src;    // the request that it is a copy of; -1: it ends
  int held;   // positions of src
  int copy;   // its place among the copies; -1: none
  int used;   // pages that it had
};

struct ForkHead {
  int status, head, count, copies;
};

struct ForkArgs {
  moe_paged_fork f;
  Divider per;      // by page_size
  int columns, blocks;   // of a block, of the tables
  Divider by_columns;
  ForkHead* top;    // work
  Goes* goes;       // work [n_req]
  int* counts;      // work [blocks] pages that come back
  int* list;        // work [n_req * max_pages] these, a block's from n_req * its first column on
};

template <int MOST>
struct ForkShared {
  int parent[MOST], held[MOST], copy[MOST];
  int wave[kN / kWave], bad;
};

// The requests, into sh: how each goes on, and whether the call can be done.  Every block of a call finds the same.
template <int MOST>
__device__ __forceinline__ ForkHead fork_requests(const ForkArgs& a, ForkShared<MOST>& sh) {
  const moe_paged_fork& f = a.f;
  const int tid = threadIdx.x, n = f.n_req;
  const long long most = (long long)f.max_pages * f.page_size;
  const int head = f.ring_at[0], count = f.ring_at[1];
  if (tid == 0) sh.bad = head < 0 || head >= f.n_pages || count < 0 || count > f.n_pages;
  for (int r = tid; r < n; r += kN) {
    sh.parent[r] = f.parent[r];
    sh.held[r] = f.held[r];
    sh.copy[r] = n;
  }
  __syncthreads();
  // the page that is not full stays with the request itself, or its first copy
  for (int r = tid; r < n; r += kN) {
    const int p = sh.parent[r], h = sh.held[r];
    if (p < -1 || p >= n || h < 0 || h > most) sh.bad = 1;
    else if (p >= 0) atomicMin(&sh.copy[p], p == r ? -1 : r);
  }
  __syncthreads();
  const bool bad = sh.bad;
  int done = 0;
  for (int r0 = 0; r0 < n; r0 += kN) {
    const int r = r0 + tid;
    bool copied = false;
    if (r < n && !bad) {
      const int p = sh.parent[r];
      if (p >= 0) {
        const int h = sh.held[p];
        copied = h != (int)divide((uint32_t)h, a.per) * f.page_size && sh.copy[p] != r && p != r;
      }
    }
    int all;
    const int at = done + block_scan<kN>(copied, sh.wave, &all);
    // (the keepers of the requests behind these are still to be read)
    if (r < n) sh.parent[r] = bad ? -1 : copied ? sh.parent[r] | at << 12 | 1 << 30 : sh.parent[r];
    done += all;
  }
  __syncthreads();
  for (int r = tid; r < n; r += kN) {
    const int x = sh.parent[r];
    const bool copied = x >= 0 && x >> 30;
    sh.copy[r] = copied ? x >> 12 & 0xfff : -1;
    if (copied) sh.parent[r] = x & 0xfff;
    if (bad) sh.held[r] = 0;
  }
  __syncthreads();
  return ForkHead{bad ? kForkBad : done > f.max_copies ? kForkCopies : done > count ? kForkNoPages : kForkOk, head, count, done};
}

template <int MOST>
__device__ __forceinline__ Goes goes_of(const ForkArgs& a, const ForkShared<MOST>& sh, int r) {
  const int p = sh.parent[r];
  return Goes{p, p >= 0 ? sh.held[p] : 0, sh.copy[r], pages_for(sh.held[r], a.per)};
}

// A thread's entries of a block's columns: entry i is column i % columns of request i / columns, counted from the first.
struct Entry {
  int r, c;
  bool in;
};
__device__ __forceinline__ Entry entry_of(const ForkArgs& a, int c0, int k) {
  const int i = k * kN + (int)threadIdx.x, r = (int)divide((uint32_t)i, a.by_columns), c = c0 + i - r * a.columns;
  return {r, c, r < a.f.n_req && c < a.f.max_pages};
}

// The pages of columns c0 .. that come back, in order of the columns, then of the requests, to `list`; their number.
template <int PER, int MOST>
__device__ __forceinline__ int fork_columns(const ForkArgs& a, ForkShared<MOST>& sh, int c0, int* list) {
  const moe_paged_fork& f = a.f;
  const int n = f.n_req, tid = threadIdx.x;
  constexpr int WORDS = PER * kN / 32;
  __shared__ uint32_t bits_s[WORDS];
  __shared__ int first_s[WORDS];
  constexpr uint32_t SLOTS = 2 * PER * kN;
  __shared__ int page_s[SLOTS], most_s[SLOTS];
  int old[PER], now[PER], slot[PER];
  for (int i = tid; i < (int)SLOTS; i += kN) page_s[i] = -1, most_s[i] = 0;
  for (int i = tid; i < WORDS; i += kN) bits_s[i] = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const Entry e = entry_of(a, c0, k);
    old[k] = now[k] = -1;
    if (!e.in) continue;
    const Goes g = goes_of(a, sh, e.r);
    const int* row = f.tables + e.c;
    if (e.c < g.used) old[k] = row[(size_t)e.r * f.max_pages];
    const int fills = pages_for(g.held, a.per);
    if (g.src >= 0 && e.c < fills && !(g.copy >= 0 && e.c == fills - 1)) now[k] = row[(size_t)g.src * f.max_pages];
  }
  // what the request before does for the same page, in a neighbouring lane, need not be done again
  const int lane = tid % kWave, from = lane - a.columns;
  auto again = [&](int x) {
    const int y = __shfl(x, max(from, 0));
    return from >= 0 && x == y;
  };
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if ((uint32_t)old[k] >= (uint32_t)f.n_pages) old[k] = -1;
    if ((uint32_t)now[k] >= (uint32_t)f.n_pages) now[k] = -1;
    const bool twice = again(old[k]), stays = old[k] == now[k];
    if (again(now[k])) now[k] = -1;
    if (twice) old[k] = -1;
    slot[k] = stays ? -1 : 0;   // (what stays with its request gives nothing back)
  }
  __syncthreads();
  auto home = [](int page) { return (uint32_t)page * 2654435761u >> (32 - __builtin_ctz(SLOTS)); };
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (old[k] < 0) continue;
    uint32_t h = home(old[k]);
    for (;;) {
      const int was = atomicCAS(&page_s[h], -1, old[k]);
      if (was == -1 || was == old[k]) break;
      h = (h + 1) % SLOTS;
    }
    if (slot[k] < 0) old[k] = -1;
    slot[k] = (int)h;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (now[k] >= 0) {
      uint32_t h = home(now[k]);
      while (page_s[h] != now[k] && page_s[h] != -1) h = (h + 1) % SLOTS;
      atomicMax(&most_s[h], kStays);
    }
    if (old[k] >= 0) atomicMax(&most_s[slot[k]], n - entry_of(a, c0, k).r);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k) now[k] = old[k] >= 0 ? most_s[slot[k]] : 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const Entry e = entry_of(a, c0, k);
    if (e.in && now[k] == n - e.r) {
      const int bit = (e.c - c0) * n + e.r;
      atomicOr(&bits_s[bit / 32], 1u << bit % 32);
    } else {
      old[k] = -1;
    }
  }
  __syncthreads();
  // a thread a word: places within the block
  static_assert(WORDS <= kN);
  int all;
  const int before = block_scan<kN>(tid < WORDS ? __popc(bits_s[tid]) : 0, sh.wave, &all);
  if (tid < WORDS) first_s[tid] = before;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (old[k] < 0) continue;
    const Entry e = entry_of(a, c0, k);
    const int bit = (e.c - c0) * n + e.r;
    list[first_s[bit / 32] + __popc(bits_s[bit / 32] & ((1u << bit % 32) - 1))] = old[k];
  }
  return all;
}

// What the call leaves: block b's columns of the tables and its pages in the ring, block 0 the rest too.
template <int PER, class GoesOf>
__device__ __forceinline__ void fork_finish(const ForkArgs& a, ForkHead top, int b, int before, int mine, int back, const int* list, GoesOf goes) {
  const moe_paged_fork& f = a.f;
  const int tid = threadIdx.x, n = f.n_req, c0 = b * a.columns;
  if ((long long)top.count + back > f.n_pages) top.status = kForkBad;
  const bool ok = top.status == kForkOk;
  if (ok || f.tables_out != f.tables) {
    int now[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const Entry e = entry_of(a, c0, k);
      if (!e.in) continue;
      const Goes g = goes(e.r);
      const int fills = pages_for(g.held, a.per);
      const bool in = ok && g.src >= 0 && e.c < fills;
      now[k] = f.tables[(size_t)(in ? g.src : e.r) * f.max_pages + e.c];
      if (in && g.copy >= 0 && e.c == fills - 1) {   // copies name their pages by the old tables
        f.copies[3 * g.copy] = now[k];
        f.copies[3 * g.copy + 1] = now[k] = f.ring[ring_place(top.head, g.copy, f.n_pages)];
        f.copies[3 * g.copy + 2] = g.held - (fills - 1) * f.page_size;
      }
    }
    stage_sync<0>();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const Entry e = entry_of(a, c0, k);
      if (e.in) f.tables_out[(size_t)e.r * f.max_pages + e.c] = now[k];
    }
  }
  if (ok) {
    const int tail = ring_place(top.head, top.count, f.n_pages);
    for (int i = tid; i < mine; i += kN) f.ring[ring_place(tail, before + i, f.n_pages)] = list[i];
  }
  if (b == 0) {
    for (int i = 3 * (ok ? top.copies : 0) + tid; i < 3 * f.max_copies; i += kN) f.copies[i] = -1;
    for (int r = tid; r < n; r += kN) f.held_out[r] = ok ? goes(r).held : f.held[r];
    if (tid == 0) {
      f.ring_at_out[0] = ok ? ring_place(top.head, top.copies, f.n_pages) : top.head;
      f.ring_at_out[1] = ok ? top.count - top.copies + back : top.count;
      *f.status = top.status;
    }
  }
}

// Few entries: all of it in one block, one launch (4 requests of 40 pages 5.0 us, 16 of 128 6.7; in columns 6.6, 7.8).
constexpr int kOnePer = 2, kFewRequests = 1024;
__global__ __launch_bounds__(kN) void fork_one_kernel(ForkArgs a) {
  __shared__ ForkShared<kFewRequests> sh;
  const ForkHead top = fork_requests(a, sh);
  const int back = fork_columns<kOnePer>(a, sh, 0, a.list);
  stage_sync<0>();
  fork_finish<kOnePer>(a, top, 0, 0, back, back, a.list, [&](int r) { return goes_of(a, sh, r); });
}

// Many: a block some columns, then, when the pages that come back are counted, the tables.
template <int PER>
__global__ __launch_bounds__(kN) void fork_columns_kernel(ForkArgs a) {
  __shared__ ForkShared<PER <= 2 ? kFewRequests : kMostRequests> sh;
  const ForkHead top = fork_requests(a, sh);
  const int c0 = (int)blockIdx.x * a.columns, back = fork_columns<PER>(a, sh, c0, a.list + (size_t)c0 * a.f.n_req);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = back;
  if (blockIdx.x == 0) {   // (held may be changed by the next kernel while its other blocks need it)
    for (int r = threadIdx.x; r < a.f.n_req; r += kN) a.goes[r] = goes_of(a, sh, r);
    if (threadIdx.x == 0) *a.top = top;
  }
}

template <int PER>
__global__ __launch_bounds__(kN) void fork_finish_kernel(ForkArgs a) {
  __shared__ int wave_s[kN / kWave], before_s, mine_s;
  int back = 0;
  for (int b0 = 0; b0 < a.blocks; b0 += kN) {
    const int b = b0 + (int)threadIdx.x, c = b < a.blocks ? a.counts[b] : 0;
    int all;
    const int at = block_scan<kN>(c, wave_s, &all);
    if (b == (int)blockIdx.x) before_s = back + at, mine_s = c;
    back += all;
  }
  __syncthreads();
  fork_finish<PER>(a, *a.top, (int)blockIdx.x, before_s, mine_s, back, a.list + (size_t)blockIdx.x * a.columns * a.f.n_req, [&](int r) { return a.goes[r]; });
}

// ------------------------------------------------------------ copies

constexpr int kLayers = 64;   // of a launch

struct CopyArgs {
  PageMap map;
  int row;       // 16-byte pieces of a row (one head's position)
  Divider by_row;
  long long page, head, slot;   // strides in bytes
  const int32_t* copies;
  char* side[2 * kLayers];
};

// A block a (copy, pool, head): the first n positions of a head of a page.  All bytes are read once and written once, which
// bounds many copies (40 copies of 9 positions or so in 48 layers of 8 heads of 128, bf16: 12 us); of one the launch does, 4.4.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
  const int32_t* c = a.copies + 3 * (size_t)blockIdx.x;
  const int src = c[0], dst = c[1], n = min(c[2], a.map.page_size);
  if (!page_ok(a.map, src) || !page_ok(a.map, dst) || n <= 0) return;
  char* pool = a.side[blockIdx.y];
  const int head = (int)blockIdx.z;
  const char* from = pool + (long long)src * a.page + (long long)head * a.head;
  char* to = pool + (long long)dst * a.page + (long long)head * a.head;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const int all = n * a.row;
  for (int i = threadIdx.x; i < all; i += 256) {
    const int off = (int)divide((uint32_t)i, a.by_row);
    const long long at = (long long)off * a.slot + (long long)(i - off * a.row) * 16;
    *(u32x4*)(to + at) = *(const u32x4*)(from + at);
  }
}

}  // namespace

moe_status check_fork(const moe_paged_fork* f) {
  if (!f) return set_error(MOE_ERR_ARG, "paged_fork: null argument");
  if (f->n_req < 0 || f->max_pages < 1 || f->n_pages < 1 || f->page_size < 1 || f->max_copies < 0)
    return set_error(MOE_ERR_ARG, "paged_fork: %d requests of %d pages, %d pages of %d, %d copies", f->n_req, f->max_pages, f->n_pages,
                     f->page_size, f->max_copies);
  if ((long long)f->n_pages * f->page_size > 0x7fffffffll || (long long)f->max_pages * f->page_size > kMostPositions)
    return set_error(MOE_ERR_ARG, "paged_fork: %d pages of %d, %d a request: past 2^31 slots or 2^30 positions", f->n_pages, f->page_size,
                     f->max_pages);
  if (f->n_req > kMostRequests || f->max_copies > kMostRows)
    return set_error(MOE_ERR_UNSUPPORTED, "paged_fork: %d requests, %d copies (at most %d, %d)", f->n_req, f->max_copies, kMostRequests, kMostRows);
  for (const void* p : {(const void*)f->ring_at, (const void*)f->ring, (const void*)f->ring_at_out, (const void*)f->status, (const void*)f->work})
    if (!p) return set_error(MOE_ERR_ARG, "paged_fork: null pointer");
  if ((f->n_req && (!f->parent || !f->held || !f->tables || !f->held_out || !f->tables_out)) || (f->max_copies && !f->copies)) return set_error(MOE_ERR_ARG, "paged_fork: null pointer");
  const size_t need = ::moe_paged_fork_work_bytes(f->n_req, f->max_pages, f->n_pages);
  if (f->work_bytes < need || (uintptr_t)f->work % 16)
    return set_error(MOE_ERR_ARG, "paged_fork: %zu bytes of work at %p, %zu needed, 16-byte aligned", f->work_bytes, f->work, need);
  return MOE_OK;
}

moe_status check_copy(const int32_t* copies, int n, const moe_pages* layers, int n_layers) {
  if (n < 0 || n_layers < 0 || n > kMostRows) return set_error(MOE_ERR_ARG, "paged_copy: %d copies in %d layers", n, n_layers);
  if (n == 0 || n_layers == 0) return MOE_OK;
  if (!copies || !layers) return set_error(MOE_ERR_ARG, "paged_copy: null pointer");
  for (int l = 0; l < n_layers; ++l) {
    PageMap map;
    moe_status st = check_pages(&layers[l], "paged_copy", &map);
    if (st) return st;
    const moe_pages &x = layers[l], &y = layers[0];
    if (x.dtype != y.dtype || x.n_pages != y.n_pages || x.page_size != y.page_size || x.n_kv != y.n_kv || x.head_dim != y.head_dim ||
        x.page_stride != y.page_stride || x.head_stride != y.head_stride || x.slot_stride != y.slot_stride)
      return set_error(MOE_ERR_UNSUPPORTED, "paged_copy: layer %d's pages are laid out otherwise than layer 0's", l);
    if (x.n_kv > 65535) return set_error(MOE_ERR_ARG, "paged_copy: %d heads", x.n_kv);
  }
  return MOE_OK;
}

}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_paged_fork_work_bytes(int n_req, int max_pages, int n_pages) {
  if (n_req < 0 || n_req > kMostRequests || max_pages < 1 || n_pages < 1) return 0;
  return sizeof(ForkHead) + (size_t)n_req * sizeof(Goes) + 4 * ((size_t)n_req * max_pages + max_pages) + 64;
}

moe_status moe_paged_fork_dev(const moe_paged_fork* f) {
  moe_status st = check_fork(f);
  if (st || (st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  ForkArgs a;
  a.f = *f;
  a.per = make_divider((uint32_t)f->page_size);
  const bool one = f->n_req <= kFewRequests && (long long)f->n_req * f->max_pages <= kOnePer * kN;
  // Entries of a thread: every block goes through all requests first, so with many of them fewer blocks are better (us with
  // one and two: 64 requests of 160 pages 8.2, 9.6; 256 of 512 9.1, 11.5; 512 of 512 11.4, 11.6; 1024 of 512 21.4, 16.8).
  // Past 1024 requests a column has to fit a block: four.
  const int per = f->n_req <= 256 ? 1 : f->n_req <= 1024 ? 2 : 4;
  a.columns = one ? f->max_pages : per * kN / f->n_req;
  if (a.columns > f->max_pages) a.columns = f->max_pages;
  a.blocks = (f->max_pages + a.columns - 1) / a.columns;
  a.by_columns = make_divider((uint32_t)a.columns);
  a.top = (ForkHead*)f->work;
  a.goes = (Goes*)(a.top + 1);
  a.counts = (int*)(a.goes + f->n_req);
  a.list = a.counts + f->max_pages;
  if (one) {
    hipLaunchKernelGGL(fork_one_kernel, dim3(1), dim3(kN), 0, stream(), a);
    return check_hip(hipGetLastError(), "paged_fork launch");
  }
  const dim3 grid((unsigned)a.blocks);
  if (per == 2) hipLaunchKernelGGL(fork_columns_kernel<2>, grid, dim3(kN), 0, stream(), a);
  else if (per == 1) hipLaunchKernelGGL(fork_columns_kernel<1>, grid, dim3(kN), 0, stream(), a);
  else hipLaunchKernelGGL(fork_columns_kernel<4>, grid, dim3(kN), 0, stream(), a);
  if ((st = check_hip(hipGetLastError(), "paged_fork launch"))) return st;
  if (per == 2) hipLaunchKernelGGL(fork_finish_kernel<2>, grid, dim3(kN), 0, stream(), a);
  else if (per == 1) hipLaunchKernelGGL(fork_finish_kernel<1>, grid, dim3(kN), 0, stream(), a);
  else hipLaunchKernelGGL(fork_finish_kernel<4>, grid, dim3(kN), 0, stream(), a);
  return check_hip(hipGetLastError(), "paged_fork launch");
}

moe_status moe_paged_copy_dev(const int32_t* copies, int n, const moe_pages* layers, int n_layers) {
  moe_status st = check_copy(copies, n, layers, n_layers);
  if (st || n == 0 || n_layers == 0) return st;
  PageMap map;
  if ((st = check_pages(&layers[0], "paged_copy", &map))) return st;
  if ((st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  const int size = type_bytes(layers[0].dtype);
  CopyArgs a;
  a.map = map;
  a.row = map.head_dim * size / 16;
  a.by_row = make_divider((uint32_t)a.row);
  a.page = map.page_stride * size, a.head = map.head_stride * size, a.slot = map.slot_stride * size;
  a.copies = copies;
  for (int l0 = 0; l0 < n_layers; l0 += kLayers) {
    const int m = n_layers - l0 < kLayers ? n_layers - l0 : kLayers;
    for (int l = 0; l < m; ++l) {
      a.side[2 * l] = (char*)layers[l0 + l].k;
      a.side[2 * l + 1] = (char*)layers[l0 + l].v;
    }
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)n, (unsigned)(2 * m), (unsigned)map.n_kv), dim3(256), 0, stream(), a);
    if ((st = check_hip(hipGetLastError(), "paged_copy launch"))) return st;
  }
  return MOE_OK;
}

}  // extern "C"
