// paged.hip - many requests over a paged key-value cache (include/moehip.h,
// "many requests over a paged cache"): the step's plan, the new rows' heads
// into their pages, and the entry points (attention: paged_attn.hip).
#include <math.h>

#include <initializer_list>
#include <type_traits>

#include "moe_device.h"
#include "moe_lib.h"
#include "paged_attn.h"

namespace moe {
namespace {

// ------------------------------------------------------------ arguments

int type_bytes(int dtype) { return dtype == MOE_PAGE_F32 ? 4 : dtype == MOE_PAGE_E4M3 ? 1 : 2; }

// Rows of a call at most: a launch holds fewer than 2^32 threads.  Positions of a request at most: what a step of the
// kernels adds to one stays far inside an int.
constexpr int kMostRows = (1 << 24) - 1;
constexpr long long kMostPositions = 1ll << 30;

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// Checks a cache's description and fills its map.
moe_status check_pages(const moe_pages* g, const char* who, PageMap* m) {
  if (!g || !g->k || !g->v) return set_error(MOE_ERR_ARG, "%s: no pages", who);
  if (g->dtype != MOE_PAGE_F32 && g->dtype != MOE_PAGE_F16 && g->dtype != MOE_PAGE_BF16 && g->dtype != MOE_PAGE_E4M3)
    return set_error(MOE_ERR_ARG, "%s: cache type %d", who, g->dtype);
  if (g->n_pages < 1 || g->page_size < 1 || g->n_kv < 1 || (long long)g->n_pages * g->page_size > 0x7fffffffll)
    return set_error(MOE_ERR_ARG, "%s: %d pages of %d positions, %d heads", who, g->n_pages, g->page_size, g->n_kv);
  if (g->head_dim < 16 || g->head_dim > 256 || g->head_dim % 16)
    return set_error(MOE_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 16 up to 256)", who, g->head_dim);
  const long long per16 = 16 / type_bytes(g->dtype);
  for (long long s : {g->page_stride, g->head_stride, g->slot_stride})
    if (s < g->head_dim || s % per16 || s > (1ll << 40))
      return set_error(MOE_ERR_ARG, "%s: stride %lld (at least head_dim, a multiple of %lld)", who, s, per16);
  if (g->page_stride > (1ll << 48) / g->n_pages)
    return set_error(MOE_ERR_ARG, "%s: %d pages of %lld elements", who, g->n_pages, g->page_stride);
  if (!aligned(g->k, 16) || !aligned(g->v, 16)) return set_error(MOE_ERR_ARG, "%s: pages not 16-byte aligned", who);
  if (g->dtype != MOE_PAGE_E4M3 && (g->k_scale || g->v_scale))
    return set_error(MOE_ERR_ARG, "%s: scales belong to 8-bit pages", who);
  *m = PageMap{g->n_pages, g->page_size, g->n_kv, g->head_dim, g->page_stride, g->head_stride, g->slot_stride,
               make_divider((uint32_t)g->page_size)};
  return MOE_OK;
}

moe_status check_plan(const moe_paged_plan* p) {
  if (!p) return set_error(MOE_ERR_ARG, "paged_plan: null argument");
  if (p->n_req < 0 || p->max_pages < 1 || p->n_pages < 1 || p->page_size < 1 || p->max_tokens < 0)
    return set_error(MOE_ERR_ARG, "paged_plan: %d requests of %d pages, %d pages of %d, %d tokens", p->n_req, p->max_pages,
                     p->n_pages, p->page_size, p->max_tokens);
  if ((long long)p->n_pages * p->page_size > 0x7fffffffll || (long long)p->max_pages * p->page_size > kMostPositions)
    return set_error(MOE_ERR_ARG, "paged_plan: %d pages of %d, %d a request: past 2^31 slots or 2^30 positions", p->n_pages,
                     p->page_size, p->max_pages);
  if (p->n_req > kMostRows || p->max_tokens > kMostRows)
    return set_error(MOE_ERR_ARG, "paged_plan: %d requests, %d tokens (%d at most)", p->n_req, p->max_tokens, kMostRows);
  for (const void* q : {(const void*)p->ring_at, (const void*)p->ring, (const void*)p->ring_at_out, (const void*)p->starts,
                        (const void*)p->status})
    if (!q) return set_error(MOE_ERR_ARG, "paged_plan: null pointer");
  if (p->n_req && (!p->fresh || !p->held || !p->tables || !p->held_out)) return set_error(MOE_ERR_ARG, "paged_plan: null pointer");
  if (p->max_tokens && (!p->req || !p->pos || !p->slot)) return set_error(MOE_ERR_ARG, "paged_plan: null pointer");
  return MOE_OK;
}

bool heads_fit(long long T, int n_q, int n_kv) { return (n_q + 2ll * n_kv) * T <= 16ll * kMostRows; }

// ------------------------------------------------------------ plan

struct PlanArgs {
  moe_paged_plan p;
  Divider per;
};

// Sums over the lanes up to each one.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

struct Request {
  int held, add, old, need, back;   // positions, new ones; pages it has, needs, gives back
};

// Tokens, pages taken and pages given back that lie before a request in its piece, and of the piece.
struct Before {
  int tok, take, back;
};

template <int N>
struct PlanShared {
  double sum[N / kWave][3];
  int odd[N / kWave];
  Before wave[N / kWave];
  int tok0[N], take0[N], back0[N], old[N], held[N];
};

template <int N>
__device__ __forceinline__ Before place_piece(const Request& r, bool in, PlanShared<N>& sh, Before* all) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const Before s = {wave_scan(r.add), wave_scan(r.need), wave_scan(r.back)};
  if (lane == kWave - 1) sh.wave[wave] = s;
  __syncthreads();
  Before at = {s.tok - r.add, s.take - r.need, s.back - r.back};
  *all = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < N / kWave; ++w) {
    const Before q = sh.wave[w];
    if (w < wave) at = {at.tok + q.tok, at.take + q.take, at.back + q.back};
    *all = {all->tok + q.tok, all->take + q.take, all->back + q.back};
  }
  constexpr int kPast = 0x7fffffff;   // behind every item
  sh.tok0[tid] = in ? at.tok : kPast;
  sh.take0[tid] = in ? at.take : kPast;
  sh.back0[tid] = in ? at.back : kPast;
  sh.old[tid] = r.old;
  sh.held[tid] = r.held;
  __syncthreads();
  return at;
}

// U neighbouring items: for each the last request that starts at or before it (first ascending, its first entry 0).
// N = 1024, where the LDS reads of sixteen waves bound it: the inner ones are sought only where the outer two differ;
// else all side by side.
template <int N, int U>
__device__ __forceinline__ void owners(const int* first, int item, int last, int (&i)[U], int (&q)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) i[u] = min(item + u, last), q[u] = 0;
#pragma unroll
  for (int s = N / 2; s; s /= 2) {
#pragma unroll
    for (int u = 0; u < U; u += N < 1024 ? 1 : U - 1)
      if (first[q[u] + s] <= i[u]) q[u] += s;
  }
  if (N < 1024) return;
  if (q[0] == q[U - 1]) {
#pragma unroll
    for (int u = 1; u < U - 1; ++u) q[u] = q[0];
  } else {
#pragma unroll
    for (int s = N / 2; s; s /= 2)
#pragma unroll
      for (int u = 1; u < U - 1; ++u)
        if (first[q[u] + s] <= i[u]) q[u] += s;
  }
}

typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));

// The first n of x to p.
template <int U>
__device__ __forceinline__ void store_items(int32_t* p, const int (&x)[U], int n) {
  if (n >= U) {
#pragma unroll
    for (int u = 0; u < U; u += 4) *(i32x4u*)(p + u) = i32x4u{x[u], x[u + 1], x[u + 2], x[u + 3]};
  } else {
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (u < n) p[u] = x[u];
  }
}

// One block, as the step is done in place: requests in pieces of one a thread.  First the totals, which say whether the
// step can be done at all; then, piece by piece, sums over the piece's requests place its tokens and page moves, which
// all threads then share, four at a time (an item finds its request by bisection of the piece's sums).  Latency bounds it:
// launch, two levels of loads, the sums and the search; 64 requests with a token each 5.6 us, 1024 requests with 16k tokens
// 14.3 us, of which the tokens' searches (the LDS reads of sixteen waves) are half.
template <int N>
__global__ __launch_bounds__(N) void plan_kernel(PlanArgs a) {
  constexpr int U = 4;   // items of a thread at once (8: 15.6 us for 1024 requests with 16k tokens, 4: 14.3)
  const moe_paged_plan& p = a.p;
  __shared__ PlanShared<N> sh;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const long long most = (long long)p.max_pages * p.page_size;
  int held0 = 0, fresh0 = 0;   // of the first piece
  if (tid < p.n_req) held0 = p.held[tid], fresh0 = p.fresh[tid];
  const int head = p.ring_at[0], count = p.ring_at[1];
  auto request = [&](int held, int fresh, int* odd) {
    Request r = {held, max(fresh, 0), 0, 0, 0};
    if (held < 0 || fresh < -1) *odd |= 1;
    else if (held + (long long)r.add > most) *odd |= 2;
    else {
      r.old = pages_for(held, a.per);
      r.need = pages_for(held + r.add, a.per) - r.old;
      r.back = fresh < 0 ? r.old : 0;
    }
    return r;
  };
  int odd = 0;
  Request first = request(held0, fresh0, &odd);
  double sum[3] = {(double)first.add, (double)first.need, (double)first.back};
  for (int r = tid + N; r < p.n_req; r += N) {
    const Request x = request(p.held[r], p.fresh[r], &odd);
    sum[0] += x.add, sum[1] += x.need, sum[2] += x.back;
  }
  const int odds = (__any(odd & 1) ? 1 : 0) | (__any(odd & 2) ? 2 : 0);
#pragma unroll
  for (int i = 0; i < 3; ++i) sum[i] = group_sum_f64<kWave>(sum[i]);   // (whole numbers below 2^53: exact)
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i) sh.sum[wave][i] = sum[i];
    sh.odd[wave] = odds;
  }
  __syncthreads();
  sum[0] = sum[1] = sum[2] = odd = 0;
#pragma unroll
  for (int w = 0; w < N / kWave; ++w) {
#pragma unroll
    for (int i = 0; i < 3; ++i) sum[i] += sh.sum[w][i];
    odd |= sh.odd[w];
  }
  const int status = plan_status(odd & 1, odd & 2, (long long)sum[0], (long long)sum[1], (long long)sum[2], head, count, p.n_pages, p.max_tokens);
  const bool ok = status == kPlanOk;
  int done_t = 0, done_n = 0, done_b = 0;   // tokens and pages of the pieces before
  for (int r0 = 0; r0 < p.n_req; r0 += N) {
    const int r = r0 + tid;
    const bool in = r < p.n_req;
    if (r0) held0 = in ? p.held[r] : 0, fresh0 = in ? p.fresh[r] : 0;
    if (!ok) {
      if (in) p.starts[r] = 0, p.held_out[r] = held0;
      continue;
    }
    const Request x = r0 ? request(held0, fresh0, &odd) : first;
    Before all;
    const Before at = place_piece<N>(x, in, sh, &all);
    if (in) {
      p.starts[r] = done_t + at.tok;
      p.held_out[r] = fresh0 < 0 ? 0 : held0 + x.add;
    }
    const int tail = ring_place(head, count, p.n_pages);
    for (int i0 = tid * U; i0 < all.tok; i0 += U * N) {   // tokens
      int i[U], q[U], page[U], pos[U];
      owners<N, U>(sh.tok0, i0, all.tok - 1, i, q);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        pos[u] = sh.held[q[u]] + i[u] - sh.tok0[q[u]];
        const int pg = (int)divide((uint32_t)pos[u], a.per), old = sh.old[q[u]];
        // a page of this step is read from the ring: its table entry may not be there yet
        page[u] = *(pg < old ? p.tables + (size_t)(r0 + q[u]) * p.max_pages + pg
                             : p.ring + ring_place(head, done_n + sh.take0[q[u]] + pg - old, p.n_pages));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        page[u] = position_slot(page[u], pos[u], p.n_pages, p.page_size, a.per);
        q[u] += r0;
      }
      store_items(p.req + done_t + i0, q, all.tok - i0);
      store_items(p.pos + done_t + i0, pos, all.tok - i0);
      store_items(p.slot + done_t + i0, page, all.tok - i0);
    }
    for (int i0 = tid * U; i0 < all.take; i0 += U * N) {   // pages taken
      int i[U], q[U], page[U];
#pragma unroll
      for (int u = 0; u < U; ++u) page[u] = p.ring[ring_place(head, done_n + min(i0 + u, all.take - 1), p.n_pages)];
      owners<N, U>(sh.take0, i0, all.take - 1, i, q);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < all.take)
          p.tables[(size_t)(r0 + q[u]) * p.max_pages + sh.old[q[u]] + i[u] - sh.take0[q[u]]] = page[u];
    }
    for (int i0 = tid * U; i0 < all.back; i0 += U * N) {   // pages given back
      int i[U], q[U], page[U];
      owners<N, U>(sh.back0, i0, all.back - 1, i, q);
#pragma unroll
      for (int u = 0; u < U; ++u) page[u] = p.tables[(size_t)(r0 + q[u]) * p.max_pages + i[u] - sh.back0[q[u]]];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < all.back) p.ring[ring_place(tail, done_b + i[u], p.n_pages)] = page[u];
    }
    done_t += all.tok;
    done_n += all.take;
    done_b += all.back;
    __syncthreads();
  }
  int none[U];
#pragma unroll
  for (int u = 0; u < U; ++u) none[u] = -1;
  for (int i = done_t + tid * U; i < p.max_tokens; i += U * N)
    for (int32_t* to : {p.req, p.pos, p.slot}) store_items(to + i, none, p.max_tokens - i);
  if (tid == 0) {
    p.starts[p.n_req] = done_t;
    p.ring_at_out[0] = ok ? ring_place(head, done_n, p.n_pages) : head;
    p.ring_at_out[1] = ok ? count - done_n + done_b : count;
    *p.status = status;
  }
}

// ------------------------------------------------------------ heads

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// V values of a cache type, stored at once.
template <int CT, int V>
__device__ __forceinline__ void store_values(void* base, long long at, const float (&x)[V]) {
  if constexpr (CT == MOE_PAGE_F32) {
    float* p = (float*)base + at;
    if constexpr (V == 4) *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
    else *p = x[0];
  } else if constexpr (CT == MOE_PAGE_E4M3) {
    // saturated here: the conversion turns what is past 448 into NaN; NaN stays one
    float c[V];
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = x[i] > 448.0f ? 448.0f : x[i] < -448.0f ? -448.0f : x[i];
    uint8_t* p = (uint8_t*)base + at;
    if constexpr (V == 4) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
      *(int*)p = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
    } else {
      *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[0], 0, false);
    }
  } else {
    uint16_t h[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
      h[i] = CT == MOE_PAGE_F16 ? __builtin_bit_cast(uint16_t, (_Float16)x[i]) : __builtin_bit_cast(uint16_t, (__bf16)x[i]);
    uint16_t* p = (uint16_t*)base + at;
    if constexpr (V == 4) *(u32x2*)p = u32x2{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
    else *p = h[0];
  }
}

struct HeadsArgs {
  moe_paged_heads h;
  PageMap map;
  void* k;
  void* v;
  const float* k_scale;
  const float* v_scale;
  Divider per;   // by the heads of a token
};

// Sum over the 16 lanes of a row of lanes.
__device__ __forceinline__ float row_sum(float x) {
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xf, 0xf, false));   // row_ror 8, 4, 2, 1
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x124, 0xf, 0xf, false));
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x122, 0xf, 0xf, false));
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x121, 0xf, 0xf, false));
  return x;
}

// (token, head) rows, 16 lanes each, 16 a block.  A lane holds V neighbouring pairs at a time: pair i is (i, i + half) of
// the turned values, then two of the rest; so norm, rotation and conversion stay in its registers, and the only sum over
// lanes is the squares', in fp32.  Bound by the bytes: 4096 tokens of 32 / 4 heads of 128 into bf16 pages 33.7 us, 4.8 TB/s.
// V = 4: every access is 16 bytes (8 or 4 into 16- or 8-bit pages); V = 1 (49.7 us) where a pointer, a stride or the
// rotation's width does not allow it.
template <int CT, int V>
__global__ __launch_bounds__(256) void heads_pages_kernel(HeadsArgs a) {
  constexpr int K = 128 / (16 * V);   // a lane's groups of pairs at most (head_dim 256)
  const moe_paged_heads& h = a.h;
  const int hd = a.map.head_dim, H = h.n_q + 2 * a.map.n_kv, lane = threadIdx.x % 16;
  const uint32_t row = blockIdx.x * 16u + threadIdx.x / 16;
  const int t = (int)divide(row, a.per), head = (int)row - t * H;
  if (t >= h.T) return;
  const int slot = h.slot[t], pos = h.pos[t];
  if (slot < 0) return;
  const bool is_q = head < h.n_q, is_v = head >= h.n_q + a.map.n_kv;
  const int kv = is_q ? 0 : is_v ? head - h.n_q - a.map.n_kv : head - h.n_q;
  long long at = 0;
  const bool in = slot_row(a.map, slot, kv, &at);
  if (!is_q && !in) return;
  const float* x = h.qkv + (size_t)t * h.ld + (size_t)head * hd;
  const float* w = is_q ? h.q_norm : is_v ? nullptr : h.k_norm;
  const int half = is_v ? 0 : h.rope_dim / 2, rest = hd / 2 - half;
  const bool turned = half == 0 || (pos >= 0 && pos < h.rope_len);
  auto get = [](const float* p, float (&y)[V]) {
    if constexpr (V == 4) {
      const f32x4 v = *(const f32x4*)p;
      y[0] = v[0], y[1] = v[1], y[2] = v[2], y[3] = v[3];
    } else {
      y[0] = *p;
    }
  };
  auto getx = [](const float* p, float (&y)[V]) {   // read once: past the caches (4096 tokens: 33.7 us, 37.5 through them)
    if constexpr (V == 4) {
      const f32x4 v = __builtin_nontemporal_load((const f32x4*)p);
      y[0] = v[0], y[1] = v[1], y[2] = v[2], y[3] = v[3];
    } else {
      y[0] = *p;
    }
  };
  float y0[K][V], y1[K][V], ss = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = (lane + 16 * k) * V;
    if (i >= hd / 2) break;
    const int e0 = i < half ? i : half + i, e1 = e0 + (i < half ? half : rest);
    getx(x + e0, y0[k]);
    getx(x + e1, y1[k]);
#pragma unroll
    for (int c = 0; c < V; ++c) ss = fmaf(y1[k][c], y1[k][c], fmaf(y0[k][c], y0[k][c], ss));
  }
  const float inv = w ? 1.0f / sqrtf(row_sum(ss) / (float)hd + h.eps) : 1.0f;
  const float* scale = is_q ? nullptr : is_v ? a.v_scale : a.k_scale;
  const float by = scale ? scale[kv] : 1.0f;
  const bool lost = !turned || (is_q && !in);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = (lane + 16 * k) * V;
    if (i >= hd / 2) break;
    const bool turn = i < half;
    const int e0 = turn ? i : half + i, e1 = e0 + (turn ? half : rest);
    if (w) {
      float w0[V], w1[V];
      get(w + e0, w0);
      get(w + e1, w1);
#pragma unroll
      for (int c = 0; c < V; ++c) y0[k][c] = y0[k][c] * inv * w0[c], y1[k][c] = y1[k][c] * inv * w1[c];
    }
    if (turn && turned) {
      float cs[V], sn[V];
      get(h.rope_cos + (size_t)pos * half + i, cs);
      get(h.rope_sin + (size_t)pos * half + i, sn);
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const float r0 = y0[k][c] * cs[c] - y1[k][c] * sn[c], r1 = y1[k][c] * cs[c] + y0[k][c] * sn[c];
        y0[k][c] = r0, y1[k][c] = r1;
      }
    }
    if (lost) {
#pragma unroll
      for (int c = 0; c < V; ++c) y0[k][c] = y1[k][c] = NAN;
    }
    if (is_q) {
      const long long o = (long long)t * h.ldq + (long long)head * hd;
      store_values<MOE_PAGE_F32>(h.q_out, o + e0, y0[k]);
      store_values<MOE_PAGE_F32>(h.q_out, o + e1, y1[k]);
    } else {
      if (CT == MOE_PAGE_E4M3 && scale) {
#pragma unroll
        for (int c = 0; c < V; ++c) y0[k][c] /= by, y1[k][c] /= by;
      }
      void* pool = is_v ? a.v : a.k;
      store_values<CT>(pool, at + e0, y0[k]);
      store_values<CT>(pool, at + e1, y1[k]);
    }
  }
}

__global__ __launch_bounds__(256) void last_rows_kernel(const float* __restrict__ x, const int32_t* __restrict__ starts,
                                                       int D, float* __restrict__ out) {
  const size_t r = blockIdx.x;
  const int first = starts[r], next = starts[r + 1];
  const float* src = x + (size_t)max(next - 1, 0) * D;
  for (int i = threadIdx.x; i < D; i += 256) out[r * D + i] = next > first ? src[i] : 0.0f;
}

// Runs f with the cache's type as a constant.
template <class F>
void with_type(int dtype, F f) {
  if (dtype == MOE_PAGE_F32) f(std::integral_constant<int, MOE_PAGE_F32>{});
  else if (dtype == MOE_PAGE_F16) f(std::integral_constant<int, MOE_PAGE_F16>{});
  else if (dtype == MOE_PAGE_BF16) f(std::integral_constant<int, MOE_PAGE_BF16>{});
  else f(std::integral_constant<int, MOE_PAGE_E4M3>{});
}

}  // namespace

hipError_t launch_last_rows(const float* x, const int32_t* starts, int n_req, int D, float* out, hipStream_t s) {
  hipLaunchKernelGGL(last_rows_kernel, dim3((unsigned)n_req), dim3(256), 0, s, x, starts, D, out);
  return hipGetLastError();
}

moe_status check_paged_step(const moe_paged_plan* plan, const moe_pages* layers, int n_layers, int n_q, int n_kv) {
  moe_status st = check_plan(plan);
  for (int l = 0; !st && l < n_layers; ++l) {
    PageMap map;
    st = check_pages(&layers[l], "step_paged", &map);
  }
  if (!st && !heads_fit(plan->max_tokens, n_q, n_kv))
    return set_error(MOE_ERR_ARG, "step_paged: %d rows of %d heads", plan->max_tokens, n_q);
  return st;
}

}  // namespace moe

using namespace moe;

extern "C" {

moe_status moe_paged_plan_dev(const moe_paged_plan* p) {
  moe_status st = check_plan(p);
  if (st || (st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  const PlanArgs args{*p, make_divider((uint32_t)p->page_size)};
  // few requests and tokens: four waves, whose sums and barriers are the shorter (64 requests 5.6 us, with sixteen 8.5);
  // past them sixteen share the tokens
  if (p->n_req <= 256 && p->max_tokens <= 2048) hipLaunchKernelGGL(plan_kernel<256>, dim3(1), dim3(256), 0, stream(), args);
  else hipLaunchKernelGGL(plan_kernel<1024>, dim3(1), dim3(1024), 0, stream(), args);
  return check_hip(hipGetLastError(), "paged_plan launch");
}

moe_status moe_paged_heads_dev(const moe_paged_heads* h, const moe_pages* g) {
  if (!h) return set_error(MOE_ERR_ARG, "paged_heads: null argument");
  PageMap map;
  moe_status st = check_pages(g, "paged_heads", &map);
  if (st) return st;
  if (h->T < 0 || h->n_q < 1 || h->n_q % map.n_kv)
    return set_error(MOE_ERR_ARG, "paged_heads: %d rows, %d query heads over %d", h->T, h->n_q, map.n_kv);
  const long long H = (long long)h->n_q + 2ll * map.n_kv;
  if (h->ld < H * map.head_dim || h->ldq < (long long)h->n_q * map.head_dim)
    return set_error(MOE_ERR_ARG, "paged_heads: rows of %lld and %lld floats", h->ld, h->ldq);
  if (h->rope_dim < 0 || h->rope_dim % 2 || h->rope_dim > map.head_dim || h->rope_len < 0)
    return set_error(MOE_ERR_ARG, "paged_heads: rope_dim %d, rope_len %d", h->rope_dim, h->rope_len);
  if (h->T == 0) return MOE_OK;
  if (!heads_fit(h->T, h->n_q, map.n_kv)) return set_error(MOE_ERR_ARG, "paged_heads: %d rows of %lld heads", h->T, H);
  if (!h->qkv || !h->pos || !h->slot || !h->q_out || (h->rope_dim && (!h->rope_cos || !h->rope_sin)))
    return set_error(MOE_ERR_ARG, "paged_heads: null pointer");
  if (h->q_out == h->qkv && h->ldq != h->ld) return set_error(MOE_ERR_ARG, "paged_heads: q_out is qkv with another stride");
  if ((st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  const HeadsArgs a{*h, map, g->k, g->v, g->k_scale, g->v_scale, make_divider((uint32_t)H)};
  const dim3 grid((unsigned)((H * h->T + 15) / 16));
  bool four = h->ld % 4 == 0 && h->ldq % 4 == 0 && h->rope_dim % 8 == 0;
  for (const void* p : {(const void*)h->qkv, (const void*)h->q_out, (const void*)h->q_norm, (const void*)h->k_norm,
                        (const void*)(h->rope_dim ? h->rope_cos : nullptr), (const void*)(h->rope_dim ? h->rope_sin : nullptr)})
    four = four && aligned(p, 16);
  with_type(g->dtype, [&](auto c) {
    if (four) hipLaunchKernelGGL((heads_pages_kernel<decltype(c)::value, 4>), grid, dim3(256), 0, stream(), a);
    else hipLaunchKernelGGL((heads_pages_kernel<decltype(c)::value, 1>), grid, dim3(256), 0, stream(), a);
  });
  return check_hip(hipGetLastError(), "paged_heads launch");
}

size_t moe_paged_attn_work_bytes(int T, int n_q, int n_kv, int head_dim) {
  if (T < 0 || n_q < 1 || n_kv < 1 || n_q % n_kv || head_dim < 1) return 0;
  return paged_attn_work(T, n_q, n_kv, head_dim);
}

moe_status moe_paged_attn_dev(const moe_paged_attn* a, const moe_pages* g) {
  if (!a) return set_error(MOE_ERR_ARG, "paged_attn: null argument");
  PageMap map;
  moe_status st = check_pages(g, "paged_attn", &map);
  if (st) return st;
  if (a->T < 0 || a->T > kMostRows || a->n_q < 1 || a->n_q % map.n_kv || a->n_q > 65535)
    return set_error(MOE_ERR_ARG, "paged_attn: %d rows, %d query heads over %d", a->T, a->n_q, map.n_kv);
  if (a->ldq < (long long)a->n_q * map.head_dim || a->ldo < (long long)a->n_q * map.head_dim)
    return set_error(MOE_ERR_ARG, "paged_attn: rows of %lld and %lld floats", a->ldq, a->ldo);
  if (a->n_req < 0 || a->max_pages < 1 || (long long)a->max_pages * map.page_size > kMostPositions)
    return set_error(MOE_ERR_ARG, "paged_attn: %d requests of %d pages", a->n_req, a->max_pages);
  if (!a->req && a->T > a->n_req) return set_error(MOE_ERR_ARG, "paged_attn: %d rows for %d requests", a->T, a->n_req);
  if (a->T == 0) return MOE_OK;
  if (!a->q || !a->pos || !a->tables || !a->out || !a->work) return set_error(MOE_ERR_ARG, "paged_attn: null pointer");
  if (a->out == a->q) return set_error(MOE_ERR_ARG, "paged_attn: out is q");
  const size_t need = moe_paged_attn_work_bytes(a->T, a->n_q, map.n_kv, map.head_dim);
  if (a->work_bytes < need || !aligned(a->work, 16))
    return set_error(MOE_ERR_ARG, "paged_attn: %zu bytes of work at %p, %zu needed, 16-byte aligned", a->work_bytes, a->work, need);
  if ((st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  return check_hip(launch_paged_attn(AttnPages{*a, map, g->k, g->v, g->k_scale, g->v_scale}, g->dtype, stream()),
                   "paged_attn launch");
}

}  // extern "C"
