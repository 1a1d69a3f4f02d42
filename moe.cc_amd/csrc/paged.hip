// paged.hip - many requests over a paged key-value cache (include/moehip.h,
// "many requests over a paged cache"): the step's plan, the new rows' heads
// into their pages, and the entry points (attention: paged_attn.hip).
#include <math.h>

#include "moe_device.h"
#include "moe_lib.h"
#include "paged_attn.h"

namespace moe {
namespace {

// ------------------------------------------------------------ arguments

// Work is queued on the library's stream whatever device the calling thread
// has current.
struct OnDevice {
  int was = -1;
  moe_status enter() {
    int d = -1;
    moe_status st = check_hip(hipGetDevice(&d), "hipGetDevice");
    if (st || d == device()) return st;
    was = d;
    return check_hip(hipSetDevice(device()), "hipSetDevice");
  }
  ~OnDevice() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

int type_bytes(int dtype) { return dtype == MOE_PAGE_F32 ? 4 : dtype == MOE_PAGE_E4M3 ? 1 : 2; }

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
  if (!aligned(g->k, 16) || !aligned(g->v, 16)) return set_error(MOE_ERR_ARG, "%s: pages not 16-byte aligned", who);
  if (g->dtype != MOE_PAGE_E4M3 && (g->k_scale || g->v_scale))
    return set_error(MOE_ERR_ARG, "%s: scales belong to 8-bit pages", who);
  *m = PageMap{g->n_pages, g->page_size, g->n_kv, g->head_dim, g->page_stride, g->head_stride, g->slot_stride,
               make_divider((uint32_t)g->page_size)};
  return MOE_OK;
}

// ------------------------------------------------------------ cache types

struct CacheF32 {
  using T = float;
  static __device__ T make(float x) { return x; }
};
struct CacheF16 {
  using T = _Float16;
  static __device__ T make(float x) { return (_Float16)x; }
};
struct CacheBF16 {
  using T = uint16_t;
  static __device__ T make(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (T)(u >> 16 | 0x40);   // NaN stays one
    return (T)((u + 0x7fffu + (u >> 16 & 1)) >> 16);
  }
};
struct CacheE4M3 {
  using T = uint8_t;
  // saturated here: the conversion itself turns what is past 448 into NaN
  static __device__ T make(float x) {
    const float c = x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x;   // NaN passes
    return (T)(__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false) & 0xff);
  }
};

// ------------------------------------------------------------ plan

constexpr int kPlanThreads = 1024;

// Exclusive sums over the block's threads of three numbers at once, and their
// totals; ends with the block in step.
__device__ int3 block_scan3(int3 v, int3* wave_sum, int3* total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int3 s = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int x = __shfl_up(s.x, d), y = __shfl_up(s.y, d), z = __shfl_up(s.z, d);
    if (lane >= d) s.x += x, s.y += y, s.z += z;
  }
  __syncthreads();
  if (lane == kWave - 1) wave_sum[wave] = s;
  __syncthreads();
  int3 base = {0, 0, 0}, all = {0, 0, 0};
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    const int3 q = wave_sum[w];
    if (w < wave) base.x += q.x, base.y += q.y, base.z += q.z;
    all.x += q.x, all.y += q.y, all.z += q.z;
  }
  *total = all;
  return {base.x + s.x - v.x, base.y + s.y - v.y, base.z + s.z - v.z};
}

// Largest i < n with first[i] <= x (first ascending from first[0] <= x).
__device__ int last_at_most(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct PlanArgs {
  moe_paged_plan p;
  Divider per;
};

// One block: requests in pieces of one a thread.  First the totals, which say
// whether the step can be done at all; then, piece by piece, sums over the
// piece's requests place its tokens and page moves, which all threads then
// share (an item finds its request by bisection of the piece's sums).
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  const moe_paged_plan& p = a.p;
  __shared__ int3 wave_sum[kPlanThreads / kWave];
  __shared__ int tok0[kPlanThreads], take0[kPlanThreads], back0[kPlanThreads], old_s[kPlanThreads], held_s[kPlanThreads];
  __shared__ unsigned long long sums[3];
  __shared__ int bad_s, long_s;
  const int tid = threadIdx.x;
  const int head = p.ring_at[0], count = p.ring_at[1];
  if (tid < 3) sums[tid] = 0;
  if (tid == 0) bad_s = long_s = 0;
  __syncthreads();
  unsigned long long nt = 0, nn = 0, nb = 0;
  for (int r = tid; r < p.n_req; r += kPlanThreads) {
    const int held = p.held[r], fresh = p.fresh[r];
    if (held < 0 || fresh < -1) {
      bad_s = 1;
      continue;
    }
    const long long old = pages_for(held, p.page_size);
    if (old > p.max_pages) long_s = 1;
    if (fresh < 0) {
      nb += old;
    } else {
      const long long now = pages_for((long long)held + fresh, p.page_size);
      if (now > p.max_pages) long_s = 1;
      nt += fresh;
      nn += now - old;
    }
  }
  atomicAdd(&sums[0], nt);
  atomicAdd(&sums[1], nn);
  atomicAdd(&sums[2], nb);
  __syncthreads();
  const int status = plan_status(bad_s, long_s, (long long)sums[0], (long long)sums[1], (long long)sums[2], head, count,
                                 p.n_pages, p.max_tokens);
  const bool ok = status == kPlanOk;
  int done_t = 0, done_n = 0, done_b = 0;   // tokens and pages of the pieces before
  for (int r0 = 0; r0 < p.n_req; r0 += kPlanThreads) {
    const int r = r0 + tid, n = min(kPlanThreads, p.n_req - r0);
    const bool in = r < p.n_req;
    const int held = in ? p.held[r] : 0;
    if (!ok) {
      if (in) p.starts[r] = 0, p.held_out[r] = held;
      continue;
    }
    const int fresh = in ? p.fresh[r] : 0, add = max(fresh, 0);
    const int old = (int)pages_for(held, p.page_size);
    const int need = (int)pages_for((long long)held + add, p.page_size) - old, back = fresh < 0 ? old : 0;
    int3 all;
    const int3 at = block_scan3({add, need, back}, wave_sum, &all);
    tok0[tid] = at.x;
    take0[tid] = at.y;
    back0[tid] = at.z;
    old_s[tid] = old;
    held_s[tid] = held;
    if (in) {
      p.starts[r] = done_t + at.x;
      p.held_out[r] = fresh < 0 ? 0 : held + add;
    }
    __syncthreads();
    for (int i = tid; i < all.y; i += kPlanThreads) {   // pages taken
      const int q = last_at_most(take0, n, i);
      p.tables[(size_t)(r0 + q) * p.max_pages + old_s[q] + i - take0[q]] =
          p.ring[ring_place(head, done_n + i, p.n_pages)];
    }
    for (int i = tid; i < all.z; i += kPlanThreads) {   // pages given back
      const int q = last_at_most(back0, n, i);
      p.ring[ring_place(head, (long long)count + done_b + i, p.n_pages)] =
          p.tables[(size_t)(r0 + q) * p.max_pages + i - back0[q]];
    }
    for (int i = tid; i < all.x; i += kPlanThreads) {   // tokens
      const int q = last_at_most(tok0, n, i);
      const int pos = held_s[q] + i - tok0[q], pg = (int)divide((uint32_t)pos, a.per);
      // a page of this step is read from the ring: its table entry may not be there yet
      const int page = pg < old_s[q] ? p.tables[(size_t)(r0 + q) * p.max_pages + pg]
                                     : p.ring[ring_place(head, (long long)done_n + take0[q] + pg - old_s[q], p.n_pages)];
      p.req[done_t + i] = r0 + q;
      p.pos[done_t + i] = pos;
      p.slot[done_t + i] = position_slot(page, pos, p.n_pages, p.page_size, a.per);
    }
    done_t += all.x;
    done_n += all.y;
    done_b += all.z;
    __syncthreads();
  }
  for (int i = done_t + tid; i < p.max_tokens; i += kPlanThreads) p.req[i] = p.pos[i] = p.slot[i] = -1;
  if (tid == 0) {
    p.starts[p.n_req] = done_t;
    p.ring_at_out[0] = ok ? ring_place(head, done_n, p.n_pages) : head;
    p.ring_at_out[1] = ok ? count - done_n + done_b : count;
    *p.status = status;
  }
}

// ------------------------------------------------------------ heads

struct HeadsArgs {
  moe_paged_heads h;
  PageMap map;
  void* k;
  void* v;
  const float* k_scale;
  const float* v_scale;
};

// A block a (token, head) row: norm, rotation, store.
template <class C>
__global__ __launch_bounds__(64) void heads_pages_kernel(HeadsArgs a) {
  const moe_paged_heads& h = a.h;
  const int lane = threadIdx.x, hd = a.map.head_dim, H = h.n_q + 2 * a.map.n_kv;
  const int t = (int)(blockIdx.x / H), head = (int)(blockIdx.x % H);
  const int slot = h.slot[t], pos = h.pos[t];
  if (slot < 0) return;
  const bool is_q = head < h.n_q, is_v = head >= h.n_q + a.map.n_kv;
  const int kv = is_q ? 0 : is_v ? head - h.n_q - a.map.n_kv : head - h.n_q;
  long long at = 0;
  const bool in = slot_row(a.map, slot, kv, &at);
  if (!is_q && !in) return;
  const float* x = h.qkv + (size_t)t * h.ld + (size_t)head * hd;
  const float* w = is_q ? h.q_norm : is_v ? nullptr : h.k_norm;
  float inv = 1.0f;
  if (w) {
    float s = 0.0f;
    for (int d = lane; d < hd; d += 64) s = fmaf(x[d], x[d], s);
    for (int d = 32; d; d /= 2) s += __shfl_xor(s, d);
    inv = 1.0f / sqrtf(s / (float)hd + h.eps);
  }
  const int half = is_v ? 0 : h.rope_dim / 2, rest = hd / 2 - half;
  const bool turned = !is_v && (half == 0 || (pos >= 0 && pos < h.rope_len));
  const float* scale = is_v ? a.v_scale : a.k_scale;
  const float sc = scale && !is_q ? scale[kv] : 1.0f;
  for (int i = lane; i < hd / 2; i += 64) {
    // pair i: turned (i, i + half) of the first rope_dim, else two of the rest
    const bool rot = i < half;
    const int e0 = rot ? i : half + i, e1 = rot ? i + half : e0 + rest;
    float y0 = x[e0], y1 = x[e1];
    if (w) y0 = y0 * inv * w[e0], y1 = y1 * inv * w[e1];
    if (rot && turned) {
      const float c = h.rope_cos[(size_t)pos * half + i], s = h.rope_sin[(size_t)pos * half + i];
      const float r0 = y0 * c - y1 * s, r1 = y1 * c + y0 * s;
      y0 = r0, y1 = r1;
    }
    if ((!is_v && !turned) || (is_q && !in)) y0 = y1 = NAN;
    if (is_q) {
      float* o = h.q_out + (size_t)t * h.ldq + (size_t)head * hd;
      o[e0] = y0;
      o[e1] = y1;
    } else {
      typename C::T* o = (typename C::T*)(is_v ? a.v : a.k) + at;
      if (scale) y0 /= sc, y1 /= sc;
      o[e0] = C::make(y0);
      o[e1] = C::make(y1);
    }
  }
}

// Runs f with the cache's type.
template <class F>
void with_type(int dtype, F f) {
  if (dtype == MOE_PAGE_F32) f(CacheF32{});
  else if (dtype == MOE_PAGE_F16) f(CacheF16{});
  else if (dtype == MOE_PAGE_BF16) f(CacheBF16{});
  else f(CacheE4M3{});
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

moe_status moe_paged_plan_dev(const moe_paged_plan* p) {
  if (!p) return set_error(MOE_ERR_ARG, "paged_plan: null argument");
  if (p->n_req < 0 || p->max_pages < 1 || p->n_pages < 1 || p->page_size < 1 || p->max_tokens < 0)
    return set_error(MOE_ERR_ARG, "paged_plan: %d requests of %d pages, %d pages of %d, %d tokens", p->n_req, p->max_pages,
                     p->n_pages, p->page_size, p->max_tokens);
  if ((long long)p->n_pages * p->page_size > 0x7fffffffll || (long long)p->max_pages * p->page_size > 0x7fffffffll)
    return set_error(MOE_ERR_ARG, "paged_plan: %d pages of %d, %d a request: past 2^31 positions", p->n_pages, p->page_size,
                     p->max_pages);
  for (const void* q : {(const void*)p->ring_at, (const void*)p->ring, (const void*)p->ring_at_out, (const void*)p->starts,
                        (const void*)p->status})
    if (!q) return set_error(MOE_ERR_ARG, "paged_plan: null pointer");
  if (p->n_req && (!p->fresh || !p->held || !p->tables || !p->held_out)) return set_error(MOE_ERR_ARG, "paged_plan: null pointer");
  if (p->max_tokens && (!p->req || !p->pos || !p->slot)) return set_error(MOE_ERR_ARG, "paged_plan: null pointer");
  moe_status st = ensure_init();
  if (st) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream(), PlanArgs{*p, make_divider((uint32_t)p->page_size)});
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
  if (H * h->T > 0x7fffffffll) return set_error(MOE_ERR_ARG, "paged_heads: %d rows of %lld heads", h->T, H);
  if (!h->qkv || !h->pos || !h->slot || !h->q_out || (h->rope_dim && (!h->rope_cos || !h->rope_sin)))
    return set_error(MOE_ERR_ARG, "paged_heads: null pointer");
  if (h->q_out == h->qkv && h->ldq != h->ld) return set_error(MOE_ERR_ARG, "paged_heads: q_out is qkv with another stride");
  if ((st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  const HeadsArgs a{*h, map, g->k, g->v, g->k_scale, g->v_scale};
  with_type(g->dtype, [&](auto c) {
    hipLaunchKernelGGL(heads_pages_kernel<decltype(c)>, dim3((unsigned)(H * h->T)), dim3(64), 0, stream(), a);
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
  if (a->T < 0 || a->n_q < 1 || a->n_q % map.n_kv || a->n_q > 65535)
    return set_error(MOE_ERR_ARG, "paged_attn: %d rows, %d query heads over %d", a->T, a->n_q, map.n_kv);
  if (a->ldq < (long long)a->n_q * map.head_dim || a->ldo < (long long)a->n_q * map.head_dim)
    return set_error(MOE_ERR_ARG, "paged_attn: rows of %lld and %lld floats", a->ldq, a->ldo);
  if (a->n_req < 0 || a->max_pages < 1 || (long long)a->max_pages * map.page_size > 0x7fffffffll)
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
