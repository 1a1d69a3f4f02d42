// paged_shared.hip - attention of rows whose requests begin in the same pages
// (moe_paged_share_dev, moe_paged_attn_shared_dev, include/moehip.h).
#include <math.h>

#include <type_traits>

#include "moe_device.h"
#include "paged_attn.h"

namespace moe {
namespace {

enum { F32 = MOE_PAGE_F32, F16 = MOE_PAGE_F16, BF16 = MOE_PAGE_BF16, E4M3 = MOE_PAGE_E4M3 };

constexpr int kMostShared = 1 << 16;   // rows, groups of a call

// ---------------------------------------------------------------- which positions groups share

struct ShareArgs {
  moe_paged_share s;
  Divider per;    // by page_size
  int* common;    // plan [T] leading pages that a row and its group's first share; kNotLive: no row to count
};
constexpr int kNotLive = 0x7fffffff;

// A wave a row: the group that holds it, that group's first live row, and how many leading pages the two have in common.
__global__ __launch_bounds__(256) void share_rows_kernel(ShareArgs a) {
  const moe_paged_share& s = a.s;
  const int t = (int)blockIdx.x * 4 + (int)threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (t >= s.T) return;
  const int positions = s.max_pages * s.page_size;
  auto length = [&](int r) { return row_length(s.req ? s.req[r] : r, s.pos[r], s.n_req, positions); };
  const int len = length(t);
  if (len <= 0) {
    if (lane == 0) a.common[t] = kNotLive;
    return;
  }
  int lo = 0, hi = s.n_groups;   // the last group that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (s.first[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  int lead = t;
  if (lo > 0 && t < s.first[lo]) {
    for (int r0 = max(s.first[lo - 1], 0); r0 < t; r0 += kWave) {
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
  if (lane == 0) a.common[t] = same;
}

// One block, a wave a group.
__global__ __launch_bounds__(1024) void share_groups_kernel(ShareArgs a) {
  const moe_paged_share& s = a.s;
  const int tid = threadIdx.x, lane = tid % kWave;
  bool bad = false;
  for (int g = tid; g < s.n_groups; g += 1024) bad |= s.first[g] < 0 || s.first[g] > s.first[g + 1] || s.first[g + 1] > s.T;
  bad = __syncthreads_or(bad);
  for (int g = tid / kWave; g < s.n_groups; g += 1024 / kWave) {
    int least = kNotLive;
    if (!bad)
      for (int r = s.first[g] + lane; r < s.first[g + 1]; r += kWave) least = min(least, a.common[r]);
#pragma unroll
    for (int c = 32; c; c /= 2) least = min(least, __shfl_xor(least, c));
    if (lane == 0) s.prefix[g] = least == kNotLive ? 0 : least * s.page_size;
  }
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

template <int CT>
__device__ __forceinline__ float value_at(const char* p, long long i) {
  if constexpr (CT == F32) return ((const float*)p)[i];
  else if constexpr (CT == F16) return (float)((const _Float16*)p)[i];
  else if constexpr (CT == BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  else return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)p)[i], 0);
}

// A wave a (row, query head): 64 positions a step, a lane each for the scores, then a lane a dimension for the values.
template <int CT>
__global__ __launch_bounds__(kWave) void shared_attn_kernel(AttnPages g) {
  constexpr int S = CT == F32 ? 4 : CT == E4M3 ? 1 : 2;
  const moe_paged_attn& a = g.a;
  const int t = (int)blockIdx.x, head = (int)blockIdx.y, lane = threadIdx.x, hd = g.map.head_dim;
  const int req = a.req ? a.req[t] : t;
  const int len = row_length(req, a.pos[t], a.n_req, a.max_pages * g.map.page_size);
  if (len == kPadding) return;
  const int kv = head / (a.n_q / g.map.n_kv);
  const float* q = a.q + (size_t)t * a.ldq + (size_t)head * hd;
  float* out = a.out + (size_t)t * a.ldo + (size_t)head * hd;
  __shared__ float q_s[256], p_s[kWave];
  __shared__ long long at_s[kWave];
  const float scale = a.scale * (g.k_scale ? g.k_scale[kv] : 1.0f), vs = g.v_scale ? g.v_scale[kv] : 1.0f;
  for (int d = lane; d < hd; d += kWave) q_s[d] = q[d] * scale;
  __syncthreads();
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
  bool bad = len == kOutside;
  for (int p0 = 0; p0 < len; p0 += kWave) {
    const int p = p0 + lane;
    float s = -INFINITY;
    long long at = 0;
    if (p < len) {
      const int page = a.tables[(size_t)req * a.max_pages + divide((uint32_t)p, g.map.per)];
      if (page_ok(g.map, page)) {
        at = page_row(g.map, page, kv, p - (int)divide((uint32_t)p, g.map.per) * g.map.page_size);
        s = 0.0f;
        for (int d = 0; d < hd; ++d) s = fmaf(q_s[d], value_at<CT>((const char*)g.k + at * S, d), s);
      } else {
        bad = true;
      }
    }
    float top = s;
#pragma unroll
    for (int c = 32; c; c /= 2) top = fmaxf(top, __shfl_xor(top, c));
    top = fmaxf(top, m);
    const float from = top == -INFINITY ? 0.0f : top, keep = expf(m - from), w = expf(s - from);
    m = top;
    float sum = w;
#pragma unroll
    for (int c = 32; c; c /= 2) sum += __shfl_xor(sum, c);
    l = l * keep + sum;
    p_s[lane] = w;
    at_s[lane] = at;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] *= keep;
      const int d = lane + kWave * i;
      if (d < hd)
        for (int j = 0; j < kWave && p0 + j < len; ++j) o[i] = fmaf(p_s[j], value_at<CT>((const char*)g.v + at_s[j] * S, d), o[i]);
    }
    __syncthreads();
  }
  if (__any(bad)) l = NAN;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + kWave * i;
    if (d < hd) out[d] = l == 0.0f ? 0.0f : o[i] / l * vs;
  }
}

hipError_t launch_shared(const AttnPages& g, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)g.a.T, (unsigned)g.a.n_q), block(kWave);
  if (dtype == F32) hipLaunchKernelGGL(shared_attn_kernel<F32>, grid, block, 0, s, g);
  else if (dtype == F16) hipLaunchKernelGGL(shared_attn_kernel<F16>, grid, block, 0, s, g);
  else if (dtype == BF16) hipLaunchKernelGGL(shared_attn_kernel<BF16>, grid, block, 0, s, g);
  else hipLaunchKernelGGL(shared_attn_kernel<E4M3>, grid, block, 0, s, g);
  return hipGetLastError();
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_paged_share_plan_bytes(int T, int n_groups, int n_q, int n_kv, int head_dim) {
  if (T < 0 || T > kMostShared || n_groups < 0 || n_groups > kMostShared || n_q < 1 || n_kv < 1 || n_q % n_kv || head_dim < 1) return 0;
  return 16 + 4 * (size_t)T;
}

moe_status moe_paged_share_dev(const moe_paged_share* s) {
  moe_status st = check_share(s, "paged_share");
  if (st || (st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  const ShareArgs a{*s, make_divider((uint32_t)s->page_size), (int*)s->plan};
  if (s->T) {
    hipLaunchKernelGGL(share_rows_kernel, dim3((unsigned)(s->T + 3) / 4), dim3(256), 0, stream(), a);
    if ((st = check_hip(hipGetLastError(), "paged_share launch"))) return st;
  }
  hipLaunchKernelGGL(share_groups_kernel, dim3(1), dim3(1024), 0, stream(), a);
  return check_hip(hipGetLastError(), "paged_share launch");
}

size_t moe_paged_attn_shared_work_bytes(int T, int n_groups, int n_q, int n_kv, int head_dim) {
  if (T < 0 || T > kMostShared || n_groups < 0 || n_groups > kMostShared || n_q < 1 || n_kv < 1 || n_q % n_kv || head_dim < 1) return 0;
  return 16;
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
  if ((st = ensure_init())) return st;
  OnDevice on;
  if ((st = on.enter())) return st;
  return check_hip(launch_shared(AttnPages{*a, map, g->k, g->v, g->k_scale, g->v_scale}, g->dtype, stream()), "paged_attn_shared launch");
}

}  // extern "C"
