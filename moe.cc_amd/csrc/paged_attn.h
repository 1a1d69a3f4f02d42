// paged_attn.h - launcher of the attention over a paged cache
// (paged_attn.hip).  Internal; the public ABI is include/moehip.h.
#pragma once
#include <hip/hip_runtime.h>

#include "moe_lib.h"
#include "paged.h"

namespace moe {

inline int type_bytes(int dtype) { return dtype == MOE_PAGE_F32 ? 4 : dtype == MOE_PAGE_E4M3 ? 1 : 2; }

// Rows of a call at most: a launch holds fewer than 2^32 threads.  Positions of a request at most: what a step of the
// kernels adds to one stays far inside an int.
constexpr int kMostRows = (1 << 24) - 1;
constexpr long long kMostPositions = 1ll << 30;

// Checks a cache's description and fills its map.
moe_status check_pages(const moe_pages* g, const char* who, PageMap* m);
// Checks moe_paged_attn_dev's arguments, without its work.
moe_status check_attn(const moe_paged_attn* a, const moe_pages* g, const char* who, PageMap* m);

struct AttnPages {
  moe_paged_attn a;
  PageMap map;
  const void* k;
  const void* v;
  const float* k_scale;
  const float* v_scale;
};

// Bytes of moe_paged_attn::work.
size_t paged_attn_work(int T, int n_q, int n_kv, int head_dim);
hipError_t launch_paged_attn(const AttnPages& p, int dtype, hipStream_t stream);

// Whether a model with n_q query heads over n_kv can take a step of this plan
// over these layers' pages: what its moe_paged_* calls would refuse.
moe_status check_paged_step(const moe_paged_plan* plan, const moe_pages* layers, int n_layers, int n_q, int n_kv);

// What moe_beam_select_dev, moe_paged_fork_dev and moe_paged_copy_dev refuse, without any GPU work.
moe_status check_select(const moe_beam_select* s);
moe_status check_fork(const moe_paged_fork* f);
moe_status check_copy(const int32_t* copies, int n, const moe_pages* layers, int n_layers);
// Rows of moe_paged_share_dev at most.
int shared_rows_max();

// x row of each request's last token (zeros for one without tokens): out
// [n_req][D] from x [.][D] at starts[r + 1] - 1.
hipError_t launch_last_rows(const float* x, const int32_t* starts, int n_req, int D, float* out, hipStream_t stream);

}  // namespace moe
