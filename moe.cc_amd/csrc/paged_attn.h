// paged_attn.h - launcher of the attention over a paged cache
// (paged_attn.hip).  Internal; the public ABI is include/moehip.h.
#pragma once
#include <hip/hip_runtime.h>

#include "moe_lib.h"
#include "paged.h"

namespace moe {

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

// x row of each request's last token (zeros for one without tokens): out
// [n_req][D] from x [.][D] at starts[r + 1] - 1.
hipError_t launch_last_rows(const float* x, const int32_t* starts, int n_req, int D, float* out, hipStream_t stream);

}  // namespace moe
