// paged.cuh -- launch interfaces of the paged KV-cache operators.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cutetts_b200.h"

namespace ctts {

constexpr int kPlanMaxBatch = 4096;  // per-request prefix sums of the plan live in shared memory

cudaError_t launch_paged_plan(const ctts_paged_plan& p, cudaStream_t s);
cudaError_t launch_paged_append(const ctts_paged_append& p, cudaStream_t s);

// Attention: how a call is laid out over the GPU; it follows from the host's
// arguments and the device alone.
struct PagedAttnPlan {
  int ctas = 0;       // persistent CTAs
  int tile_rows = 0;  // packed rows (token-major, query heads of a KV head inside) per work item
  size_t ws_bytes = 0;  // of this call
};
PagedAttnPlan paged_attn_plan(const ctts_paged_attn& p);
size_t paged_attn_ws_bytes(const ctts_paged_attn& p);  // that serve calls with up to p.max_new new rows
cudaError_t launch_paged_attn(const ctts_paged_attn& p, cudaStream_t s);

}  // namespace ctts
