// nvfp4_route_experts: argument checks and dispatch.  The kernels are in
// route.cuh; those for more than 256 experts are compiled by route_wide.cu.
#include "route.cuh"

namespace nvfp4 {
int launch_route_wide(const void* args, int registers, bool softmax, cudaStream_t stream);   // args: a RouteArgs
}

extern "C" int nvfp4_route_experts(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, const float* bias,
                                   int score, int64_t k, int64_t groups, int64_t top_groups, int group_top,
                                   int renorm, float scale, float* weights, int32_t* ids, void* stream) {
  using namespace nvfp4;
  if (T < 0 || E < 1 || E > kMaxExperts) return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: need T >= 0 and 1..%d experts", kMaxExperts);
  if (k < 1 || k > kMaxTopK || k > E) return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: top_k must be 1..min(%d, experts)", kMaxTopK);
  if (groups < 1 || groups > kMaxGroups || E % groups || top_groups < 1 || top_groups > groups)
    return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: 1..%d groups that divide the experts, of which 1..groups may be used", kMaxGroups);
  if (group_top < 1 || group_top > 2) return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: a group's score sums its 1 or 2 best experts");
  if (score < 0 || score > 1) return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: unknown score function");
  if (dtype < 0 || dtype > 2) return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: logits must be float32, float16 or bfloat16");
  if (ld < E && T > 1) return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: row stride below the number of experts");
  if (T == 0) return NVFP4_OK;
  if (!logits || !weights || !ids) return fail(NVFP4_ERR_INVALID, "nvfp4_route_experts: null pointer");
  const uintptr_t size = dtype == 0 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size || (reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(weights) |
                                                     reinterpret_cast<uintptr_t>(ids)) % 4)
    return fail(NVFP4_ERR_ALIGNMENT, "nvfp4_route_experts: a pointer is not aligned to its element");
  RouteArgs p;
  p.logits = logits; p.bias = bias; p.weights = weights; p.ids = ids;
  p.T = T; p.ld = ld;
  p.E = (int)E; p.k = (int)k; p.groups = (int)groups; p.top_groups = (int)top_groups;
  p.group_top = group_top; p.group_size = (int)(E / groups);
  p.renorm = renorm; p.scale = scale;
  p.dtype = dtype;
  p.vec = aligned16(logits) && (ld * (int64_t)size % 16 == 0 || T == 1);
  p.group_lanes = 0;
  p.batch = 1;
  const bool softmax = score == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int vpl = (p.E + 31) / 32;
  if (vpl <= 1) return launch_route<1>(p, softmax, st);
  if (vpl <= 2) return launch_route<2>(p, softmax, st);
  if (vpl <= 4) return launch_route<4>(p, softmax, st);
  if (vpl <= 8) return launch_route<8>(p, softmax, st);
  return launch_route_wide(&p, vpl, softmax, st);
}
