// grouped_topk routing: one warp per token.
//
// Rule (grouped_topk/v0/grouped_topk.py:91-132 of the reference, plus the
// DeepSeek-V3 bias / top-2-sum extension):
//   scores  = softmax(g) | sigmoid(g)
//   choice  = scores (+ bias)
//   gscore  = max(choice in group) | sum of the two largest choice in group
//   keep the topk_group best groups; top-k experts of the kept groups by choice
//   weights = scores of the chosen experts, renormalised, times the scale
// Ordering is the strict total order (value descending, index ascending), the
// rank rule of grouped_topk/v1/grouped_topk.py:94.
//
// Layout: lane l holds experts [l*VPL, l*VPL + VPL) of its token in registers
// (VPL = 8 for E = 256: two 128-bit loads per lane, one coalesced 1 KiB row per
// warp). Group scores go through a per-warp shared-memory row so that any
// group size works; the top-k is k rounds of a warp arg-max over
// (choice, -index) carrying the unbiased score. HBM-bound at large M.
#include "common.cuh"
#include "routing.cuh"

namespace moe {
namespace {

constexpr int kWarpsPerBlock = 8;

template <int VPL, bool VEC>
__global__ void __launch_bounds__(kWarpsPerBlock * 32)
grouped_topk_kernel(const float* __restrict__ gating, const float* __restrict__ bias, int64_t M, int E,
                    int topk, int renormalize, int n_group, int topk_group, int scoring, int gmode,
                    float scale, float* __restrict__ out_w, int32_t* __restrict__ out_ids) {
  __shared__ float s_choice[kWarpsPerBlock][kRouteMaxExperts];
  const int warp = threadIdx.x >> 5;
  const int64_t tok = (int64_t)blockIdx.x * kWarpsPerBlock + warp;
  if (tok >= M) return;  // whole warp exits together

  route_token_general<VPL, VEC>(gating + tok * (int64_t)E, bias, tok, E, topk, renormalize, n_group, topk_group, scoring,
                                gmode, scale, out_w, out_ids, s_choice[warp]);
}

template <int VPL, int LPG>
__global__ void __launch_bounds__(kWarpsPerBlock * 32)
grouped_topk_lanes_kernel(const float* __restrict__ gating, const float* __restrict__ bias, int64_t M, int topk,
                          int renormalize, int n_group, int topk_group, int scoring, int gmode, float scale,
                          float* __restrict__ out_w, int32_t* __restrict__ out_ids) {
  __shared__ RouteScratch s_scr[kWarpsPerBlock];
  const int64_t tok = (int64_t)blockIdx.x * kWarpsPerBlock + (threadIdx.x >> 5);
  if (tok >= M) return;  // whole warp exits together
  route_token_lanes<VPL, LPG, false>(gating + tok * (int64_t)(32 * VPL), bias, tok, topk, renormalize, n_group,
                                     topk_group, scoring, gmode, scale, out_w, out_ids,
                                     &s_scr[threadIdx.x >> 5]);
}

template <int VPL>
cudaError_t launch_vpl(bool vec, const float* g, const float* bias, int64_t M, int E, int topk, int renorm,
                       int n_group, int topk_group, int scoring, int gmode, float scale, float* w,
                       int32_t* ids, cudaStream_t st) {
  const dim3 block(kWarpsPerBlock * 32);
  const dim3 grid((unsigned)ceil_div(M, kWarpsPerBlock));
  if constexpr (VPL % 4 == 0) {
    if (vec) {
      grouped_topk_kernel<VPL, true><<<grid, block, 0, st>>>(g, bias, M, E, topk, renorm, n_group, topk_group,
                                                             scoring, gmode, scale, w, ids);
      return cudaGetLastError();
    }
  }
  grouped_topk_kernel<VPL, false><<<grid, block, 0, st>>>(g, bias, M, E, topk, renorm, n_group, topk_group,
                                                          scoring, gmode, scale, w, ids);
  return cudaGetLastError();
}

}  // namespace
}  // namespace moe

extern "C" int moe_grouped_topk(const float* gating_output, const float* bias, int64_t num_tokens,
                                int num_experts, int topk, int renormalize, int num_expert_group,
                                int topk_group, int scoring_func, int group_score_mode,
                                float routed_scaling_factor, float* topk_weights, int32_t* topk_ids,
                                void* stream) {
  using namespace moe;
  if (num_tokens < 0 || num_experts <= 0 || topk <= 0 || num_expert_group <= 0 || topk_group <= 0)
    return MOE_ERR_INVALID_ARG;
  if (scoring_func != MOE_SCORING_SOFTMAX && scoring_func != MOE_SCORING_SIGMOID) return MOE_ERR_INVALID_ARG;
  if (group_score_mode != MOE_GROUP_SCORE_MAX && group_score_mode != MOE_GROUP_SCORE_TOP2_SUM)
    return MOE_ERR_INVALID_ARG;
  if (num_experts > kRouteMaxExperts || num_expert_group > 32 || topk > 32) return MOE_ERR_BAD_SHAPE;
  if (num_experts % num_expert_group != 0 || topk_group > num_expert_group) return MOE_ERR_BAD_SHAPE;
  const int epg = num_experts / num_expert_group;
  if (topk > topk_group * epg) return MOE_ERR_BAD_SHAPE;
  if (group_score_mode == MOE_GROUP_SCORE_TOP2_SUM && epg < 2) return MOE_ERR_BAD_SHAPE;
  if (num_tokens == 0) return MOE_OK;
  if (!gating_output || !topk_weights || !topk_ids) return MOE_ERR_INVALID_ARG;
  if (num_tokens > (int64_t)INT32_MAX * kWarpsPerBlock) return MOE_ERR_BAD_SHAPE;

  const int vpl_needed = (int)ceil_div(num_experts, 32);
  {
    // register-only variant: every lane full, 16-byte aligned rows, groups of whole lanes
    const bool aligned = ((reinterpret_cast<uintptr_t>(gating_output) & 15u) == 0) &&
                         (bias == nullptr || (reinterpret_cast<uintptr_t>(bias) & 15u) == 0);
    const bool grouped = topk_group < num_expert_group;
    const int lpg = (num_experts / num_expert_group) / 8;  // lanes per group at VPL = 8
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (aligned && num_experts == 256 && topk <= 32 &&
        (!grouped || ((num_experts / num_expert_group) % 8 == 0 && (lpg & (lpg - 1)) == 0))) {
      const dim3 block(kWarpsPerBlock * 32);
      const dim3 grid((unsigned)ceil_div(num_tokens, kWarpsPerBlock));
#define MOE_GTL_ARGS gating_output, bias, num_tokens, topk, renormalize, num_expert_group, topk_group, \
                     scoring_func, group_score_mode, routed_scaling_factor, topk_weights, topk_ids
      switch (grouped ? lpg : 1) {
        case 1: grouped_topk_lanes_kernel<8, 1><<<grid, block, 0, st>>>(MOE_GTL_ARGS); break;
        case 2: grouped_topk_lanes_kernel<8, 2><<<grid, block, 0, st>>>(MOE_GTL_ARGS); break;
        case 4: grouped_topk_lanes_kernel<8, 4><<<grid, block, 0, st>>>(MOE_GTL_ARGS); break;
        case 8: grouped_topk_lanes_kernel<8, 8><<<grid, block, 0, st>>>(MOE_GTL_ARGS); break;
        case 16: grouped_topk_lanes_kernel<8, 16><<<grid, block, 0, st>>>(MOE_GTL_ARGS); break;
        default: grouped_topk_lanes_kernel<8, 32><<<grid, block, 0, st>>>(MOE_GTL_ARGS); break;
      }
#undef MOE_GTL_ARGS
      return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
    }
  }
  const bool vec = (num_experts % 4 == 0) && ((reinterpret_cast<uintptr_t>(gating_output) & 15u) == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t err;
#define MOE_GT_ARGS vec, gating_output, bias, num_tokens, num_experts, topk, renormalize, num_expert_group, \
                    topk_group, scoring_func, group_score_mode, routed_scaling_factor, topk_weights, topk_ids, st
  if (vpl_needed <= 1) err = launch_vpl<1>(MOE_GT_ARGS);
  else if (vpl_needed <= 2) err = launch_vpl<2>(MOE_GT_ARGS);
  else if (vpl_needed <= 4) err = launch_vpl<4>(MOE_GT_ARGS);
  else if (vpl_needed <= 8) err = launch_vpl<8>(MOE_GT_ARGS);
  else err = launch_vpl<16>(MOE_GT_ARGS);
#undef MOE_GT_ARGS
  return err == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}
