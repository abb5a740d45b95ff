// Launch interface of the mixture-of-experts and orthogonalisation kernels.
#pragma once

#include "ckan_kernels.hpp"

namespace ckan {

// ---- routing (ckan_route.hip) -----------------------------------------------
constexpr int kRouteMaxExperts = 512;  // 8 experts a lane
constexpr int kRouteMaxTopK = 64;      // lane j holds the j-th chosen expert
constexpr int kRouteMaxGroups = 64;    // a lane a group
// Added to the sum that renormalised weights are divided by: a row whose chosen
// scores all underflow gets zero weights instead of NaN.
constexpr float kRouteEps = 1e-20f;

struct RouteArgs {
  const void* logits;  // [rows, E], row pitch ld
  const float* bias;   // [E] or NULL
  float* weights;      // [rows, top_k]
  int64_t* indices;    // [rows, top_k] (read by the backward)
  const float* dweights;
  void* dlogits;       // [rows, E]
  int64_t rows, ld;
  int E, top_k, groups, top_groups;
  int softmax, renormalize, bf16;
  float scale;
};
void launch_route(const RouteArgs& a, bool backward, hipStream_t st);

}  // namespace ckan
