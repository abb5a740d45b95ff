// C-ABI entry points of the mixture-of-experts and orthogonalisation operators
// (include/chebykan.h): argument checks on the host, then the launches on the
// caller's stream.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "chebykan.h"
#include "ckan_mix.hpp"

using namespace ckan;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(CKAN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return CKAN_OK;
}

int route_args(const ckan_route_desc* d, RouteArgs* a) {
  if (!d) return fail(CKAN_ERR_INVALID_ARG, "route desc is NULL");
  if (d->rows < 0) return fail(CKAN_ERR_INVALID_ARG, "rows must be >= 0 (got %lld)", (long long)d->rows);
  if (d->rows > ((int64_t)1 << 31))
    return fail(CKAN_ERR_UNSUPPORTED, "rows above 2^31 are not supported (got %lld)", (long long)d->rows);
  if (d->experts < 1) return fail(CKAN_ERR_INVALID_ARG, "experts must be >= 1 (got %d)", d->experts);
  if (d->experts > kRouteMaxExperts)
    return fail(CKAN_ERR_UNSUPPORTED, "experts above %d are not supported (got %d)", kRouteMaxExperts, d->experts);
  if (d->logits_ld < d->experts)
    return fail(CKAN_ERR_INVALID_ARG, "logits_ld %lld is below experts %d", (long long)d->logits_ld, d->experts);
  if (d->dtype != CKAN_DTYPE_F32 && d->dtype != CKAN_DTYPE_BF16)
    return fail(CKAN_ERR_INVALID_ARG, "unknown logits dtype %d", d->dtype);
  if (d->score != CKAN_SCORE_SOFTMAX && d->score != CKAN_SCORE_SIGMOID)
    return fail(CKAN_ERR_INVALID_ARG, "unknown score function %d", d->score);
  if (d->groups < 1 || d->experts % d->groups)
    return fail(CKAN_ERR_INVALID_ARG, "groups must divide experts %d (got %d)", d->experts, d->groups);
  if (d->groups > kRouteMaxGroups)
    return fail(CKAN_ERR_UNSUPPORTED, "groups above %d are not supported (got %d)", kRouteMaxGroups, d->groups);
  if (d->top_groups < 1 || d->top_groups > d->groups)
    return fail(CKAN_ERR_INVALID_ARG, "top_groups must lie in [1, %d] (got %d)", d->groups, d->top_groups);
  const int open = d->experts / d->groups * d->top_groups;
  if (d->top_k < 1 || d->top_k > open)
    return fail(CKAN_ERR_INVALID_ARG, "top_k must lie in [1, %d], the experts of the kept groups (got %d)", open, d->top_k);
  if (d->top_k > kRouteMaxTopK)
    return fail(CKAN_ERR_UNSUPPORTED, "top_k above %d is not supported (got %d)", kRouteMaxTopK, d->top_k);
  if (!isfinite(d->scale)) return fail(CKAN_ERR_INVALID_ARG, "scale must be finite");
  *a = RouteArgs{};
  a->rows = d->rows;
  a->ld = d->logits_ld;
  a->E = d->experts;
  a->top_k = d->top_k;
  a->groups = d->groups;
  a->top_groups = d->top_groups;
  a->softmax = d->score == CKAN_SCORE_SOFTMAX;
  a->renormalize = d->renormalize != 0;
  a->bf16 = d->dtype == CKAN_DTYPE_BF16;
  a->scale = d->scale;
  return CKAN_OK;
}

}  // namespace

extern "C" {

int ckan_route(const ckan_route_desc* desc, const void* logits, const float* bias, float* weights,
               int64_t* indices, void* stream) {
  RouteArgs a;
  if (const int rc = route_args(desc, &a)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  if (!logits || !weights || !indices) return fail(CKAN_ERR_INVALID_ARG, "route: NULL pointer");
  a.logits = logits;
  a.bias = bias;
  a.weights = weights;
  a.indices = indices;
  launch_route(a, false, reinterpret_cast<hipStream_t>(stream));
  return check_launch("route");
}

int ckan_route_backward(const ckan_route_desc* desc, const void* logits, const int64_t* indices,
                        const float* dweights, void* dlogits, void* stream) {
  RouteArgs a;
  if (const int rc = route_args(desc, &a)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  if (!logits || !indices || !dweights || !dlogits)
    return fail(CKAN_ERR_INVALID_ARG, "route_backward: NULL pointer");
  a.logits = logits;
  a.indices = const_cast<int64_t*>(indices);
  a.dweights = dweights;
  a.dlogits = dlogits;
  launch_route(a, true, reinterpret_cast<hipStream_t>(stream));
  return check_launch("route_backward");
}

}  // extern "C"
