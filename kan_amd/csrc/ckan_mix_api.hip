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
  // a wave a row: a launch holds fewer than 2^32 threads
  if (d->rows >= ((int64_t)1 << 26))
    return fail(CKAN_ERR_UNSUPPORTED, "2^26 rows or more are not supported (got %lld)", (long long)d->rows);
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
  // as many lanes a group as 64 lanes have for all of them, a power of two
  while ((2 << a->lanes_log2) * d->groups <= 64) ++a->lanes_log2;
  a->inv_size = (float)d->groups / (float)d->experts;
  a->softmax = d->score == CKAN_SCORE_SOFTMAX;
  a->renormalize = d->renormalize != 0;
  a->bf16 = d->dtype == CKAN_DTYPE_BF16;
  a->scale = d->scale;
  return CKAN_OK;
}

int experts_check(const ckan_experts_desc* d) {
  if (!d) return fail(CKAN_ERR_INVALID_ARG, "experts desc is NULL");
  if (d->rows < 0) return fail(CKAN_ERR_INVALID_ARG, "rows must be >= 0 (got %lld)", (long long)d->rows);
  if (d->experts < 1 || d->top_k < 1 || d->in_dim < 1 || d->out_dim < 1)
    return fail(CKAN_ERR_INVALID_ARG, "experts, top_k, in_dim and out_dim must be >= 1 (got %d, %d, %d, %d)", d->experts,
                d->top_k, d->in_dim, d->out_dim);
  if (d->degree < 0) return fail(CKAN_ERR_INVALID_ARG, "degree must be >= 0 (got %d)", d->degree);
  if (d->dtype != CKAN_DTYPE_F32 && d->dtype != CKAN_DTYPE_BF16) return fail(CKAN_ERR_INVALID_ARG, "unknown dtype %d", d->dtype);
  if (d->wdtype != CKAN_DTYPE_F32 && d->wdtype != CKAN_DTYPE_BF16)
    return fail(CKAN_ERR_INVALID_ARG, "unknown weights dtype %d", d->wdtype);
  if (d->experts > kExpertsMax) return fail(CKAN_ERR_UNSUPPORTED, "experts above %d are not supported (got %d)", kExpertsMax, d->experts);
  if (d->top_k > kExpertsMaxTopK) return fail(CKAN_ERR_UNSUPPORTED, "top_k above %d is not supported (got %d)", kExpertsMaxTopK, d->top_k);
  if (d->degree < 1 || d->degree > kExpertsMaxDegree)
    return fail(CKAN_ERR_UNSUPPORTED, "experts have degree 1 to %d (got %d)", kExpertsMaxDegree, d->degree);
  if (d->in_dim > 65536 || d->out_dim > 65536)
    return fail(CKAN_ERR_UNSUPPORTED, "in_dim and out_dim above 65536 are not supported (got %d, %d)", d->in_dim, d->out_dim);
  // a launch holds fewer than 2^32 threads: 32 a slot, one for four values of a row
  if (d->rows > ((int64_t)1 << 26) / d->top_k)
    return fail(CKAN_ERR_UNSUPPORTED, "rows * top_k above 2^26 is not supported");
  if (d->rows > ((int64_t)1 << 33) / (d->in_dim > d->out_dim ? d->in_dim : d->out_dim))
    return fail(CKAN_ERR_UNSUPPORTED, "rows times in_dim or out_dim above 2^33 is not supported");
  return CKAN_OK;
}

ExpertsPlan experts_plan(const ckan_experts_desc* d) {
  return make_experts_plan(d->rows, d->experts, d->top_k, d->in_dim, d->out_dim, d->degree,
                           d->dtype == CKAN_DTYPE_BF16, d->wdtype == CKAN_DTYPE_BF16);
}

// Without a saved buffer its parts that the forward itself needs (all before the
// packed dx operand) lead the workspace.
size_t experts_fwd_ws(const ExpertsPlan& p, bool without_saved) {
  if (without_saved && p.stream) return p.stream_bytes;
  return p.fwd_bytes + (without_saved ? p.cb_off : 0);
}

ckan_experts_desc mixture_experts(const ckan_mixture_desc* d) {
  return ckan_experts_desc{d->rows, d->experts, d->top_k, d->in_dim, d->out_dim, d->degree, d->coeff_dtype, CKAN_DTYPE_F32};
}

int mixture_args(const ckan_mixture_desc* d, FewArgs* a) {
  if (!d) return fail(CKAN_ERR_INVALID_ARG, "mixture desc is NULL");
  for (const int t : {d->x_dtype, d->gate_dtype, d->coeff_dtype})
    if (t != CKAN_DTYPE_F32 && t != CKAN_DTYPE_BF16) return fail(CKAN_ERR_INVALID_ARG, "unknown dtype %d", t);
  const ckan_experts_desc e = mixture_experts(d);
  if (const int rc = experts_check(&e)) return rc;
  const ckan_route_desc r = {d->rows, d->experts, d->experts, d->top_k, d->score, d->groups, d->top_groups, d->renormalize,
                             CKAN_DTYPE_F32, d->scale};
  *a = FewArgs{};
  if (const int rc = route_args(&r, &a->route)) return rc;
  a->x_bf16 = d->x_dtype == CKAN_DTYPE_BF16;
  a->gate_bf16 = d->gate_dtype == CKAN_DTYPE_BF16;
  a->coeff_bf16 = d->coeff_dtype == CKAN_DTYPE_BF16;
  a->I = d->in_dim;
  a->O = d->out_dim;
  a->D = d->degree + 1;
  few_plan(a);
  return CKAN_OK;
}

// The largest |b s^2 + c s^4| and |a + b s^2 + c s^4|, the iteration's matrices, that
// singular values in [0, 1] can reach over all steps, by sampling the interval.
double ortho_reach(const ckan_ortho_desc* d) {
  double top = 1.0, most = 0.0;
  for (int s = 0; s < d->steps && most < 1e6; ++s) {
    double next = 0.0;
    for (int i = 0; i <= 1024; ++i) {
      const double x = top * i / 1024, y = x * x, bv = d->b * y + d->c * y * y;
      most = fmax(most, fmax(fabs(bv), fabs(d->a + bv)));
      next = fmax(next, fabs(x * (d->a + bv)));
    }
    top = fmax(next, 1e-30);
  }
  return fmax(most, 2.0 * top * top);  // A = X X^T has to fit with it
}

int ortho_check(const ckan_ortho_desc* d) {
  if (!d) return fail(CKAN_ERR_INVALID_ARG, "ortho desc is NULL");
  if (d->batch < 0 || d->batch > 65535)
    return fail(CKAN_ERR_INVALID_ARG, "batch must lie in [0, 65535] (got %d)", d->batch);
  if (d->rows < 1 || d->cols < 1)
    return fail(CKAN_ERR_INVALID_ARG, "rows and cols must be >= 1 (got %d, %d)", d->rows, d->cols);
  const int m = d->rows < d->cols ? d->rows : d->cols, n = d->rows < d->cols ? d->cols : d->rows;
  if (m > 16384) return fail(CKAN_ERR_UNSUPPORTED, "the smaller dimension above 16384 is not supported (got %d)", m);
  if (n > (1 << 24)) return fail(CKAN_ERR_UNSUPPORTED, "dimensions above 2^24 are not supported (got %d)", n);
  if (d->inner < 1 || d->cols % d->inner)
    return fail(CKAN_ERR_INVALID_ARG, "inner must divide cols %d (got %d)", d->cols, d->inner);
  if (d->batch_stride < 0 || d->row_stride < 0 || d->outer_stride < 0 || d->inner_stride < 0)
    return fail(CKAN_ERR_INVALID_ARG, "strides must be >= 0");
  if (d->batch > 1 && d->batch_stride < (int64_t)d->rows * d->cols)
    return fail(CKAN_ERR_INVALID_ARG, "batch_stride %lld is below a matrix's %lld elements", (long long)d->batch_stride,
                (long long)d->rows * d->cols);
  const bool rows_first = d->inner == 1 && d->outer_stride == 1 && d->row_stride == d->cols;
  const bool cols_first = d->inner == 1 && d->row_stride == 1 && d->outer_stride == d->rows;
  const bool coeffs = d->inner > 1 && d->inner_stride == 1 && d->row_stride == d->inner &&
                      d->outer_stride == (int64_t)d->rows * d->inner;
  const bool vector = d->inner == 1 && (d->rows == 1 || d->cols == 1) && (d->rows == 1 ? d->outer_stride : d->row_stride) == 1;
  if (!rows_first && !cols_first && !coeffs && !vector)
    return fail(CKAN_ERR_UNSUPPORTED, "the matrices have to be dense: row-major, column-major or [cols / inner, rows, inner]");
  if (d->steps < 0 || d->steps > 100) return fail(CKAN_ERR_INVALID_ARG, "steps must lie in [0, 100] (got %d)", d->steps);
  if (d->dtype != CKAN_DTYPE_F32 && d->dtype != CKAN_DTYPE_BF16)
    return fail(CKAN_ERR_INVALID_ARG, "unknown dtype %d", d->dtype);
  if (!isfinite(d->a) || !isfinite(d->b) || !isfinite(d->c) || !(d->eps >= 0.0f) || !isfinite(d->eps))
    return fail(CKAN_ERR_INVALID_ARG, "the coefficients and eps must be finite, eps >= 0");
  if (!(ortho_reach(d) < 15.0))
    return fail(CKAN_ERR_UNSUPPORTED, "coefficients (%g, %g, %g) leave the products' range within %d steps", d->a,
                d->b, d->c, d->steps);
  return CKAN_OK;
}

OrthoArgs ortho_args(const ckan_ortho_desc* d) {
  OrthoArgs a{};
  a.batch = d->batch;
  a.rows = d->rows;
  a.cols = d->cols;
  a.steps = d->steps;
  a.a = d->a;
  a.b = d->b;
  a.c = d->c;
  a.eps = d->eps;
  a.bf16 = d->dtype == CKAN_DTYPE_BF16;
  a.view = MatView{d->batch_stride, d->row_stride, d->outer_stride, d->inner_stride, d->inner};
  return a;
}

int ortho_ws(const ckan_ortho_desc* d, void* ws, size_t ws_bytes) {
  const size_t need = ortho_workspace_bytes(ortho_args(d));
  if (ws_bytes < need) return fail(CKAN_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", ws_bytes, need);
  if (!ws || !is_al16(ws)) return fail(CKAN_ERR_INVALID_ARG, "workspace is NULL or not 16-byte aligned");
  return CKAN_OK;
}

}  // namespace

extern "C" {

size_t ckan_experts_saved_bytes(const ckan_experts_desc* desc) {
  return experts_check(desc) || desc->rows == 0 ? 0 : experts_plan(desc).saved_bytes;
}

size_t ckan_experts_workspace_bytes(const ckan_experts_desc* desc, int backward, int without_saved) {
  if (experts_check(desc) || desc->rows == 0) return 0;
  const ExpertsPlan p = experts_plan(desc);
  return backward ? p.bwd_bytes : experts_fwd_ws(p, without_saved != 0);
}

int ckan_experts_forward(const ckan_experts_desc* desc, const void* x, const void* coeffs, const int64_t* indices,
                         const void* weights, void* y, void* saved, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = experts_check(desc)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  if (!x || !coeffs || !indices || !weights || !y) return fail(CKAN_ERR_INVALID_ARG, "experts_forward: NULL pointer");
  ExpertsArgs a{};
  a.p = experts_plan(desc);
  const size_t need = experts_fwd_ws(a.p, !saved);
  if (ws_bytes < need) return fail(CKAN_ERR_WORKSPACE, "experts forward workspace too small: %zu < %zu bytes", ws_bytes, need);
  if (!ws || !is_al16(ws) || !is_al16(saved))
    return fail(CKAN_ERR_INVALID_ARG, "experts_forward: workspace is NULL, or workspace or saved not 16-byte aligned");
  if (!is_al16(x) || !is_al16(coeffs) || !is_al16(y))
    return fail(CKAN_ERR_INVALID_ARG, "experts_forward: x, coeffs and y must be 16-byte aligned");
  a.x = x;
  a.coeffs = coeffs;
  a.indices = indices;
  a.weights = weights;
  a.y = y;
  if (!saved && a.p.stream) {
    a.ws = (char*)ws;
    launch_experts_stream(a, reinterpret_cast<hipStream_t>(stream));
    return check_launch("experts_forward");
  }
  a.saved = saved ? (char*)saved : (char*)ws;
  a.ws = (char*)ws + (saved ? 0 : a.p.cb_off);
  launch_experts_forward(a, saved != nullptr, reinterpret_cast<hipStream_t>(stream));
  return check_launch("experts_forward");
}

int ckan_experts_backward(const ckan_experts_desc* desc, const int64_t* indices, const void* weights, void* saved,
                          const void* dy, void* dx, void* dcoeffs, void* dweights, void* ws, size_t ws_bytes,
                          void* stream) {
  if (const int rc = experts_check(desc)) return rc;
  if (desc->rows == 0) {
    if (dcoeffs) return fail(CKAN_ERR_INVALID_ARG, "experts_backward: no rows, the caller fills dcoeffs with zeros");
    return CKAN_OK;
  }
  if (!dx && !dcoeffs && !dweights) return CKAN_OK;
  if (!indices || !weights || !saved || !dy) return fail(CKAN_ERR_INVALID_ARG, "experts_backward: NULL pointer");
  ExpertsArgs a{};
  a.p = experts_plan(desc);
  if (ws_bytes < a.p.bwd_bytes)
    return fail(CKAN_ERR_WORKSPACE, "experts backward workspace too small: %zu < %zu bytes", ws_bytes, a.p.bwd_bytes);
  if (!ws || !is_al16(ws) || !is_al16(saved))
    return fail(CKAN_ERR_INVALID_ARG, "experts_backward: workspace is NULL, or workspace or saved not 16-byte aligned");
  if (!is_al16(dy) || !is_al16(dx) || !is_al16(dcoeffs))
    return fail(CKAN_ERR_INVALID_ARG, "experts_backward: dy, dx and dcoeffs must be 16-byte aligned");
  a.indices = indices;
  a.weights = weights;
  a.dy = dy;
  a.dx = dx;
  a.dcoeffs = dcoeffs;
  a.dweights = dweights;
  a.saved = (char*)saved;
  a.ws = (char*)ws;
  launch_experts_backward(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch("experts_backward");
}

size_t ckan_orthogonalize_workspace_bytes(const ckan_ortho_desc* desc) {
  return ortho_check(desc) ? 0 : ortho_workspace_bytes(ortho_args(desc));
}

int ckan_orthogonalize(const ckan_ortho_desc* desc, const void* in, void* out, void* ws, size_t ws_bytes,
                       void* stream) {
  if (const int rc = ortho_check(desc)) return rc;
  if (desc->batch == 0) return CKAN_OK;
  if (!in || !out) return fail(CKAN_ERR_INVALID_ARG, "orthogonalize: NULL pointer");
  if (const int rc = ortho_ws(desc, ws, ws_bytes)) return rc;
  OrthoArgs a = ortho_args(desc);
  a.in = in;
  a.out = out;
  launch_ortho(a, ws, reinterpret_cast<hipStream_t>(stream));
  return check_launch("orthogonalize");
}

int ckan_muon_step(const ckan_ortho_desc* desc, float* p, const float* g, float* buf, float lr, float momentum,
                   float weight_decay, float scale, int nesterov, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = ortho_check(desc)) return rc;
  if (desc->dtype != CKAN_DTYPE_F32) return fail(CKAN_ERR_INVALID_ARG, "muon_step: fp32 only");
  if (!(momentum >= 0.0f && momentum < 1.0f))
    return fail(CKAN_ERR_INVALID_ARG, "momentum must lie in [0, 1) (got %g)", momentum);
  if (!isfinite(lr) || !isfinite(weight_decay) || !isfinite(scale))
    return fail(CKAN_ERR_INVALID_ARG, "lr, weight_decay and scale must be finite");
  if (desc->batch == 0) return CKAN_OK;
  if (!p || !g || !buf) return fail(CKAN_ERR_INVALID_ARG, "muon_step: NULL pointer");
  if (const int rc = ortho_ws(desc, ws, ws_bytes)) return rc;
  OrthoArgs a = ortho_args(desc);
  a.p = p;
  a.g = g;
  a.buf = buf;
  a.lr = lr;
  a.momentum = momentum;
  a.decay = weight_decay;
  a.scale = scale;
  a.nesterov = nesterov != 0;
  launch_ortho(a, ws, reinterpret_cast<hipStream_t>(stream));
  return check_launch("muon_step");
}

int ckan_mixture_few(const ckan_mixture_desc* desc) {
  FewArgs a;
  return mixture_args(desc, &a) == CKAN_OK && a.few;
}

size_t ckan_mixture_workspace_bytes(const ckan_mixture_desc* desc) {
  FewArgs a;
  return mixture_args(desc, &a) || !a.few ? 0 : a.ws_bytes;
}

int ckan_mixture_forward(const ckan_mixture_desc* desc, const void* x, const void* gate, const void* coeffs,
                         const float* bias, void* y, float* weights, int64_t* indices, void* ws, size_t ws_bytes,
                         void* stream) {
  FewArgs a;
  if (const int rc = mixture_args(desc, &a)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  if (!a.few) return fail(CKAN_ERR_UNSUPPORTED, "mixture_forward: too many rows for its form, use the parts' entry points");
  if (!x || !gate || !coeffs || !y || !weights || !indices) return fail(CKAN_ERR_INVALID_ARG, "mixture_forward: NULL pointer");
  const size_t need = a.ws_bytes;
  if (ws_bytes < need) return fail(CKAN_ERR_WORKSPACE, "mixture workspace too small: %zu < %zu bytes", ws_bytes, need);
  if (!ws || !is_al16(ws)) return fail(CKAN_ERR_INVALID_ARG, "mixture_forward: workspace is NULL or not 16-byte aligned");
  if (!is_al16(x) || !is_al16(gate) || !is_al16(coeffs) || !is_al16(y))
    return fail(CKAN_ERR_INVALID_ARG, "mixture_forward: x, gate, coeffs and y must be 16-byte aligned");
  a.x = x;
  a.gate = gate;
  a.coeffs = coeffs;
  a.y = y;
  a.ws = (char*)ws;
  a.route.bias = bias;
  a.route.weights = weights;
  a.route.indices = indices;
  launch_few(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch("mixture_forward");
}

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
