// C-ABI entry points of the residual-block, dropout and log-probability operators
// (include/chebykan.h): argument checks on the host, then the launches on the caller's
// stream.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "chebykan.h"
#include "ckan_block.hpp"

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

bool known_dtype(int d) { return d == CKAN_DTYPE_F32 || d == CKAN_DTYPE_BF16; }

// An address that elements of the type may have.
bool aligned_to(const void* p, int dtype) { return ((uintptr_t)p & (dtype == CKAN_DTYPE_BF16 ? 1 : 3)) == 0; }

int drop_args(double p, uint64_t seed, uint64_t offset, const int64_t* state, DropArgs* d) {
  if (!(p >= 0.0 && p <= 1.0)) return fail(CKAN_ERR_INVALID_ARG, "the dropout probability must lie in [0, 1] (got %g)", p);
  if ((uintptr_t)state & 7) return fail(CKAN_ERR_INVALID_ARG, "the dropout state must be 8-byte aligned");
  const uint64_t threshold = (uint64_t)nearbyint(p * 4294967296.0);
  const uint32_t high = (uint32_t)(threshold >> 16);
  *d = DropArgs{state, seed, offset, high, (uint32_t)(threshold & 0xffff), high && !(high >> 16) ? high : 1,
                p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f, p > 0.0, (int)(high >> 16)};
  return CKAN_OK;
}

int residual_check(const ckan_residual_desc* d) {
  if (!d) return fail(CKAN_ERR_INVALID_ARG, "residual desc is NULL");
  if (d->rows < 0) return fail(CKAN_ERR_INVALID_ARG, "rows must be >= 0 (got %lld)", (long long)d->rows);
  if (d->rows >= kDropMaxRows) return fail(CKAN_ERR_UNSUPPORTED, "2^32 rows or more are not supported");
  if (d->dim < 1) return fail(CKAN_ERR_INVALID_ARG, "dim must be >= 1 (got %d)", d->dim);
  if (d->dim > kResMaxDim) return fail(CKAN_ERR_UNSUPPORTED, "dim above 2^20 is not supported (got %d)", d->dim);
  for (const int t : {d->x_dtype, d->y_dtype, d->gate_dtype, d->post_weight_dtype, d->post_bias_dtype, d->next_weight_dtype,
                      d->next_bias_dtype})
    if (!known_dtype(t)) return fail(CKAN_ERR_INVALID_ARG, "unknown dtype %d", t);
  if (d->norm != CKAN_NORM_RMS && d->norm != CKAN_NORM_LAYER) return fail(CKAN_ERR_INVALID_ARG, "unknown norm %d", d->norm);
  if (d->gate_rows != 0 && d->gate_rows != 1) return fail(CKAN_ERR_INVALID_ARG, "gate_rows must be 0 or 1");
  if (!(d->eps >= 0.0f) || !isfinite(d->eps) || !isfinite(d->scale))
    return fail(CKAN_ERR_INVALID_ARG, "eps and scale must be finite, eps >= 0");
  for (const int64_t ld : {d->x_ld, d->y_ld, d->gate_ld})
    if (ld < 0) return fail(CKAN_ERR_INVALID_ARG, "row pitches must be >= 0");
  return CKAN_OK;
}

int residual_args(const ckan_residual_desc* d, const ckan_residual_buffers* b, bool backward, ResidualArgs* a) {
  if (const int rc = residual_check(d)) return rc;
  if (!b) return fail(CKAN_ERR_INVALID_ARG, "residual buffers are NULL");
  *a = ResidualArgs{};
  if (const int rc = drop_args(d->dropout, b->dropout_seed, b->dropout_offset, b->dropout_state, &a->drop)) return rc;
  if (d->rows == 0) return CKAN_OK;
  if (!b->x) return fail(CKAN_ERR_INVALID_ARG, "residual: x is NULL");
  if (backward && (b->dout_ld < 0 || b->dh_ld < 0)) return fail(CKAN_ERR_INVALID_ARG, "row pitches must be >= 0");
  if (!b->y && (b->gate || b->post_weight || b->dout || d->dropout > 0.0))
    return fail(CKAN_ERR_INVALID_ARG, "residual: without y there is no gate, post norm, dropout or out");
  if (!b->y && !b->next_weight) return fail(CKAN_ERR_INVALID_ARG, "residual: neither y nor next_weight");
  if ((b->post_bias && !b->post_weight) || (b->next_bias && !b->next_weight))
    return fail(CKAN_ERR_INVALID_ARG, "residual: a norm's bias without its weight");
  if (!backward && ((b->y && !b->out) || (b->next_weight && !b->h)))
    return fail(CKAN_ERR_INVALID_ARG, "residual_forward: out or h is NULL");
  if (!backward && ((!b->y && b->out) || (!b->next_weight && b->h)))
    return fail(CKAN_ERR_INVALID_ARG, "residual_forward: out without y, or h without next_weight");
  if (backward && !b->stats) return fail(CKAN_ERR_INVALID_ARG, "residual_backward: stats is NULL");
  if (b->dh && !b->next_weight) return fail(CKAN_ERR_INVALID_ARG, "residual_backward: dh without next_weight");
  if (!is_al16(b->stats)) return fail(CKAN_ERR_INVALID_ARG, "residual: stats must be 16-byte aligned");
  const struct { const void* p; int dtype; const char* name; } typed[] = {
      {b->x, d->x_dtype, "x"}, {b->out, d->x_dtype, "out"}, {b->dout, d->x_dtype, "dout"}, {b->dx, d->x_dtype, "dx"},
      {b->y, d->y_dtype, "y"}, {b->h, d->y_dtype, "h"}, {b->dh, d->y_dtype, "dh"}, {b->dy, d->y_dtype, "dy"},
      {b->gate, d->gate_dtype, "gate"}, {b->dgate, d->gate_dtype, "dgate"},
      {b->post_weight, d->post_weight_dtype, "post_weight"}, {b->dpost_weight, d->post_weight_dtype, "dpost_weight"},
      {b->post_bias, d->post_bias_dtype, "post_bias"}, {b->dpost_bias, d->post_bias_dtype, "dpost_bias"},
      {b->next_weight, d->next_weight_dtype, "next_weight"}, {b->dnext_weight, d->next_weight_dtype, "dnext_weight"},
      {b->next_bias, d->next_bias_dtype, "next_bias"}, {b->dnext_bias, d->next_bias_dtype, "dnext_bias"}};
  for (const auto& t : typed)
    if (!aligned_to(t.p, t.dtype)) return fail(CKAN_ERR_INVALID_ARG, "residual: %s is not aligned to its elements", t.name);
  // a wanted gradient needs what it is the gradient of
  if ((b->dy && !b->y) || (b->dgate && !b->gate) || (b->dpost_weight && !b->post_weight) || (b->dpost_bias && !b->post_bias) ||
      (b->dnext_weight && !b->next_weight) || (b->dnext_bias && !b->next_bias))
    return fail(CKAN_ERR_INVALID_ARG, "residual_backward: the gradient of an absent input is wanted");
  a->rows = d->rows;
  a->x_ld = d->x_ld;
  a->y_ld = d->y_ld;
  a->gate_ld = d->gate_ld;
  a->dout_ld = b->dout_ld;
  a->dh_ld = b->dh_ld;
  a->dim = d->dim;
  a->x_bf16 = d->x_dtype == CKAN_DTYPE_BF16;
  a->y_bf16 = d->y_dtype == CKAN_DTYPE_BF16;
  a->layer = d->norm == CKAN_NORM_LAYER;
  a->gate_rows = d->gate_rows && b->gate;  // a NULL gate is 1 in either form
  a->eps = d->eps;
  a->scale = d->scale;
  a->x = b->x;
  a->y = b->y;
  a->gate = AnyPtr{b->gate, d->gate_dtype == CKAN_DTYPE_BF16};
  a->post_w = AnyPtr{b->post_weight, d->post_weight_dtype == CKAN_DTYPE_BF16};
  a->post_b = AnyPtr{b->post_bias, d->post_bias_dtype == CKAN_DTYPE_BF16};
  a->next_w = AnyPtr{b->next_weight, d->next_weight_dtype == CKAN_DTYPE_BF16};
  a->next_b = AnyPtr{b->next_bias, d->next_bias_dtype == CKAN_DTYPE_BF16};
  a->stats = (float*)b->stats;
  if (!backward) {
    a->out = b->out;
    a->h = b->h;
    return CKAN_OK;
  }
  // the forward's seed and call
  if (a->drop.on) a->drop.state = (const int64_t*)(a->stats + a->rows * 4);
  a->drop.offset = 0;
  a->dout = b->dout;
  a->dh = b->dh;
  a->dx = b->dx;
  a->dy = b->dy;
  a->dgate = b->dgate;
  a->dpost_w = b->dpost_weight;
  a->dpost_b = b->dpost_bias;
  a->dnext_w = b->dnext_weight;
  a->dnext_b = b->dnext_bias;
  return CKAN_OK;
}

// The workspace of a backward that wants every gradient.
size_t residual_ws(const ckan_residual_desc* d) {
  ResidualArgs a{};
  a.rows = d->rows;
  a.dim = d->dim;
  a.x_bf16 = d->x_dtype == CKAN_DTYPE_BF16;
  a.y_bf16 = d->y_dtype == CKAN_DTYPE_BF16;
  a.dnext_w = &a;
  return residual_workspace_bytes(a);
}

int logp_check(const ckan_log_probs_desc* d) {
  if (!d) return fail(CKAN_ERR_INVALID_ARG, "log_probs desc is NULL");
  if (d->rows < 0) return fail(CKAN_ERR_INVALID_ARG, "rows must be >= 0 (got %lld)", (long long)d->rows);
  if (d->rows >= (int64_t)1 << 31) return fail(CKAN_ERR_UNSUPPORTED, "2^31 rows or more are not supported");
  if (d->classes < 1) return fail(CKAN_ERR_INVALID_ARG, "classes must be >= 1 (got %d)", d->classes);
  if (d->classes > 1 << 30) return fail(CKAN_ERR_UNSUPPORTED, "classes above 2^30 are not supported (got %d)", d->classes);
  if (d->top < 0 || d->top > d->classes)
    return fail(CKAN_ERR_INVALID_ARG, "top must lie in [0, %d] (got %d)", d->classes, d->top);
  if (d->top > kLogpMaxTop) return fail(CKAN_ERR_UNSUPPORTED, "top above %d is not supported (got %d)", kLogpMaxTop, d->top);
  if (!known_dtype(d->dtype)) return fail(CKAN_ERR_INVALID_ARG, "unknown dtype %d", d->dtype);
  if (d->logits_ld < 0) return fail(CKAN_ERR_INVALID_ARG, "logits_ld must be >= 0");
  return CKAN_OK;
}

LogpArgs logp_args(const ckan_log_probs_desc* d) {
  LogpArgs a{};
  a.rows = d->rows;
  a.ld = d->logits_ld;
  a.classes = d->classes;
  a.top = d->top;
  a.bf16 = d->dtype == CKAN_DTYPE_BF16;
  return a;
}

}  // namespace

extern "C" {

size_t ckan_residual_stats_bytes(const ckan_residual_desc* desc) {
  return residual_check(desc) ? 0 : (size_t)desc->rows * 16 + 16;
}

size_t ckan_residual_workspace_bytes(const ckan_residual_desc* desc) {
  return residual_check(desc) || desc->rows == 0 ? 0 : residual_ws(desc);
}

int ckan_residual_forward(const ckan_residual_desc* desc, const ckan_residual_buffers* buffers, void* stream) {
  ResidualArgs a;
  if (const int rc = residual_args(desc, buffers, false, &a)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  launch_residual_forward(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch("residual_forward");
}

int ckan_residual_backward(const ckan_residual_desc* desc, const ckan_residual_buffers* buffers, void* ws,
                           size_t ws_bytes, void* stream) {
  ResidualArgs a;
  if (const int rc = residual_args(desc, buffers, true, &a)) return rc;
  if (desc->rows == 0) {
    if (buffers->dpost_weight || buffers->dpost_bias || buffers->dnext_weight || buffers->dnext_bias ||
        (buffers->dgate && !desc->gate_rows))
      return fail(CKAN_ERR_INVALID_ARG, "residual_backward: no rows, the caller fills the parameters' gradients with zeros");
    return CKAN_OK;
  }
  const size_t need = residual_ws(desc);
  if (ws_bytes < need) return fail(CKAN_ERR_WORKSPACE, "residual backward workspace too small: %zu < %zu bytes", ws_bytes, need);
  if (!ws || !is_al16(ws)) return fail(CKAN_ERR_INVALID_ARG, "residual_backward: workspace is NULL or not 16-byte aligned");
  a.ws = (float*)ws;
  launch_residual_backward(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch("residual_backward");
}

int ckan_dropout(const ckan_dropout_desc* desc, const int64_t* state, const void* x, void* y, int64_t* used,
                 void* stream) {
  if (!desc) return fail(CKAN_ERR_INVALID_ARG, "dropout desc is NULL");
  if (desc->rows < 0 || desc->dim < 1 || desc->x_ld < 0)
    return fail(CKAN_ERR_INVALID_ARG, "rows and x_ld must be >= 0, dim >= 1 (got %lld, %lld, %lld)", (long long)desc->rows,
                (long long)desc->x_ld, (long long)desc->dim);
  if (desc->rows >= kDropMaxRows || desc->dim > kDropMaxDim)
    return fail(CKAN_ERR_UNSUPPORTED, "2^32 rows or more, or rows above 2^34 values, are not supported");
  if (!known_dtype(desc->dtype)) return fail(CKAN_ERR_INVALID_ARG, "unknown dtype %d", desc->dtype);
  DropoutArgs a{};
  if (const int rc = drop_args(desc->p, desc->seed, desc->offset, state, &a.drop)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  if (!x || !y) return fail(CKAN_ERR_INVALID_ARG, "dropout: NULL pointer");
  if (!aligned_to(x, desc->dtype) || !aligned_to(y, desc->dtype) || ((uintptr_t)used & 7))
    return fail(CKAN_ERR_INVALID_ARG, "dropout: a buffer is not aligned to its elements");
  a.x = x;
  a.y = y;
  a.rows = desc->rows;
  a.dim = desc->dim;
  a.ld = desc->x_ld;
  a.bf16 = desc->dtype == CKAN_DTYPE_BF16;
  a.used = used;
  launch_dropout(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch("dropout");
}

size_t ckan_log_probs_workspace_bytes(const ckan_log_probs_desc* desc) {
  return logp_check(desc) || desc->rows == 0 ? 0 : logprobs_workspace_bytes(logp_args(desc));
}

int ckan_log_probs(const ckan_log_probs_desc* desc, const void* logits, const int64_t* targets, float* logp,
                   float* entropy, float* top_logp, int64_t* top_indices, float* stats, void* ws, size_t ws_bytes,
                   void* stream) {
  if (const int rc = logp_check(desc)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  if (!logits || !targets || !logp || !entropy) return fail(CKAN_ERR_INVALID_ARG, "log_probs: NULL pointer");
  if (desc->top && (!top_logp || !top_indices)) return fail(CKAN_ERR_INVALID_ARG, "log_probs: top_logp or top_indices is NULL");
  if (!aligned_to(logits, desc->dtype)) return fail(CKAN_ERR_INVALID_ARG, "log_probs: logits are not aligned to their elements");
  LogpArgs a = logp_args(desc);
  const size_t need = logprobs_workspace_bytes(a);
  if (ws_bytes < need) return fail(CKAN_ERR_WORKSPACE, "log_probs workspace too small: %zu < %zu bytes", ws_bytes, need);
  if (need && (!ws || !is_al16(ws))) return fail(CKAN_ERR_INVALID_ARG, "log_probs: workspace is NULL or not 16-byte aligned");
  a.logits = logits;
  a.targets = targets;
  a.logp = logp;
  a.entropy = entropy;
  a.top_logp = top_logp;
  a.top_idx = top_indices;
  a.stats = stats;
  a.ws = (char*)ws;
  launch_logprobs(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch("log_probs");
}

int ckan_log_probs_backward(const ckan_log_probs_desc* desc, const void* logits, const int64_t* targets,
                            const float* stats, const float* dlogp, const float* dentropy, void* dlogits, void* stream) {
  if (const int rc = logp_check(desc)) return rc;
  if (desc->rows == 0) return CKAN_OK;
  if (!logits || !targets || !stats || !dlogits) return fail(CKAN_ERR_INVALID_ARG, "log_probs_backward: NULL pointer");
  if (!aligned_to(logits, desc->dtype) || !aligned_to(dlogits, desc->dtype))
    return fail(CKAN_ERR_INVALID_ARG, "log_probs_backward: logits or dlogits are not aligned to their elements");
  LogpArgs a = logp_args(desc);
  a.logits = logits;
  a.targets = targets;
  a.stats = const_cast<float*>(stats);
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  a.dlogits = dlogits;
  launch_logprobs_backward(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch("log_probs_backward");
}

}  // extern "C"
