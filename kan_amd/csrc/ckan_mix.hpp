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

// ---- orthogonalisation (ckan_ortho.hip) ---------------------------------------
// A batch of matrices in memory: element (r, c) of matrix b lies at
// b sb + r sr + (c / inner) so + (c % inner) si.  inner = 1 is an ordinary
// strided matrix; a ChebyKAN layer's [in, out, D] coefficients as the matrix
// [out, in D] have inner = D, sr = D, so = out D, si = 1.
struct MatView {
  int64_t sb, sr, so, si;
  int inner;
};

struct OrthoArgs {
  int batch, rows, cols;
  int steps;
  float a, b, c, eps;
  int bf16;            // element type of in and out (orthogonalize)
  MatView view;        // of in, out / of p, g, buf
  const void* in;      // orthogonalize: the matrices
  void* out;
  float *p, *buf;      // Muon step (in == nullptr): all fp32, one view
  const float* g;
  float lr, momentum, decay, scale;
  int nesterov;
};
size_t ortho_workspace_bytes(int batch, int rows, int cols);
void launch_ortho(const OrthoArgs& a, void* ws, hipStream_t st);

}  // namespace ckan
