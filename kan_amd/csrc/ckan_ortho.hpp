// What the orthogonalisation kernels share: addressing a matrix, what enters the
// iteration and where its results go.
#pragma once

#include "ckan_mix.hpp"

namespace ckan {

__device__ __forceinline__ int64_t view_at(const MatView& v, int b, int r, int c) {
  const int q = v.inner == 1 ? c : c / v.inner;
  return b * v.sb + r * v.sr + q * v.so + (v.inner == 1 ? 0 : (c - q * v.inner) * v.si);
}

// The matrix entry that enters the iteration: the input, or Muon's update
// direction from the gradient and the (already updated) momentum.
__device__ __forceinline__ float muon_dir(float g, float buf, const OrthoArgs& a) {
  return a.nesterov ? fmaf(a.momentum, buf, (1.0f - a.momentum) * g) : buf;
}
__device__ __forceinline__ float entry(const OrthoArgs& a, int64_t at) {
  if (!a.in) return muon_dir(a.g[at], a.buf[at], a);
  return a.bf16 ? (float)((const __bf16*)a.in)[at] : ((const float*)a.in)[at];
}

// Muon's parameter from its old value and the update.
__device__ __forceinline__ float muon_param(const OrthoArgs& a, float old, float o) {
  return fmaf(-a.lr * a.scale, o, old * (1.0f - a.lr * a.decay));
}
__device__ __forceinline__ void put(const OrthoArgs& a, int64_t e, float o) {
  if (!a.in)
    a.p[e] = muon_param(a, a.p[e], o);
  else if (a.bf16)
    ((__bf16*)a.out)[e] = (__bf16)o;
  else
    ((float*)a.out)[e] = o;
}

// Whether memory runs along m: the columns of a tall matrix in row-major order, the
// rows of a wide one in column-major order.
__device__ __forceinline__ bool runs_along_m(const OrthoArgs& a) {
  return (a.rows > a.cols) == (a.view.so == 1 || a.view.inner != 1);
}

}  // namespace ckan
