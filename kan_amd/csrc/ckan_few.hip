// A whole mixture layer for few rows (ckan_mixture_forward): the gate's logits, the
// choice, the chosen experts' products and their weighted sum.
#include "ckan_mix.hpp"

namespace ckan {
namespace {

constexpr int kGateRows = 8;  // rows a pass over the gate serves

// logits[t, e] = sum_i x[t, i] gate[e, i], a wave an expert.  The products of fp32 values are
// exact in 64 bits and so, nearly, is their sum: rounded once, a logit does not depend on
// the order of the sum.
template <typename TX, typename TG>
__global__ __launch_bounds__(256) void k_few_logits(FewArgs a) {
  const int lane = threadIdx.x & 63, e = blockIdx.x * 4 + (threadIdx.x >> 6), I = a.p.I;
  if (e >= a.route.E) return;
  const TG* g = (const TG*)a.gate + (int64_t)e * I;
  const int64_t t0 = (int64_t)blockIdx.y * kGateRows;
  const int n = a.route.rows - t0 < kGateRows ? (int)(a.route.rows - t0) : kGateRows;
  double sum[kGateRows] = {};
  for (int i = lane; i < I; i += 64) {
    const double w = (double)(float)g[i];
#pragma unroll
    for (int r = 0; r < kGateRows; ++r)
      if (r < n) sum[r] = fma((double)(float)((const TX*)a.x)[(t0 + r) * I + i], w, sum[r]);
  }
#pragma unroll
  for (int r = 0; r < kGateRows; ++r) {
    double v = sum[r];
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) v += __shfl_xor(v, w);
    if (lane == 0 && r < n) ((float*)a.ws)[(t0 + r) * a.route.E + e] = (float)v;
  }
}

}  // namespace

void launch_few(const FewArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.route.E, 4), (unsigned)ceil_div(a.route.rows, kGateRows)), block(256);
  if (a.x_bf16) {
    if (a.gate_bf16)
      hipLaunchKernelGGL((k_few_logits<__bf16, __bf16>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((k_few_logits<__bf16, float>), grid, block, 0, st, a);
  } else {
    if (a.gate_bf16)
      hipLaunchKernelGGL((k_few_logits<float, __bf16>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((k_few_logits<float, float>), grid, block, 0, st, a);
  }
  RouteArgs r = a.route;
  r.logits = a.ws;
  launch_route(r, false, st);
  ExpertsArgs x{};
  x.p = a.p;
  x.x = a.x;
  x.coeffs = a.coeffs;
  x.indices = r.indices;
  x.weights = r.weights;
  x.y = a.y;
  x.ws = a.ws + few_logits_bytes(a);
  launch_experts_stream(x, a.x_bf16 != 0, st);
}

}  // namespace ckan
