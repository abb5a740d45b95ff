// Routing of rows to experts and its gradient (ckan_route, ckan_route_backward).
//
// A row of logits l[0..E) gives scores s (softmax or sigmoid), selection keys
// s + bias, optionally a choice of whole groups of experts by the sum of their
// two largest keys, the top_k largest keys among the kept groups (ties to the
// lowest index), and the chosen experts' weights.  One wave takes one row: lane
// j holds the J = ceil(E / 64) consecutive experts from j J on in registers, so
// a row is read once and the lowest index among equal keys is the lowest lane's
// lowest register.
#include "ckan_route_row.hpp"

namespace ckan {
namespace {

constexpr int kRowsPerBlock = 4;  // one wave a row

template <int J, typename T>
__device__ __forceinline__ void row_logits(const T* row, int E, int lane, float (&l)[J]) {
#pragma unroll
  for (int q = 0; q < J; ++q) {
    const int e = lane * J + q;
    const float v = (float)row[e < E ? e : E - 1];
    l[q] = e < E ? eligible_logit(v) : -INFINITY;
  }
}

template <int J, typename T>
__global__ __launch_bounds__(64 * kRowsPerBlock) void k_route(RouteArgs a) {
  extern __shared__ float sm[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + wave;
  if (row >= a.rows) return;  // no block-wide barrier below: each wave keeps to its own LDS
  float l[J];
  row_logits<J>((const T*)a.logits + row * a.ld, a.E, lane, l);
  int mine;
  float w;
  route_row<J>(a, lane, l, sm + wave * (64 * J + 64), mine, w);
  if (lane < a.top_k) {
    a.weights[row * a.top_k + lane] = w;
    a.indices[row * a.top_k + lane] = mine;
  }
}

// dlogits of a row from the chosen experts' weight gradients.  The scores are
// computed again from the logits (reading them twice costs less than keeping a
// [rows, E] tensor).  With r = sum over the chosen of s ds: softmax
// dl = s (ds - r), sigmoid dl = s (1 - s) ds, ds being 0 off the chosen.
template <int J, typename T>
__global__ __launch_bounds__(64 * kRowsPerBlock) void k_route_backward(RouteArgs a) {
  extern __shared__ float sm[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + wave;
  if (row >= a.rows) return;
  float* lds = sm + wave * (64 * J);
  float l[J], s[J];
  row_logits<J>((const T*)a.logits + row * a.ld, a.E, lane, l);
  row_scores<J>(l, a.softmax, s);
#pragma unroll
  for (int q = 0; q < J; ++q) lds[lane * J + q] = s[q];
  __builtin_amdgcn_wave_barrier();
  int64_t e = -1;
  float sj = 0.0f, dw = 0.0f;
  if (lane < a.top_k) {
    e = a.indices[row * a.top_k + lane];
    if (e >= 0 && e < a.E) {
      sj = lds[e];
      dw = a.dweights[row * a.top_k + lane];
    } else {
      e = -1;
    }
  }
  __builtin_amdgcn_wave_barrier();
  float ds, r = 0.0f;
  if (a.renormalize) {
    // ds_j = scale (dw_j - mean) / total, mean = sum w_j dw_j.  From the differences to the
    // first slot's dw: what all dw of a row share leaves no rounding, and one slot alone,
    // whose weight is 1, gets 0.  short_of_one = 1 - sum w_j, of which that share is left.
    const float own = wave_sum(sj), total = own + kRouteEps, short_of_one = total > own ? kRouteEps / total : 0.0f;
    const float base = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(dw)));
    const float diff = e >= 0 ? dw - base : 0.0f, mean = wave_sum(diff * sj) / total;
    ds = a.scale * ((diff - mean) + base * short_of_one) / total;
    r = a.scale * (mean + base * (1.0f - short_of_one)) * short_of_one;  // sum s ds
  } else {
    ds = a.scale * dw;
    r = wave_sum(sj * ds);
  }
  // the chosen experts' ds to the lanes that hold them
#pragma unroll
  for (int q = 0; q < J; ++q) lds[lane * J + q] = 0.0f;
  __builtin_amdgcn_wave_barrier();
  if (e >= 0) lds[e] = ds;
  __builtin_amdgcn_wave_barrier();
  T* out = (T*)a.dlogits + row * a.E;
#pragma unroll
  for (int q = 0; q < J; ++q) {
    const int i = lane * J + q;
    if (i >= a.E) continue;
    const float d = lds[i];
    float v;
    if (a.softmax) {
      v = s[q] * (d - r);
    } else {
      // s (1 - s) without the cancellation of 1 - s near s = 1
      const float x = expf(-fabsf(l[q]));
      v = l[q] > -INFINITY ? x / ((1.0f + x) * (1.0f + x)) * d : 0.0f;
    }
    out[i] = (T)v;
  }
}

template <typename T>
void launch_typed(const RouteArgs& a, bool backward, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.rows, kRowsPerBlock)), block(64 * kRowsPerBlock);
  const int J = (a.E + 63) / 64;
#define CKAN_ROUTE_CASE(N)                                                                     \
  if (J <= N) {                                                                                \
    const size_t lds = (size_t)kRowsPerBlock * (64 * N + (backward ? 0 : 64)) * sizeof(float); \
    if (backward)                                                                              \
      hipLaunchKernelGGL((k_route_backward<N, T>), grid, block, lds, st, a);                   \
    else                                                                                       \
      hipLaunchKernelGGL((k_route<N, T>), grid, block, a.groups > 1 ? lds : 0, st, a);         \
    return;                                                                                    \
  }
  CKAN_ROUTE_CASE(1)
  CKAN_ROUTE_CASE(2)
  CKAN_ROUTE_CASE(4)
  CKAN_ROUTE_CASE(8)
#undef CKAN_ROUTE_CASE
}

}  // namespace

void launch_route(const RouteArgs& a, bool backward, hipStream_t st) {
  if (a.bf16)
    launch_typed<__bf16>(a, backward, st);
  else
    launch_typed<float>(a, backward, st);
}

}  // namespace ckan
