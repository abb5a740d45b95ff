// Routing of one row by one wave: scores, choice and weights from the row's logits in
// registers.
#pragma once

#include <float.h>
#include <math.h>

#include "ckan_mix.hpp"

namespace ckan {

// The scores of a row in registers: s[q] of expert lane * J + q, 0 for an
// expert that is not eligible (logit -inf or NaN) or past E.  The softmax's
// exponentials are summed in 64 bits and the sum rounded once to 32: the score
// of an expert then does not depend on the order of the sum, and keys that are
// near one another compare the same way wherever the row is computed.
template <int J>
__device__ __forceinline__ void row_scores(const float (&l)[J], int softmax, float (&s)[J]) {
  if (softmax) {
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < J; ++q) m = fmaxf(m, l[q]);
    m = fmaxf(wave_max(m), -FLT_MAX);
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < J; ++q) {
      s[q] = expf(l[q] - m);
      sum += (double)s[q];
    }
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) sum += __shfl_xor(sum, w);
    const float total = (float)sum;
#pragma unroll
    for (int q = 0; q < J; ++q) s[q] = total > 0.0f ? s[q] / total : 0.0f;
  } else {
#pragma unroll
    for (int q = 0; q < J; ++q) s[q] = 1.0f / (1.0f + expf(-l[q]));
  }
}

// A logit as the choice takes it. NaN: not eligible; +inf as the largest finite value, so that the
// row's scores are the limit (all weight on it) and not NaN.
__device__ __forceinline__ float eligible_logit(float v) { return v > -INFINITY ? fminf(v, FLT_MAX) : -INFINITY; }

// What follows the logits: l[q] is that of expert lane * J + q, -inf where the expert is not
// eligible. `keys` is LDS of the wave's own (64 J + 64 floats), touched with groups only. Lane j
// gets the j-th chosen expert (-1: none) and its weight.
template <int J>
__device__ __forceinline__ void route_row(const RouteArgs& a, int lane, const float (&l)[J], float* keys, int& mine, float& w) {
  float s[J], key[J];
  row_scores<J>(l, a.softmax, s);
#pragma unroll
  for (int q = 0; q < J; ++q) {
    const int e = lane * J + q;
    const float k = a.bias ? s[q] + a.bias[e < a.E ? e : a.E - 1] : s[q];
    key[q] = l[q] > -INFINITY && k > -INFINITY ? k : -INFINITY;  // nor with a NaN bias
  }
  if (a.groups > 1) {
    // lane (g, u) of LG lanes a group takes every LG-th key of group g for the
    // group's two largest, then the lanes of a group merge theirs
    float* kept = keys + 64 * J;
#pragma unroll
    for (int q = 0; q < J; ++q) keys[lane * J + q] = key[q];
    __builtin_amdgcn_wave_barrier();
    const int G = a.groups, size = a.E / G, LG = 1 << a.lanes_log2;
    const int g = lane >> a.lanes_log2, u = lane & (LG - 1);
    float b1 = -INFINITY, b2 = -INFINITY;
    if (g < G)
      for (int e = u; e < size; e += LG) {
        const float k = keys[g * size + e];
        b2 = fmaxf(b2, fminf(b1, k));
        b1 = fmaxf(b1, k);
      }
    for (int w = 1; w < LG; w <<= 1) {
      const float o1 = __shfl_xor(b1, w), o2 = __shfl_xor(b2, w);
      b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
      b1 = fmaxf(b1, o1);
    }
    const float value = b1 + (b2 > -INFINITY ? b2 : 0.0f);
    int ahead = 0;  // groups before this one in the order of the choice
    for (int h = 0; h < G; ++h) {
      const float v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(value), h * LG));
      ahead += v > value || (v == value && h < g);
    }
    if (g < G && u == 0) kept[g] = ahead < a.top_groups ? 1.0f : 0.0f;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < J; ++q) {
      const int e = lane * J + q;
      if (e < a.E && kept[(int)(((float)e + 0.5f) * a.inv_size)] == 0.0f) key[q] = -INFINITY;
    }
  }
  // top_k rounds: the largest key left, then its lowest index
  mine = -1;
  float chosen = 0.0f;
  for (int j = 0; j < a.top_k; ++j) {
    float own = key[0];
#pragma unroll
    for (int q = 1; q < J; ++q) own = fmaxf(own, key[q]);
    const float best = wave_max(own);
    if (!(best > -INFINITY)) break;  // uniform: no eligible expert is left
    // the lowest lane that holds it, and its lowest register
    const int from = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(own == best)) - 1);
    int at = J - 1;
    float score = s[J - 1];
#pragma unroll
    for (int q = J - 2; q >= 0; --q) {
      const bool here = key[q] == best;
      at = here ? q : at;
      score = here ? s[q] : score;
    }
    at = __builtin_amdgcn_readlane(at, from);
    score = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(score), from));
    mine = lane == j ? from * J + at : mine;
    chosen = lane == j ? score : chosen;
#pragma unroll
    for (int q = 0; q < J; ++q) key[q] = lane == from && q == at ? -INFINITY : key[q];
  }
  w = chosen;
  if (a.renormalize) w = chosen / (wave_sum(chosen) + kRouteEps);
  if (a.scale != 1.0f) w *= a.scale;
}

}  // namespace ckan
