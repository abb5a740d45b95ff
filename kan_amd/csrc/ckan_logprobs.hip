// Log probabilities of given classes, entropies and the likeliest classes of rows of
// logits (ckan_log_probs), and the gradient (ckan_log_probs_backward).
//
// One pass over a row keeps four numbers: the largest logit m so far, how many equal it
// (n), the sum s of e = exp(l - m) over the others and a = sum e (l - m).  They give
//   log Z - m = log n + log1p(s / n),   log p_t = (l_t - m) - (log Z - m),
//   H = -sum p log p = (log Z - m) - a / (n + s).
// The largest apart from the rest keeps both exact in rows that are sure of one class,
// where 1 + s would round to 1.  A logit of -inf has no probability; with d = l - m held
// above kFar its products stay 0 instead of 0 inf.  The gradient of a row is
//   dl_j = dlogp (delta_jt - p_j) - dH p_j (log p_j + H).
#include "ckan_block.hpp"
#include "ckan_mix.hpp"

namespace ckan {
namespace {

constexpr float kFar = -200.0f;  // exp(kFar) is 0 in fp32
constexpr float kLog2e = 1.44269504088896341f;

struct RowSum {
  float m, n, s, a;
};
__device__ __forceinline__ RowSum empty_sum() { return {-FLT_MAX, 0.0f, 0.0f, 0.0f}; }

// exp(d) in two instructions: off by |d| 2^-24 or so, which sums weighted by it do not see.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }
// A probability that is a result's own factor: as exact as its type.
__device__ __forceinline__ float prob_of(float d, float) { return expf(d); }
__device__ __forceinline__ float prob_of(float d, __bf16) { return exp_of(d); }

// The sums with their largest moved up to m (NaN logits never move it, but leave s NaN).
__device__ __forceinline__ void raise(RowSum& r, float m) {
  const float d = r.m - m, c = exp_of(d);
  const float all = r.n + r.s;
  const bool same = r.m == m;
  r.a = same ? r.a : c * fmaf(all, fmaxf(d, kFar), r.a);
  r.s = same ? r.s : c * all;
  r.n = same ? r.n : 0.0f;
  r.m = m;
}
__device__ __forceinline__ RowSum merged(RowSum x, RowSum y) {
  const float m = fmaxf(x.m, y.m);
  raise(x, m);
  raise(y, m);
  return {m, x.n + y.n, x.s + y.s, x.a + y.a};
}
template <int N>
__device__ __forceinline__ void add_logits(RowSum& r, const float (&l)[N]) {
  float m = r.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, l[i]);
  raise(r, m);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = l[i] - m, e = exp_of(d);
    const bool top = l[i] == m;
    r.n += top ? 1.0f : 0.0f;
    r.s += top ? 0.0f : e;
    r.a = fmaf(e, fmaxf(d, kFar), r.a);
  }
}

// What a row's sums say: its shift, log of the sum and entropy.
struct RowResult {
  float m, logs, entropy;
  bool empty;
};
__device__ __forceinline__ RowResult row_result(const RowSum& r) {
  RowResult q;
  q.empty = r.n == 0.0f && r.s == 0.0f;  // nothing above -inf (a NaN leaves s NaN)
  q.m = r.m;
  q.logs = q.empty ? INFINITY : logf(r.n) + log1pf(r.s / r.n);
  if ((r.n == 0.0f && !q.empty) || r.m == INFINITY) q.logs = NAN;  // NaN alone, or +inf
  q.entropy = q.empty ? 0.0f : q.logs - r.a / (r.n + r.s);
  return q;
}

// ---- the likeliest classes ---------------------------------------------------------
// A logit's place in the order: larger first, equal ones by the lower index; 0 for what
// is never chosen (-inf, NaN).
__device__ __forceinline__ uint64_t top_key(float l, uint32_t index) {
  if (!(l > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(l + 0.0f);  // -0 and 0 are equal
  return (uint64_t)(b ^ (b >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int w = 32; w; w >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, w);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ void write_row(const LogpArgs& a, int64_t row, const RowResult& r) {
  const int64_t t = a.targets[row];
  float logp = 0.0f;
  if (t >= 0 && t < a.classes) {
    const float l = a.bf16 ? (float)((const __bf16*)a.logits)[row * a.ld + t] : ((const float*)a.logits)[row * a.ld + t];
    logp = r.empty ? -INFINITY : (l - r.m) - r.logs;
  }
  a.logp[row] = logp;
  a.entropy[row] = r.entropy;
  if (a.stats) {
    a.stats[row * 3] = r.m;
    a.stats[row * 3 + 1] = r.logs;
    a.stats[row * 3 + 2] = r.entropy;
  }
}
__device__ __forceinline__ void write_top(const LogpArgs& a, int64_t row, int j, uint64_t key, const RowResult& r) {
  a.top_logp[row * a.top + j] = key ? (key_logit(key) - r.m) - r.logs : -INFINITY;
  a.top_idx[row * a.top + j] = key ? (int64_t)key_index(key) : -1;
}

constexpr int kThreads = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprobs_any(LogpArgs a) {
  __shared__ RowSum sums[kThreads / 64];
  __shared__ uint64_t best[kThreads / 64];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
  const T* l = (const T*)a.logits + row * a.ld;
  RowSum r = empty_sum();
  for (int64_t c = (int64_t)tid * kChunk; c < a.classes; c += kThreads * kChunk) {
    float v[kChunk];
    load8(l + c, a.classes - c, v);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = c + i < a.classes ? v[i] : -INFINITY;
    add_logits(r, v);
  }
#pragma unroll
  for (int w = 1; w < 64; w <<= 1)
    r = merged(r, RowSum{__shfl_xor(r.m, w), __shfl_xor(r.n, w), __shfl_xor(r.s, w), __shfl_xor(r.a, w)});
  if (lane == 0) sums[wave] = r;
  __syncthreads();
  r = sums[0];
  for (int w = 1; w < kThreads / 64; ++w) r = merged(r, sums[w]);
  const RowResult q = row_result(r);
  if (tid == 0) write_row(a, row, q);
  uint64_t last = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    uint64_t mine = 0;
    for (int c = tid; c < a.classes; c += kThreads) {
      const uint64_t k = top_key((float)l[c], c);
      mine = k < last && k > mine ? k : mine;
    }
    mine = wave_max64(mine);
    __syncthreads();
    if (lane == 0) best[wave] = mine;
    __syncthreads();
    last = best[0];
    for (int w = 1; w < kThreads / 64; ++w) last = best[w] > last ? best[w] : last;
    if (tid == 0) write_top(a, row, j, last, q);
  }
  __syncthreads();
  }
}

// ---- gradient ------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprobs_backward(LogpArgs a) {
  const int64_t chunks = ((int64_t)a.classes + kChunk - 1) / kChunk;
  for (int64_t row = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row < a.rows; row += (int64_t)gridDim.y * blockDim.y) {
    const float m = a.stats[row * 3], logs = a.stats[row * 3 + 1], H = a.stats[row * 3 + 2];
    const int64_t t = a.targets[row];
    // a row without any class has no gradient
    const bool has = t >= 0 && t < a.classes && logs != INFINITY;
    const float g = has && a.dlogp ? a.dlogp[row] : 0.0f, dH = a.dentropy ? a.dentropy[row] : 0.0f;
    const T* l = (const T*)a.logits + row * a.ld;
    T* out = (T*)a.dlogits + row * (int64_t)a.classes;
    for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < chunks; c += (int64_t)gridDim.x * blockDim.x) {
      float v[kChunk];
      const int64_t at = c * kChunk, left = a.classes - at;
      load8(l + at, left, v);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const float lp = (v[i] - m) - logs, p = prob_of(lp, T());
        v[i] = -p * fmaf(dH, fmaxf(lp, kFar) + H, g);
        // 1 - p without its cancellation near p = 1
        if (has && at + i == t) v[i] = -fmaf(p * dH, fmaxf(lp, kFar) + H, g * expm1f(lp));
      }
      store8(out + at, left, v);
    }
  }
}

}  // namespace

size_t logprobs_workspace_bytes(const LogpArgs&) { return 0; }

void launch_logprobs(const LogpArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows < 65536 ? a.rows : 65536));
  if (a.bf16)
    hipLaunchKernelGGL((k_logprobs_any<__bf16>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((k_logprobs_any<float>), grid, dim3(kThreads), 0, st, a);
}

void launch_logprobs_backward(const LogpArgs& a, hipStream_t st) {
  const int64_t chunks = ceil_div(a.classes, kChunk);
  int lanes = kThreads;
  while (lanes > 1 && lanes / 2 >= chunks) lanes /= 2;
  const dim3 block(lanes, kThreads / lanes);
  const int64_t gx = ceil_div(chunks, lanes), gy = ceil_div(a.rows, block.y);
  const dim3 grid((unsigned)(gx < 4096 ? gx : 4096), (unsigned)(gy < 65535 ? gy : 65535));
  if (a.bf16)
    hipLaunchKernelGGL((k_logprobs_backward<__bf16>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((k_logprobs_backward<float>), grid, block, 0, st, a);
}

}  // namespace ckan
