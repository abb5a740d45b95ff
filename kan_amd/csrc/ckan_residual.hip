// Norms around a residual block (ckan_residual_forward, ckan_residual_backward):
//
//   u = drop(post(y)),  out = x + scale gate u,  h = next(out)
//
// with post and next a row's (v - mean) r w + b, r = 1 / sqrt(mean((v - mean)^2) + eps)
// (mean 0 in the rms form), and either of them absent.  Backward, with o^ = (out - mean) r
// and y^ likewise:
//
//   g = dh w_next,  dx = dout + r (g - o^ mean(g o^) - mean(g)),     dw_next = sum dh o^
//   dgate = scale dx u,  e = drop(scale gate dx),                    dw_post = sum e y^
//   dy = r (e w_post - y^ mean(e w_post y^) - mean(e w_post))
//
// out is made again from x and y, unrounded, so that no gradient sees its rounding: the
// same bytes as reading out.  Sums over a row and over rows are in fp32, in a fixed order.
#include "ckan_block.hpp"

namespace ckan {
namespace {

constexpr int kStats = 4;  // floats a row keeps for the backward

// ---- any width: a block a row, the row read again for every sum ------------------

constexpr int kAnyThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int w = 32; w; w >>= 1) v += __shfl_xor(v, w);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

struct RowStats {
  float m1, r1, m2, r2;
};

// One chunk of a row: u (after dropout), y^ and out's unrounded value.
template <typename TX, typename TY>
__device__ __forceinline__ uint32_t chunk_values(const ResidualArgs& a, const DropKey& key, int64_t row, int c,
                                                 const RowStats& st, float (&yh)[kChunk], float (&u)[kChunk],
                                                 float (&gate)[kChunk], float (&o)[kChunk]) {
  const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
  load8((const TX*)a.x + row * a.x_ld + at, left, o);
  uint32_t keep = 0xff;
  if (!a.y) return keep;
  load8((const TY*)a.y + row * a.y_ld + at, left, yh);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) u[i] = yh[i];
  if (a.post_w.p) {
    float w[kChunk], b[kChunk] = {};
    load8(a.post_w, at, left, w);
    if (a.post_b.p) load8(a.post_b, at, left, b);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      yh[i] = i < left ? (yh[i] - st.m1) * st.r1 : 0.0f;
      u[i] = fmaf(yh[i], w[i], b[i]);
    }
  }
  if (a.drop.on) {
    keep = drop_keep(a.drop, key, (uint32_t)row, (uint32_t)c);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) u[i] = keep >> i & 1 ? u[i] * a.drop.scale : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) gate[i] = 1.0f;
  if (a.gate.p) load8(a.gate, (a.gate_rows ? row * a.gate_ld : 0) + at, left, gate);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    gate[i] *= a.scale;
    o[i] = fmaf(gate[i], u[i], o[i]);
  }
  return keep;
}

template <typename TX, typename TY>
__global__ __launch_bounds__(kAnyThreads) void k_residual_any(ResidualArgs a) {
  __shared__ float red[kAnyThreads / 64];
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const int chunks = (a.dim + kChunk - 1) / kChunk, tid = threadIdx.x;
  const float inv = 1.0f / (float)a.dim;
  if (a.stats && a.drop.on && blockIdx.x == 0 && tid == 0) {
    int64_t* used = (int64_t*)(a.stats + a.rows * kStats);
    used[0] = a.drop.state ? a.drop.state[0] : (int64_t)a.drop.seed;
    used[1] = (int64_t)(((uint64_t)key.call1 << 32) | key.call0);
  }
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    RowStats st = {};
    float yh[kChunk], u[kChunk], gate[kChunk], o[kChunk];
    if (a.y && a.post_w.p) {
      for (int pass = a.layer ? 0 : 1; pass < 2; ++pass) {
        float sum = 0.0f;
        for (int c = tid; c < chunks; c += kAnyThreads) {
          const int64_t left = a.dim - (int64_t)c * kChunk;
          load8((const TY*)a.y + row * a.y_ld + (int64_t)c * kChunk, left, yh);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            const float d = i < left ? yh[i] - st.m1 : 0.0f;
            sum += pass ? d * d : d;
          }
        }
        sum = block_sum(sum, red) * inv;
        if (pass)
          st.r1 = 1.0f / sqrtf(sum + a.eps);
        else
          st.m1 = sum;
      }
    }
    if (a.next_w.p) {
      for (int pass = a.layer ? 0 : 1; pass < 2; ++pass) {
        float sum = 0.0f;
        for (int c = tid; c < chunks; c += kAnyThreads) {
          const int64_t left = a.dim - (int64_t)c * kChunk;
          chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            const float d = i < left ? o[i] - st.m2 : 0.0f;
            sum += pass ? d * d : d;
          }
        }
        sum = block_sum(sum, red) * inv;
        if (pass)
          st.r2 = 1.0f / sqrtf(sum + a.eps);
        else
          st.m2 = sum;
      }
    }
    for (int c = tid; c < chunks; c += kAnyThreads) {
      const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
      chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
      if (a.out) store8((TX*)a.out + row * a.dim + at, left, o);
      if (a.next_w.p) {
        float w[kChunk], b[kChunk] = {};
        load8(a.next_w, at, left, w);
        if (a.next_b.p) load8(a.next_b, at, left, b);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) o[i] = fmaf((o[i] - st.m2) * st.r2, w[i], b[i]);
        store8((TY*)a.h + row * a.dim + at, left, o);
      }
    }
    if (a.stats && tid == 0) {
      float* s = a.stats + row * kStats;
      s[0] = st.m1;
      s[1] = st.r1;
      s[2] = st.m2;
      s[3] = st.r2;
    }
  }
}

// A chunk's gradients: dx, e (the gradient of post's result) and o^.
struct RowMeans {
  float go, g, ey, e;  // mean(g o^), mean(g), mean(e w y^), mean(e w)
};

template <typename TX, typename TY>
__device__ __forceinline__ void chunk_dx(const ResidualArgs& a, int64_t row, int c, const RowStats& st, const RowMeans& mean,
                                         const float (&o)[kChunk], float (&oh)[kChunk], float (&dh)[kChunk],
                                         float (&dx)[kChunk]) {
  const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) oh[i] = dh[i] = dx[i] = 0.0f;
  if (a.dout) load8((const TX*)a.dout + row * a.dout_ld + at, left, dx);
  if (a.next_w.p && a.dh) {
    float w[kChunk];
    load8((const TY*)a.dh + row * a.dh_ld + at, left, dh);
    load8(a.next_w, at, left, w);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      oh[i] = i < left ? (o[i] - st.m2) * st.r2 : 0.0f;
      dx[i] += st.r2 * (dh[i] * w[i] - oh[i] * mean.go - mean.g);
    }
  }
}

// dx, dy and a row gate's gradient; the row's means to the workspace for the sums over rows.
template <typename TX, typename TY>
__global__ __launch_bounds__(kAnyThreads) void k_residual_any_dx(ResidualArgs a) {
  __shared__ float red[kAnyThreads / 64];
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const int chunks = (a.dim + kChunk - 1) / kChunk, tid = threadIdx.x;
  const float inv = 1.0f / (float)a.dim;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* s = a.stats + row * kStats;
    const RowStats st = {s[0], s[1], s[2], s[3]};
    RowMeans mean = {};
    float yh[kChunk], u[kChunk], gate[kChunk], o[kChunk], oh[kChunk], dh[kChunk], dx[kChunk], w[kChunk];
    if (a.next_w.p && a.dh) {
      float go = 0.0f, g = 0.0f;
      for (int c = tid; c < chunks; c += kAnyThreads) {
        chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
        chunk_dx<TX, TY>(a, row, c, st, mean, o, oh, dh, dx);
        load8(a.next_w, (int64_t)c * kChunk, a.dim - (int64_t)c * kChunk, w);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          go = fmaf(dh[i] * w[i], oh[i], go);
          g = fmaf(dh[i], w[i], g);
        }
      }
      mean.go = block_sum(go, red) * inv;
      if (a.layer) mean.g = block_sum(g, red) * inv;
    }
    const bool post = a.y && a.post_w.p;
    for (int pass = post && a.dy ? 0 : 1; pass < 2; ++pass) {
      float ey = 0.0f, e = 0.0f;
      for (int c = tid; c < chunks; c += kAnyThreads) {
        const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
        const uint32_t keep = chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
        chunk_dx<TX, TY>(a, row, c, st, mean, o, oh, dh, dx);
        if (pass && a.dx) store8((TX*)a.dx + row * a.dim + at, left, dx);
        if (!a.y) continue;
        if (pass && a.gate_rows && a.dgate) {
          float dg[kChunk];
#pragma unroll
          for (int i = 0; i < kChunk; ++i) dg[i] = a.scale * dx[i] * u[i];
          if (a.gate.bf16)
            store8((__bf16*)a.dgate + row * a.dim + at, left, dg);
          else
            store8((float*)a.dgate + row * a.dim + at, left, dg);
        }
        if (post) load8(a.post_w, at, left, w);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          float v = gate[i] * dx[i];
          if (a.drop.on) v = keep >> i & 1 ? v * a.drop.scale : 0.0f;
          if (post) {
            v *= w[i];
            ey = fmaf(v, yh[i], ey);
            e += v;
            v = st.r1 * (v - yh[i] * mean.ey - mean.e);
          }
          dx[i] = v;
        }
        if (pass && a.dy) store8((TY*)a.dy + row * a.dim + at, left, dx);
      }
      if (!pass) {
        mean.ey = block_sum(ey, red) * inv;
        if (a.layer) mean.e = block_sum(e, red) * inv;
      }
    }
    if (tid == 0) {
      a.ws[row * 2] = mean.go;
      a.ws[row * 2 + 1] = mean.g;
    }
  }
}

// Sums over rows of the parameters' gradients: a thread a column chunk, a block 64
// chunks by four rows at a time of its slab; partial sums [slab, 5, dim].
constexpr int kSums = 5;  // dpost_w, dpost_b, dgate, dnext_w, dnext_b
constexpr int kAnySlabs = 256;

template <typename TX, typename TY>
__global__ __launch_bounds__(kAnyThreads) void k_residual_any_sums(ResidualArgs a, float* part) {
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const int c = blockIdx.x * kAnyThreads + threadIdx.x;
  const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
  if (left <= 0) return;
  const int64_t per = (a.rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
  float s[kSums][kChunk] = {};
  for (int64_t row = r0; row < r1; ++row) {
    const float* q = a.stats + row * kStats;
    const RowStats st = {q[0], q[1], q[2], q[3]};
    RowMeans mean = {};
    mean.go = a.ws[row * 2];
    mean.g = a.ws[row * 2 + 1];
    float yh[kChunk], u[kChunk], gate[kChunk], o[kChunk], oh[kChunk], dh[kChunk], dx[kChunk];
    const uint32_t keep = chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
    chunk_dx<TX, TY>(a, row, c, st, mean, o, oh, dh, dx);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      s[3][i] = fmaf(dh[i], oh[i], s[3][i]);
      s[4][i] += dh[i];
      if (!a.y) continue;
      s[2][i] = fmaf(a.scale * dx[i], u[i], s[2][i]);
      float v = gate[i] * dx[i];
      if (a.drop.on) v = keep >> i & 1 ? v * a.drop.scale : 0.0f;
      s[0][i] = fmaf(v, yh[i], s[0][i]);
      s[1][i] += v;
    }
  }
  float* p = part + (int64_t)blockIdx.y * kSums * a.dim + at;
#pragma unroll
  for (int k = 0; k < kSums; ++k) store8(p + (int64_t)k * a.dim, left, s[k]);
}

// The partial sums of one column of one parameter, in order.
__global__ __launch_bounds__(256) void k_residual_sums(ResidualArgs a, const float* part, int slabs) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.y;
  void* outs[kSums] = {a.dpost_w, a.dpost_b, a.gate_rows ? nullptr : a.dgate, a.dnext_w, a.dnext_b};
  const int types[kSums] = {a.post_w.bf16, a.post_b.bf16, a.gate.bf16, a.next_w.bf16, a.next_b.bf16};
  void* out = outs[k];
  if (!out) return;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (col < a.dim)
    for (int s = wave; s < slabs; s += 4) v += part[((int64_t)s * kSums + k) * a.dim + col];
  red[wave][lane] = v;
  __syncthreads();
  if (wave || col >= a.dim) return;
  v = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
  if (types[k])
    ((__bf16*)out)[col] = (__bf16)v;
  else
    ((float*)out)[col] = v;
}

bool wants_sums(const ResidualArgs& a) {
  return a.dpost_w || a.dpost_b || a.dnext_w || a.dnext_b || (a.dgate && !a.gate_rows);
}

int any_slabs(const ResidualArgs& a) {
  const int64_t wide = ceil_div(a.dim, kChunk * kAnyThreads);
  int64_t slabs = ceil_div(4 * kNumCUs, wide);
  if (slabs > kAnySlabs) slabs = kAnySlabs;
  if (slabs > a.rows) slabs = a.rows;
  return (int)slabs;
}

template <typename TX, typename TY>
void forward_typed(const ResidualArgs& a, hipStream_t st) {
  const int64_t blocks = a.rows < 8 * kNumCUs ? a.rows : 8 * kNumCUs;
  hipLaunchKernelGGL((k_residual_any<TX, TY>), dim3((unsigned)blocks), dim3(kAnyThreads), 0, st, a);
}

template <typename TX, typename TY>
void backward_typed(const ResidualArgs& a, hipStream_t st) {
  const int64_t blocks = a.rows < 8 * kNumCUs ? a.rows : 8 * kNumCUs;
  hipLaunchKernelGGL((k_residual_any_dx<TX, TY>), dim3((unsigned)blocks), dim3(kAnyThreads), 0, st, a);
  if (!wants_sums(a)) return;
  const int slabs = any_slabs(a);
  float* part = a.ws + round_up(a.rows * 2, 4);
  hipLaunchKernelGGL((k_residual_any_sums<TX, TY>), dim3((unsigned)ceil_div(a.dim, kChunk * kAnyThreads), (unsigned)slabs),
                     dim3(kAnyThreads), 0, st, a, part);
  hipLaunchKernelGGL(k_residual_sums, dim3((unsigned)ceil_div(a.dim, 64), kSums), dim3(256), 0, st, a, part, slabs);
}

}  // namespace

size_t residual_workspace_bytes(const ResidualArgs& a) {
  return align256((round_up(a.rows * 2, 4) + (wants_sums(a) ? (int64_t)any_slabs(a) * kSums * a.dim : 0)) * sizeof(float));
}

void launch_residual_forward(const ResidualArgs& a, hipStream_t st) {
  if (a.x_bf16)
    a.y_bf16 ? forward_typed<__bf16, __bf16>(a, st) : forward_typed<__bf16, float>(a, st);
  else
    a.y_bf16 ? forward_typed<float, __bf16>(a, st) : forward_typed<float, float>(a, st);
}

void launch_residual_backward(const ResidualArgs& a, hipStream_t st) {
  if (a.x_bf16)
    a.y_bf16 ? backward_typed<__bf16, __bf16>(a, st) : backward_typed<__bf16, float>(a, st);
  else
    a.y_bf16 ? backward_typed<float, __bf16>(a, st) : backward_typed<float, float>(a, st);
}

}  // namespace ckan
