// Orthogonalisation of matrices with a side m <= 64, in 64 bits and three launches.
//
// With G = [m, n] (transposed where rows < cols fails), every iterate is Q_s G, Q_s a
// polynomial in A = G G^T / |G|^2, and |G|^2 is the trace of G G^T:
//   1. G G^T in parts of n (and Muon's momentum on the way: each entry is read once),
//   2. one workgroup a matrix sums the parts, scales by the trace and iterates
//        P = a I + b A + c A^2,  Q <- Q P,  A <- P A P
//      on 64 x 64 matrices in LDS,
//   3. Q G, to where it belongs.
// In fp32 this form loses the small singular values (their error grows by 3.4^2 a step);
// in fp64 it is exact to fp32's last bits, and at these sizes the fp64 matrix
// instructions cost less than the launches they save: [64, 3920] took 20 launches and
// 167 us step by step.  What bounds it: step 2, 17 dependent products on one CU.
#include "ckan_ortho.hpp"

namespace ckan {
namespace {

typedef __attribute__((ext_vector_type(4))) double f64x4_t;
constexpr int kM = 64, kTiles = 10;  // 16 x 16 tiles on and below the diagonal
constexpr int kPitch = 68;           // of the LDS matrices: a fragment's 16 rows x 4 k on distinct banks
constexpr int kMaxChunks = 32;

struct SmallPlan {
  int m, n, chunks, chunk_cols;
  size_t part_off, q_off, bytes;
};
SmallPlan make_small_plan(int batch, int rows, int cols) {
  SmallPlan p{};
  p.m = rows < cols ? rows : cols;
  p.n = rows < cols ? cols : rows;
  p.chunk_cols = (int)round_up(ceil_div(p.n, kMaxChunks), 64);
  p.chunks = (int)ceil_div(p.n, p.chunk_cols);
  p.part_off = 0;
  p.q_off = align256((size_t)batch * p.chunks * kTiles * 256 * sizeof(double));
  p.bytes = p.q_off + align256((size_t)batch * kM * kM * sizeof(double));
  return p;
}

// v_mfma_f64_16x16x4: lane l holds row l % 16 and k = l / 16 of either operand;
// accumulator value v is row 4 v + l / 16, column l % 16.
__device__ __forceinline__ f64x4_t mma(double a, double b, f64x4_t c) {
  return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void tile_of(int t, int& tm, int& tn) {
  tm = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
  tn = t - tm * (tm + 1) / 2;
}

// Calls f(mi, ni, inside, element) for the 64 x 64 tile of columns n0.., in the order of
// memory, 16 entries a thread; an entry outside the matrix gets the matrix's first
// element as its address.
template <typename F>
__device__ __forceinline__ void each_entry(const OrthoArgs& a, int m, int n, int b, int n0, const F& f) {
  const bool tall = a.rows > a.cols, along_m = runs_along_m(a);
  const bool inner = a.view.inner != 1 && !tall;
  const int64_t base = b * a.view.sb;
  if (inner) {
    const int D = a.view.inner, i0 = n0 / D, i1 = (n0 + 63) / D;
#pragma unroll 4
    for (int q = threadIdx.x; q < (i1 - i0 + 1) * kM * D; q += 256) {
      const int i = q / (kM * D), in = q - i * kM * D, r = in / D, d = in - r * D, c = (i0 + i) * D + d;
      if (c < n0 || c >= n0 + 64) continue;
      const bool ok = r < m && c < n;
      f(r, c - n0, ok, ok ? base + r * a.view.sr + (int64_t)(i0 + i) * a.view.so + d * a.view.si : base);
    }
    return;
  }
#pragma unroll 8
  for (int u = 0; u < 16; ++u) {
    const int q = threadIdx.x + u * 256, x = q & 63, y = q >> 6;
    const int mi = along_m ? x : y, ni = along_m ? y : x, c = n0 + ni;
    const bool ok = mi < m && c < n;
    f(mi, ni, ok, !ok ? base : tall ? view_at(a.view, b, c, mi) : view_at(a.view, b, mi, c));
  }
}

// What a kernel reads: the compiler batches a tile's loads only where their type is
// no question at run time.
enum SmallKind { kSmallF32, kSmallBf16, kSmallMuon };
template <int KIND>
__device__ __forceinline__ float small_entry(const OrthoArgs& a, int64_t e) {
  if constexpr (KIND == kSmallMuon) return muon_dir(a.g[e], a.buf[e], a);
  if constexpr (KIND == kSmallBf16) return (float)((const __bf16*)a.in)[e];
  return ((const float*)a.in)[e];
}

template <int KIND>
__global__ __launch_bounds__(256) void k_small_gram(OrthoArgs a, SmallPlan p, double* part) {
  __shared__ float tile[kM * kPitch];
  const int b = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n_end = (int)(blockIdx.x + 1) * p.chunk_cols < p.n ? (int)(blockIdx.x + 1) * p.chunk_cols : p.n;
  f64x4_t acc[3] = {};  // tiles wave, wave + 4, wave + 8
  for (int n0 = blockIdx.x * p.chunk_cols; n0 < n_end; n0 += 64) {
    __syncthreads();
    each_entry(a, p.m, p.n, b, n0, [&](int mi, int ni, bool ok, int64_t e) {
      float v;
      if constexpr (KIND == kSmallMuon) {
        const float g = a.g[e], nb = fmaf(a.momentum, a.buf[e], (1.0f - a.momentum) * g);
        if (ok) a.buf[e] = nb;
        v = muon_dir(g, nb, a);
      } else {
        v = small_entry<KIND>(a, e);
      }
      tile[mi * kPitch + ni] = ok ? v : 0.0f;
    });
    __syncthreads();
    // the wave's tiles take turns, so that no instruction waits for the last one's sum
    const float *x[3], *y[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      int tm, tn;
      tile_of(wave + 4 * s < kTiles ? wave + 4 * s : wave, tm, tn);
      x[s] = tile + (tm * 16 + (lane & 15)) * kPitch + (lane >> 4);
      y[s] = tile + (tn * 16 + (lane & 15)) * kPitch + (lane >> 4);
    }
#pragma unroll
    for (int k = 0; k < 64; k += 4)
#pragma unroll
      for (int s = 0; s < 3; ++s) acc[s] = mma((double)x[s][k], (double)y[s][k], acc[s]);
  }
#pragma unroll
  for (int s = 0; s < 3; ++s)
    if (wave + 4 * s < kTiles)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        part[(((size_t)b * p.chunks + blockIdx.x) * kTiles + wave + 4 * s) * 256 + v * 64 + lane] = acc[s][v];
}

// One workgroup a matrix, one wave a tile on or below the diagonal; the tiles above
// are their mirror images (every matrix here is symmetric).
__global__ __launch_bounds__(64 * kTiles) void k_small_chain(OrthoArgs a, SmallPlan p, const double* part, double* q) {
  extern __shared__ double lds[];
  constexpr int kMat = kM * kPitch;
  double *A = lds, *P = lds + kMat, *W = lds + 2 * kMat, *Q = lds + 3 * kMat;
  __shared__ double trace;
  const int b = blockIdx.x, t = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int tm, tn;
  tile_of(t, tm, tn);
  const int ks = (p.m + 15) / 16 * 16;
  const bool live = tm * 16 < p.m;  // wave-uniform; the barriers below are outside it
  auto product = [&](const double* X, const double* Y) {
    f64x4_t acc = {};
    if (live) {
      const double *x = X + (tm * 16 + (lane & 15)) * kPitch + (lane >> 4), *y = Y + (tn * 16 + (lane & 15)) * kPitch + (lane >> 4);
#pragma unroll 4
      for (int k = 0; k < ks; k += 4) acc = mma(x[k], y[k], acc);
    }
    return acc;
  };
  auto store = [&](double* Z, f64x4_t v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = tm * 16 + 4 * i + (lane >> 4), c = tn * 16 + (lane & 15);
      if (r >= c) Z[r * kPitch + c] = Z[c * kPitch + r] = v[i];
    }
  };
  f64x4_t v = {};
  const double* src = part + ((size_t)b * p.chunks * kTiles + t) * 256 + lane;
#pragma unroll 8
  for (int c = 0; c < p.chunks; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += src[(size_t)c * kTiles * 256 + i * 64];
  store(A, v);
  __syncthreads();
  if (t == 0) {
    double d = A[lane * kPitch + lane];
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) d += __shfl_xor(d, w);
    if (lane == 0) trace = d;
  }
  __syncthreads();
  const double s = 1.0 / (sqrt(trace) + (double)a.eps);
  // the identity, and this tile's A
  f64x4_t one, self;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = tm * 16 + 4 * i + (lane >> 4), c = tn * 16 + (lane & 15);
    one[i] = r == c && r < p.m ? 1.0 : 0.0;
    self[i] = v[i] * s * s;
  }
  f64x4_t mine = one;  // this tile of Q
  __syncthreads();
  store(A, self);
  store(Q, one);
  __syncthreads();
  for (int step = 0; step < a.steps; ++step) {
    const f64x4_t h = product(A, A);
    f64x4_t pt;
#pragma unroll
    for (int i = 0; i < 4; ++i) pt[i] = (double)a.a * one[i] + (double)a.b * self[i] + (double)a.c * h[i];
    store(P, pt);
    __syncthreads();
    mine = step ? product(Q, P) : pt;
    const bool more = step + 1 < a.steps;
    if (more) store(W, product(P, A));
    __syncthreads();
    store(Q, mine);
    if (more) {
      self = product(W, P);
      store(A, self);  // A's last readers are past the barrier
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = tm * 16 + 4 * i + (lane >> 4), c = tn * 16 + (lane & 15);
    if (r >= c) q[((size_t)b * kM + r) * kM + c] = q[((size_t)b * kM + c) * kM + r] = mine[i] * s;
  }
}

// 64 columns of Q G a block, a wave 16 rows.
template <int KIND>
__global__ __launch_bounds__(256) void k_small_apply(OrthoArgs a, SmallPlan p, const double* q) {
  __shared__ float tile[kM * kPitch];
  __shared__ double Q[kM * kPitch];
  const int b = blockIdx.y, n0 = blockIdx.x * 64, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int e = threadIdx.x + u * 256;
    Q[(e >> 6) * kPitch + (e & 63)] = q[(size_t)b * kM * kM + e];
  }
  each_entry(a, p.m, p.n, b, n0, [&](int mi, int ni, bool ok, int64_t e) { 
    const float v = small_entry<KIND>(a, e);
    tile[mi * kPitch + ni] = ok ? v : 0.0f;
  });
  __syncthreads();
  f64x4_t acc[4] = {};
  const int ks = (p.m + 3) / 4 * 4;
  for (int k = 0; k < ks; k += 4) {
    const double x = Q[(wave * 16 + (lane & 15)) * kPitch + k + (lane >> 4)];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = mma(x, (double)tile[(k + (lane >> 4)) * kPitch + j * 16 + (lane & 15)], acc[j]);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v) tile[(wave * 16 + 4 * v + (lane >> 4)) * kPitch + j * 16 + (lane & 15)] = (float)acc[j][v];
  __syncthreads();
  each_entry(a, p.m, p.n, b, n0, [&](int mi, int ni, bool ok, int64_t e) {
    const float o = tile[mi * kPitch + ni];
    if constexpr (KIND == kSmallMuon) {
      const float old = a.p[e];
      if (ok) a.p[e] = muon_param(a, old, o);
    } else if constexpr (KIND == kSmallBf16) {
      if (ok) ((__bf16*)a.out)[e] = (__bf16)o;
    } else {
      if (ok) ((float*)a.out)[e] = o;
    }
  });
}

}  // namespace

size_t ortho_small_workspace_bytes(int batch, int rows, int cols) { return make_small_plan(batch, rows, cols).bytes; }

namespace {
template <int KIND>
void launch_kind(const OrthoArgs& a, const SmallPlan& p, double* part, double* q, hipStream_t st) {
  hipLaunchKernelGGL(k_small_gram<KIND>, dim3(p.chunks, a.batch), dim3(256), 0, st, a, p, part);
  constexpr int lds = 4 * kM * kPitch * (int)sizeof(double);
  static std::atomic<uint32_t> done;
  ensure_lds_limit((const void*)k_small_chain, lds, done);
  hipLaunchKernelGGL(k_small_chain, dim3(a.batch), dim3(64 * kTiles), lds, st, a, p, part, q);
  hipLaunchKernelGGL(k_small_apply<KIND>, dim3((unsigned)ceil_div(p.n, 64), a.batch), dim3(256), 0, st, a, p, q);
}
}  // namespace

void launch_ortho_small(const OrthoArgs& a, void* ws, hipStream_t st) {
  const SmallPlan p = make_small_plan(a.batch, a.rows, a.cols);
  double *part = (double*)((char*)ws + p.part_off), *q = (double*)((char*)ws + p.q_off);
  if (!a.in)
    launch_kind<kSmallMuon>(a, p, part, q, st);
  else if (a.bf16)
    launch_kind<kSmallBf16>(a, p, part, q, st);
  else
    launch_kind<kSmallF32>(a, p, part, q, st);
}

}  // namespace ckan
