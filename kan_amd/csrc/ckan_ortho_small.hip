// Orthogonalisation of matrices with a side m <= 64, in 64 bits and three launches.
//
// With G = [m, n] (transposed where rows < cols fails), every iterate is Q_s G, Q_s a
// polynomial in A = G G^T / |G|^2, and |G|^2 is the trace of G G^T:
//   1. G G^T in parts of n (and Muon's momentum on the way: each entry is read once),
//   2. one workgroup a matrix sums the parts, scales by the trace and iterates
//        P = a I + b A + c A^2,  Q <- Q P,  A <- P A P
//      on 64 x 64 matrices in LDS, the identity's share of P and Q apart from them,
//   3. Q G, to where it belongs.
// A is not made from the iterate between the steps, so that its error in the directions of
// small singular values grows by a^2 = 11.9 a step (by a in the iteration itself): in fp32
// five steps lose them, in fp64 nine leave 2^-22 of them at worst.  Longer iterations go in
// runs of at most that many steps, the iterate between two runs in 64 bits.  At these
// sizes the fp64 matrix instructions cost less than the launches they save: [64, 3920] took
// 20 launches and 167 us step by step.  What bounds it: step 2, 17 dependent products on
// one CU.
#include <math.h>

#include <type_traits>

#include "ckan_ortho.hpp"

namespace ckan {
namespace {

typedef __attribute__((ext_vector_type(4))) double f64x4_t;
constexpr int kM = 64, kTiles = 10;  // 16 x 16 tiles on and below the diagonal
constexpr int kPitch = 68;           // of the LDS matrices: a fragment's 16 rows x 4 k on distinct banks
constexpr int kMaxChunks = 32;

struct SmallPlan {
  int m, n, chunks, chunk_cols;
  int runs;
  size_t part_off, q_off, share_off, x_off, bytes;
};

// The most steps whose product leaves an error of A's 2^-53 below 2^-22 (the slope of
// y p(y)^2 a step, along the singular values in [0, 1]).
int longest_run(const OrthoArgs& a) {
  double grown[65];
  int most = a.steps > 1 ? a.steps : 1;
  for (double& g : grown) g = 1.0;
  for (int i = 0; i < 65; ++i) {
    double x = i / 64.0;
    for (int s = 0; s + 1 < most; ++s) {
      const double y = x * x, p = a.a + a.b * y + a.c * y * y;
      grown[i] *= fmax(fabs(p * (p + 2.0 * y * (a.b + 2.0 * a.c * y))), p * p);
      if (!(grown[i] <= 0x1p31)) most = s + 1;
      x *= p;
    }
  }
  return most;
}

SmallPlan make_small_plan(const OrthoArgs& a) {
  SmallPlan p{};
  p.m = a.rows < a.cols ? a.rows : a.cols;
  p.n = a.rows < a.cols ? a.cols : a.rows;
  p.chunk_cols = (int)round_up(ceil_div(p.n, kMaxChunks), 64);
  p.chunks = (int)ceil_div(p.n, p.chunk_cols);
  p.runs = a.steps > 0 ? (int)ceil_div(a.steps, longest_run(a)) : 1;
  p.part_off = 0;
  p.q_off = align256((size_t)a.batch * p.chunks * kTiles * 256 * sizeof(double));
  p.share_off = p.q_off + align256((size_t)a.batch * kM * kM * sizeof(double));
  p.x_off = p.share_off + align256((size_t)a.batch * sizeof(double));
  p.bytes = p.x_off + (p.runs > 1 ? align256((size_t)a.batch * p.m * p.n * sizeof(double)) : 0);
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

// The same for the iterate between two runs, [batch, m, n] in 64 bits.
template <typename F>
__device__ __forceinline__ void each_between(const SmallPlan& p, int b, int n0, const F& f) {
#pragma unroll 8
  for (int u = 0; u < 16; ++u) {
    const int q = threadIdx.x + u * 256, ni = q & 63, mi = q >> 6, c = n0 + ni;
    const bool ok = mi < p.m && c < p.n;
    f(mi, ni, ok, ((int64_t)b * p.m + (ok ? mi : 0)) * p.n + (ok ? c : 0));
  }
}

// What a kernel reads or writes: the compiler batches a tile's loads only where their type
// is no question at run time.
enum SmallKind { kSmallF32, kSmallBf16, kSmallMuon, kSmallBetween };
template <int KIND> using SmallElem = typename std::conditional<KIND == kSmallBetween, double, float>::type;
template <int KIND>
__device__ __forceinline__ float small_entry(const OrthoArgs& a, int64_t e) {
  if constexpr (KIND == kSmallMuon) return muon_dir(a.g[e], a.buf[e], a);
  if constexpr (KIND == kSmallBf16) return (float)((const __bf16*)a.in)[e];
  return ((const float*)a.in)[e];
}

template <int KIND>
__global__ __launch_bounds__(256) void k_small_gram(OrthoArgs a, SmallPlan p, double* part, const double* between) {
  typedef SmallElem<KIND> E;
  __shared__ E tile[kM * kPitch];
  const int b = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n_end = (int)(blockIdx.x + 1) * p.chunk_cols < p.n ? (int)(blockIdx.x + 1) * p.chunk_cols : p.n;
  f64x4_t acc[3] = {};  // tiles wave, wave + 4, wave + 8
  for (int n0 = blockIdx.x * p.chunk_cols; n0 < n_end; n0 += 64) {
    __syncthreads();
    if constexpr (KIND == kSmallBetween) {
      each_between(p, b, n0, [&](int mi, int ni, bool ok, int64_t e) { tile[mi * kPitch + ni] = ok ? between[e] : 0.0; });
    } else {
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
    }
    __syncthreads();
    // the wave's tiles take turns, so that no instruction waits for the last one's sum
    const E *x[3], *y[3];
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

// One workgroup a matrix: `steps` steps from the Gram matrix's parts, scaled by the trace
// where it is the input's (first).  Q = share I + R, R to q.  One wave a tile on or below
// the diagonal, the tiles above being their mirror images (every matrix here is symmetric);
// or, WHOLE, a wave for each of the 16: two products of commuting matrices that are each
// other's mirror image differ in a last bit, which tells equal rows of the input apart, and
// over several runs that grows by a a step where the rows of the result are equal too.
template <bool WHOLE>
__global__ __launch_bounds__(64 * (WHOLE ? 16 : kTiles)) void k_small_chain(OrthoArgs a, SmallPlan p, const double* part,
                                                                            double* q, double* shares, int steps, int first) {
  extern __shared__ double lds[];
  constexpr int kMat = kM * kPitch;
  double *A = lds, *P = lds + kMat, *W = lds + 2 * kMat, *Q = lds + 3 * kMat;
  __shared__ double trace;
  const int b = blockIdx.x, t = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int tm, tn;
  auto mirrored = [&](double* Z, f64x4_t v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = tm * 16 + 4 * i + (lane >> 4), c = tn * 16 + (lane & 15);
      if (r >= c) Z[r * kPitch + c] = Z[c * kPitch + r] = v[i];
    }
  };
  tile_of(t, tm, tn);
  f64x4_t v = {};
  if (t < kTiles) {
    const double* src = part + ((size_t)b * p.chunks * kTiles + t) * 256 + lane;
#pragma unroll 8
    for (int c = 0; c < p.chunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += src[(size_t)c * kTiles * 256 + i * 64];
    mirrored(A, v);
  }
  __syncthreads();
  if (first && t == 0) {
    double d = A[lane * kPitch + lane];
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) d += __shfl_xor(d, w);
    if (lane == 0) trace = d;
  }
  if constexpr (WHOLE) {
    tm = t >> 2;
    tn = t & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = A[(tm * 16 + 4 * i + (lane >> 4)) * kPitch + tn * 16 + (lane & 15)];
  }
  __syncthreads();
  const int ks = (p.m + 15) / 16 * 16;
  const bool live = tm * 16 < p.m && tn * 16 < p.m;  // wave-uniform; the barriers below are outside it
  auto product = [&](const double* X, const double* Y, f64x4_t acc) {
    if (live) {
      const double *x = X + (tm * 16 + (lane & 15)) * kPitch + (lane >> 4), *y = Y + (tn * 16 + (lane & 15)) * kPitch + (lane >> 4);
#pragma unroll 4
      for (int k = 0; k < ks; k += 4) acc = mma(x[k], y[k], acc);
    }
    return acc;
  };
  auto store = [&](double* Z, f64x4_t z) {
    if constexpr (WHOLE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) Z[(tm * 16 + 4 * i + (lane >> 4)) * kPitch + tn * 16 + (lane & 15)] = z[i];
    } else {
      mirrored(Z, z);
    }
  };
  const double s = first ? 1.0 / (sqrt(trace) + (double)a.eps) : 1.0, ca = a.a, cb = a.b, cc = a.c;
  f64x4_t self, mine = {};  // this tile of A, of R
#pragma unroll
  for (int i = 0; i < 4; ++i) self[i] = v[i] * s * s;
  double share = 1.0;
  store(A, self);
  __syncthreads();
  for (int step = 0; step < steps; ++step) {
    f64x4_t bt = product(A, A, f64x4_t{});  // B = P - a I
#pragma unroll
    for (int i = 0; i < 4; ++i) bt[i] = cb * self[i] + cc * bt[i];
    store(P, bt);
    __syncthreads();
    const bool more = step + 1 < steps;
    if (step) {  // R P + share B
      f64x4_t r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = ca * mine[i] + share * bt[i];
      mine = product(Q, P, r);
    } else {
      mine = bt;
    }
    share *= ca;
    f64x4_t w;  // P A
    if (more) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = ca * self[i];
      w = product(P, A, w);
      store(W, w);
    }
    __syncthreads();
    store(Q, mine);
    if (more) {
#pragma unroll
      for (int i = 0; i < 4; ++i) self[i] = ca * w[i];
      self = product(W, P, self);
      store(A, self);  // A's last readers are past the barrier
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) shares[b] = share * s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = tm * 16 + 4 * i + (lane >> 4), c = tn * 16 + (lane & 15);
    if constexpr (WHOLE)
      q[((size_t)b * kM + r) * kM + c] = mine[i] * s;
    else if (r >= c)
      q[((size_t)b * kM + r) * kM + c] = q[((size_t)b * kM + c) * kM + r] = mine[i] * s;
  }
}

// 64 columns of Q G a block, a wave 16 rows.
template <int SRC, int DST>
__global__ __launch_bounds__(256) void k_small_apply(OrthoArgs a, SmallPlan p, const double* q, const double* shares,
                                                     double* between) {
  typedef SmallElem<(SRC == kSmallBetween ? SRC : DST)> E;
  extern __shared__ double lds[];
  double* Q = lds;
  E* tile = (E*)(lds + kM * kPitch);
  const int b = blockIdx.y, n0 = blockIdx.x * 64, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int e = threadIdx.x + u * 256;
    Q[(e >> 6) * kPitch + (e & 63)] = q[(size_t)b * kM * kM + e];
  }
  if constexpr (SRC == kSmallBetween) {
    each_between(p, b, n0, [&](int mi, int ni, bool ok, int64_t e) { tile[mi * kPitch + ni] = ok ? between[e] : 0.0; });
  } else {
    each_entry(a, p.m, p.n, b, n0, [&](int mi, int ni, bool ok, int64_t e) {
      const float v = small_entry<SRC>(a, e);
      tile[mi * kPitch + ni] = ok ? v : 0.0f;
    });
  }
  __syncthreads();
  const double share = shares[b];
  f64x4_t acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[j][v] = share * (double)tile[(wave * 16 + 4 * v + (lane >> 4)) * kPitch + j * 16 + (lane & 15)];
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
    for (int v = 0; v < 4; ++v) tile[(wave * 16 + 4 * v + (lane >> 4)) * kPitch + j * 16 + (lane & 15)] = (E)acc[j][v];
  __syncthreads();
  if constexpr (DST == kSmallBetween) {
    each_between(p, b, n0, [&](int mi, int ni, bool ok, int64_t e) {
      if (ok) between[e] = tile[mi * kPitch + ni];
    });
  } else {
    each_entry(a, p.m, p.n, b, n0, [&](int mi, int ni, bool ok, int64_t e) {
      const float o = (float)tile[mi * kPitch + ni];
      if constexpr (DST == kSmallMuon) {
        const float old = a.p[e];
        if (ok) a.p[e] = muon_param(a, old, o);
      } else if constexpr (DST == kSmallBf16) {
        if (ok) ((__bf16*)a.out)[e] = (__bf16)o;
      } else {
        if (ok) ((float*)a.out)[e] = o;
      }
    });
  }
}

}  // namespace

size_t ortho_small_workspace_bytes(const OrthoArgs& a) { return make_small_plan(a).bytes; }

namespace {
struct SmallBuffers {
  double *part, *q, *shares, *between;
};

template <int KIND>
void launch_gram(const OrthoArgs& a, const SmallPlan& p, const SmallBuffers& w, hipStream_t st) {
  hipLaunchKernelGGL(k_small_gram<KIND>, dim3(p.chunks, a.batch), dim3(256), 0, st, a, p, w.part, w.between);
}

template <bool WHOLE>
void launch_chain(const OrthoArgs& a, const SmallPlan& p, const SmallBuffers& w, int steps, bool first, hipStream_t st) {
  constexpr int lds = 4 * kM * kPitch * (int)sizeof(double);
  static std::atomic<uint32_t> done;
  ensure_lds_limit((const void*)k_small_chain<WHOLE>, lds, done);
  hipLaunchKernelGGL(k_small_chain<WHOLE>, dim3(a.batch), dim3(64 * (WHOLE ? 16 : kTiles)), lds, st, a, p, w.part, w.q, w.shares,
                     steps, (int)first);
}

template <int SRC, int DST>
void launch_apply(const OrthoArgs& a, const SmallPlan& p, const SmallBuffers& w, hipStream_t st) {
  constexpr int lds = kM * kPitch * (int)(sizeof(double) + sizeof(SmallElem<(SRC == kSmallBetween ? SRC : DST)>));
  static std::atomic<uint32_t> done;
  ensure_lds_limit((const void*)k_small_apply<SRC, DST>, lds, done);
  hipLaunchKernelGGL((k_small_apply<SRC, DST>), dim3((unsigned)ceil_div(p.n, 64), a.batch), dim3(256), lds, st, a, p, w.q, w.shares,
                     w.between);
}

template <int KIND>
void launch_kind(const OrthoArgs& a, const SmallPlan& p, const SmallBuffers& w, hipStream_t st) {
  if (p.runs == 1) {
    launch_gram<KIND>(a, p, w, st);
    launch_chain<false>(a, p, w, a.steps, true, st);
    launch_apply<KIND, KIND>(a, p, w, st);
    return;
  }
  for (int run = 0; run < p.runs; ++run) {
    const bool first = run == 0;
    if (first)
      launch_gram<KIND>(a, p, w, st);
    else
      launch_gram<kSmallBetween>(a, p, w, st);
    launch_chain<true>(a, p, w, a.steps / p.runs + (run < a.steps % p.runs), first, st);
    if (first)
      launch_apply<KIND, kSmallBetween>(a, p, w, st);
    else if (run + 1 < p.runs)
      launch_apply<kSmallBetween, kSmallBetween>(a, p, w, st);
    else
      launch_apply<kSmallBetween, KIND>(a, p, w, st);
  }
}
}  // namespace

void launch_ortho_small(const OrthoArgs& a, void* ws, hipStream_t st) {
  const SmallPlan p = make_small_plan(a);
  char* w = (char*)ws;
  const SmallBuffers buf{(double*)(w + p.part_off), (double*)(w + p.q_off), (double*)(w + p.share_off), (double*)(w + p.x_off)};
  if (!a.in)
    launch_kind<kSmallMuon>(a, p, buf, st);
  else if (a.bf16)
    launch_kind<kSmallBf16>(a, p, buf, st);
  else
    launch_kind<kSmallF32>(a, p, buf, st);
}

}  // namespace ckan
