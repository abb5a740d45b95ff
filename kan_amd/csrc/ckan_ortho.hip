// Orthogonalisation of matrices by Newton-Schulz products, and Muon's step.
//
// X0 = G / (|G|_F + eps), then `steps` times X <- a X + (b A + c A^2) X with
// A = X X^T.  m = the smaller, n = the larger dimension; the matrix is taken
// with its m-side as rows (the iteration of the transpose is the transpose).
//
// The products run on two fp16 planes (ckan_planes.hpp), all values scaled by
// 2^12: |X| and |A| stay below 1.5 and |b A + c A^2| below 7, far inside fp16's
// range, and the planes keep 22 bits of entries down to 2^-15 of the largest.
// X is held twice, as the operand with rows m and k = n (Xr, for A = X X^T) and
// as the operand with rows n and k = m (Xc, for the product with X).
#include "ckan_mix.hpp"
#include "ckan_planes.hpp"

namespace ckan {
namespace {

constexpr float kS = 4096.0f, kInvS = 1.0f / 4096.0f;  // the planes' scale
constexpr int kNormBlocks = 256;                       // partial sums of squares a matrix
constexpr int kTile = 128;

// Sizes of one matrix's buffers in the workspace.
struct OrthoPlan {
  int batch, m, n;
  bool tall;           // rows > cols: m runs along the columns
  int m32, n32;        // k extents
  int m128, n128;      // row extents
  int splits, kb_per_split;
  size_t norm_off, xr_off, xc_off[2], part_off, a_off, b_off, bytes;
  size_t xr_bytes, xc_bytes, a_bytes, part_elems;  // a matrix
};

OrthoPlan make_ortho_plan(int batch, int rows, int cols) {
  OrthoPlan p{};
  p.batch = batch;
  p.tall = rows > cols;
  p.m = p.tall ? cols : rows;
  p.n = p.tall ? rows : cols;
  p.m32 = (int)round_up(p.m, 32);
  p.n32 = (int)round_up(p.n, 32);
  p.m128 = (int)round_up(p.m, kTile);
  p.n128 = (int)round_up(p.n, kTile);
  // A = X X^T has few tiles and a long k: enough splits of k to give every CU a
  // block, none shorter than 256 (16 k-blocks)
  const int T = p.m128 / kTile;
  const int64_t tiles = (int64_t)batch * T * (T + 1) / 2;
  int64_t splits = ceil_div(kNumCUs, tiles);
  const int kb = p.n32 / 16;
  if (splits > kb / 16) splits = kb / 16;
  if (splits < 1) splits = 1;
  p.kb_per_split = (int)round_up(ceil_div(kb, splits), 2);
  p.splits = (int)ceil_div(kb, p.kb_per_split);
  p.xr_bytes = (size_t)p.m128 * p.n32 * 4;
  p.xc_bytes = (size_t)p.n128 * p.m32 * 4;
  p.a_bytes = (size_t)p.m128 * p.m32 * 4;
  p.part_elems = (size_t)p.m128 * p.m128;
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off = align256(off + n);
    return at;
  };
  p.norm_off = take((size_t)batch * kNormBlocks * sizeof(double));
  p.xr_off = take(p.xr_bytes * batch);
  p.xc_off[0] = take(p.xc_bytes * batch);
  p.xc_off[1] = take(p.xc_bytes * batch);
  p.part_off = take(p.part_elems * batch * p.splits * sizeof(float));
  p.a_off = take(p.a_bytes * batch);
  p.b_off = take(p.a_bytes * batch);
  p.bytes = off;
  return p;
}

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

// Sums of squares in 64 bits, kNormBlocks partials a matrix; Muon's momentum is
// updated on the way (buf = mu buf + (1 - mu) g).  Element order follows memory:
// inner, then rows, then outer columns where a view has an inner dimension.
__global__ __launch_bounds__(256) void k_ortho_norm(OrthoArgs a, double* part) {
  const int b = blockIdx.y;
  const int64_t total = (int64_t)a.rows * a.cols;
  const int inner = a.view.inner;
  double s = 0.0;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)kNormBlocks * 256) {
    int64_t at;
    if (inner == 1) {
      const int64_t r = e / a.cols;
      at = b * a.view.sb + r * a.view.sr + (e - r * a.cols) * a.view.so;
    } else {  // (outer column, row, inner)
      const int64_t q = e / inner, i = q / a.rows;
      at = b * a.view.sb + (q - i * a.rows) * a.view.sr + i * a.view.so + (e - q * inner) * a.view.si;
    }
    float v;
    if (a.in) {
      v = entry(a, at);
    } else {
      const float g = a.g[at];
      const float nb = fmaf(a.momentum, a.buf[at], (1.0f - a.momentum) * g);
      a.buf[at] = nb;
      v = muon_dir(g, nb, a);
    }
    s += (double)v * v;
  }
  __shared__ double red[256];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) part[b * kNormBlocks + blockIdx.x] = red[0];
}

// X0 in both operand forms: one block a 64 x 64 tile (m x n), through LDS.
__global__ __launch_bounds__(256) void k_ortho_pack(OrthoArgs a, OrthoPlan p, const double* part, char* xr,
                                                    char* xc) {
  __shared__ float tile[64][65];
  __shared__ double red[256];
  const int b = blockIdx.z, m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tid = threadIdx.x;
  red[tid] = part[b * kNormBlocks + tid];
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (tid < w) red[tid] += red[tid + w];
    __syncthreads();
  }
  const float f = kS / ((float)sqrt(red[0]) + a.eps);
  // memory runs along n for an ordinary matrix with rows m, along m for the
  // transposed, and along (row, inner) for a view with an inner dimension
  for (int e = tid; e < 64 * 64; e += 256) {
    int mi = e >> 6, ni = e & 63;
    if (p.tall || a.view.inner != 1) {
      mi = e & 63;
      ni = e >> 6;
    }
    const int m = m0 + mi, n = n0 + ni;
    float v = 0.0f;
    if (m < p.m && n < p.n) v = f * entry(a, p.tall ? view_at(a.view, b, n, m) : view_at(a.view, b, m, n));
    tile[mi][ni] = v;
  }
  __syncthreads();
  // 64 rows x 8 groups of 8 k of each form: 512 lanes' values, two a thread
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int q = tid + half * 256, r = q & 63, k8 = q >> 6;
    float v[8];
    if (m0 + r < p.m128 && n0 + k8 * 8 < p.n32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = tile[r][k8 * 8 + j];
      const Planes8<2> f8 = to_planes8<2>(v);
      const int row = m0 + r, kb = (n0 + k8 * 8) >> 4, g = k8 & 1;
      char* d = xr + b * p.xr_bytes + ((size_t)(row >> 5) * (p.n32 / 16) + kb) * 2 * kPlaneBytes + ((row & 31) + 32 * g) * 16;
      *(f16x8_t*)d = f8.p[0];
      *(f16x8_t*)(d + kPlaneBytes) = f8.p[1];
    }
    if (n0 + r < p.n128 && m0 + k8 * 8 < p.m32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = tile[k8 * 8 + j][r];
      const Planes8<2> f8 = to_planes8<2>(v);
      const int row = n0 + r, kb = (m0 + k8 * 8) >> 4, g = k8 & 1;
      char* d = xc + b * p.xc_bytes + ((size_t)(row >> 5) * (p.m32 / 16) + kb) * 2 * kPlaneBytes + ((row & 31) + 32 * g) * 16;
      *(f16x8_t*)d = f8.p[0];
      *(f16x8_t*)(d + kPlaneBytes) = f8.p[1];
    }
  }
}

typedef NtTile<2, 2, 2, 2, 2, 2, 2, 2> Tile22;  // 128 x 128, 64 KiB of LDS

// Partial sums of A = X X^T (scale kS^2): the tiles on and below the diagonal,
// each stored with its mirror image, k split over blocks.
__global__ __launch_bounds__(256, 2) void k_ortho_gram(OrthoPlan p, const char* xr, float* part) {
  extern __shared__ char lds[];
  const int T = p.m128 / kTile, pairs = T * (T + 1) / 2;
  int id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  const int pair = id % pairs, b = id / pairs;
  int tm = 0;
  while ((tm + 1) * (tm + 2) / 2 <= pair) ++tm;
  const int tn = pair - tm * (tm + 1) / 2;
  const int KB = p.n32 / 16, kb0 = split * p.kb_per_split;
  const int kbs = KB - kb0 < p.kb_per_split ? KB - kb0 : p.kb_per_split;
  const size_t pitch = (size_t)KB * 2 * kPlaneBytes;
  const char* x = xr + b * p.xr_bytes;
  f32x16_t acc[2][2] = {};
  Tile22::run(RowBlocks{x + tm * 4 * pitch, pitch}, RowBlocks{x + tn * 4 * pitch, pitch}, kb0, kbs / 2, lds, acc);
  float* out = part + ((size_t)split * p.batch + b) * p.part_elems;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 5;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int row = tm * kTile + (wave >> 1) * 64 + m * 32, col = tn * kTile + (wave & 1) * 64 + n * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = acc[m][n][q * 4 + j];
          if (tm != tn) out[(size_t)(row + 8 * q + 4 * g + j) * p.m128 + col] = v[j];
        }
        *(f32x4_t*)(out + (size_t)col * p.m128 + row + 8 * q + 4 * g) = v;
      }
    }
}

// A in planes from the partial sums: a thread a row and 8 k.
__global__ __launch_bounds__(256) void k_ortho_gram_sum(OrthoPlan p, const float* part, char* A) {
  const int b = blockIdx.y;
  const int k8s = p.m32 / 8;
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (q >= (int64_t)p.m128 * k8s) return;
  const int k8 = (int)(q % k8s), row = (int)(q / k8s);
  float v[8] = {};
  if (row < p.m) {
    for (int s = 0; s < p.splits; ++s) {
      const float* src = part + ((size_t)s * p.batch + b) * p.part_elems + (size_t)row * p.m128 + k8 * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += src[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k8 * 8 + j < p.m ? v[j] * kInvS : 0.0f;
  }
  const Planes8<2> f = to_planes8<2>(v);
  char* d = A + b * p.a_bytes + ((size_t)(row >> 5) * (p.m32 / 16) + (k8 >> 1)) * 2 * kPlaneBytes + ((row & 31) + 32 * (k8 & 1)) * 16;
  *(f16x8_t*)d = f.p[0];
  *(f16x8_t*)(d + kPlaneBytes) = f.p[1];
}

// The 8-byte half of a lane's planes that an accumulator quad (4 consecutive
// rows of the product) is in the operand whose k runs along those rows.
__device__ __forceinline__ size_t quad_at(int row, int k, int KB) {
  return ((size_t)(row >> 5) * KB + (k >> 4)) * 2 * kPlaneBytes + ((row & 31) + 32 * ((k >> 3) & 1)) * 16 + (k & 4) * 2;
}

// B = b A + c A^2 (A symmetric: A A = A A^T); B is symmetric too, so the product's
// rows are stored as the operand's k.
__global__ __launch_bounds__(256, 2) void k_ortho_poly(OrthoPlan p, const char* A, char* B, float cb, float cc) {
  extern __shared__ char lds[];
  const int T = p.m128 / kTile, b = blockIdx.x / (T * T), t = blockIdx.x % (T * T), tm = t / T, tn = t % T;
  const int KB = p.m32 / 16;
  const size_t pitch = (size_t)KB * 2 * kPlaneBytes;
  const char* x = A + b * p.a_bytes;
  f32x16_t acc[2][2] = {};
  Tile22::run(RowBlocks{x + tm * 4 * pitch, pitch}, RowBlocks{x + tn * 4 * pitch, pitch}, 0, KB / 2, lds, acc);
  char* out = B + b * p.a_bytes;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 5;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int row0 = tm * kTile + (wave >> 1) * 64 + m * 32, col = tn * kTile + (wave & 1) * 64 + n * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = row0 + 8 * q + 4 * g;
        if (k >= p.m32) continue;
        const size_t at = quad_at(col, k, KB);
        const f16x4_t h = *(const f16x4_t*)(x + at), l = *(const f16x4_t*)(x + at + kPlaneBytes);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = cb * ((float)h[j] + (float)l[j]) + cc * (acc[m][n][q * 4 + j] * kInvS);
          if (k + j >= p.m || col >= p.m) v[j] = 0.0f;
        }
        const Planes4<2> f = to_planes4<2>(v);
        *(f16x4_t*)(out + at) = f.p[0];
        *(f16x4_t*)(out + at + kPlaneBytes) = f.p[1];
      }
    }
}

// X' = a X + B X.  The product's rows are m, its columns n: an accumulator quad is 4
// consecutive k of Xc, where the old X is read and the new one stored; Xr goes
// through LDS.  The last step writes the result instead (or Muon's parameters).
__global__ __launch_bounds__(256, 2) void k_ortho_update(OrthoArgs a, OrthoPlan p, const char* B, const char* xc,
                                                         char* xc_new, char* xr, int last) {
  extern __shared__ char lds[];
  const int TM = p.m128 / kTile, TN = p.n128 / kTile;
  int id = blockIdx.x;
  const int tm = id % TM;
  id /= TM;
  const int tn = id % TN, b = id / TN;
  const int KB = p.m32 / 16;
  const size_t pitch = (size_t)KB * 2 * kPlaneBytes;
  const char* x = xc + b * p.xc_bytes;
  f32x16_t acc[2][2] = {};
  Tile22::run(RowBlocks{B + b * p.a_bytes + tm * 4 * pitch, pitch}, RowBlocks{x + tn * 4 * pitch, pitch}, 0, KB / 2, lds, acc);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 5;
  constexpr int kPitch = (kTile + 8) * 2;  // bytes of a row of the LDS tile
  char* plane1 = lds + kTile * kPitch;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r0 = (wave >> 1) * 64 + m * 32, c = (wave & 1) * 64 + n * 32 + (lane & 31);
      const int col = tn * kTile + c;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = r0 + 8 * q + 4 * g, k = tm * kTile + r;
        float v[4] = {};
        const size_t at = quad_at(col, k, KB);
        if (k < p.m32) {
          const f16x4_t h = *(const f16x4_t*)(x + at), l = *(const f16x4_t*)(x + at + kPlaneBytes);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k + j < p.m && col < p.n) v[j] = a.a * ((float)h[j] + (float)l[j]) + acc[m][n][q * 4 + j] * kInvS;
        }
        if (last) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (k + j >= p.m || col >= p.n) continue;
            const float o = v[j] * kInvS;
            const int64_t e = p.tall ? view_at(a.view, b, col, k + j) : view_at(a.view, b, k + j, col);
            if (!a.in)
              a.p[e] = fmaf(-a.lr * a.scale, o, a.p[e] * (1.0f - a.lr * a.decay));
            else if (a.bf16)
              ((__bf16*)a.out)[e] = (__bf16)o;
            else
              ((float*)a.out)[e] = o;
          }
          continue;
        }
        const Planes4<2> f = to_planes4<2>(v);
        if (k < p.m32) {
          char* d = xc_new + b * p.xc_bytes + at;
          *(f16x4_t*)d = f.p[0];
          *(f16x4_t*)(d + kPlaneBytes) = f.p[1];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          *(_Float16*)(lds + (r + j) * kPitch + c * 2) = f.p[0][j];
          *(_Float16*)(plane1 + (r + j) * kPitch + c * 2) = f.p[1][j];
        }
      }
    }
  if (last) return;
  __syncthreads();
  // Xr: 128 rows x 16 groups of 8 k, 8 a thread
  const int KBr = p.n32 / 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = threadIdx.x + i * 256, r = q & 127, k8 = q >> 7;
    const int row = tm * kTile + r, k = tn * kTile + k8 * 8;
    if (k >= p.n32) continue;
    char* d = xr + b * p.xr_bytes + ((size_t)(row >> 5) * KBr + (k >> 4)) * 2 * kPlaneBytes + ((row & 31) + 32 * (k8 & 1)) * 16;
    *(f16x8_t*)d = *(const f16x8_t*)(lds + r * kPitch + k8 * 16);
    *(f16x8_t*)(d + kPlaneBytes) = *(const f16x8_t*)(plane1 + r * kPitch + k8 * 16);
  }
}

constexpr int kUpdateLds = 2 * kTile * (kTile + 8) * 2 > Tile22::kLdsBytes ? 2 * kTile * (kTile + 8) * 2 : Tile22::kLdsBytes;

// steps == 0: the normalised matrix itself.
__global__ __launch_bounds__(256) void k_ortho_scale(OrthoArgs a, const double* part) {
  __shared__ double red[256];
  const int b = blockIdx.y, tid = threadIdx.x;
  red[tid] = part[b * kNormBlocks + tid];
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (tid < w) red[tid] += red[tid + w];
    __syncthreads();
  }
  const float f = (float)sqrt(red[0]) + a.eps;
  const int64_t total = (int64_t)a.rows * a.cols;
  for (int64_t e = (int64_t)blockIdx.x * 256 + tid; e < total; e += (int64_t)gridDim.x * 256) {
    const int r = (int)(e / a.cols), c = (int)(e % a.cols);
    const int64_t at = view_at(a.view, b, r, c);
    const float o = entry(a, at) / f;
    if (!a.in)
      a.p[at] = fmaf(-a.lr * a.scale, o, a.p[at] * (1.0f - a.lr * a.decay));
    else if (a.bf16)
      ((__bf16*)a.out)[at] = (__bf16)o;
    else
      ((float*)a.out)[at] = o;
  }
}

}  // namespace

size_t ortho_workspace_bytes(int batch, int rows, int cols) { return make_ortho_plan(batch, rows, cols).bytes; }

void launch_ortho(const OrthoArgs& a, void* ws, hipStream_t st) {
  const OrthoPlan p = make_ortho_plan(a.batch, a.rows, a.cols);
  char* w = (char*)ws;
  double* norm = (double*)(w + p.norm_off);
  char *xr = w + p.xr_off, *A = w + p.a_off, *B = w + p.b_off;
  char* xc[2] = {w + p.xc_off[0], w + p.xc_off[1]};
  float* part = (float*)(w + p.part_off);
  static std::atomic<uint32_t> done[3];
  ensure_lds_limit((const void*)k_ortho_gram, Tile22::kLdsBytes, done[0]);
  ensure_lds_limit((const void*)k_ortho_poly, Tile22::kLdsBytes, done[1]);
  ensure_lds_limit((const void*)k_ortho_update, kUpdateLds, done[2]);
  hipLaunchKernelGGL(k_ortho_norm, dim3(kNormBlocks, a.batch), dim3(256), 0, st, a, norm);
  if (a.steps == 0) {
    hipLaunchKernelGGL(k_ortho_scale, dim3(kNormBlocks, a.batch), dim3(256), 0, st, a, norm);
    return;
  }
  hipLaunchKernelGGL(k_ortho_pack, dim3(p.n128 / 64, p.m128 / 64, a.batch), dim3(256), 0, st, a, p, norm, xr, xc[0]);
  const int T = p.m128 / kTile, TN = p.n128 / kTile;
  for (int s = 0; s < a.steps; ++s) {
    hipLaunchKernelGGL(k_ortho_gram, dim3(a.batch * (T * (T + 1) / 2) * p.splits), dim3(256), Tile22::kLdsBytes, st, p,
                       xr, part);
    hipLaunchKernelGGL(k_ortho_gram_sum, dim3((unsigned)ceil_div((int64_t)p.m128 * (p.m32 / 8), 256), a.batch),
                       dim3(256), 0, st, p, part, A);
    hipLaunchKernelGGL(k_ortho_poly, dim3(a.batch * T * T), dim3(256), Tile22::kLdsBytes, st, p, A, B, a.b, a.c);
    hipLaunchKernelGGL(k_ortho_update, dim3(a.batch * T * TN), dim3(256), kUpdateLds, st, a, p, B, xc[s & 1],
                       xc[(s + 1) & 1], xr, s == a.steps - 1);
  }
}

}  // namespace ckan
