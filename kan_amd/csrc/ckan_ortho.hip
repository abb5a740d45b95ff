// Orthogonalisation of matrices by Newton-Schulz products, and Muon's step.
//
// X0 = G / (|G|_F + eps), then `steps` times X <- a X + (b A + c A^2) X with
// A = X X^T.  m = the smaller, n = the larger dimension; the matrix is taken
// with its m-side as rows (the iteration of the transpose is the transpose).
//
// The products run on fp16 planes (ckan_planes.hpp), X and A scaled by 2^12: |X| and
// |A| stay below 1.5 and |b A + c A^2| below 7, far inside fp16's range, and two
// planes keep 22 bits of entries down to 2^-15 of the largest.  A matrix whose norm is
// far below eps enters with |X0| far below 1: it is lifted by a power of two of its own, which
// its steps use up again as X grows (lift_at below).
//
// Matrices with a side of at most 64 are ckan_ortho_small.hip's.  Of the others,
// fp32 matrices take the iteration on two planes, as it is written or, where they are
// wide, two steps at a time (pairs() below).  X is held
// twice, as the operand with rows m and k = n (Xr, for A = X X^T) and as the one
// with rows n and k = m (Xc, for the product with X).
//
// bf16 matrices begin in the m x m domain.  Every factor is a polynomial in A_0:
//   P_s = a I + b A_s + c A_s^2,   A_{s+1} = P_s A_s P_s,   Q = P_{r-1} .. P_1 P_0,
// and Q X0 are r steps in one: two products with the long side instead of 3 r, and X0,
// scaled by a power of two, is exact in one plane.  But A is not made from X again
// between them: what A has as noise in the directions of small singular values grows by
// a^2 = 11.9 a step (by a in the iteration itself), so only as many steps are taken this
// way as keep it below bf16's own rounding (product_run() below: 3 of 5), and the rest
// as fp32 matrices do.  All five in one product left a matrix of rank one 1.9e-2 off, more
// of them anything.
#include <math.h>

#include "ckan_ortho.hpp"
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
  int run;             // steps at first in the m x m domain, of X0 in one plane
  int np;              // planes that X's buffers have room for
  int mk, n32;         // k extents: m in whole stages of the m x m products, n in 32
  int m128, n128;      // row extents
  int splits, kb_per_split;
  float qscale;        // the scale of Q's planes
  size_t norm_off, xr_off, xc_off[2], part_off, mm_off[5], bytes;
  size_t xr_bytes, xc_bytes, a_bytes, part_elems;  // a matrix
};

// Two steps as one product with the long side:
//   X'' = P_1 P_0 X,  P_s = a I + B_s,  B_s = b A_s + c A_s^2,  A_1 = P_0 A_0 P_0,
// five m x m products more and one pass over X and one X X^T less.  At n = 4 m the trade
// in multiply-adds is 11 m^3 more for 12 m^3 less: 8 x [512, 4608] 776 us against 997,
// [256, 2304] 192 against 209.  The errors are 1.2 to 3 times the iteration's (the result is
// a difference of a^2 X and the rest), 2.1-2.8e-6 of a random matrix whatever its size,
// where plain fp32 products' grow with their sums: 1.3-1.7e-6 with m = 80 to 192, 2.1e-6
// with 256, 4.4e-6 with 512.  So fp32 matrices take it from m = 256 on; results in bf16 do
// not see it.
bool pairs(int m, int n, bool bf16) { return n >= 4 * (int64_t)m && n >= 2048 && (bf16 || m >= 256); }

// How many steps a bf16 matrix takes in the m x m domain: all of them, or the most (three
// at least) that leave the result's error below 2^-9, half of a rounding to bf16 at its
// largest.  The noise is 2^-20 of A, from the fp32 sums of X X^T and of a A and
// b A^2 + c A^3, which cancel in A_1 (rank one, 1024 x 4608: 1.8e-2 after five steps,
// 2^-20 11.9^4; shorter sums, or the product of the low planes too, change nothing).  A
// step in the m x m domain takes an error of A by the slope of y p(y)^2, each later one
// that of X by the slope of x p(x^2).  0: the iteration on two planes.  1024 x 9216, five
// steps: three of them this way 498 us, none 693, all 356 (and wrong).
int product_run(const OrthoArgs& a) {
  constexpr int kSamples = 64;
  if (!a.bf16) return 0;
  double worst[101] = {};  // of a run of r steps
  for (int i = 0; i <= kSamples; ++i) {
    double x = (double)i / kSamples, in_a[101], in_x[101], prefix = 1.0, suffix = 1.0;
    for (int s = 0; s < a.steps; ++s) {
      const double y = x * x, p = a.a + a.b * y + a.c * y * y, slope = p + 2.0 * y * (a.b + 2.0 * a.c * y);
      in_a[s] = fmax(fabs(p * slope), p * p);
      in_x[s] = fmax(fabs(slope), fabs(p));
      x *= p;
    }
    double after[101];
    for (int s = a.steps; s >= 0; --s) {
      after[s] = suffix;
      if (s > 0) suffix = fmin(suffix * in_x[s - 1], 1e100);
    }
    for (int r = 1; r <= a.steps; ++r) {
      if (r > 1) prefix = fmin(prefix * in_a[r - 2], 1e100);
      worst[r] = fmax(worst[r], prefix * after[r]);
    }
  }
  for (int r = a.steps; r > 0; r = r > 3 ? r - 1 : 0)
    if (worst[r] <= 2048.0) return r;
  return 0;
}

OrthoPlan make_ortho_plan(const OrthoArgs& a) {
  const int batch = a.batch, rows = a.rows, cols = a.cols;
  OrthoPlan p{};
  p.batch = batch;
  p.run = product_run(a);
  p.np = p.run > 0 && p.run == a.steps ? 1 : 2;
  p.tall = rows > cols;
  p.m = p.tall ? cols : rows;
  p.n = p.tall ? rows : cols;
  p.mk = (int)round_up(p.m, 64);
  p.n32 = (int)round_up(p.n, 32);
  p.m128 = (int)round_up(p.m, kTile);
  p.n128 = (int)round_up(p.n, kTile);
  // A = X X^T has few tiles and a long k: enough splits of k to give every CU a block,
  // none shorter than 256 (16 k-blocks).  Two blocks a CU (8 x [512, 4608]): the products
  // 50 us instead of 54, the sum of the splits 12 instead of 9.
  const int T = p.m128 / kTile;
  const int64_t tiles = (int64_t)batch * T * (T + 1) / 2;
  int64_t splits = ceil_div(kNumCUs, tiles);
  const int kb = p.n32 / 16;
  if (splits > kb / 16) splits = kb / 16;
  if (splits < 1) splits = 1;
  p.kb_per_split = (int)round_up(ceil_div(kb, splits), 2);
  p.splits = (int)ceil_div(kb, p.kb_per_split);
  p.xr_bytes = (size_t)p.m128 * p.n32 * 2 * p.np;
  p.xc_bytes = (size_t)p.n128 * p.mk * 2 * p.np;
  p.a_bytes = (size_t)p.m128 * p.mk * 4;
  p.part_elems = (size_t)p.m128 * p.m128;
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off = align256(off + n);
    return at;
  };
  p.norm_off = take((size_t)batch * (kNormBlocks + 2) * sizeof(double));
  p.xr_off = take(p.xr_bytes * batch);
  p.xc_off[0] = take(p.xc_bytes * batch);
  p.xc_off[1] = p.np == 1 ? 0 : take(p.xc_bytes * batch);
  p.part_off = take(p.part_elems * batch * p.splits * sizeof(float));
  for (int i = 0; i < (p.run > 0 || pairs(p.m, p.n, a.bf16 != 0) ? 5 : 2); ++i) p.mm_off[i] = take(p.a_bytes * batch);
  p.bytes = off;
  return p;
}

// Sums of squares in 64 bits, kNormBlocks partials a matrix; Muon's momentum is
// updated on the way (buf = mu buf + (1 - mu) g).  A matrix is dense in memory, so
// its elements are read as they lie, 16 bytes a load, four loads in flight.
enum NormKind { kNormF32, kNormBf16, kNormMuon };
template <int KIND>
__global__ __launch_bounds__(256) void k_ortho_norm(OrthoArgs a, double* part) {
  constexpr int N = KIND == kNormBf16 ? 8 : 4;
  const int b = blockIdx.y;
  const int64_t total = (int64_t)a.rows * a.cols, step = (int64_t)kNormBlocks * 256;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, base = b * a.view.sb;
  const char* src = (KIND == kNormMuon ? (const char*)a.g : (const char*)a.in) + base * (16 / N);
  float* buf = a.buf + base;
  double s = 0.0;
  auto muon = [&](float g, float& m) {
    m = fmaf(a.momentum, m, (1.0f - a.momentum) * g);
    const float v = muon_dir(g, m, a);
    s += (double)v * v;
  };
  // vectors where the matrix (and Muon's momentum) begin at a 16-byte boundary
  const uintptr_t at = (uintptr_t)src | (KIND == kNormMuon ? (uintptr_t)buf : 0);
  const int64_t nv = at & 15 ? 0 : total / N;
  for (int64_t i = first; i < nv; i += 4 * step) {
    u32x4_t w[4], m[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * step < nv) {
        w[u] = ((const u32x4_t*)src)[i + u * step];
        if constexpr (KIND == kNormMuon) m[u] = ((const u32x4_t*)buf)[i + u * step];
      }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + u * step >= nv) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (KIND == kNormBf16) {
          const float x = __uint_as_float(w[u][j] << 16), y = __uint_as_float(w[u][j] & 0xffff0000u);
          s += (double)x * x;
          s += (double)y * y;
        } else if constexpr (KIND == kNormF32) {
          const float v = __uint_as_float(w[u][j]);
          s += (double)v * v;
        } else {
          float nb = __uint_as_float(m[u][j]);
          muon(__uint_as_float(w[u][j]), nb);
          m[u][j] = __float_as_uint(nb);
        }
      }
      if constexpr (KIND == kNormMuon) ((u32x4_t*)buf)[i + u * step] = m[u];
    }
  }
  for (int64_t e = nv * N + first; e < total; e += step) {
    if constexpr (KIND == kNormMuon) {
      float nb = buf[e];
      muon(((const float*)src)[e], nb);
      buf[e] = nb;
    } else {
      const float v = entry(a, base + e);
      s += (double)v * v;
    }
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

__device__ __forceinline__ double norm_sum(const double* part, int b, double* red) {
  red[threadIdx.x] = part[b * kNormBlocks + threadIdx.x];
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  return red[0];
}

// The lift of X after some steps: the matrix's own, less what the steps may have grown X
// by (`used`, at most 1), and none below 1.
__device__ __forceinline__ float lift_at(const double* lift, int b, float used) { return fmaxf((float)lift[b] * used, 1.0f); }

// X0 in both operand forms: one block a 64 x 64 tile (m x n), through LDS.  In one
// plane the scale is a power of two and what it leaves goes to rest[b]: the matrix is then
// X0 / rest exactly.
template <int NP>
__global__ __launch_bounds__(256) void k_ortho_pack(OrthoArgs a, OrthoPlan p, const double* part, double* rest,
                                                    double* lift, char* xr, char* xc) {
  __shared__ float tile[64][65];
  __shared__ double red[256];
  const int b = blockIdx.z, m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tid = threadIdx.x;
  const float norm = (float)sqrt(norm_sum(part, b, red));
  float f = kS / (norm + a.eps);
  // the largest power of two that leaves |X0| below 1, and f below 2^120
  int up = 0, top = 0;
  if (norm > 0.0f && norm < a.eps) {
    frexpf(fminf((norm + a.eps) / norm, 0x1p100f), &up);
    frexpf(f, &top);
    up = up - 1 < 120 - top ? up - 1 : 120 - top;
    up = up > 0 ? up : 0;
  }
  const float own = ldexpf(1.0f, up);
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) lift[b] = (double)own;
  if constexpr (NP == 1) {
    int x;
    frexpf(f * own, &x);
    const float two = ldexpf(1.0f, x - 1);
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) rest[b] = (double)f / (double)two;
    f = two;
  } else {
    f *= own;
  }
  if (a.view.inner != 1 && !p.tall) {
    // memory runs along (row, inner column): 64 rows of each outer column in the tile
    const int D = a.view.inner, i0 = n0 / D, i1 = (n0 + 63) / D;
    for (int q = tid; q < 64 * 64; q += 256) tile[q >> 6][q & 63] = 0.0f;
    __syncthreads();
    for (int q = tid; q < (i1 - i0 + 1) * 64 * D; q += 256) {
      const int i = q / (64 * D), in = q - i * 64 * D, r = in / D, c = (i0 + i) * D + in - r * D;
      if (c < n0 || c >= n0 + 64 || c >= p.n || m0 + r >= p.m) continue;
      tile[r][c - n0] = f * entry(a, b * a.view.sb + (int64_t)(m0 + r) * a.view.sr + (int64_t)(i0 + i) * a.view.so +
                                         (int64_t)(in - r * D) * a.view.si);
    }
  } else {
    // memory runs along n for an ordinary matrix with rows m, along m for a transposed one
    const bool along_m = runs_along_m(a);
    for (int e = tid; e < 64 * 64; e += 256) {
      const int mi = along_m ? e & 63 : e >> 6, ni = along_m ? e >> 6 : e & 63;
      const int m = m0 + mi, n = n0 + ni;
      float v = 0.0f;
      if (m < p.m && n < p.n) v = f * entry(a, p.tall ? view_at(a.view, b, n, m) : view_at(a.view, b, m, n));
      tile[mi][ni] = v;
    }
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
      const Planes8<NP> f8 = to_planes8<NP>(v);
      const int row = m0 + r, kb = (n0 + k8 * 8) >> 4, g = k8 & 1;
      char* d = xr + b * p.xr_bytes + ((size_t)(row >> 5) * (p.n32 / 16) + kb) * NP * kPlaneBytes + ((row & 31) + 32 * g) * 16;
#pragma unroll
      for (int k = 0; k < NP; ++k) *(f16x8_t*)(d + k * kPlaneBytes) = f8.p[k];
    }
    if (n0 + r < p.n128 && m0 + k8 * 8 < p.mk) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = tile[k8 * 8 + j][r];
      const Planes8<NP> f8 = to_planes8<NP>(v);
      const int row = n0 + r, kb = (m0 + k8 * 8) >> 4, g = k8 & 1;
      char* d = xc + b * p.xc_bytes + ((size_t)(row >> 5) * (p.mk / 16) + kb) * NP * kPlaneBytes + ((row & 31) + 32 * g) * 16;
#pragma unroll
      for (int k = 0; k < NP; ++k) *(f16x8_t*)(d + k * kPlaneBytes) = f8.p[k];
    }
  }
}

// 128 x 128, 64 KiB of LDS.  On two planes each of the three plane products has its own
// sum: an entry then does not depend on which of its two rows is the tile's (h l and l h
// change places).  With one sum it did, equal rows of X in different tiles got rows of A
// that differed in a last bit, and what is no singular vector grew from there by
// 3.4 a step: 200 x 1500, rows 0-99 twice, was 4e-3 off after 12 steps and 0.7 after 20.
template <int NP> struct GramTile {
  static constexpr int kSums = NP == 1 ? 1 : 3;
  typedef NtTile<NP, NP, 2, 2, 2, 2, 2, NP == 1 ? 4 : 2, kSums> Tile;
};

// Partial sums of A = X X^T (scale kS^2): the tiles on and below the diagonal,
// each stored with its mirror image, k split over blocks.
template <int NP>
__global__ __launch_bounds__(256, 2) void k_ortho_gram(OrthoPlan p, const char* xr, float* part) {
  extern __shared__ char lds[];
  typedef typename GramTile<NP>::Tile Tile;
  constexpr int NC = GramTile<NP>::kSums;
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
  const size_t pitch = (size_t)KB * NP * kPlaneBytes;
  const char* x = xr + b * p.xr_bytes;
  f32x16_t acc[NC * 2][2] = {};
  Tile::run(RowBlocks{x + tm * 4 * pitch, pitch}, RowBlocks{x + tn * 4 * pitch, pitch}, kb0, kbs / Tile::kStageBlocks, lds, acc);
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
          const int r = q * 4 + j;
          v[j] = NC == 1 ? acc[m][n][r] : (acc[m][n][r] + acc[NC / 3 * 2 + m][n][r]) + acc[NC / 3 * 4 + m][n][r];
          if (tm != tn) out[(size_t)(row + 8 * q + 4 * g + j) * p.m128 + col] = v[j];
        }
        *(f32x4_t*)(out + (size_t)col * p.m128 + row + 8 * q + 4 * g) = v;
      }
    }
}

// A in planes from the partial sums: a thread a row and 8 k.  rest: X is X0 / rest of
// one plane; else X is lifted.
__global__ __launch_bounds__(256) void k_ortho_gram_sum(OrthoPlan p, const float* part, const double* rest, const double* lift,
                                                        float used, char* A) {
  const int b = blockIdx.y;
  const int k8s = p.mk / 8;
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (q >= (int64_t)p.m128 * k8s) return;
  const int k8 = (int)(q % k8s), row = (int)(q / k8s);
  const double u = rest ? rest[b] : 1.0 / (double)lift_at(lift, b, used);
  const float f = (float)(u * u) * kInvS;
  float v[8] = {};
  if (row < p.m) {
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
      const float* src = part + ((size_t)s * p.batch + b) * p.part_elems + (size_t)row * p.m128 + k8 * 8;
      const f32x4_t lo = *(const f32x4_t*)src, hi = *(const f32x4_t*)(src + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] += lo[j];
        v[4 + j] += hi[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k8 * 8 + j < p.m ? v[j] * f : 0.0f;
  }
  const Planes8<2> o = to_planes8<2>(v);
  char* d = A + b * p.a_bytes + ((size_t)(row >> 5) * (p.mk / 16) + (k8 >> 1)) * 2 * kPlaneBytes + ((row & 31) + 32 * (k8 & 1)) * 16;
  *(f16x8_t*)d = o.p[0];
  *(f16x8_t*)(d + kPlaneBytes) = o.p[1];
}

// The 8-byte half of a lane's planes that an accumulator quad (4 consecutive
// rows of the product) is in the operand whose k runs along those rows.
template <int NP>
__device__ __forceinline__ size_t quad_at(int row, int k, int KB) {
  return ((size_t)(row >> 5) * KB + (k >> 4)) * NP * kPlaneBytes + ((row & 31) + 32 * ((k >> 3) & 1)) * 16 + (k & 4) * 2;
}

// One product of m x m matrices: out = alpha L R^T + beta R + delta L + gamma I in planes
// (out2 the same times `two`).  All of them are symmetric, polynomials in one matrix, so
// the product's rows are stored as the operand's k.
struct MmJob {
  const char *l, *r;
  char *out, *out2;
  float alpha, beta, delta, gamma, two;
};
struct MmJobs { MmJob j[2]; };

// 64 x 64 tiles (128 x 128 ones leave most CUs without a block at these sizes): one
// block a CU, so kMmGroups groups of four waves divide a stage's k-blocks to have
// work while others wait.  At m = 1024 a launch takes 14-17 us, 13 of them its copies
// (16 KiB a k-block and CU): rings of 2 to 4 buffers, stages of 2 or 4 k-blocks, one
// or three accumulators and one or two groups all measure within 1 us.
constexpr int kMmGroups = 2;
typedef NtTile<2, 2, 2, 2, 1, 1, 4, 2, 3, kMmGroups> MmTile;  // 64 KiB of LDS

__global__ __launch_bounds__(256 * kMmGroups) void k_ortho_mm(OrthoPlan p, MmJobs jobs) {
  extern __shared__ char lds[];
  const MmJob& j = jobs.j[blockIdx.y];
  const int T = p.mk / 64, b = blockIdx.x / (T * T), t = blockIdx.x % (T * T);
  int tm = t / T, tn = t % T;
  if (T % 4 == 0) {
    // a patch of T/2 x T/4 tiles an XCD: 3/4 of the operands through its L2, where rows
    // of tiles in turn take 9/8 and more
    const int x = t & 7, u = t >> 3;
    tm = (x >> 2) * (T / 2) + u / (T / 4);
    tn = (x & 3) * (T / 4) + u % (T / 4);
  }
  const int KB = p.mk / 16;
  const size_t pitch = (size_t)KB * 2 * kPlaneBytes, at0 = b * p.a_bytes;
  f32x16_t acc[3][1] = {};
  MmTile::run(RowBlocks{j.l + at0 + tm * 2 * pitch, pitch}, RowBlocks{j.r + at0 + tn * 2 * pitch, pitch}, 0,
              KB / MmTile::kStageBlocks, lds, acc);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 5, quad = wave & 3, group = wave >> 2;
  f32x16_t sum;
#pragma unroll
  for (int q = 0; q < 16; ++q) sum[q] = (acc[0][0][q] + acc[1][0][q]) + acc[2][0][q];
  float* share = (float*)lds;  // the later groups' sums
  if (group > 0)
#pragma unroll
    for (int q = 0; q < 16; ++q) share[(((group - 1) * 4 + quad) * 16 + q) * 64 + lane] = sum[q];
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int s = 0; s < kMmGroups - 1; ++s)
#pragma unroll
    for (int q = 0; q < 16; ++q) sum[q] += share[((s * 4 + quad) * 16 + q) * 64 + lane];
  const int row0 = tm * 64 + (quad >> 1) * 32, col = tn * 64 + (quad & 1) * 32 + (lane & 31);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int k = row0 + 8 * q + 4 * g;
    const size_t at = at0 + quad_at<2>(col, k, KB);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = j.alpha * sum[q * 4 + i] + (k + i == col ? j.gamma : 0.0f);
    if (j.beta != 0.0f) {
      const f16x4_t h = *(const f16x4_t*)(j.r + at), l = *(const f16x4_t*)(j.r + at + kPlaneBytes);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fmaf(j.beta, (float)h[i] + (float)l[i], v[i]);
    }
    if (j.delta != 0.0f) {
      const f16x4_t h = *(const f16x4_t*)(j.l + at), l = *(const f16x4_t*)(j.l + at + kPlaneBytes);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fmaf(j.delta, (float)h[i] + (float)l[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i >= p.m || col >= p.m) v[i] = 0.0f;
    Planes4<2> f = to_planes4<2>(v);
    *(f16x4_t*)(j.out + at) = f.p[0];
    *(f16x4_t*)(j.out + at + kPlaneBytes) = f.p[1];
    if (j.out2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] *= j.two;
      f = to_planes4<2>(v);
      *(f16x4_t*)(j.out2 + at) = f.p[0];
      *(f16x4_t*)(j.out2 + at + kPlaneBytes) = f.p[1];
    }
  }
}

// Where entry (m, n) of a 128 x 128 result tile is staged in LDS: the direction in
// which it is stored is the contiguous one, except for a view with an inner
// dimension, whose outer columns are gathered at an odd pitch.
constexpr int kPutPitch = kTile + 4;
__device__ __forceinline__ int tile_at(bool along_m, bool gathered, int m, int n) {
  return gathered ? n * (kTile + 1) + m : along_m ? n * kPutPitch + m : m * kPutPitch + n;
}

// The staged tile to where it belongs.  Four elements a thread and step along the
// contiguous direction, in one access where the addresses allow; one element at a
// time cost the bf16 result's launch 40 of its 77 us.
__device__ __forceinline__ void put_tile(const OrthoArgs& a, const OrthoPlan& p, const float* tile, int b, int m0, int n0) {
  if (a.view.inner != 1 && !p.tall) {
    constexpr int U = 8;
    const int D = a.view.inner, i0 = n0 / D, i1 = (n0 + kTile - 1) / D;
    for (int in = threadIdx.x; in < kTile * D; in += 256) {
      const int r = in / D, d = in - r * D;
      if (m0 + r >= p.m) continue;
      const int64_t at = b * a.view.sb + (int64_t)(m0 + r) * a.view.sr + (int64_t)d * a.view.si;
      for (int i = i0; i <= i1; i += U) {
        float old[U];  // Muon's parameters, asked for before any of them is needed
        if (!a.in)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = (i + u) * D + d;
            if (i + u <= i1 && c >= n0 && c < n0 + kTile && c < p.n) old[u] = a.p[at + (int64_t)(i + u) * a.view.so];
          }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = (i + u) * D + d;
          if (i + u > i1 || c < n0 || c >= n0 + kTile || c >= p.n) continue;
          const float o = tile[tile_at(false, true, r, c - n0)];
          const int64_t e = at + (int64_t)(i + u) * a.view.so;
          if (!a.in)
            a.p[e] = muon_param(a, old[u], o);
          else
            put(a, e, o);
        }
      }
    }
    return;
  }
  const bool along_m = runs_along_m(a);
  const int c0 = along_m ? m0 : n0, r0 = along_m ? n0 : m0, cn = along_m ? p.m : p.n, rn = along_m ? p.n : p.m;
  // stride of the slow direction; the fast one is 1 (or `inner` runs of a tall view)
  const int64_t slow = p.tall == along_m ? a.view.sr : a.view.so;
  const int64_t base = b * a.view.sb + r0 * slow;
  const bool vec = a.view.inner == 1 && slow % 4 == 0 && (a.view.sb % 4 == 0 || p.batch == 1) &&
                   (((uintptr_t)(a.in ? a.out : (void*)a.p)) & 15) == 0;
#pragma unroll 4
  for (int q = threadIdx.x; q < kTile * kTile / 4; q += 256) {
    const int r = q / (kTile / 4), c = q % (kTile / 4) * 4;
    if (r0 + r >= rn || c0 + c >= cn) continue;
    const f32x4_t v = *(const f32x4_t*)(tile + r * kPutPitch + c);
    if (vec && c0 + c + 4 <= cn) {
      const int64_t e = base + r * slow + c0 + c;
      if (!a.in) {
        f32x4_t w = *(const f32x4_t*)(a.p + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = muon_param(a, w[j], v[j]);
        *(f32x4_t*)(a.p + e) = w;
      } else if (a.bf16) {
        bf16x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (__bf16)v[j];
        *(bf16x4_t*)((__bf16*)a.out + e) = w;
      } else {
        *(f32x4_t*)((float*)a.out + e) = v;
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = along_m ? c0 + c + j : r0 + r, n = along_m ? r0 + r : c0 + c + j;
      if (c0 + c + j < cn) put(a, p.tall ? view_at(a.view, b, n, m) : view_at(a.view, b, m, n), v[j]);
    }
  }
}
constexpr int kPutLds = kTile * kPutPitch * 4;

// X' = ax X + inv B X.  The product's rows are m, its columns n: an accumulator quad is 4
// consecutive k of Xc, where the old X is read and the new one stored; Xr goes
// through LDS.  The last step writes the result instead (or Muon's parameters).
// On one plane (NB = 1) X is X0 / rest and B the whole factor Q of the run's steps.
// 8 x [512, 4608]: 128 us for 300 MB of X read and written and 58 GFLOP of plane
// products, 1152 blocks in 512 places, the matrix pipe 19 % busy; 1024 x 9216 on one
// plane: 63 us, 620 TFLOP/s on its two products.
template <int NB> struct UpdateTile {
  typedef NtTile<2, NB, 2, 2, 2, 2, 2, NB == 1 ? 3 : 2> Tile;  // 72 or 64 KiB of LDS
  static constexpr int kLds = Tile::kLdsBytes > kPutLds ? Tile::kLdsBytes : kPutLds;
};
template <int NB>
__global__ __launch_bounds__(256, 2) void k_ortho_update(OrthoArgs a, OrthoPlan p, const char* B, const char* xc,
                                                         char* xc_new, char* xr, float ax, float inv, const double* rest,
                                                         const double* lift, float before, float after, int last) {
  extern __shared__ char lds[];
  typedef typename UpdateTile<NB>::Tile Tile;
  const int TM = p.m128 / kTile, TN = p.n128 / kTile;
  int id = blockIdx.x;
  const int tm = id % TM;
  id /= TM;
  const int tn = id % TN, b = id / TN;
  const int KB = p.mk / 16;
  const size_t pb = (size_t)KB * 2 * kPlaneBytes, px = (size_t)KB * NB * kPlaneBytes;
  const char* x = xc + b * p.xc_bytes;
  f32x16_t acc[2][2] = {};
  Tile::run(RowBlocks{B + b * p.a_bytes + tm * 4 * pb, pb}, RowBlocks{x + tn * 4 * px, px}, 0, KB / Tile::kStageBlocks, lds, acc);
  // from the lift before to the one after, or to the result
  const float to = last ? 1.0f : lift_at(lift, b, after);
  if constexpr (NB == 1) {
    inv *= (float)(rest[b] * (double)to);
  } else {
    const float by = to / lift_at(lift, b, before);
    ax *= by;
    inv *= by;
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 5;
  const bool gathered = a.view.inner != 1 && !p.tall, along_m = runs_along_m(a);
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
        const size_t at = quad_at<2>(col, k, KB);
        if constexpr (NB == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k + j < p.m && col < p.n) v[j] = acc[m][n][q * 4 + j] * inv;
        } else if (k < p.mk) {
          const f16x4_t h = *(const f16x4_t*)(x + at), l = *(const f16x4_t*)(x + at + kPlaneBytes);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k + j < p.m && col < p.n) v[j] = ax * ((float)h[j] + (float)l[j]) + acc[m][n][q * 4 + j] * inv;
        }
        if (last) {
#pragma unroll
          for (int j = 0; j < 4; ++j) ((float*)lds)[tile_at(along_m, gathered, r + j, c)] = v[j] * kInvS;
          continue;
        }
        const Planes4<2> f = to_planes4<2>(v);
        if (k < p.mk) {
          char* d = xc_new + b * p.xc_bytes + at;
          *(f16x4_t*)d = f.p[0];
          *(f16x4_t*)(d + kPlaneBytes) = f.p[1];
        }
        // both planes of an element in one LDS word: half the stores of two planes
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const _Float16 h = f.p[0][j], l = f.p[1][j];  // a bit cast of a vector's element takes the first one
          ((uint32_t*)lds)[(r + j) * kPutPitch + c] =
              (uint32_t)__builtin_bit_cast(uint16_t, h) | (uint32_t)__builtin_bit_cast(uint16_t, l) << 16;
        }
      }
    }
  __syncthreads();
  if (last) {
    put_tile(a, p, (const float*)lds, b, tm * kTile, tn * kTile);
    return;
  }
  // Xr: 128 rows x 16 groups of 8 k, 8 a thread
  const int KBr = p.n32 / 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = threadIdx.x + i * 256, r = q & 127, k8 = q >> 7;
    const int row = tm * kTile + r, k = tn * kTile + k8 * 8;
    if (k >= p.n32) continue;
    char* d = xr + b * p.xr_bytes + ((size_t)(row >> 5) * KBr + (k >> 4)) * 2 * kPlaneBytes + ((row & 31) + 32 * (k8 & 1)) * 16;
    const u32x4_t* src = (const u32x4_t*)((const uint32_t*)lds + r * kPutPitch + k8 * 8);
    const u32x4_t w0 = src[0], w1 = src[1];
    u32x4_t h, l;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      h[j] = (w0[2 * j] & 0xffffu) | w0[2 * j + 1] << 16;
      l[j] = w0[2 * j] >> 16 | (w0[2 * j + 1] & 0xffff0000u);
      h[j + 2] = (w1[2 * j] & 0xffffu) | w1[2 * j + 1] << 16;
      l[j + 2] = w1[2 * j] >> 16 | (w1[2 * j + 1] & 0xffff0000u);
    }
    *(u32x4_t*)d = h;
    *(u32x4_t*)(d + kPlaneBytes) = l;
  }
}

// steps == 0: the normalised matrix itself.
__global__ __launch_bounds__(256) void k_ortho_scale(OrthoArgs a, const double* part) {
  __shared__ double red[256];
  const int b = blockIdx.y;
  const float f = (float)sqrt(norm_sum(part, b, red)) + a.eps;
  const int64_t total = (int64_t)a.rows * a.cols;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256)
    put(a, b * a.view.sb + e, entry(a, b * a.view.sb + e) / f);
}

// The largest value of Q that singular values in [0, 1] give in a run of steps, by sampling.
float largest_q(const OrthoArgs& a, int run) {
  double most = 0.0;
  for (int i = 0; i <= 1024; ++i) {
    double x = i / 1024.0, q = 1.0;
    for (int s = 0; s < run; ++s) {
      const double f = a.a + a.b * x * x + a.c * x * x * x * x;
      q *= f;
      x *= f;
      most = fmax(most, fabs(q));
    }
  }
  return (float)most;
}

// 2^-k with 2^k at least what a step multiplies X by.
float step_use(const OrthoArgs& a) {
  double most = 1.0;
  for (int i = 0; i <= 1024; ++i) {
    double x = i / 1024.0;
    for (int s = 0; s < a.steps; ++s) {
      const double f = a.a + a.b * x * x + a.c * x * x * x * x;
      most = fmax(most, fabs(f));
      x *= f;
    }
  }
  int e;
  frexp(most, &e);
  return ldexpf(1.0f, -e);
}

// The largest |P_1 P_0 - a^2| of two steps in a row.
float largest_pair(const OrthoArgs& a) {
  double most = 0.0;
  for (int i = 0; i <= 1024; ++i) {
    double x = i / 1024.0, before = 1.0;
    for (int s = 0; s < a.steps; ++s) {
      const double f = a.a + a.b * x * x + a.c * x * x * x * x;
      if (s) most = fmax(most, fabs(before * f - (double)a.a * a.a));
      before = f;
      x *= f;
    }
  }
  return (float)most;
}

}  // namespace

size_t ortho_workspace_bytes(const OrthoArgs& a) {
  if (ortho_small(a.rows, a.cols)) return ortho_small_workspace_bytes(a);
  return make_ortho_plan(a).bytes;
}

void launch_ortho(const OrthoArgs& a, void* ws, hipStream_t st) {
  if (ortho_small(a.rows, a.cols)) {
    launch_ortho_small(a, ws, st);
    return;
  }
  OrthoPlan p = make_ortho_plan(a);
  char* w = (char*)ws;
  double *norm = (double*)(w + p.norm_off), *rest = norm + (size_t)a.batch * kNormBlocks, *lift = rest + a.batch;
  char* xr = w + p.xr_off;
  char* xc[2] = {w + p.xc_off[0], w + p.xc_off[1]};
  float* part = (float*)(w + p.part_off);
  char* mm[5];
  for (int i = 0; i < 5; ++i) mm[i] = w + p.mm_off[i];
  static std::atomic<uint32_t> done[5];
  ensure_lds_limit((const void*)k_ortho_gram<1>, GramTile<1>::Tile::kLdsBytes, done[0]);
  ensure_lds_limit((const void*)k_ortho_gram<2>, GramTile<2>::Tile::kLdsBytes, done[1]);
  ensure_lds_limit((const void*)k_ortho_mm, MmTile::kLdsBytes, done[2]);
  ensure_lds_limit((const void*)k_ortho_update<1>, UpdateTile<1>::kLds, done[3]);
  ensure_lds_limit((const void*)k_ortho_update<2>, UpdateTile<2>::kLds, done[4]);
  const dim3 norm_grid(kNormBlocks, a.batch);
  if (!a.in)
    hipLaunchKernelGGL(k_ortho_norm<kNormMuon>, norm_grid, dim3(256), 0, st, a, norm);
  else if (a.bf16)
    hipLaunchKernelGGL(k_ortho_norm<kNormBf16>, norm_grid, dim3(256), 0, st, a, norm);
  else
    hipLaunchKernelGGL(k_ortho_norm<kNormF32>, norm_grid, dim3(256), 0, st, a, norm);
  if (a.steps == 0) {
    hipLaunchKernelGGL(k_ortho_scale, dim3(kNormBlocks, a.batch), dim3(256), 0, st, a, norm);
    return;
  }
  const dim3 pack_grid(p.n128 / 64, p.m128 / 64, a.batch), block(256);
  const int T = p.m128 / kTile, TN = p.n128 / kTile, T64 = p.mk / 64;
  const dim3 gram_grid(a.batch * (T * (T + 1) / 2) * p.splits);
  const dim3 sum_grid((unsigned)ceil_div((int64_t)p.m128 * (p.mk / 8), 256), a.batch);
  auto products = [&](const MmJob& one, const MmJob* two) {
    MmJobs jobs{{one, two ? *two : one}};
    hipLaunchKernelGGL(k_ortho_mm, dim3(a.batch * T64 * T64, two ? 2 : 1), dim3(256 * kMmGroups), MmTile::kLdsBytes, st, p,
                       jobs);
  };
  const dim3 update_grid(a.batch * T * TN);
  char* x = xc[0];
  char* xn = xc[1];
  const float use = step_use(a);
  auto used = [&](int steps) {  // all of it where the power leaves fp32
    const int e = ilogbf(use) * steps;
    return e > -126 ? ldexpf(1.0f, e) : 0.0f;
  };
  int s = p.run;
  if (p.run == 0) {
    hipLaunchKernelGGL(k_ortho_pack<2>, pack_grid, block, 0, st, a, p, norm, rest, lift, xr, x);
  } else {
    int exponent;  // |Q| below 2^14 in its planes
    frexpf(largest_q(a, p.run), &exponent);
    p.qscale = ldexpf(1.0f, 14 - exponent > 12 ? 12 : 14 - exponent);
    hipLaunchKernelGGL(k_ortho_pack<1>, pack_grid, block, 0, st, a, p, norm, rest, lift, xr, x);
    hipLaunchKernelGGL(k_ortho_gram<1>, gram_grid, block, GramTile<1>::Tile::kLdsBytes, st, p, xr, part);
    hipLaunchKernelGGL(k_ortho_gram_sum, sum_grid, block, 0, st, p, part, rest, lift, 1.0f, mm[0]);
    char *A = mm[0], *P = mm[1], *W = mm[2], *Q = mm[3], *Qn = mm[4];
    for (int i = 0; i < p.run; ++i) {
      const bool more = i + 1 < p.run;
      products(MmJob{A, A, P, i == 0 ? Q : nullptr, a.c * kInvS, a.b, 0.0f, a.a * kS, p.qscale * kInvS}, nullptr);
      const MmJob pa{P, A, W, nullptr, kInvS, 0.0f, 0.0f, 0.0f, 0.0f}, qp{Q, P, Qn, nullptr, kInvS, 0.0f, 0.0f, 0.0f, 0.0f};
      if (i == 0) {
        if (more) products(pa, nullptr);
      } else {
        products(qp, more ? &pa : nullptr);
        char* q = Q;
        Q = Qn;
        Qn = q;
      }
      if (more) products(MmJob{W, P, A, nullptr, kInvS, 0.0f, 0.0f, 0.0f, 0.0f}, nullptr);
    }
    hipLaunchKernelGGL(k_ortho_update<1>, update_grid, block, UpdateTile<1>::kLds, st, a, p, Q, x, xn, xr, 0.0f,
                       1.0f / p.qscale, rest, lift, 1.0f, used(s), s == a.steps);
    x = xc[1];
    xn = xc[0];
  }
  const bool two = pairs(p.m, p.n, a.bf16 != 0) && largest_pair(a) < 31.0f;  // its planes at 2^11 hold 31.98
  constexpr float kS2 = 2048.0f;
  while (s < a.steps) {
    const int taken = two && s + 1 < a.steps ? 2 : 1;
    hipLaunchKernelGGL(k_ortho_gram<2>, gram_grid, block, GramTile<2>::Tile::kLdsBytes, st, p, xr, part);
    hipLaunchKernelGGL(k_ortho_gram_sum, sum_grid, block, 0, st, p, part, nullptr, lift, used(s), mm[0]);
    // B_s = b A_s + c A_s^2 = P_s - a I: the identity stays out of the planes
    const MmJob poly{mm[0], mm[0], mm[1], nullptr, a.c * kInvS, a.b, 0.0f, 0.0f, 0.0f};
    products(poly, nullptr);  // B_0
    if (taken == 2) {
      products(MmJob{mm[1], mm[0], mm[2], nullptr, kInvS, a.a, 0.0f, 0.0f, 0.0f}, nullptr);  // P_0 A_0 = a A_0 + B_0 A_0
      products(MmJob{mm[1], mm[2], mm[0], nullptr, kInvS, a.a, 0.0f, 0.0f, 0.0f}, nullptr);  // A_1 = P_0 (A_0 P_0)
      MmJob second = poly;
      second.out = mm[3];
      products(second, nullptr);  // B_1
      // P_1 P_0 - a^2 I = B_1 B_0 + a (B_0 + B_1); X itself enters with a^2 in fp32
      products(MmJob{mm[3], mm[1], mm[4], nullptr, kS2 * kInvS * kInvS, a.a * kS2 * kInvS, a.a * kS2 * kInvS, 0.0f, 0.0f},
               nullptr);
    }
    const int from = s;
    s += taken;
    hipLaunchKernelGGL(k_ortho_update<2>, update_grid, block, UpdateTile<2>::kLds, st, a, p, mm[taken == 1 ? 1 : 4], x, xn, xr,
                       taken == 1 ? a.a : a.a * a.a, taken == 1 ? kInvS : 1.0f / kS2, rest, lift, used(from), used(s), s == a.steps);
    char* o = x;
    x = xn;
    xn = o;
  }
}

}  // namespace ckan
