// The products of a mixture of ChebyKAN experts, forward and backward.
//
//   y[t] = sum_j w[t, j] f_e(x[t]),  e = idx[t, j],  f_e(x) = sum_{i, d} T_d(tanh x_i) C_e[i, :, d].
//
// The slots (t, j) are sorted by expert on the device, each expert's run padded to
// 32 rows, so one launch a product covers every expert and nothing is read back
// by the host.  All three products run on fp16 planes (ckan_planes.hpp): one
// plane for bf16 tensors (the basis values then carry 11 bits, more than a bf16
// result), two for fp32.  fp16's range is met by powers of two: one an expert for the
// coefficients; for the upstream gradients one a row in dx, where rows stay apart, and
// one an expert in dC, where they are summed; the basis values lie in [-1, 1].
//
//   forward  z[row, o] = sum_k phi[row, k] Cf[o, k]: phi is made in registers from
//            the row's tanh values, k = (input, degree 1..P); T_0 is a bias.
//   dx       per row and input the degrees' sums over o of g[row, o] d C[i, o, d]
//            stand in separate accumulators; the epilogue weights them by
//            U_{d-1}(t) (1 - t^2).
//   dC       sum over rows of T_d(t) g: phi is made into LDS, k = the rows.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "ckan_mix.hpp"
#include "ckan_planes.hpp"

namespace ckan {

ExpertsPlan make_experts_plan(int64_t T, int E, int k, int I, int O, int deg, bool bf16, bool wbf16) {
  ExpertsPlan p{};
  p.T = T;
  p.S = T * k;
  p.E = E;
  p.k = k;
  p.I = I;
  p.O = O;
  p.deg = deg;
  p.D = deg + 1;
  p.P = deg <= 4 ? 4 : deg <= 8 ? 8 : 16;
  p.NP = bf16 ? 1 : 2;
  p.bf16 = bf16;
  p.wbf16 = wbf16;
  p.Ip = (int)round_up(I, 32);
  p.Op = (int)round_up(O, 32);
  p.R = round_up(p.S + (int64_t)31 * (E < p.S ? E : p.S), 128) + 128;
  p.tiles = (int)(ceil_div(p.S, 128) + (E < p.S ? E : p.S));
  p.plan_chunk = round_up(ceil_div(p.S, kPlanBlocks), kPlanThreads);
  p.plan_blocks = (int)ceil_div(p.S, p.plan_chunk);
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off = align256(off + n);
    return at;
  };
  p.off_off = take((size_t)(E + 2) * 4);
  p.tok_off = take((size_t)p.R * 4);
  p.slot_off = take((size_t)p.R * 4);
  p.row_off = take((size_t)p.S * 4);
  p.tiles_off = take((size_t)p.tiles * 8);
  p.order_off = take((size_t)E * 4);
  p.scale_off = take((size_t)E * 4);
  p.t_off = take((size_t)p.T * p.Ip * 4);
  p.z_off = take((size_t)p.R * O * 4);
  p.cb_off = take((size_t)E * p.Ip * deg * p.Op * 2 * p.NP);
  p.saved_bytes = off;
  off = 0;
  // inputs a block of the pack takes: 128, fewer where that leaves under four blocks a CU
  // (6 experts, 500 -> 300, degree 5, fp32: 32 inputs 14 us, 128 20)
  p.pack_inputs = 128;
  while (p.pack_inputs > 32 && ceil_div(p.Ip, p.pack_inputs) * (p.Op / 32) * E < 4 * kNumCUs) p.pack_inputs /= 2;
  p.bias_parts = (int)ceil_div(p.Ip, p.pack_inputs);
  p.hist_off = take((size_t)p.plan_blocks * E * 4);
  p.cmax_off = take((size_t)E * kMaxParts * 4);
  p.cf_off = take((size_t)E * p.Op * p.Ip * p.P * 2 * p.NP);
  p.bias_off = take((size_t)p.bias_parts * E * p.Op * 4);
  p.fpart_off = take((size_t)512 * 128 * 256 * 4);
  p.fwd_bytes = off;
  off = 0;
  p.gmax_off = take((size_t)(p.R / 32) * 4);
  p.gscale_off = take((size_t)E * 4);
  p.rscale_off = take((size_t)p.R * 4);
  p.gr_off = take((size_t)p.R * p.Op * 2 * p.NP);
  p.gt_off = take((size_t)p.R * p.Op * 2 * p.NP);
  p.gsum_off = take((size_t)(p.R / 32) * p.Op * 4);
  p.gtot_off = take((size_t)E * p.Op * 4);
  p.ts_off = take((size_t)p.R * p.Ip * 4);
  p.dxs_off = take((size_t)p.R * I * 4);
  p.bpart_off = take((size_t)512 * 128 * 64 * 4);
  p.bwd_bytes = off;
  // Streaming: up to 16 slots an expert on average.  Its blocks read the coefficients
  // as they lie, once for 8 rows; the tile path reads them twice and packs them
  // before its products start.
  const int64_t active = E < p.S ? E : p.S, oc = ceil_div(O, 64);
  p.stream = p.S <= kStreamMaxSlots && p.S <= 16 * active;
  int64_t chunks = ceil_div(8 * kNumCUs, active * oc);
  if (chunks > ceil_div(I, 16)) chunks = ceil_div(I, 16);
  if (chunks < ceil_div(I, kStreamInputs)) chunks = ceil_div(I, kStreamInputs);
  p.chunk_inputs = (int)round_up(ceil_div(I, chunks), 4);
  if (p.chunk_inputs > kStreamInputs) p.chunk_inputs = kStreamInputs;
  p.chunks = (int)ceil_div(I, p.chunk_inputs);
  p.part_off = 0;
  p.stream_bytes = p.stream ? align256((size_t)p.chunks * p.S * O * 4) : 0;
  return p;
}

namespace {

// ---- the plan: slots sorted by expert ----------------------------------------

__device__ __forceinline__ int slot_expert(const ExpertsArgs& a, int64_t s) {
  const int64_t e = a.indices[s];
  return e >= 0 && e < a.p.E ? (int)e : -1;
}

__global__ __launch_bounds__(kPlanThreads) void k_plan_count(ExpertsArgs a) {
  __shared__ int count[kExpertsMax];
  const ExpertsPlan& p = a.p;
  for (int e = threadIdx.x; e < p.E; e += kPlanThreads) count[e] = 0;
  __syncthreads();
  const int64_t s0 = blockIdx.x * p.plan_chunk;
  for (int64_t s = s0 + threadIdx.x; s < s0 + p.plan_chunk && s < p.S; s += kPlanThreads) {
    const int e = slot_expert(a, s);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  int* hist = (int*)(a.ws + p.hist_off) + (size_t)blockIdx.x * p.E;
  for (int e = threadIdx.x; e < p.E; e += kPlanThreads) hist[e] = count[e];
}

// Each block scans the counts again (a few kilobytes from the L2) instead of
// waiting for a launch that does, then places its own slots: within a wave
// by the lanes before it of the same expert (one ballot a bit of the number),
// among the waves of the block by their counts.  The order within an expert is
// the slots' order, whatever the blocks' timing.
__global__ __launch_bounds__(kPlanThreads) void k_plan_place(ExpertsArgs a) {
  constexpr int kWaves = kPlanThreads / 64;
  __shared__ int next[kExpertsMax], scan[2][kExpertsMax], wave_count[kWaves][kExpertsMax];
  const ExpertsPlan& p = a.p;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int* hist = (const int*)(a.ws + p.hist_off);
  int total = 0, before = 0;
  if (tid < p.E)
    for (int b = 0; b < p.plan_blocks; ++b) {
      const int h = hist[(size_t)b * p.E + tid];
      total += h;
      if (b < (int)blockIdx.x) before += h;
    }
  const int padded = (total + 31) / 32 * 32, ntiles = (total + 127) / 128;
  if (blockIdx.x == 0) {  // the experts by falling row count
    if (tid < p.E) next[tid] = total;
    __syncthreads();
    if (tid < p.E) {
      int ahead = 0;
      for (int e = 0; e < p.E; ++e) ahead += next[e] > total || (next[e] == total && e < tid);
      ((int*)(a.saved + p.order_off))[ahead] = tid;
    }
    __syncthreads();
  }
  int sum[2] = {padded, ntiles};  // inclusive sums over the experts of rows and of tiles
  for (int which = 0; which < 2; ++which) {
    if (tid < kExpertsMax) scan[0][tid] = tid < p.E ? sum[which] : 0;
    __syncthreads();
    int cur = 0;
    for (int w = 1; w < p.E; w <<= 1) {
      if (tid < kExpertsMax) scan[cur ^ 1][tid] = scan[cur][tid] + (tid >= w ? scan[cur][tid - w] : 0);
      __syncthreads();
      cur ^= 1;
    }
    if (tid < p.E) sum[which] = scan[cur][tid];
    __syncthreads();
  }
  int* off = (int*)(a.saved + p.off_off);
  int* tok = (int*)(a.saved + p.tok_off);
  int* slot = (int*)(a.saved + p.slot_off);
  int* row = (int*)(a.saved + p.row_off);
  if (tid < p.E) {
    next[tid] = sum[0] - padded + before;
    if (blockIdx.x == 0) {
      off[tid + 1] = sum[0];
      if (tid == 0) off[0] = 0;
      for (int r = sum[0] - padded + total; r < sum[0]; ++r) tok[r] = slot[r] = -1;
      int2* tiles = (int2*)(a.saved + p.tiles_off);
      for (int i = 0; i < ntiles; ++i) tiles[sum[1] - ntiles + i] = make_int2(tid, sum[0] - padded + i * 128);
      if (tid == p.E - 1) off[p.E + 1] = sum[1];
    }
  }
  const int64_t s0 = blockIdx.x * p.plan_chunk;
  for (int64_t s = s0; s < s0 + p.plan_chunk && s < p.S; s += kPlanThreads) {
    for (int e = lane; e < p.E; e += 64) wave_count[wave][e] = 0;
    __syncthreads();
    const int64_t mine = s + tid;
    const int e = mine < p.S ? slot_expert(a, mine) : -1;
    unsigned long long same = __ballot(e >= 0);
    for (int bit = 1; bit < p.E; bit <<= 1) {
      const unsigned long long has = __ballot(e & bit);
      same &= (e & bit) ? has : ~has;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (e >= 0 && rank == 0) wave_count[wave][e] = __popcll(same);
    __syncthreads();
    if (tid < p.E) {
      int at = next[tid];
      for (int w = 0; w < kWaves; ++w) {
        const int c = wave_count[w][tid];
        wave_count[w][tid] = at;
        at += c;
      }
      next[tid] = at;
    }
    __syncthreads();
    if (mine < p.S) {
      int r = -1;
      if (e >= 0) {
        r = wave_count[wave][e] + rank;
        tok[r] = (int)(mine / p.k);
        slot[r] = (int)mine;
      }
      row[mine] = r;
    }
    __syncthreads();
  }
}

// ---- tanh, scales, packed coefficients ----------------------------------------

// Sixteen bytes of T as floats: 8 bf16 or 4 fp32 values.
template <typename T> struct Vec16 { static constexpr int N = 16 / (int)sizeof(T); };
__device__ __forceinline__ void widen(u32x4_t q, float (&v)[4], const float*) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(q[j]);
}
__device__ __forceinline__ void widen(u32x4_t q, float (&v)[8], const __bf16*) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(q[j] << 16);
    v[2 * j + 1] = __uint_as_float(q[j] & 0xffff0000u);
  }
}

// Four consecutive values of a row, from a vector load where every row begins at a
// multiple of four values (n the row's length, the values past it zeros).
__device__ __forceinline__ f32x4_t load4(const float* row, int c, int n, bool vec) {
  if (vec) return *(const f32x4_t*)(row + c);
  f32x4_t v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = c + j < n ? row[c + j] : 0.0f;
  return v;
}
__device__ __forceinline__ f32x4_t load4(const __bf16* row, int c, int n, bool vec) {
  f32x4_t v;
  if (vec) {
    const bf16x4_t b = *(const bf16x4_t*)(row + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)b[j];
    return v;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = c + j < n ? (float)row[c + j] : 0.0f;
  return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* row, int c, int n, bool vec, f32x4_t v) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *(f32x4_t*)(row + c) = v;
    } else {
      bf16x4_t b;
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = (__bf16)v[j];
      *(bf16x4_t*)(row + c) = b;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < n) row[c + j] = (T)v[j];
}

template <typename T>
__global__ __launch_bounds__(256) void k_experts_tanh(ExpertsArgs a) {
  const ExpertsPlan& p = a.p;
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = p.Ip / 4;
  const int64_t r = q / per;
  if (r >= p.T) return;
  const int i = (int)(q - r * per) * 4;
  f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (i < p.I) v = load4((const T*)a.x + r * p.I, i, p.I, p.I % 4 == 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = tanhf(v[j]);
  *(f32x4_t*)((float*)(a.saved + p.t_off) + r * p.Ip + i) = v;
}

// The power of two that brings a largest magnitude m into [2^(e-1), 2^e).
__device__ __forceinline__ float range_scale(float m, int e) {
  if (!(m > 0.0f)) return 1.0f;
  int x;
  frexpf(m, &x);
  x = e - x;
  return ldexpf(1.0f, x > 126 ? 126 : x < -126 ? -126 : x);
}
__device__ __forceinline__ float finite_abs(float v) {
  const float m = fabsf(v);
  return m <= FLT_MAX ? m : 0.0f;  // infinities and NaN set no scale; on two planes both come out as NaN (inf - inf)
}
__device__ __forceinline__ float block_max_256(float v, float* red) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) v = fmaxf(v, __shfl_xor(v, w));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  return v;
}

// The largest finite |C| of each expert by blocks; four 16-byte loads in flight a
// thread (2-byte loads took 450 us for 151 MB where these take 35).
template <typename T>
__global__ __launch_bounds__(256) void k_experts_cmax(ExpertsArgs a) {
  __shared__ float red[4];
  constexpr int N = Vec16<T>::N;
  const ExpertsPlan& p = a.p;
  const int e = blockIdx.y;
  const int64_t n = (int64_t)p.I * p.O * p.D;
  const T* c = (const T*)a.coeffs + e * n;
  // the elements before the expert's first 16-byte boundary and past its last
  int64_t head = ((16 - ((uintptr_t)c & 15)) & 15) / sizeof(T);
  if (head > n) head = n;
  const int64_t nv = (n - head) / N, step = (int64_t)kMaxParts * 256;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const u32x4_t* q = (const u32x4_t*)(c + head);
  float m = 0.0f;
  for (int64_t i = first; i < nv; i += 4 * step) {
    u32x4_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * step < nv) w[u] = q[i + u * step];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * step < nv) {
        float v[N];
        widen(w[u], v, c);
#pragma unroll
        for (int j = 0; j < N; ++j) m = fmaxf(m, finite_abs(v[j]));
      }
  }
  if (first < head) m = fmaxf(m, finite_abs((float)c[first]));
  if (head + nv * N + first < n) m = fmaxf(m, finite_abs((float)c[head + nv * N + first]));
  m = block_max_256(m, red);
  if (threadIdx.x == 0) ((float*)(a.ws + p.cmax_off))[e * kMaxParts + blockIdx.x] = m;
}

int64_t xcd_grid(int64_t n) { return (n + 7) / 8 * 8; }

// The share of a product over W equal output tiles that a block takes.  Blocks are
// spread over the eight XCDs in turn; XCD x gets the x-th eighth of the tiles, so that
// blocks which share operands share an L2.  64 blocks run on an XCD at once: its
// tiles past the last whole round of 64 are each split along k into up to
// kMaxSplits parts (few tiles altogether are the same case), whose partial
// results a second launch sums in order.  528 tiles in 512 places took the time of
// two whole rounds.
constexpr int kMaxSplits = 8, kXcdBlocks = 64;
struct Share {
  int v;            // the tile; -1: none
  int part, parts;  // this block's part of its k
  int place;        // of the partial result among kXcdBlocks of the XCD
};
__device__ __forceinline__ Share split_rule(int xcd, int W, int& full, int& rest, int& parts) {
  const int per = (W + 7) / 8, n = W - xcd * per < per ? W - xcd * per : per;
  full = n > 0 ? n / kXcdBlocks * kXcdBlocks : 0;
  rest = n > 0 ? n - full : 0;
  parts = rest ? kXcdBlocks / rest : 1;
  parts = parts < kMaxSplits ? parts : kMaxSplits;
  return Share{xcd * per, 0, 1, 0};
}
__device__ __forceinline__ Share block_share(int block, int W) {
  int full, rest, parts;
  Share s = split_rule(block & 7, W, full, rest, parts);
  const int j = block >> 3;
  if (j < full) {
    s.v += j;
  } else if (j - full < rest * parts) {
    s.place = j - full;
    s.part = s.place % parts;
    s.parts = parts;
    s.v += full + s.place / parts;
  } else {
    s.v = -1;
  }
  return s;
}
// The time of W tiles shared out so, in rounds of whole tiles.
double share_rounds(int64_t W) {
  const int64_t n = ceil_div(W, 8), rest = n % kXcdBlocks;
  const int64_t parts = rest ? kXcdBlocks / rest : 1;
  return (double)(n / kXcdBlocks) + (rest ? 1.0 / (parts < kMaxSplits ? parts : kMaxSplits) : 0.0);
}
int64_t share_grid(int64_t most) { return 8 * (ceil_div(most, 8) + kXcdBlocks); }

// (tile, column block) of a product's block: 16 tiles go through one column block
// before the next, so the 64 blocks that an XCD runs at once read about four
// column blocks of the packed coefficients and 16 tiles of rows.
__device__ __forceinline__ void tile_and_column(int v, int tiles, int cols, int& tile, int& col) {
  constexpr int G = 16;
  const int group = v / (G * cols), in = v - group * G * cols;
  const int size = tiles - group * G < G ? tiles - group * G : G;
  col = in / size;
  tile = group * G + in - col * size;
}

// The forward's stages: KS k-blocks, the IN inputs that they hold, and the ring of
// LDS buffers.  One plane: short stages, three ahead (the copies of a stage take
// longer than its products); two planes: a stage's products take three times as
// long and one ahead is enough.
template <int NP, int P> struct FwdStage {
  static constexpr int KS = P == 16 ? 4 : 2;
  static constexpr int IN = KS * 16 / P;
  static constexpr int NBUF = NP == 1 && P < 16 ? 4 : 2;
};

// Cf: the forward's operand, rows o, k in stages of IN inputs: half g of a lane
// pair holds inputs g IN/2.., P degrees each, eight values a k-block.  Cb: the dx
// operand, rows i and k = o for each degree d, scaled by d.  And the sums over the
// inputs of the T_0 coefficients.  A block takes 32 outputs and p.pack_inputs inputs of
// an expert, 16 inputs at a time through LDS, the next 16 inputs' loads in flight
// meanwhile.
template <typename T, int NP, int P, bool VEC>
__global__ __launch_bounds__(256) void k_experts_pack(ExpertsArgs a, bool backward) {
  extern __shared__ float sm[];
  __shared__ float red[4];
  using FS = FwdStage<NP, P>;
  constexpr int N = VEC ? Vec16<T>::N : 1;
  constexpr int kLoads = 16 * 32 * (P + 1) / N / 256 + 1;  // vectors a thread, at degree P
  const ExpertsPlan& p = a.p;
  const int e = blockIdx.z, ob = blockIdx.y, tid = threadIdx.x;
  const int D = p.D, W = 32 * D + 1;  // a row of the tile: 32 outputs, D coefficients each
  const float* cmax = (const float*)(a.ws + p.cmax_off) + e * kMaxParts;
  // d C with d <= 16 has to fit too: the largest |C| below 2^11
  const float scale = range_scale(block_max_256(cmax[tid % kMaxParts], red), 11);
  if (blockIdx.x == 0 && ob == 0 && tid == 0) ((float*)(a.saved + p.scale_off))[e] = scale;
  const T* C = (const T*)a.coeffs + (int64_t)e * p.I * p.O * D;
  char* cf = a.ws + p.cf_off + (size_t)e * p.Op * p.Ip * P * 2 * NP;
  char* cb = a.saved + p.cb_off + (size_t)e * p.Ip * p.deg * p.Op * 2 * NP;
  const int KBf = p.Ip * P / 16, KBo = p.Op / 16;
  const int o0 = ob * 32, no = p.O - o0 < 32 ? p.O - o0 : 32;
  const int vrow = 32 * D / N;  // vectors of an input
  float bias = 0.0f;
  const int i_end = (int)(blockIdx.x + 1) * p.pack_inputs < p.Ip ? (int)(blockIdx.x + 1) * p.pack_inputs : p.Ip;
  u32x4_t w[VEC ? kLoads : 1];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int q = tid + u * 256, i = q / vrow, f = (q - i * vrow) * N;
      w[u] = u32x4_t{0, 0, 0, 0};
      if (i < 16 && i0 + i < p.I && f < no * D) w[u] = *(const u32x4_t*)(C + ((int64_t)(i0 + i) * p.O + o0) * D + f);
    }
  };
  if constexpr (VEC) load((int)blockIdx.x * p.pack_inputs);
  for (int i0 = (int)blockIdx.x * p.pack_inputs; i0 < i_end; i0 += 16) {
    __syncthreads();
    if constexpr (VEC) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
          const int q = tid + u * 256, i = q / vrow, f = (q - i * vrow) * N;
        if (i >= 16) continue;
        float v[N];
        widen(w[u], v, C);
#pragma unroll
        for (int j = 0; j < N; ++j) sm[i * W + f + j] = v[j];
      }
    } else {
      for (int q = tid; q < 16 * 32 * D; q += 256) {
        const int i = q / (32 * D), f = q - i * 32 * D;
        sm[i * W + f] = i0 + i < p.I && f < no * D ? (float)C[((int64_t)(i0 + i) * p.O + o0) * D + f] : 0.0f;
      }
    }
    __syncthreads();
    if constexpr (VEC)
      if (i0 + 16 < i_end) load(i0 + 16);
    if (tid < 32)
      for (int i = 0; i < 16; ++i) bias += sm[i * W + tid * D];
    // Cf: P k-blocks of 64 lanes
    for (int q = tid; q < 64 * P; q += 256) {
      const int lane = q & 63, kb = q >> 6;  // k-block of the 16 inputs
      const int stage = kb / FS::KS, j = kb % FS::KS;
      float v[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const int u = j * 8 + s;
        const int i = stage * FS::IN + (lane >> 5) * (FS::IN / 2) + u / P, d = u % P + 1;
        v[s] = d < D ? scale * sm[i * W + (lane & 31) * D + d] : 0.0f;
      }
      const Planes8<NP> f = to_planes8<NP>(v);
      char* dst = cf + (((size_t)ob * KBf + i0 * P / 16 + kb) * NP) * kPlaneBytes + lane * 16;
#pragma unroll
      for (int k = 0; k < NP; ++k) *(f16x8_t*)(dst + k * kPlaneBytes) = f.p[k];
    }
    // Cb: for each degree 16 rows (half a row block) x 4 groups of 8 outputs
    if (backward)
      for (int q = tid; q < 64 * p.deg; q += 256) {
        const int i = q & 15, k8 = (q >> 4) & 3, d = (q >> 6) + 1;
        float v[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) v[s] = (float)d * scale * sm[i * W + (k8 * 8 + s) * D + d];
        const Planes8<NP> f = to_planes8<NP>(v);
        const int row = i0 + i;
        char* dst = cb + (((((size_t)(row >> 5) * p.deg + d - 1) * KBo) + ob * 2 + (k8 >> 1)) * NP) * kPlaneBytes +
                    ((row & 31) + 32 * (k8 & 1)) * 16;
#pragma unroll
        for (int k = 0; k < NP; ++k) *(f16x8_t*)(dst + k * kPlaneBytes) = f.p[k];
      }
  }
  if (tid < 32) ((float*)(a.ws + p.bias_off))[((size_t)blockIdx.x * p.E + e) * p.Op + o0 + tid] = bias;
}

// ---- forward ------------------------------------------------------------------

// 128 rows x 64 FN columns a block, four waves of 64 x 32 FN.  Each stage copies the
// rows' tanh values of IN inputs (gathered by token) and KS k-blocks of Cf to LDS;
// a wave makes its rows' basis values in registers, eight values of one or two
// inputs a lane and k-block: a fragment of 12 vector instructions serves four
// matrix ones.  16384 slots, 1024 -> 1024, degree 8, bf16: 340 us within a step
// (808 TFLOP/s), 317 at best, the matrix pipe 45 % busy; of 311 in an early trial without
// its copies 278, without the recurrence 301.
// Shorter stages than these wait at their barriers.  FN = 2 (128 columns) where wide tiles
// would be few.
template <int NP, int P, int FN>
__global__ __launch_bounds__(256, 2) void k_experts_fwd(ExpertsArgs a) {
  extern __shared__ char lds[];
  using FS = FwdStage<NP, P>;
  constexpr int KS = FS::KS, IN = FS::IN, NBUF = FS::NBUF;
  constexpr int TB = IN * 4;  // bytes of a row's tanh values a stage
  constexpr int kT = 128 * TB, kB = 2 * FN * KS * NP;  // bytes, 1 KiB chunks
  constexpr int kStage = kT + kB * kPlaneBytes;
  const ExpertsPlan& p = a.p;
  const int cols = (p.O + 64 * FN - 1) / (64 * FN), tiles = ((const int*)(a.saved + p.off_off))[p.E + 1];
  const Share share = block_share(blockIdx.x, tiles * cols);
  if (share.v < 0) return;
  int ti, cb;
  tile_and_column(share.v, tiles, cols, ti, cb);
  const int2 tile = ((const int2*)(a.saved + p.tiles_off))[ti];
  const int e = tile.x, row0 = tile.y;
  const int end = ((const int*)(a.saved + p.off_off))[e + 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave >> 1, wn = wave & 1, g = lane >> 5;
  const int* tok = (const int*)(a.saved + p.tok_off);
  const float* t = (const float*)(a.saved + p.t_off);
  const int KB = p.Ip * P / 16, nb = p.Op / 32;
  const int s0 = KB / KS * share.part / share.parts, nst = KB / KS * (share.part + 1) / share.parts - s0;
  const char* cf = a.ws + p.cf_off + (size_t)e * p.Op * p.Ip * P * 2 * NP;
  const size_t pitch = (size_t)KB * NP * kPlaneBytes;
  const uint32_t l0 = lds_address(lds);
  // this wave's tanh copies: its 32 rows of the tile, 16 bytes a lane (half the lanes
  // where a row has 16), the same count for every wave
  constexpr int kTPer = (32 * TB + 1023) / 1024;
  const float* tsrc[kTPer];
#pragma unroll
  for (int i = 0; i < kTPer; ++i) {
    const int byte = i * 1024 + lane * 16, r = row0 + wave * 32 + byte / TB % 32;
    int k = r < end ? tok[r] : 0;
    if (k < 0) k = 0;  // a pad row: any values, its results are not stored
    tsrc[i] = t + (int64_t)k * p.Ip + byte % TB / 4;
  }
  auto copy = [&](int s, uint32_t at) {
#pragma unroll
    for (int i = 0; i < kTPer; ++i)
      if (32 * TB >= 1024 || lane * 16 < 32 * TB) dma16v(tsrc[i] + (s0 + s) * IN, at + wave * 32 * TB + i * 1024);
#pragma unroll
    for (int i = 0; i < kB / 4; ++i) {
      const int c = i * 4 + wave;
      int rb = cb * 2 * FN + c / (KS * NP);
      rb = rb < nb ? rb : nb - 1;  // past the outputs: any, not stored
      dma16s(cf + rb * pitch + ((size_t)(s0 + s) * KS * NP + c % (KS * NP)) * kPlaneBytes, lane * 16, at + kT + c * kPlaneBytes);
    }
  };
  constexpr int kPer = kTPer + kB / 4;  // copies a wave and stage
  f32x16_t acc[2][FN] = {};
#pragma unroll
  for (int s = 0; s < NBUF - 1; ++s)
    if (s < nst) copy(s, l0 + s * kStage);
  int cur = 0;
  for (int s = 0; s < nst; ++s) {
    if (NBUF > 2 && nst - 1 - s >= NBUF - 2)
      wait_vm<kPer * (NBUF - 2)>();
    else
      wait_vm<0>();
    wait_lds();
    block_barrier();
    if (s + NBUF - 1 < nst) copy(s + NBUF - 1, l0 + (cur == 0 ? NBUF - 1 : cur - 1) * kStage);
    const char* buf = lds + cur * kStage;
    if (++cur == NBUF) cur = 0;
    float tv[2][IN / 2], pa[2], pb[2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int q = 0; q < IN / 2; ++q)
        tv[m][q] = ((const float*)(buf + (wm * 64 + m * 32 + (lane & 31)) * TB + g * (TB / 2)))[q];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      f16x8_t fa[2][NP], fb[FN][NP];
#pragma unroll
      for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int q = 0; q < NP; ++q)
          fb[n][q] = lds_frag(buf + kT + (((wn * FN + n) * KS + k) * NP + q) * kPlaneBytes, lane);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int d = (k * 8 + u) % P;  // T_{d+1} of input (k 8 + u) / P
          const float x = tv[m][(k * 8 + u) / P];
          if (d == 0) {
            pa[m] = 1.0f;
            pb[m] = x;
          } else {
            const float c = fmaf(x + x, pb[m], -pa[m]);
            pa[m] = pb[m];
            pb[m] = c;
          }
          v[u] = pb[m];
        }
        const Planes8<NP> f = to_planes8<NP>(v);
#pragma unroll
        for (int q = 0; q < NP; ++q) fa[m][q] = f.p[q];
      }
      mfma_planes<NP, NP, 2, FN>(fa, fb, acc);
    }
  }
  const float inv = 1.0f / ((const float*)(a.saved + p.scale_off))[e];
  if (share.parts > 1) {
    float* part = (float*)(a.ws + p.fpart_off) + ((size_t)(blockIdx.x & 7) * kXcdBlocks + share.place) * 128 * 256;
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int q = 0; q < 16; ++q)
          part[(wm * 64 + m * 32 + acc_row(q, g)) * 256 + (wn * FN + n) * 32 + (lane & 31)] = acc[m][n][q] * inv;
    return;
  }
  const float* bias = (const float*)(a.ws + p.bias_off);
  float* z = (float*)(a.saved + p.z_off);
#pragma unroll
  for (int n = 0; n < FN; ++n) {
    const int o = (cb * 2 * FN + wn * FN + n) * 32 + (lane & 31);
    if (o >= p.O) continue;
    float b = 0.0f;
    for (int k = 0; k < p.bias_parts; ++k) b += bias[((size_t)k * p.E + e) * p.Op + o];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const int r = row0 + wm * 64 + m * 32 + acc_row(q, g);
        if (r < end) z[(size_t)r * p.O + o] = fmaf(acc[m][n][q], inv, b);
      }
  }
}

// The tiles that block_share split: the sum of their parts, in order, four columns a
// thread.  dx: the inputs' gradients of 64 columns a tile; else the forward's outputs
// of `width` columns and their bias.
template <bool DX>
__global__ __launch_bounds__(256) void k_experts_parts(ExpertsArgs a, int width) {
  const ExpertsPlan& p = a.p;
  const int n = DX ? p.I : p.O, cols = ((DX ? p.Ip : p.O) + width - 1) / width;
  const int tiles = ((const int*)(a.saved + p.off_off))[p.E + 1];
  const int xcd = blockIdx.x & 7, u = blockIdx.x >> 3;
  int full, rest, parts;
  const Share s = split_rule(xcd, tiles * cols, full, rest, parts);
  if (u >= rest || parts < 2) return;
  int ti, cb;
  tile_and_column(s.v + full + u, tiles, cols, ti, cb);
  const int2 tile = ((const int2*)(a.saved + p.tiles_off))[ti];
  const int end = ((const int*)(a.saved + p.off_off))[tile.x + 1];
  const int pitch = DX ? 64 : 256;
  const int r = (blockIdx.y * 256 + threadIdx.x) / (width / 4), c = (int)threadIdx.x % (width / 4) * 4, col = cb * width + c;
  if (tile.y + r >= end || col >= n) return;
  const float* part = (const float*)(a.ws + (DX ? p.bpart_off : p.fpart_off)) +
                      ((size_t)xcd * kXcdBlocks + u * parts) * 128 * pitch + r * pitch + c;
  f32x4_t w[kMaxSplits], v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < kMaxSplits; ++k)
    if (k < parts) w[k] = *(const f32x4_t*)(part + (size_t)k * 128 * pitch);
  if constexpr (!DX) {
    const float* bias = (const float*)(a.ws + p.bias_off) + (size_t)tile.x * p.Op + col;  // padded to 32 columns
#pragma unroll 4
    for (int k = 0; k < p.bias_parts; ++k) {
      const f32x4_t b = *(const f32x4_t*)(bias + (size_t)k * p.E * p.Op);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += b[j];
    }
  }
#pragma unroll
  for (int k = 0; k < kMaxSplits; ++k)
    if (k < parts)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += w[k][j];
  store4((float*)(DX ? a.ws + p.dxs_off : a.saved + p.z_off) + (size_t)(tile.y + r) * n, col, n, n % 4 == 0, v);
}

__device__ __forceinline__ float load_weight(const ExpertsArgs& a, int64_t s) {
  return a.p.wbf16 ? (float)((const __bf16*)a.weights)[s] : ((const float*)a.weights)[s];
}

// out[t, c] = sum over the token's kept slots of (weight) src[row, c], in slot order;
// four columns a thread.
template <typename T, bool WEIGHTED>
__global__ __launch_bounds__(256) void k_experts_gather(ExpertsArgs a, const float* src, void* out, int width) {
  const ExpertsPlan& p = a.p;
  const int* row = (const int*)(a.saved + p.row_off);
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = (width + 3) / 4;
  const int64_t t = q / per;
  if (t >= p.T) return;
  const int c = (int)(q - t * per) * 4;
  const bool vec = width % 4 == 0;
  f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
  for (int j = 0; j < p.k; ++j) {
    const int r = row[t * p.k + j];
    const float w = WEIGHTED ? load_weight(a, t * p.k + j) : 1.0f;
    if (r < 0) continue;
    const f32x4_t z = load4(src + (size_t)r * width, c, width, vec);
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = WEIGHTED ? fmaf(w, z[u], v[u]) : v[u] + z[u];
  }
  store4((T*)out + t * width, c, width, vec, v);
}

// ---- backward -------------------------------------------------------------------

// dweights of each slot, the inverse of the scale of each row's w dy, and the largest of each block of 32
// rows; 16 waves a block, two rows each.
template <typename T>
__global__ __launch_bounds__(1024) void k_experts_dweights(ExpertsArgs a) {
  __shared__ float most[16];
  const ExpertsPlan& p = a.p;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, rb = blockIdx.x;
  const int* off = (const int*)(a.saved + p.off_off);
  const int* slot = (const int*)(a.saved + p.slot_off);
  const int* row = (const int*)(a.saved + p.row_off);
  const float* z = (const float*)(a.saved + p.z_off);
  if (a.dweights)  // slots without an expert
    for (int64_t s = (int64_t)rb * 1024 + threadIdx.x; s < p.S; s += (int64_t)gridDim.x * 1024)
      if (row[s] < 0) {
        if (p.wbf16)
          ((__bf16*)a.dweights)[s] = (__bf16)0.0f;
        else
          ((float*)a.dweights)[s] = 0.0f;
      }
  if (rb * 32 >= off[p.E]) return;
  const bool vec = p.O % 4 == 0;
  float dot[2] = {}, m[2] = {};
  int s[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) s[h] = slot[rb * 32 + wave * 2 + h];
  for (int o = lane * 4; o < p.O; o += 256)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (s[h] < 0) continue;
      const f32x4_t d = load4((const T*)a.dy + (int64_t)(s[h] / p.k) * p.O, o, p.O, vec);
      const f32x4_t v = load4(z + (size_t)(rb * 32 + wave * 2 + h) * p.O, o, p.O, vec);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dot[h] = fmaf(d[j], v[j], dot[h]);
        m[h] = fmaxf(m[h], finite_abs(d[j]));
      }
    }
  float big = 0.0f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (s[h] < 0) continue;
    const float sum = wave_sum(dot[h]), most_g = finite_abs(wave_max(m[h]) * load_weight(a, s[h]));
    if (lane == 0) ((float*)(a.ws + p.rscale_off))[rb * 32 + wave * 2 + h] = 1.0f / range_scale(most_g, 14);
    big = fmaxf(big, most_g);
    if (lane == 0 && a.dweights) {
      if (p.wbf16)
        ((__bf16*)a.dweights)[s[h]] = (__bf16)sum;
      else
        ((float*)a.dweights)[s[h]] = sum;
    }
  }
  if (lane == 0) most[wave] = big;
  __syncthreads();
  if (wave == 0) {
    const float v = wave_max(lane < 16 ? most[lane] : 0.0f);
    if (lane == 0) ((float*)(a.ws + p.gmax_off))[rb] = v;
  }
}

__device__ __forceinline__ int row_expert(const int* off, int E, int r) {
  int lo = 0, hi = E;  // the last e with off[e] <= r
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  while (lo + 1 < E && off[lo + 1] <= r) ++lo;
  return lo;
}

// g = w dy (scaled) of 32 rows x 64 outputs in both operand forms: rows = slots and
// k = o for dx (scaled by the row), rows = o and k = slots for dC (by the expert); and
// the rows' sum for each output.
template <typename T, int NP>
__global__ __launch_bounds__(256) void k_experts_gpack(ExpertsArgs a) {
  __shared__ float tile[32][65], red[4];
  const ExpertsPlan& p = a.p;
  const int* off = (const int*)(a.saved + p.off_off);
  const int rb = blockIdx.x, o0 = blockIdx.y * 64, tid = threadIdx.x;
  if (rb * 32 >= off[p.E]) return;
  const int e = row_expert(off, p.E, rb * 32);
  const float* gmax = (const float*)(a.ws + p.gmax_off);
  float m = 0.0f;
  for (int b = off[e] / 32 + tid; b < off[e + 1] / 32; b += 256) m = fmaxf(m, gmax[b]);
  m = block_max_256(m, red);
  const float scale = range_scale(m, 14);
  if (rb * 32 == off[e] && blockIdx.y == 0 && tid == 0) ((float*)(a.ws + p.gscale_off))[e] = scale;
  const int* slot = (const int*)(a.saved + p.slot_off);
  {  // eight values a thread
    const int r = tid >> 3, c = (tid & 7) * 8, s = slot[rb * 32 + r];
    const float w = s >= 0 ? load_weight(a, s) : 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int o = o0 + c + h * 4;
      f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (s >= 0 && o < p.O) v = load4((const T*)a.dy + (int64_t)(s / p.k) * p.O, o, p.O, p.O % 4 == 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) tile[r][c + h * 4 + j] = s >= 0 ? w * v[j] : 0.0f;
    }
  }
  __syncthreads();
  if (tid < 64 && o0 + tid < p.Op) {
    float sum = 0.0f;
    for (int r = 0; r < 32; ++r) sum += tile[r][tid];
    ((float*)(a.ws + p.gsum_off))[(size_t)rb * p.Op + o0 + tid] = sum;
  }
  float v[8];
  const int KBo = p.Op / 16;
  {  // rows = slots: 32 rows x 8 groups of 8 outputs
    const int r = tid & 31, k8 = tid >> 5, o = o0 + k8 * 8;
    if (o < p.Op) {
      const float own = slot[rb * 32 + r] >= 0 ? 1.0f / ((const float*)(a.ws + p.rscale_off))[rb * 32 + r] : 1.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = own * tile[r][k8 * 8 + j];
      const Planes8<NP> f = to_planes8<NP>(v);
      char* d = a.ws + p.gr_off + (((size_t)rb * KBo + (o >> 4)) * NP) * kPlaneBytes + (r + 32 * (k8 & 1)) * 16;
#pragma unroll
      for (int k = 0; k < NP; ++k) *(f16x8_t*)(d + k * kPlaneBytes) = f.p[k];
    }
  }
  {  // rows = o: 64 rows x 4 groups of 8 slots
    const int oo = tid & 63, k8 = tid >> 6, o = o0 + oo;
    if (o < p.Op) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = scale * tile[k8 * 8 + j][oo];
      const Planes8<NP> f = to_planes8<NP>(v);
      const int KBr = (int)(p.R / 16);
      char* d = a.ws + p.gt_off + (((size_t)(o >> 5) * KBr + rb * 2 + (k8 >> 1)) * NP) * kPlaneBytes +
                ((o & 31) + 32 * (k8 & 1)) * 16;
#pragma unroll
      for (int k = 0; k < NP; ++k) *(f16x8_t*)(d + k * kPlaneBytes) = f.p[k];
    }
  }
}

// dx += sum over j < nd of acc[.][j] U_{N+j}(x), the degrees N + 1 .. N + 4.  By Clenshaw's
// recurrence in the run of four,
//   sum_j g_j U_{N+j} = U_N B_0 - U_{N-1} B_1,   B_j = g_j + 2 x B_{j+1} - B_{j+2},
// with U_N and U_{N-1} from products (U_{2n} = U_n^2 - U_{n-1}^2, U_{2n+1} = U_n (U_{n+1} -
// U_{n-1})): straight code, so that the 32 elements of a lane hide one another's
// latency; a loop over the degrees an element took 112 us of 398.
template <int N>
__device__ __forceinline__ void weigh_by_u(const f32x16_t (&acc)[2][4], int nd, const float (&x)[2][16], float (&dx)[2][16]) {
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      // volatile: what depends on x alone is made here, not kept in registers through
      // the products of every run (240 registers more than there are)
      float xv = x[m][q];
      asm volatile("" : "+v"(xv));
      const float y = xv + xv;
      const float g1 = nd > 1 ? acc[m][1][q] : 0.0f, g2 = nd > 2 ? acc[m][2][q] : 0.0f, b3 = nd > 3 ? acc[m][3][q] : 0.0f;
      const float b2 = fmaf(y, b3, g2), b1 = fmaf(y, b2, g1 - b3), b0 = fmaf(y, b1, acc[m][0][q] - b2);
      if constexpr (N == 0) {
        dx[m][q] += b0;
      } else {
        const float u2 = fmaf(y, y, -1.0f), u3 = fmaf(y, u2, -y), u4 = fmaf(y, u3, -u2);
        float un = u4, um = u3;  // U_N, U_{N-1}
        if constexpr (N == 8) {
          un = fmaf(u4, u4, -u3 * u3);
          um = u3 * (u4 - u2);
        } else if constexpr (N == 12) {
          const float u5 = fmaf(y, u4, -u3), u6 = fmaf(y, u5, -u4);
          un = fmaf(u6, u6, -u5 * u5);
          um = u5 * (u6 - u4);
        }
        dx[m][q] += fmaf(un, b0, -um * b1);
      }
    }
}

// dx of 128 rows x 64 inputs a block, waves of 64 rows x 32 inputs: four degrees a
// pass over the outputs stand in four accumulator fragments; between passes only
// their weighted sum is kept.  16384 slots, 1024 -> 1024, degree 8, bf16: 315 us
// within a step (873 TFLOP/s), 293 at best, the matrix pipe 44 % busy; bound by the copies
// (24 KiB for 2.1 MFLOP a stage): with two or six buffers instead of three 418 and 413
// where three took 398.  All 256 registers are taken (the accumulators 128, the tanh
// values and sums 64) and 12 more live in scratch on one plane, 18 on two.
template <int NP> using DxTile = NtTile<NP, NP, 2, 2, 2, 4, NP == 1 ? 2 : 1, 3>;  // 72 KiB of LDS

template <int NP>
__global__ __launch_bounds__(256, 2) void k_experts_dx(ExpertsArgs a) {
  extern __shared__ char lds[];
  typedef DxTile<NP> Tile;
  constexpr int KS = Tile::kStageBlocks;
  const ExpertsPlan& p = a.p;
  const int cols = (p.Ip + 63) / 64, tiles = ((const int*)(a.saved + p.off_off))[p.E + 1];
  const Share share = block_share(blockIdx.x, tiles * cols);
  if (share.v < 0) return;
  int ti, cb;
  tile_and_column(share.v, tiles, cols, ti, cb);
  const int2 tile = ((const int2*)(a.saved + p.tiles_off))[ti];
  const int e = tile.x, row0 = tile.y, ib0 = cb * 2;
  const int end = ((const int*)(a.saved + p.off_off))[e + 1];
  const int KB = p.Op / 16, nib = p.Ip / 32;
  const int s0 = KB / KS * share.part / share.parts, nst = KB / KS * (share.part + 1) / share.parts - s0;
  const size_t pitch = (size_t)KB * NP * kPlaneBytes;
  const char* cbase = a.saved + p.cb_off + (size_t)e * p.Ip * p.deg * p.Op * 2 * NP;
  const RowBlocks A{a.ws + p.gr_off + (row0 >> 5) * pitch, pitch};
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 5;
  const int i = (ib0 + (wave & 1)) * 32 + (lane & 31);
  const int* tok = (const int*)(a.saved + p.tok_off);
  const float* t = (const float*)(a.saved + p.t_off);
  // every tanh value of the epilogue, asked for before the products (32 loads in
  // flight; one at a time behind a branch they took longer than the products)
  float x[2][16], dx[2][16] = {};
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      int r = row0 + (wave >> 1) * 64 + m * 32 + acc_row(q, g);
      r = r < end ? r : end - 1;
      const int k = tok[r];
      x[m][q] = t[(int64_t)(k >= 0 ? k : 0) * p.Ip + (i < p.Ip ? i : p.Ip - 1)];
    }
  for (int d0 = 0; d0 < p.deg; d0 += 4) {
    f32x16_t acc[2][4] = {};
    Tile::run(A, [&](int r) {
      int ib = ib0 + (r >> 2), d = d0 + (r & 3);
      ib = ib < nib ? ib : nib - 1;     // past the inputs or degrees: any, not used
      d = d < p.deg ? d : p.deg - 1;
      return cbase + ((size_t)ib * p.deg + d) * pitch;
    }, s0 * KS, nst, lds, acc);
    const int nd = p.deg - d0 < 4 ? p.deg - d0 : 4;
    if (d0 == 0)
      weigh_by_u<0>(acc, nd, x, dx);
    else if (d0 == 4)
      weigh_by_u<4>(acc, nd, x, dx);
    else if (d0 == 8)
      weigh_by_u<8>(acc, nd, x, dx);
    else
      weigh_by_u<12>(acc, nd, x, dx);
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int q = 0; q < 16; ++q) dx[m][q] *= fmaf(-x[m][q], x[m][q], 1.0f);
  const float ic = 1.0f / ((const float*)(a.saved + p.scale_off))[e];
  // the rows' scales undone; pad rows, and rows past the expert's, have any: they are not used
  const float* rinv = (const float*)(a.ws + p.rscale_off) + row0 + (wave >> 1) * 64;
  asm volatile("" ::: "memory");  // read here, not held in registers through the products
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int q = 0; q < 16; ++q) dx[m][q] = dx[m][q] * ic * rinv[m * 32 + acc_row(q, g)];
  if (share.parts > 1) {
    float* part = (float*)(a.ws + p.bpart_off) + ((size_t)(blockIdx.x & 7) * kXcdBlocks + share.place) * 128 * 64;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int q = 0; q < 16; ++q)
        part[((wave >> 1) * 64 + m * 32 + acc_row(q, g)) * 64 + (wave & 1) * 32 + (lane & 31)] = dx[m][q];
    return;
  }
  if (i >= p.I) return;
  float* out = (float*)(a.ws + p.dxs_off);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int r = row0 + (wave >> 1) * 64 + m * 32 + acc_row(q, g);
      if (r < end) out[(size_t)r * p.I + i] = dx[m][q];
    }
}

// The T_0 column of dC: each expert's sum of g over its rows, from the row blocks'
// sums; four running sums a column, eight loads in flight.
__global__ __launch_bounds__(256) void k_experts_gsum(ExpertsArgs a) {
  __shared__ float red[4][64];
  const ExpertsPlan& p = a.p;
  const int* off = (const int*)(a.saved + p.off_off);
  const int e = blockIdx.x, o = blockIdx.y * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const float* src = (const float*)(a.ws + p.gsum_off) + o;
  float s = 0.0f;
  if (o < p.Op) {
#pragma unroll 8
    for (int rb = off[e] / 32 + w; rb < off[e + 1] / 32; rb += 4) s += src[(size_t)rb * p.Op];
  }
  red[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && o < p.Op)
    ((float*)(a.ws + p.gtot_off))[(size_t)e * p.Op + o] =
        (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// The rows' tanh values in the order that dC reads them: for 32 inputs and 32 rows one
// run of [4 row groups][32 inputs][8 rows], zeros for pad rows.
__global__ __launch_bounds__(256) void k_experts_tsort(ExpertsArgs a) {
  __shared__ float tile[32][33];
  const ExpertsPlan& p = a.p;
  const int rb = blockIdx.x, ib = blockIdx.y, tid = threadIdx.x;
  if (rb * 32 >= ((const int*)(a.saved + p.off_off))[p.E]) return;
  const int* tok = (const int*)(a.saved + p.tok_off) + rb * 32;
  const float* t = (const float*)(a.saved + p.t_off) + ib * 32;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = u * 8 + (tid >> 5), k = tok[r];
    tile[r][tid & 31] = k >= 0 ? t[(int64_t)k * p.Ip + (tid & 31)] : 0.0f;
  }
  __syncthreads();
  f32x4_t v;
  const int g = tid >> 6, i = (tid >> 1) & 31, h = tid & 1;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = tile[g * 8 + h * 4 + j][i];
  ((f32x4_t*)(a.ws + p.ts_off))[((size_t)ib * (p.R / 32) + rb) * 256 + tid] = v;
}

// dC of NI x 32 inputs x DB degrees x 128 outputs of an expert a block (NI DB = 8 row
// blocks); waves of 4 row blocks x 64 outputs.  A stage is 32 rows.  The tanh
// values and g arrive by copies; each thread makes the basis values of 32 (row,
// degree) pairs of one input into LDS for the next stage while the matrix
// instructions work on this one.  16384 slots, 1024 -> 1024, degree 8, bf16: 362 us
// within a step (759 TFLOP/s), 330 at best, the matrix pipe 42 % busy; of 324 in one trial
// without making the basis 275, of 353 in another without the copies 346, without the
// last store 341.
//
// On two planes the basis values have one LDS buffer and a barrier more, so that two
// blocks share a CU: 16384 slots of 16 experts, 512 -> 512, degree 8, 241 us where one
// block a CU with two buffers took 314; 8 experts, 1024 -> 1024, degree 4, 472 and 572.
// With fewer blocks than CUs the barrier costs 2 %.
template <int NP> struct DcRing { static constexpr int kA = NP == 1 ? 2 : 1; };

template <typename T, int NP, int DB, bool HIGH>
__global__ __launch_bounds__(256, 2) void k_experts_dc(ExpertsArgs a) {
  extern __shared__ char lds[];
  constexpr int d0 = HIGH ? 8 : 0;  // the degrees d0 + 1 .. d0 + DB
  constexpr int KS = 2, NI = 8 / DB, kA = 8 * KS * NP, kB = 4 * KS * NP, kT = 4 * NI;  // 1 KiB chunks of a stage
  constexpr int NA = DcRing<NP>::kA;
  constexpr int kBAt = NA * kA * kPlaneBytes, kTAt = kBAt + 2 * kB * kPlaneBytes;
  const ExpertsPlan& p = a.p;
  const int nob = (p.O + 127) / 128, nib = p.Ip / 32, nbi = (nib + NI - 1) / NI;
  // Every XCD takes an eighth of each expert's blocks (whole columns of outputs, so
  // that they share g in its L2), the experts with most rows first: one expert an
  // XCD left the seven others waiting for the largest.
  const int per = (nbi * nob + 7) / 8, turn = (blockIdx.x >> 3) / per;
  const int id = ((blockIdx.x + turn) & 7) * per + (blockIdx.x >> 3) % per;
  if (id >= nbi * nob) return;
  const int ob = id % nob, ib0 = id / nob * NI, e = ((const int*)(a.saved + p.order_off))[turn];
  const int* off = (const int*)(a.saved + p.off_off);
  const int row0 = off[e], nst = (off[e + 1] - row0) / 32;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wd = wave >> 1, wo = wave & 1;
  const uint32_t l0 = lds_address(lds);
  const int KBr = (int)(p.R / 16), nb = p.Op / 32;
  const size_t pitch = (size_t)KBr * NP * kPlaneBytes;
  const char* gt = a.ws + p.gt_off + ((size_t)(row0 / 16) * NP) * kPlaneBytes;
  const char* ts = a.ws + p.ts_off + ((size_t)(row0 / 32)) * 4096;
  // the making thread's input, and its rows: DB 8: four rows of a group of eight,
  // DB 4: the whole group
  const int mq = DB == 8 ? tid >> 1 : tid;
  const int mi = mq & 31, mr = (mq >> 5) & 3, mib = mq >> 7, mh = DB == 8 ? tid & 1 : 0;
  constexpr int MR = DB == 8 ? 4 : 8;
  typedef typename std::conditional<MR == 8, Planes8<NP>, Planes4<NP>>::type Made;
  auto make = [&](int s, Made (&f)[DB]) {
    const float* src = (const float*)(lds + kTAt + (s & 1) * kT * kPlaneBytes) + ((mib * 4 + mr) * 32 + mi) * 8 + mh * 4;
    float tv[MR], ta[MR], tb[MR];
#pragma unroll
    for (int j = 0; j < MR; ++j) {
      tv[j] = src[j];
      ta[j] = 1.0f;
      tb[j] = tv[j];
    }
    if constexpr (HIGH) {  // T_8 and T_9 by products, T_{m+n} = 2 T_m T_n - T_{m-n}
#pragma unroll
      for (int j = 0; j < MR; ++j) {
        const float x = tv[j], t2 = fmaf(x + x, x, -1.0f), t3 = fmaf(x + x, t2, -x), t4 = fmaf(t2 + t2, t2, -1.0f);
        ta[j] = fmaf(t4 + t4, t4, -1.0f);
        tb[j] = fmaf(t4 + t4, fmaf(t2 + t2, t3, -x), -x);
      }
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      if constexpr (MR == 8)
        f[d] = to_planes8<NP>(tb);
      else
        f[d] = to_planes4<NP>(tb);
#pragma unroll
      for (int j = 0; j < MR; ++j) {
        const float c = fmaf(tv[j] + tv[j], tb[j], -ta[j]);
        ta[j] = tb[j];
        tb[j] = c;
      }
    }
  };
  auto keep = [&](int s, const Made (&f)[DB]) {
    char* dst = lds + s % NA * kA * kPlaneBytes + (mi + 32 * (mr & 1)) * 16 + mh * 8;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int k = 0; k < NP; ++k)
        *(typename Made::part*)(dst + (((mib * DB + d) * KS + (mr >> 1)) * NP + k) * kPlaneBytes) = f[d].p[k];
  };
  auto copy_g = [&](int s) {
#pragma unroll
    for (int i = 0; i < kB / 4; ++i) {
      const int c = i * 4 + wave;
      int rb = ob * 4 + c / (KS * NP);
      rb = rb < nb ? rb : nb - 1;
      dma16s(gt + rb * pitch + ((size_t)s * KS * NP + c % (KS * NP)) * kPlaneBytes, lane * 16,
             l0 + kBAt + ((s & 1) * kB + c) * kPlaneBytes);
    }
  };
  auto copy_t = [&](int s) {
#pragma unroll
    for (int i = 0; i < kT / 4; ++i) {
      int ib = ib0 + i;
      ib = ib < nib ? ib : nib - 1;
      dma16s(ts + ((size_t)ib * (p.R / 32) + s) * 4096 + wave * 1024, lane * 16,
             l0 + kTAt + ((s & 1) * kT + i * 4 + wave) * kPlaneBytes);
    }
  };
  f32x16_t acc[4][2] = {};
  if (nst > 0) {
    copy_t(0);
    copy_g(0);
    if (nst > 1) copy_t(1);
    wait_vm<0>();
    block_barrier();
    Made first[DB];
    make(0, first);
    keep(0, first);
  }
  for (int s = 0; s < nst; ++s) {
    wait_vm<0>();
    wait_lds();
    block_barrier();
    if (s + 1 < nst) copy_g(s + 1);
    if (s + 2 < nst) copy_t(s + 2);  // over stage s, which was made from before the barrier
    // the next stage's basis values in registers while the matrix instructions run, to
    // LDS behind them (past the last stage: of stale tanh values, not read)
    Made next[DB];
    make(s + 1, next);
    const char* buf = lds + s % NA * kA * kPlaneBytes;
    const char* bufb = lds + kBAt + (s & 1) * kB * kPlaneBytes;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      f16x8_t fa[4][NP], fb[2][NP];
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int q = 0; q < NP; ++q) fa[m][q] = lds_frag(buf + (((wd * 4 + m) * KS + k) * NP + q) * kPlaneBytes, lane);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int q = 0; q < NP; ++q) fb[n][q] = lds_frag(bufb + (((wo * 2 + n) * KS + k) * NP + q) * kPlaneBytes, lane);
      mfma_planes<NP, NP, 4, 2>(fa, fb, acc);
    }
    // a matrix instruction, then vector ones in its shadow
#pragma unroll
    for (int i = 0; i < KS * 8 * (NP == 2 ? 3 : 1); ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, NP == 2 ? 5 : 7, 0);
    }
    if constexpr (NA == 1) {  // over this stage's values, once every wave has read them
      wait_lds();
      block_barrier();
    }
    keep(s + 1, next);
  }
  // The tile leaves through LDS, 8 inputs (of each row block) at a time, so that an
  // input's coefficients of 128 outputs are stored as they lie in memory.
  wait_lds();
  block_barrier();
  const int nd = p.deg - d0 < DB ? p.deg - d0 : DB, lead = d0 == 0 ? 1 : 0, w = nd + lead;  // columns here, T_0 first
  const int no = p.O - ob * 128 < 128 ? p.O - ob * 128 : 128;
  const float inv = nst > 0 ? 1.0f / ((const float*)(a.ws + p.gscale_off))[e] : 1.0f;
  const float* gtot = (const float*)(a.ws + p.gtot_off) + (size_t)e * p.Op + ob * 128;
  T* out = (T*)a.dcoeffs + (int64_t)e * p.I * p.O * p.D;
  float* tile = (float*)lds;  // [NI][8][128][w]
  const bool whole = w == p.D && (int64_t)p.O * p.D % 4 == 0 && no * w % 4 == 0;
  const int wib = DB == 8 ? 0 : wd, wd1 = DB == 8 ? wd * 4 : 0;  // the wave's row block of inputs, its degrees
#pragma unroll
  for (int h = 0; h < 4; ++h) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (wd1 + m < nd)
            tile[((wib * 8 + g * 4 + j) * 128 + wo * 64 + n * 32 + (lane & 31)) * w + lead + wd1 + m] = acc[m][n][h * 4 + j] * inv;
    if (lead)
      for (int q = tid; q < NI * 8 * 128; q += 256) tile[q * w] = (q & 127) < no ? gtot[q & 127] : 0.0f;
    __syncthreads();
    for (int r = wave; r < NI * 8; r += 4) {
      const int i = (ib0 + (r >> 3)) * 32 + 8 * h + (r & 7);
      if (i >= p.I) continue;
      const float* src = tile + r * 128 * w;
      T* dst = out + ((int64_t)i * p.O + ob * 128) * p.D;
      if (whole) {
        for (int q = lane * 4; q < no * w; q += 256) {
          const f32x4_t v = *(const f32x4_t*)(src + q);
          if constexpr (sizeof(T) == 4) {
            *(f32x4_t*)(dst + q) = v;
          } else {
            bf16x4_t b;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = (__bf16)v[j];
            *(bf16x4_t*)(dst + q) = b;
          }
        }
      } else {
        for (int q = lane; q < no * w; q += 64) {
          const int o = q / w;
          dst[(int64_t)o * p.D + d0 + (1 - lead) + q - o * w] = (T)src[q];
        }
      }
    }
    __syncthreads();
  }
}

// ---- forward of few slots ---------------------------------------------------------

// The D coefficients of lane o of one input's row [O, D], through a bounds-checked
// buffer (lanes past O read zeros).  bf16 rows may begin, and coefficients lie, on
// odd halves of a dword: the dwords that cover them are read and shifted.
template <int D>
__device__ __forceinline__ void stream_load(const float* row, int bytes, int o, uint32_t (&w)[D]) {
  const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(row, bytes);
  constexpr int kQ = D / 4 * 4;
#pragma unroll
  for (int v = 0; v < kQ; v += 4) {
    const u32x4_t q = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (o * D + v) * 4, 0, 0));
#pragma unroll
    for (int j = 0; j < 4; ++j) w[v + j] = q[j];
  }
#pragma unroll
  for (int v = kQ; v < D; ++v) w[v] = __builtin_amdgcn_raw_buffer_load_b32(rs, (o * D + v) * 4, 0, 0);
}
template <int D> struct StreamRow {  // dwords a lane holds of an input
  static constexpr int kF32 = D, kBf16 = D % 2 ? (D + 1) / 2 : D / 2;
};
template <int D>
__device__ __forceinline__ void stream_load(const __bf16* row, int bytes, int o, uint32_t (&w)[StreamRow<D>::kBf16]) {
  const uintptr_t at = (uintptr_t)row;
  const int odd = (int)(at & 2);
  const __amdgpu_buffer_rsrc_t rs = buffer_rsrc((const void*)(at & ~(uintptr_t)3), (bytes + odd + 3) & ~3);
  const int byte = o * D * 2 + odd;
  constexpr int N = StreamRow<D>::kBf16, kQ = N / 4 * 4;
#pragma unroll
  for (int v = 0; v < kQ; v += 4) {
    const u32x4_t q = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (byte & ~3) + v * 4, 0, 0));
#pragma unroll
    for (int j = 0; j < 4; ++j) w[v + j] = q[j];
  }
#pragma unroll
  for (int v = kQ; v < N; ++v) w[v] = __builtin_amdgcn_raw_buffer_load_b32(rs, (byte & ~3) + v * 4, 0, 0);
}
template <int D>
__device__ __forceinline__ void stream_unpack(const float*, int, const uint32_t (&w)[D], float (&c)[D]) {
#pragma unroll
  for (int d = 0; d < D; ++d) c[d] = __uint_as_float(w[d]);
}
// D odd: D + 1 halves cover the D coefficients from either half of the first dword.
template <int D>
__device__ __forceinline__ void stream_unpack(const __bf16* row, int o, const uint32_t (&w)[StreamRow<D>::kBf16],
                                              float (&c)[D]) {
  const bool odd = D % 2 && ((((uintptr_t)row & 2) + o * D * 2) & 2);
#pragma unroll
  for (int d = 0; d < D; ++d) {
    const float lo = __uint_as_float(d & 1 ? w[d / 2] & 0xffff0000u : w[d / 2] << 16);
    if constexpr (D % 2) {
      const float hi = __uint_as_float(d & 1 ? w[(d + 1) / 2] << 16 : w[d / 2] & 0xffff0000u);
      c[d] = odd ? hi : lo;
    } else {
      c[d] = lo;
    }
  }
}

// part[chunk, slot, o] = the slot's expert output over one chunk of inputs.  A block
// takes one expert, 64 outputs (a lane each) and a chunk; it finds its expert's
// slots itself, makes the basis values of up to 8 rows in LDS (read as
// broadcasts), and its four waves stream the chunk's coefficients.  Bound by the
// coefficients' stream: two experts of 2048 -> 2048, degree 8, bf16, for one row 30 us
// (5.0 TB/s; a large copy reaches 5.15), 96 slots of 16 experts of 512 -> 512 in fp32
// 34 us (4.5 TB/s).
template <typename T, int D>
__global__ __launch_bounds__(256) void k_experts_stream(ExpertsArgs a) {
  constexpr int kDeg = D - 1, kW = (kDeg + 3) / 4 * 4, kU = 4;
  constexpr int kN = sizeof(T) == 4 ? StreamRow<D>::kF32 : StreamRow<D>::kBf16;
  __shared__ int slots[kStreamMaxSlots], counts[4];
  __shared__ __align__(16) float basis[kStreamInputs * kStreamRows * kW];
  __shared__ float red[4][kStreamRows][64];
  const ExpertsPlan& p = a.p;
  const int oc = (p.O + 63) / 64;
  int id = blockIdx.x;
  const int chunk = id % p.chunks;
  id /= p.chunks;
  const int o = id % oc * 64 + (threadIdx.x & 63), e = id / oc;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  int n = 0;
  for (int s0 = 0; s0 < (int)p.S; s0 += 256) {
    const int s = s0 + tid;
    const bool mine = s < (int)p.S && a.indices[s] == e;
    const unsigned long long has = __ballot(mine);
    if (lane == 0) counts[wave] = __popcll(has);
    __syncthreads();
    int at = n;
    for (int w = 0; w < wave; ++w) at += counts[w];
    if (mine) slots[at + __popcll(has & ((1ull << lane) - 1))] = s;
    n += counts[0] + counts[1] + counts[2] + counts[3];
    __syncthreads();
  }
  const int i0 = chunk * p.chunk_inputs, ni = p.I - i0 < p.chunk_inputs ? p.I - i0 : p.chunk_inputs;
  const T* C = (const T*)a.coeffs + ((int64_t)e * p.I + i0) * p.O * D;
  const int row_elems = p.O * D;
  float* part = (float*)(a.ws + p.part_off) + (size_t)chunk * p.S * p.O;
  for (int r0 = 0; r0 < n; r0 += kStreamRows) {
    const int nr = n - r0 < kStreamRows ? n - r0 : kStreamRows;
    for (int q = tid; q < ni * nr; q += 256) {
      const int r = q / ni, i = q - r * ni;
      const float t = tanhf((float)((const T*)a.x)[(int64_t)(slots[r0 + r] / p.k) * p.I + i0 + i]);
      float* b = basis + (i * kStreamRows + r) * kW;
      float ta = 1.0f, tb = t;
#pragma unroll
      for (int d = 0; d < kDeg; ++d) {
        b[d] = tb;
        const float tc = fmaf(t + t, tb, -ta);
        ta = tb;
        tb = tc;
      }
    }
    __syncthreads();
    float acc[kStreamRows] = {};
    for (int i = wave; i < ni; i += 4 * kU) {
      uint32_t w[kU][kN];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (i + 4 * u < ni) stream_load<D>(C + (int64_t)(i + 4 * u) * row_elems, row_elems * (int)sizeof(T), o, w[u]);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (i + 4 * u >= ni) break;
        float c[D];
        stream_unpack<D>(C + (int64_t)(i + 4 * u) * row_elems, o, w[u], c);
        const float* b = basis + (i + 4 * u) * kStreamRows * kW;
#pragma unroll
        for (int r = 0; r < kStreamRows; ++r) {
          if (r >= nr) break;
          float s = c[0];
#pragma unroll
          for (int d = 0; d < kDeg; ++d) s = fmaf(c[d + 1], b[r * kW + d], s);
          acc[r] += s;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kStreamRows; ++r) red[wave][r][lane] = acc[r];
    __syncthreads();
    for (int r = wave; r < nr; r += 4)
      if (o < p.O)
        part[(size_t)slots[r0 + r] * p.O + o] = (red[0][r][lane] + red[1][r][lane]) + (red[2][r][lane] + red[3][r][lane]);
    __syncthreads();
  }
}

// y from the chunks' partial sums.
template <typename T>
__global__ __launch_bounds__(256) void k_experts_stream_sum(ExpertsArgs a) {
  const ExpertsPlan& p = a.p;
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (q >= p.T * p.O) return;
  const int64_t t = q / p.O;
  const int o = (int)(q - t * p.O);
  const float* part = (const float*)(a.ws + p.part_off);
  float v = 0.0f;
  for (int j = 0; j < p.k; ++j) {
    const int64_t s = t * p.k + j;
    if (slot_expert(a, s) < 0) continue;
    float z = 0.0f;
#pragma unroll 8
    for (int c = 0; c < p.chunks; ++c) z += part[((size_t)c * p.S + s) * p.O + o];
    v += load_weight(a, s) * z;
  }
  ((T*)a.y)[q] = (T)v;
}

template <typename T>
void stream_typed(const ExpertsArgs& a, hipStream_t st) {
  const ExpertsPlan& p = a.p;
  const dim3 grid((unsigned)(p.chunks * ((p.O + 63) / 64) * p.E)), block(256);
  switch (p.D) {
#define CKAN_STREAM_CASE(N) \
  case N: hipLaunchKernelGGL((k_experts_stream<T, N>), grid, block, 0, st, a); break;
    CKAN_STREAM_CASE(2) CKAN_STREAM_CASE(3) CKAN_STREAM_CASE(4) CKAN_STREAM_CASE(5) CKAN_STREAM_CASE(6)
    CKAN_STREAM_CASE(7) CKAN_STREAM_CASE(8) CKAN_STREAM_CASE(9) CKAN_STREAM_CASE(10) CKAN_STREAM_CASE(11)
    CKAN_STREAM_CASE(12) CKAN_STREAM_CASE(13) CKAN_STREAM_CASE(14) CKAN_STREAM_CASE(15) CKAN_STREAM_CASE(16)
    CKAN_STREAM_CASE(17)
#undef CKAN_STREAM_CASE
  }
  hipLaunchKernelGGL((k_experts_stream_sum<T>), dim3((unsigned)ceil_div(p.T * p.O, 256)), block, 0, st, a);
}

template <int NP, int P, int FN>
void launch_fwd(const ExpertsArgs& a, hipStream_t st) {
  using FS = FwdStage<NP, P>;
  constexpr int lds = FS::NBUF * (128 * FS::IN * 4 + 2 * FN * FS::KS * NP * kPlaneBytes);
  static std::atomic<uint32_t> done;
  ensure_lds_limit((const void*)k_experts_fwd<NP, P, FN>, lds, done);
  const int64_t cols = ceil_div(a.p.O, 64 * FN);
  hipLaunchKernelGGL((k_experts_fwd<NP, P, FN>), dim3((unsigned)share_grid(a.p.tiles * cols)), dim3(256), lds, st, a);
  hipLaunchKernelGGL((k_experts_parts<false>), dim3(8 * kXcdBlocks, 8 * FN), dim3(256), 0, st, a, 64 * FN);
}

template <typename T, int NP, int P>
void forward_typed(const ExpertsArgs& a, bool keep, hipStream_t st) {
  const ExpertsPlan& p = a.p;
  hipLaunchKernelGGL(k_plan_count, dim3(p.plan_blocks), dim3(kPlanThreads), 0, st, a);
  hipLaunchKernelGGL(k_plan_place, dim3(p.plan_blocks), dim3(kPlanThreads), 0, st, a);
  hipLaunchKernelGGL((k_experts_tanh<T>), dim3((unsigned)ceil_div(p.T * (p.Ip / 4), 256)), dim3(256), 0, st, a);
  hipLaunchKernelGGL((k_experts_cmax<T>), dim3(kMaxParts, p.E), dim3(256), 0, st, a);
  const size_t pack_lds = (size_t)16 * (32 * p.D + 1) * sizeof(float);
  const dim3 pack_grid(p.bias_parts, p.Op / 32, p.E);
  // 16-byte loads where every input's row of coefficients begins at such a boundary
  if (p.O * p.D % Vec16<T>::N == 0)
    hipLaunchKernelGGL((k_experts_pack<T, NP, P, true>), pack_grid, dim3(256), pack_lds, st, a, keep);
  else
    hipLaunchKernelGGL((k_experts_pack<T, NP, P, false>), pack_grid, dim3(256), pack_lds, st, a, keep);
  // Tiles of 256 or of 128 columns: the narrow ones make the basis twice as often (some
  // 10 % a tile), and of few tiles they leave fewer places empty.  In fp32, 16384 slots of
  // 16 experts, 512 -> 512: 224 us narrow, 301 wide; 8 experts, 1024 -> 1024: 789 and
  // 747; bf16, 8000 slots, 300 -> 500, degree 12: 104 and 60.  On two planes of 16
  // degrees two blocks' rings of wide tiles would not share a CU.
  const double narrow = 1.1 * share_rounds(p.tiles * ceil_div(p.O, 128)), wide = 2 * share_rounds(p.tiles * ceil_div(p.O, 256));
  if ((NP == 2 && P == 16) || narrow < wide)
    launch_fwd<NP, P, 2>(a, st);
  else if constexpr (NP == 1 || P < 16)
    launch_fwd<NP, P, 4>(a, st);
  hipLaunchKernelGGL((k_experts_gather<T, true>), dim3((unsigned)ceil_div(p.T * ((p.O + 3) / 4), 256)), dim3(256), 0, st, a,
                     (const float*)(a.saved + p.z_off), a.y, p.O);
}

template <typename T, int NP, int DB, bool HIGH>
void launch_dc(const ExpertsArgs& a, hipStream_t st) {
  constexpr int NI = 8 / DB, ring = (DcRing<NP>::kA * 8 * 2 * NP + 2 * (4 * 2 * NP + 4 * NI)) * kPlaneBytes;
  constexpr int tile = NI * 8 * 128 * (DB + 1) * 4, lds = ring > tile ? ring : tile;
  static std::atomic<uint32_t> done;
  ensure_lds_limit((const void*)k_experts_dc<T, NP, DB, HIGH>, lds, done);
  const int64_t blocks = a.p.E * xcd_grid(ceil_div(a.p.Ip / 32, NI) * ceil_div(a.p.O, 128));
  hipLaunchKernelGGL((k_experts_dc<T, NP, DB, HIGH>), dim3((unsigned)blocks), dim3(256), lds, st, a);
}

template <typename T, int NP>
void backward_typed(const ExpertsArgs& a, hipStream_t st) {
  const ExpertsPlan& p = a.p;
  hipLaunchKernelGGL((k_experts_dweights<T>), dim3((unsigned)(p.R / 32)), dim3(1024), 0, st, a);
  if (!a.dx && !a.dcoeffs) return;
  hipLaunchKernelGGL((k_experts_gpack<T, NP>), dim3((unsigned)(p.R / 32), (p.Op + 63) / 64), dim3(256), 0, st, a);
  if (a.dx) {
    constexpr int lds = DxTile<NP>::kLdsBytes;
    static std::atomic<uint32_t> done;
    ensure_lds_limit((const void*)k_experts_dx<NP>, lds, done);
    hipLaunchKernelGGL((k_experts_dx<NP>), dim3((unsigned)share_grid((int64_t)p.tiles * ((p.Ip + 63) / 64))), dim3(256), lds,
                       st, a);
    hipLaunchKernelGGL((k_experts_parts<true>), dim3(8 * kXcdBlocks, 8), dim3(256), 0, st, a, 64);
    hipLaunchKernelGGL((k_experts_gather<T, false>), dim3((unsigned)ceil_div(p.T * ((p.I + 3) / 4), 256)), dim3(256), 0, st, a,
                       (const float*)(a.ws + p.dxs_off), a.dx, p.I);
  }
  if (a.dcoeffs) {
    hipLaunchKernelGGL(k_experts_gsum, dim3(p.E, (p.Op + 63) / 64), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_experts_tsort, dim3((unsigned)(p.R / 32), p.Ip / 32), dim3(256), 0, st, a);
    // runs of 8 degrees, and of 4 where no more are left
    if (p.deg > 4)
      launch_dc<T, NP, 8, false>(a, st);
    else
      launch_dc<T, NP, 4, false>(a, st);
    if (p.deg > 12)
      launch_dc<T, NP, 8, true>(a, st);
    else if (p.deg > 8)
      launch_dc<T, NP, 4, true>(a, st);
  }
}

}  // namespace

void launch_experts_forward(const ExpertsArgs& a, bool keep, hipStream_t st) {
  if (a.p.bf16) {
    if (a.p.P == 4) forward_typed<__bf16, 1, 4>(a, keep, st);
    if (a.p.P == 8) forward_typed<__bf16, 1, 8>(a, keep, st);
    if (a.p.P == 16) forward_typed<__bf16, 1, 16>(a, keep, st);
  } else {
    if (a.p.P == 4) forward_typed<float, 2, 4>(a, keep, st);
    if (a.p.P == 8) forward_typed<float, 2, 8>(a, keep, st);
    if (a.p.P == 16) forward_typed<float, 2, 16>(a, keep, st);
  }
}

void launch_experts_stream(const ExpertsArgs& a, hipStream_t st) {
  if (a.p.bf16)
    stream_typed<__bf16>(a, st);
  else
    stream_typed<float>(a, st);
}

void launch_experts_backward(const ExpertsArgs& a, hipStream_t st) {
  if (a.p.bf16)
    backward_typed<__bf16, 1>(a, st);
  else
    backward_typed<float, 2>(a, st);
}

}  // namespace ckan
