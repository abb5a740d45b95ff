// Kernels of a whole mixture layer for few rows (ckan_mixture_forward): the gate's logits, the
// choice, the chosen experts' products and their weighted sum, in two or three launches.
//
// What bounds it is the chosen experts' coefficients, read once as they lie, [in, out, D].
// The kernels of each type of coefficients are a source file of their own.
#pragma once

#include <type_traits>

#include "ckan_block.hpp"
#include "ckan_route_row.hpp"

namespace ckan {
namespace {

// ---- gate and choice -------------------------------------------------------------------

constexpr int kGateThreads = 1024, kGateWaves = kGateThreads / 64, kGateExperts = 4;

// Dot products of one row with kGateExperts rows of the gate over chunks [c0, c1), a lane's share.
// The products of fp32 values are exact in 64 bits and so, nearly, is their sum: rounded once, a
// logit does not depend on the order of the sum.
template <typename TX, typename TG>
__device__ __forceinline__ void gate_dots(const FewArgs& a, int64_t row, int e0, int c0, int c1, int lane,
                                          double (&sum)[kGateExperts]) {
  const TX* x = (const TX*)a.x + row * a.I;
  const int last = a.route.E - 1;
#pragma unroll 2
  for (int c = c0 + lane; c < c1; c += 64) {
    const int at = c * kChunk, left = a.I - at;
    const auto xr = load_raw8(x + at, (int64_t)left);
    typename RawOf<TG>::type gr[kGateExperts];
#pragma unroll
    for (int q = 0; q < kGateExperts; ++q)
      gr[q] = load_raw8((const TG*)a.gate + (int64_t)(e0 + q < last ? e0 + q : last) * a.I + at, (int64_t)left);
    float xv[kChunk];
    unpack8(xr, xv);
#pragma unroll
    for (int q = 0; q < kGateExperts; ++q) {
      float g[kChunk];
      unpack8(gr[q], g);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) sum[q] = fma((double)xv[i], (double)g[i], sum[q]);
    }
  }
}
// The sum over a wave, in every lane, by butterflies on the vector ALU as lanes_sum's. Through LDS (__shfl_xor) the exchanges
// of many experts' sums share a CU's one LDS: 128 rows of 128 inputs by 512 experts 13.5 -> 10.2 us.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true);
  return v + __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v = dpp_add<0xb1>(v);
  v = dpp_add<0x4e>(v);
  v = dpp_add<0x141>(v);
  v = dpp_add<0x140>(v);
  auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
  auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
  v = __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
  lo = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(v), false, false);
  hi = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(v), false, false);
  return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}

struct GateShared {
  double part[kRouteMaxExperts];
  float keys[kRouteMaxExperts + 64];
};

// The row's choice by a block of kGateWaves waves; lane j of wave 0 gets the j-th expert and its weight.
template <typename TX, typename TG>
__device__ __forceinline__ void gate_row(const FewArgs& a, int64_t row, GateShared& sh, int& mine, float& weight) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.route.E;
  const int groups = (E + kGateExperts - 1) / kGateExperts, chunks = (a.I + kChunk - 1) / kChunk;
  // fewer groups of experts than waves: waves share a group, a slice of the inputs each
  const int slices = groups < kGateWaves ? kGateWaves / groups : 1, per = (chunks + slices - 1) / slices;
  for (int g = wave; g < groups * slices; g += kGateWaves) {
    const int e0 = g / slices * kGateExperts, slice = g % slices, c0 = slice * per, c1 = c0 + per < chunks ? c0 + per : chunks;
    double sum[kGateExperts] = {};
    gate_dots<TX, TG>(a, row, e0, c0, c1, lane, sum);
#pragma unroll
    for (int q = 0; q < kGateExperts; ++q) {
      const double v = wave_sum64(sum[q]);
      if (lane == 0 && e0 + q < E) sh.part[(e0 + q) * slices + slice] = v;
    }
  }
  __syncthreads();
  if (wave) return;
  const auto choose = [&](auto j) {
    constexpr int J = decltype(j)::value;
    float l[J];
#pragma unroll
    for (int q = 0; q < J; ++q) {
      const int e = lane * J + q;
      double v = 0.0;
      for (int s = 0; s < slices && e < E; ++s) v += sh.part[e * slices + s];
      l[q] = e < E ? eligible_logit((float)v) : -INFINITY;
    }
    route_row<J>(a.route, lane, l, sh.keys, mine, weight);
  };
  if (E <= 64)
    choose(std::integral_constant<int, 1>());
  else if (E <= 128)
    choose(std::integral_constant<int, 2>());
  else if (E <= 256)
    choose(std::integral_constant<int, 4>());
  else
    choose(std::integral_constant<int, 8>());
}

// ---- the experts' products ---------------------------------------------------------------

// The D coefficients of one input and output, at any element's address.
template <typename T, int D>
struct __attribute__((packed)) Coefs {
  T v[D];
};

// s[p] = sum_d c[p D + d] T_d(t), T_d by the recurrence.
template <typename T, int D, int P>
__device__ __forceinline__ void series(const Coefs<T, D * P>& c, float t, float (&s)[P]) {
  float ta = 1.0f, tb = t;
#pragma unroll
  for (int p = 0; p < P; ++p) s[p] = (float)c.v[p * D];
#pragma unroll
  for (int d = 1; d < D; ++d) {
#pragma unroll
    for (int p = 0; p < P; ++p) s[p] = fmaf((float)c.v[p * D + d], tb, s[p]);
    const float tc = fmaf(t + t, tb, -ta);
    ta = tb;
    tb = tc;
  }
}

// Up to 8 rows: a block takes 64 P outputs (a lane P of them: bf16 in pairs, whose coefficients begin
// at whole dwords) and a chunk of inputs of every chosen expert, its 16 waves an input each a
// step, and leaves part[chunk, row, o], the experts summed. The rows' shares stay in registers; an
// expert's coefficients serve the rows that chose it. Bound by the coefficients' stream: two experts of
// 2048 -> 2048, degree 8, for one row 30 us in bf16 (5.0 TB/s) and 54 in fp32 (5.6), and in all with
// gate and sum 40 and 64. Blocks that own 8 outputs over all inputs, which leave no sum, read 144 bytes at
// a place in bf16 and reach 3.9 TB/s (45 us in all).
constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kRowTanh = 512;  // inputs of a chunk
constexpr int kRowsMax = 8;  // 16 rows' shares do not fit the registers: 8 rows 67 us in their form, 48 in this

// GATED, one row and a small gate: every block makes the choice itself, the first one stores it. That costs
// each block the gate's values from the L2 and saves a launch and its drain: 40.3 -> 38.3 us in all for the
// bf16 case above, 63.5 -> 60.7 for fp32, 27.7 -> 26.6 with a gate of 2^16 entries.
template <typename TX, typename TC, int D, int R, bool GATED>
__global__ __launch_bounds__(kRowThreads) void k_few_rows(FewArgs a) {
  static_assert(!GATED || (R == 1 && kRowThreads == kGateThreads));
  constexpr int P = 4 / sizeof(TC);
  constexpr int kList = R * kRouteMaxTopK < kRouteMaxExperts ? R * kRouteMaxTopK : kRouteMaxExperts;
  __shared__ float t[R][kRowTanh];
  __shared__ float red[kRowWaves][64 * P];
  __shared__ unsigned chosen[kRouteMaxExperts / 32];
  __shared__ int expert[kList], mask[kList];  // the chosen experts, and who chose them
  __shared__ float weight[kList][R];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunk = blockIdx.y, o = (blockIdx.x * 64 + lane) * P, T = (int)a.route.rows;
  const bool real = o < a.O, all = o + P <= a.O;
  const int i0 = chunk * a.chunk_inputs, ni = a.I - i0 < a.chunk_inputs ? a.I - i0 : a.chunk_inputs;
  if (tid < kRouteMaxExperts / 32) chosen[tid] = 0;
  if (tid < kList) mask[tid] = 0;
  int64_t e = -1;
  float w = 0.0f;
  if constexpr (GATED) {
    __shared__ GateShared sh;
    int mine = -1;
    if (a.gate_bf16)
      gate_row<TX, __bf16>(a, 0, sh, mine, w);
    else
      gate_row<TX, float>(a, 0, sh, mine, w);
    if (tid < a.S) {
      e = mine;
      if (blockIdx.x == 0 && blockIdx.y == 0) {
        a.route.weights[tid] = w;
        a.route.indices[tid] = mine;
      }
    }
  } else if (tid < a.S) {
    e = a.route.indices[tid];
    w = a.route.weights[tid];
    if (e >= a.route.E) e = -1;
  }
  for (int q = tid; q < ni * T; q += kRowThreads) {
    const int r = q / ni, i = q - r * ni;
    t[r][i] = tanhf((float)((const TX*)a.x)[(int64_t)r * a.I + i0 + i]);
  }
  __syncthreads();
  if (e >= 0) atomicOr(&chosen[e >> 5], 1u << (e & 31));
  __syncthreads();
  int nj = 0;
  if (e >= 0) {
    int rank = __popc(chosen[e >> 5] & ((1u << (e & 31)) - 1));
    for (int q = 0; q < (int)(e >> 5); ++q) rank += __popc(chosen[q]);
    expert[rank] = (int)e;
    const int r = tid / a.route.top_k;
    weight[rank][r] = w;
    atomicOr(&mask[rank], 1 << r);
  }
  for (int q = 0; q < (a.route.E + 31) / 32; ++q) nj += __popc(chosen[q]);
  __syncthreads();
  const int64_t pitch = (int64_t)a.O * D;
  const TC* C = (const TC*)a.coeffs + (int64_t)(real ? o : 0) * D + (int64_t)i0 * pitch;
  float y[R][P] = {};
  // kU inputs' coefficients on their way while kU are worked on; where a reader or worker is: an
  // expert and an input, uniform over the wave
  constexpr int kU = D <= 10 ? 2 : 1;
  Coefs<TC, D * P> c[2][kU];
  int fj = 0, fi = wave, wj = 0, wi = wave;
  const TC* base = nj ? C + (int64_t)expert[0] * a.I * pitch : C;
  int who = nj ? __builtin_amdgcn_readfirstlane(mask[0]) : 0;
  const auto fetch = [&](Coefs<TC, D * P>(&to)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (fj >= nj) break;
      if (fi < ni) {
        const TC* at = base + (int64_t)fi * pitch;
        if (all) {
          to[u] = *(const Coefs<TC, D * P>*)at;
        } else if (real) {
          to[u] = Coefs<TC, D * P>{};
          *(Coefs<TC, D>*)&to[u] = *(const Coefs<TC, D>*)at;
        }
      }
      fi += kRowWaves;
      if (fi >= ni) {
        fi = wave;
        if (++fj < nj) base = C + (int64_t)expert[fj] * a.I * pitch;
      }
    }
  };
  const auto work = [&](const Coefs<TC, D * P>(&from)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (wj >= nj) break;
      if (wi < ni && real) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (!(who >> r & 1)) continue;
          float z[P];
          series<TC, D, P>(from[u], t[r][wi], z);
#pragma unroll
          for (int p = 0; p < P; ++p) y[r][p] = fmaf(weight[wj][r], z[p], y[r][p]);
        }
      }
      wi += kRowWaves;
      if (wi >= ni) {
        wi = wave;
        if (++wj < nj) who = __builtin_amdgcn_readfirstlane(mask[wj]);
      }
    }
  };
  fetch(c[0]);
  while (wj < nj) {
    fetch(c[1]);
    work(c[0]);
    fetch(c[0]);
    work(c[1]);
  }
  const int out = blockIdx.x * 64 * P + tid;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= T) break;
    if (r) __syncthreads();
#pragma unroll
    for (int p = 0; p < P; ++p) red[wave][lane * P + p] = y[r][p];
    __syncthreads();
    if (tid < 64 * P && out < a.O) {
      float v = 0.0f;
#pragma unroll
      for (int q = 0; q < kRowWaves; ++q) v += red[q][tid];
      if (a.chunks == 1)
        ((TX*)a.y)[(int64_t)r * a.O + out] = (TX)v;
      else
        ((float*)(a.ws + a.part_off))[((size_t)chunk * T + r) * a.O + out] = v;
    }
  }
}

// y from the chunks: a block 64 values, its waves every fourth chunk each.
template <typename TX>
__global__ __launch_bounds__(256) void k_few_rows_sum(FewArgs a) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = a.route.rows * a.O, q = (int64_t)blockIdx.x * 64 + lane;
  const float* part = (const float*)(a.ws + a.part_off) + (q < n ? q : 0);
  float v = 0.0f;
#pragma unroll 8
  for (int c = wave; c < a.chunks; c += 4) v += part[(size_t)c * n];
  red[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && q < n) ((TX*)a.y)[q] = (TX)((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
}

// More rows: a block takes up to kFewUnit slots of one of the chosen experts, 64 outputs and a chunk of inputs, and leaves
// part[chunk, slot, o] of up to kFewRows rows at a time. It finds its expert and that expert's slots itself. Rows that crowd
// on few experts thus spread over more blocks: 500 rows on two of 16 experts of 512 -> 512, degree 8, 85 us in fp32 and 61 in
// bf16 (a block an expert, however many its slots: 216 and 165), 200 on two of 8 of 1024 -> 1024 113 and 78 (180 and 132);
// where no expert has more than kFewUnit slots nothing changes.
//
// The products run on the matrix cores: on the vector ALU 64 rows, two of 8 experts of 1024 -> 1024, degree 8, took 112 us
// in bf16 and 131 in fp32 (here 52 and 85, of which the coefficients' stream is 29 and 59 and the launches of gate and sum
// 13); 20 rows, one of 8 of 2048 -> 2048, degree 4, 75 and 139 (57 and 131). In an instruction of 16 outputs by 16
// rows by 32 products a lane holds eight coefficients of one input and output, as they lie, and against them eight basis values of that input for one
// row, made in registers: bf16 coefficients are an operand as they are, fp32 ones and the basis values three bf16
// planes (24 bits), of whose products those below 2^-24 are left out. T_0 = 1 is a sum of coefficients beside them;
// degrees above 8 take a second run of eight basis values, padded with zeros.
constexpr int kFewMaxSlots = 1024, kFewInputs = 128, kFewRows = 32, kFewUnit = 2 * kFewRows;

// The eight coefficients of an output (its T_0 at `from`) from 8 G + 1 on as an operand.
template <int D, int G>
__device__ __forceinline__ Frag<kBf16> coef_frag(const __bf16* from) {
  Frag<kBf16> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = 8 * G + j + 1 < D ? from[8 * G + j + 1 < D ? 8 * G + j + 1 : 0] : (__bf16)0.0f;
  return f;
}
template <int D, int G>
__device__ __forceinline__ Frag<kSplit> coef_frag(const float* from) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 8 * G + j + 1 < D ? from[8 * G + j + 1 < D ? 8 * G + j + 1 : 0] : 0.0f;
  return make_frag_split_any(v);
}
__device__ __forceinline__ void add_products(f32x4_t& acc, const Frag<kBf16>& c, const Frag<kSplit>& b) {
#pragma unroll
  for (int k = 2; k >= 0; --k) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c.v, b.p[k], acc, 0, 0, 0);
}
__device__ __forceinline__ void add_products(f32x4_t& acc, const Frag<kSplit>& c, const Frag<kSplit>& b) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int k = 0; k <= s; ++k) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c.p[k], b.p[s - k], acc, 0, 0, 0);
}

// A lane's coefficients are those of P outputs next to each other, which go to tiles of their own: pairs in bf16, where
// outputs are even, so that they begin at whole dwords (20 rows of the case above: 75 us, one by one 99).
template <typename TX, typename TC, int D, int P>
__global__ __launch_bounds__(256, sizeof(TC) == 2 || D <= 12 ? 3 : 2) void k_few_stream(FewArgs a) {
  constexpr int kTiles = 4, kCols = kFewRows / 16, kPitch = 64 + 4;
  __shared__ int slots[kFewMaxSlots], counts[4], mine_e, mine_r;
  __shared__ unsigned chosen[kRouteMaxExperts / 32];
  __shared__ float t[kFewRows][kFewInputs + 1];
  __shared__ __align__(16) float red[4][16][kPitch];
  __shared__ float first[4][64];
  const int oc = (a.O + 63) / 64;
  int id = blockIdx.x;
  const int chunk = id % a.chunks;
  id /= a.chunks;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int o0 = id % oc * 64;
  int nth = id / oc;
  // the nth run of kFewUnit slots of an expert, and where it begins among them
  int e = -1, begin = 0;
  if (a.route.rows <= kFewUnit) {  // one an expert: the nth of the chosen experts
    if (tid < kRouteMaxExperts / 32) chosen[tid] = 0;
    __syncthreads();
    for (int s = tid; s < a.S; s += 256) {
      const int64_t x = a.route.indices[s];
      if (x >= 0 && x < a.route.E) atomicOr(&chosen[x >> 5], 1u << (x & 31));
    }
    __syncthreads();
    for (int w = 0; w < (a.route.E + 31) / 32; ++w) {
      unsigned bits = chosen[w];
      const int n = __popc(bits);
      if (nth < n) {
        for (; nth; --nth) bits &= bits - 1;
        e = w * 32 + __ffs(bits) - 1;
        break;
      }
      nth -= n;
    }
  } else {
    static_assert(kRouteMaxExperts == 2 * 256);
    int* load = (int*)&red[0][0][0];  // an expert's slots, until the first sums
    load[tid] = load[tid + 256] = 0;
    if (tid == 0) mine_e = -1;
    __syncthreads();
    for (int s = tid; s < a.S; s += 256) {
      const int64_t x = a.route.indices[s];
      if (x >= 0 && x < a.route.E) atomicAdd(&load[x], 1);
    }
    __syncthreads();
    // the runs of the experts before this thread's two
    const int own = (load[2 * tid] + kFewUnit - 1) / kFewUnit, both = own + (load[2 * tid + 1] + kFewUnit - 1) / kFewUnit;
    int before = both;
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) {
      const int o = __shfl_up(before, w);
      before += lane >= w ? o : 0;
    }
    if (lane == 63) counts[wave] = before;
    __syncthreads();
    before -= both;
    for (int w = 0; w < wave; ++w) before += counts[w];
    if (nth >= before && nth < before + both) {
      const int q = nth >= before + own;
      mine_e = 2 * tid + q;
      mine_r = (nth - before - (q ? own : 0)) * kFewUnit;
    }
    __syncthreads();
    e = mine_e;
    begin = mine_r;
  }
  if (e < 0) return;  // uniform: fewer runs than there are blocks for
  e = __builtin_amdgcn_readfirstlane(e);
  int n = 0;
  for (int s0 = 0; s0 < a.S; s0 += 256) {
    const int s = s0 + tid;
    const bool mine = s < a.S && a.route.indices[s] == e;
    const unsigned long long has = __ballot(mine);
    if (lane == 0) counts[wave] = __popcll(has);
    __syncthreads();
    int at = n;
    for (int w = 0; w < wave; ++w) at += counts[w];
    if (mine) slots[at + __popcll(has & ((1ull << lane) - 1))] = s;
    n += counts[0] + counts[1] + counts[2] + counts[3];
    __syncthreads();
  }
  const int i0 = chunk * a.chunk_inputs, ni = a.I - i0 < a.chunk_inputs ? a.I - i0 : a.chunk_inputs;
  const int64_t pitch = (int64_t)a.O * D;
  // a lane's outputs o0 + (16 q + lane % 16) P and on, its inputs i + lane / 16
  const int col = lane & 15, sub = lane >> 4;
  // (loads past the ends go to the last ones: a branch around a load makes the compiler wait for it at once)
  const TC* C = (const TC*)a.coeffs + ((int64_t)e * a.I + i0) * pitch;
  int off[kTiles / P];
#pragma unroll
  for (int q = 0; q < kTiles / P; ++q) {
    const int o = o0 + (q * 16 + col) * P;
    off[q] = (o < a.O ? o : a.O - P) * D;
  }
  float* part = (float*)(a.ws + a.part_off) + (size_t)chunk * a.S * a.O;
  if (n > begin + kFewUnit) n = begin + kFewUnit;
  for (int r0 = begin; r0 < n; r0 += kFewRows) {
    const int nr = n - r0 < kFewRows ? n - r0 : kFewRows;
    Coefs<TC, D * P> c[kTiles / P];
    const auto fetch = [&](int i, int q) {  // inputs from i on
      const TC* at = C + (int64_t)(i + sub < ni ? i + sub : ni - 1) * pitch;
      c[q] = *(const Coefs<TC, D * P>*)(at + off[q]);
    };
#pragma unroll
    for (int q = 0; q < kTiles / P; ++q) fetch(wave * 4, q);
    for (int q = tid; q < ni * nr; q += 256) {
      const int r = q / ni, i = q - r * ni;
      t[r][i] = tanhf((float)((const TX*)a.x)[(int64_t)(slots[r0 + r] / a.route.top_k) * a.I + i0 + i]);
    }
    __syncthreads();
    f32x4_t acc[kTiles][kCols] = {};
    float ones[kTiles] = {};
    for (int i = wave * 4; i < ni; i += 16) {
      // inputs past the end count as 0; rows past the end have columns of their own, which nobody reads
      if (i + 4 > ni && i + sub >= ni)
#pragma unroll
        for (int q = 0; q < kTiles / P; ++q) c[q] = Coefs<TC, D * P>{};
      float u[kCols], ta[kCols], tb[kCols];
#pragma unroll
      for (int k = 0; k < kCols; ++k) {
        u[k] = i + sub < ni ? t[k * 16 + col][i + sub] : 0.0f;
        ta[k] = 1.0f;
        tb[k] = u[k];
      }
      const auto group = [&](auto g) {
        constexpr int G = decltype(g)::value;
        Frag<kSplit> b[kCols];
#pragma unroll
        for (int k = 0; k < kCols; ++k) {
          if (k && nr <= 16) break;
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = 0.0f;
            if (8 * G + j + 1 >= D) continue;
            v[j] = tb[k];
            const float next = fmaf(u[k] + u[k], tb[k], -ta[k]);
            ta[k] = tb[k];
            tb[k] = next;
          }
          b[k] = make_frag_split(v);
        }
#pragma unroll
        for (int tile = 0; tile < kTiles; ++tile) {
          const TC* from = c[tile / P].v + tile % P * D;
          const auto f = coef_frag<D, G>(from);
          if (G == 0) ones[tile] += (float)from[0];
          if (8 * G + 9 >= D && tile % P == P - 1) fetch(i + 16, tile / P);
          add_products(acc[tile][0], f, b[0]);
          if (nr > 16) add_products(acc[tile][1], f, b[1]);
        }
      };
      group(std::integral_constant<int, 0>());
      if constexpr (D > 9) group(std::integral_constant<int, 1>());
    }
#pragma unroll
    for (int tile = 0; tile < kTiles; ++tile) {  // over the lanes of an output
      auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(ones[tile]), __float_as_uint(ones[tile]), false, false);
      const float v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      if (sub == 0) first[wave][(tile / P * 16 + col) * P + tile % P] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    // the waves' sums: a lane has outputs (16 (tile / P) + 4 sub + j) P + tile % P of row col
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      if (k * 16 >= nr) break;
      if (k) __syncthreads();
#pragma unroll
      for (int tile = 0; tile < kTiles; tile += P) {
        f32x4_t* to = (f32x4_t*)&red[wave][col][(tile * 16 + sub * 4 * P)];
        if constexpr (P == 1) {
          to[0] = acc[tile][k];
        } else {
          const f32x4_t u = acc[tile][k], v = acc[tile + 1][k];
          to[0] = f32x4_t{u[0], v[0], u[1], v[1]};
          to[1] = f32x4_t{u[2], v[2], u[3], v[3]};
        }
      }
      __syncthreads();
      const int r = k * 16 + (tid >> 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int o = j * 16 + (tid & 15);
        const float v = (red[0][tid >> 4][o] + red[1][tid >> 4][o]) + (red[2][tid >> 4][o] + red[3][tid >> 4][o]) +
                        ((first[0][o] + first[1][o]) + (first[2][o] + first[3][o]));
        if (r < nr && o0 + o < a.O) part[(size_t)slots[r0 + r] * a.O + o0 + o] = v;
      }
    }
    __syncthreads();
  }
}

// y from the parts: a block a row's 64 outputs, its waves every fourth part each.
template <typename TX>
__global__ __launch_bounds__(256) void k_few_sum(FewArgs a) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = a.route.top_k;
  const int64_t row = blockIdx.y;
  const int o = blockIdx.x * 64 + lane;
  const float* part = (const float*)(a.ws + a.part_off) + (o < a.O ? o : 0);
  float v = 0.0f;
  for (int j = 0; j < k; ++j) {
    const int64_t s = row * k + j;
    const int64_t e = a.route.indices[s];
    if (e < 0 || e >= a.route.E) continue;
    float z = 0.0f;
#pragma unroll 8
    for (int c = wave; c < a.chunks; c += 4) z += part[((size_t)c * a.S + s) * a.O];
    v = fmaf(a.route.weights[s], z, v);
  }
  red[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && o < a.O) ((TX*)a.y)[row * a.O + o] = (TX)((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
}

template <typename TX, typename TC, int D>
void launch_products(const FewArgs& a, hipStream_t st) {
  if (!a.by_row) {
    const dim3 grid((unsigned)((int64_t)a.chunks * ceil_div(a.O, 64) * a.runs));
    if (sizeof(TC) == 2 && a.O % 2 == 0)
      hipLaunchKernelGGL((k_few_stream<TX, TC, D, 4 / sizeof(TC)>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((k_few_stream<TX, TC, D, 1>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL((k_few_sum<TX>), dim3((unsigned)ceil_div(a.O, 64), (unsigned)a.route.rows), dim3(256), 0, st, a);
    return;
  }
  const dim3 grid((unsigned)ceil_div(a.O, a.coeff_bf16 ? 128 : 64), (unsigned)a.chunks), block(kRowThreads);
  if (a.gated)
    hipLaunchKernelGGL((k_few_rows<TX, TC, D, 1, true>), grid, block, 0, st, a);
  else if (a.route.rows <= 4)
    hipLaunchKernelGGL((k_few_rows<TX, TC, D, 4, false>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((k_few_rows<TX, TC, D, kRowsMax, false>), grid, block, 0, st, a);
  if (a.chunks > 1)
    hipLaunchKernelGGL((k_few_rows_sum<TX>), dim3((unsigned)ceil_div(a.route.rows * a.O, 64)), dim3(256), 0, st, a);
}

template <typename TX, typename TC>
void launch_degree(const FewArgs& a, hipStream_t st) {
  switch (a.D) {
#define CKAN_FEW_CASE(N) case N: launch_products<TX, TC, N>(a, st); break;
    CKAN_FEW_CASE(2) CKAN_FEW_CASE(3) CKAN_FEW_CASE(4) CKAN_FEW_CASE(5) CKAN_FEW_CASE(6) CKAN_FEW_CASE(7)
    CKAN_FEW_CASE(8) CKAN_FEW_CASE(9) CKAN_FEW_CASE(10) CKAN_FEW_CASE(11) CKAN_FEW_CASE(12) CKAN_FEW_CASE(13)
    CKAN_FEW_CASE(14) CKAN_FEW_CASE(15) CKAN_FEW_CASE(16) CKAN_FEW_CASE(17)
#undef CKAN_FEW_CASE
  }
}

}  // namespace
}  // namespace ckan
