// A whole mixture layer for few rows (ckan_mixture_forward): plan, gate and choice, and the
// products on fp32 coefficients.
#include "ckan_few.hpp"

namespace ckan {
namespace {

template <typename TX, typename TG>
__global__ __launch_bounds__(kGateThreads) void k_few_gate(FewArgs a) {
  __shared__ GateShared sh;
  int mine = -1;
  float weight = 0.0f;
  const int64_t row = blockIdx.x;
  gate_row<TX, TG>(a, row, sh, mine, weight);
  if ((int)threadIdx.x < a.route.top_k) {
    a.route.weights[row * a.route.top_k + threadIdx.x] = weight;
    a.route.indices[row * a.route.top_k + threadIdx.x] = mine;
  }
}

// The logits alone, where a gate is too large for one block a row: a wave four experts.
template <typename TX, typename TG>
__global__ __launch_bounds__(256) void k_few_logits(FewArgs a) {
  const int lane = threadIdx.x & 63, e0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kGateExperts;
  if (e0 >= a.route.E) return;
  const int64_t row = blockIdx.y;
  double sum[kGateExperts] = {};
  gate_dots<TX, TG>(a, row, e0, 0, (a.I + kChunk - 1) / kChunk, lane, sum);
#pragma unroll
  for (int q = 0; q < kGateExperts; ++q) {
    const double v = wave_sum64(sum[q]);
    if (lane == 0 && e0 + q < a.route.E) ((float*)a.ws)[row * a.route.E + e0 + q] = (float)v;
  }
}

template <typename TX, typename TG>
void launch_gate(const FewArgs& a, hipStream_t st) {
  if (a.gated) return;
  if (!a.apart) {
    hipLaunchKernelGGL((k_few_gate<TX, TG>), dim3((unsigned)a.route.rows), dim3(kGateThreads), 0, st, a);
    return;
  }
  hipLaunchKernelGGL((k_few_logits<TX, TG>), dim3((unsigned)ceil_div(a.route.E, 4 * kGateExperts), (unsigned)a.route.rows), dim3(256),
                     0, st, a);
  RouteArgs r = a.route;
  r.logits = a.ws;
  launch_route(r, false, st);
}

}  // namespace

void few_plan(FewArgs* a) {
  const int64_t rows = a->route.rows, S = rows * a->route.top_k, E = a->route.E;
  const int64_t active = E < S ? E : S;
  // fewer than 64 slots an expert on average, two passes of kFewRows: 240 rows, two of 8 experts of 1024 -> 1024, degree
  // 8, 105 us in bf16 and 174 in fp32 (the parts' entry points, which pack the coefficients, 173 and 279), 64 rows 53 and 88
  // (110 and 137); 500 rows of 512 -> 512, two of 16, 73 and 108 (111 and 161), all on the same two 61 and 85 (103 and 150)
  a->few = rows > 0 && S <= kFewMaxSlots && S < 64 * active;
  if (!a->few) return;
  a->S = (int)S;
  // runs of kFewUnit slots of one expert: at most one begun an expert and one for every kFewUnit slots
  a->runs = (int)(rows > kFewUnit ? active + S / kFewUnit : active);
  // a gate of 2^16 entries: one launch 20.0 us (1 row) to 26.8 (64 rows), two 22.3 to 26.9; of 2^18
  // entries 22.6 to 41.7 and 22.1 to 35.4
  // and where a block's waves would take their four experts in two rounds or more, the GPU's time in one launch and in two: 128
  // experts of 128 inputs 14.1 and 12.6 (2 rows), 17.2 and 16.2 (64), 512 of 128 28.0 and 14.2, 32.1 and 21.5; 96 of 128 9.7 and
  // 11.3 (1 row), 12.7 and 12.5, 15.7 and 15.8
  a->apart = E * a->I > (1 << 16) || E >= 2 * kGateWaves * kGateExperts;
  a->gated = rows == 1 && !a->apart;
  // a block of k_few_rows visits every chosen expert in turn, some 0.5 us each where its coefficients are few: 8 rows of 16 of 128
  // experts of 64 -> 64, degree 3, 57 us (k_few_stream 26), 5 rows of 16 of 384 of 128 -> 128, degree 4, 55 (40), but 8 rows of 16 of
  // 128 of 512 -> 512, degree 4, 87 (107), in bf16 79 (57), of 12 of 32 of 1024 -> 1024 122 (151), in bf16 81 (87)
  const int64_t expert_bytes = (int64_t)a->I * a->O * a->D * (a->coeff_bf16 ? 2 : 4);
  const bool by_row = a->by_row = rows <= kRowsMax && (S <= 64 || expert_bytes >= 5 << 20);
  // k_few_stream makes fp32 coefficients of degree 9 and more operands in two runs of three planes, whether two rows or 32 meet them:
  // where few do and the coefficients are many, the parts' vector ALU is as fast or faster (12 rows, three of 12 experts of 300 ->
  // 700, degree 16, 62 us and 56, 24 rows 72 and 62, 48 rows 75 and 84; 16 rows, two of 32 of 700 -> 300, 92 and 75; two of 8 of 512 ->
  // 512 52 and 48). Of fewer coefficients their launches take longer (two of 8 of 512 -> 512, degree 12, 43 and 45)
  if (!by_row && !a->coeff_bf16 && a->D > 9 && S < 8 * active && active * a->I * a->O * a->D >= (int64_t)1 << 25) {
    a->few = false;
    return;
  }
  // chunks of inputs: a block of k_few_rows a CU, four of k_few_stream's (64 rows, two of 8 experts of 1024 -> 1024 in
  // bf16: four 52 us, six 58, eight 55; 2048 -> 700, degree 16, 121, 128 and 127), at least an input a wave, at most
  // what a block holds
  const int64_t oc = ceil_div(a->O, by_row && a->coeff_bf16 ? 128 : 64), hold = by_row ? kRowTanh : kFewInputs;
  int64_t chunks = by_row ? ceil_div(kNumCUs, oc) : ceil_div(4 * kNumCUs, active * oc);
  if (chunks > ceil_div(a->I, 16)) chunks = ceil_div(a->I, 16);
  if (chunks < ceil_div(a->I, hold)) chunks = ceil_div(a->I, hold);
  a->chunk_inputs = (int)ceil_div(a->I, chunks);
  a->chunks = (int)ceil_div(a->I, a->chunk_inputs);
  // a launch holds fewer than 2^32 threads
  if (!by_row && a->chunks * oc * a->runs >= ((int64_t)1 << 24)) a->few = false;
  a->part_off = align256(a->apart ? (size_t)rows * E * sizeof(float) : 1);
  a->ws_bytes = a->part_off + align256((size_t)a->chunks * (by_row ? rows : S) * a->O * sizeof(float));
}

void launch_few(const FewArgs& a, hipStream_t st) {
  if (a.x_bf16)
    a.gate_bf16 ? launch_gate<__bf16, __bf16>(a, st) : launch_gate<__bf16, float>(a, st);
  else
    a.gate_bf16 ? launch_gate<float, __bf16>(a, st) : launch_gate<float, float>(a, st);
  if (a.coeff_bf16)
    launch_few_bf16(a, st);
  else
    a.x_bf16 ? launch_degree<__bf16, float>(a, st) : launch_degree<float, float>(a, st);
}

}  // namespace ckan
