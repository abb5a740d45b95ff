// Launch interface of the mixture-of-experts and orthogonalisation kernels.
#pragma once

#include "ckan_kernels.hpp"

namespace ckan {

// The largest value and the sum over a wave, uniform: within rows of 16 lanes and then
// across them by data-parallel moves on the vector ALU.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_from(float fallback, float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(__float_as_int(fallback), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
// A lane whose move has no source keeps its value.  Two wait states lie between a
// vector write and its read by a move across lanes.  In assembly: from fmaxf and the
// builtin come five instructions a step.
__device__ __forceinline__ float wave_max(float v) {
  asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t"
      "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf"
      : "+v"(v));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp_from<0x111, 0xf>(0.0f, v);
  v += dpp_from<0x112, 0xf>(0.0f, v);
  v += dpp_from<0x114, 0xf>(0.0f, v);
  v += dpp_from<0x118, 0xf>(0.0f, v);
  v += dpp_from<0x142, 0xa>(0.0f, v);
  v += dpp_from<0x143, 0xc>(0.0f, v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// ---- routing (ckan_route.hip) -----------------------------------------------
constexpr int kRouteMaxExperts = 512;  // 8 experts a lane
constexpr int kRouteMaxTopK = 64;      // lane j holds the j-th chosen expert
constexpr int kRouteMaxGroups = 64;    // a lane a group
// Added to the sum that renormalised weights are divided by: a row whose chosen
// scores all underflow gets zero weights instead of NaN.
constexpr float kRouteEps = 1e-20f;

struct RouteArgs {
  const void* logits;  // [rows, E], row pitch ld
  const float* bias;   // [E] or NULL
  float* weights;      // [rows, top_k]
  int64_t* indices;    // [rows, top_k] (read by the backward)
  const float* dweights;
  void* dlogits;       // [rows, E]
  int64_t rows, ld;
  int E, top_k, groups, top_groups;
  int lanes_log2;      // lanes a group in the choice of groups
  float inv_size;      // 1 / (experts a group): an expert's group is (e + 0.5) times it
  int softmax, renormalize, bf16;
  float scale;
};
void launch_route(const RouteArgs& a, bool backward, hipStream_t st);

// ---- orthogonalisation (ckan_ortho.hip) ---------------------------------------
// A batch of matrices in memory: element (r, c) of matrix b lies at
// b sb + r sr + (c / inner) so + (c % inner) si.  inner = 1 is an ordinary
// strided matrix; a ChebyKAN layer's [in, out, D] coefficients as the matrix
// [out, in D] have inner = D, sr = D, so = out D, si = 1.
struct MatView {
  int64_t sb, sr, so, si;
  int inner;
};

struct OrthoArgs {
  int batch, rows, cols;
  int steps;
  float a, b, c, eps;
  int bf16;            // element type of in and out (orthogonalize)
  MatView view;        // of in, out / of p, g, buf
  const void* in;      // orthogonalize: the matrices
  void* out;
  float *p, *buf;      // Muon step (in == nullptr): all fp32, one view
  const float* g;
  float lr, momentum, decay, scale;
  int nesterov;
};
// ---- ChebyKAN experts (ckan_experts.hip) ---------------------------------------
constexpr int kExpertsMax = 512;       // a thread of the plan's scan an expert
constexpr int kExpertsMaxDegree = 16;
constexpr int kExpertsMaxTopK = 64;
constexpr int kPlanThreads = 1024;
constexpr int kPlanBlocks = 256;       // at most: a block's share of the slots grows past that
constexpr int kMaxParts = 128;         // blocks an expert that look for its largest coefficient

// Sizes and the layout of the buffers.  "Rows" are the kept slots sorted by expert,
// each expert's run padded to a multiple of 32; "slots" are the T top_k entries of
// the caller's indices.
struct ExpertsPlan {
  int64_t T, S;        // tokens, slots
  int E, k, I, O, deg, D;
  int P;               // degrees a forward reduction group holds (deg padded to 4, 8 or 16)
  int NP;              // fp16 planes an operand: 1 for bf16 tensors, 2 for fp32
  bool bf16, wbf16;
  int Ip;              // I padded to 32: pitch of the tanh cache, inputs of the packs
  int Op;              // O padded to 32
  int64_t R;           // rows allocated (a multiple of 128)
  int tiles;           // 128-row tiles at most
  int plan_blocks;
  int64_t plan_chunk;  // slots a plan block takes (a multiple of kPlanThreads)
  // saved from the forward to the backward
  size_t off_off, tok_off, slot_off, row_off, tiles_off, order_off, scale_off, t_off, z_off, cb_off, saved_bytes;
  // forward workspace
  size_t hist_off, cmax_off, cf_off, bias_off, fpart_off, fwd_bytes;
  // backward workspace
  size_t gmax_off, gscale_off, rscale_off, gr_off, gt_off, gsum_off, gtot_off, ts_off, dxs_off, bpart_off, bwd_bytes;
  int pack_inputs;     // inputs a block of the pack takes
  int bias_parts;      // input chunks of the pack's sums of T_0 coefficients
  // the streaming forward (few slots): input chunks, inputs a chunk, partial sums
  bool stream;
  int chunks, chunk_inputs;
  size_t part_off, stream_bytes;
};
constexpr int kStreamMaxSlots = 1024;  // a block keeps its expert's slots in LDS
constexpr int kStreamInputs = 64;      // inputs whose basis values a block holds at once
constexpr int kStreamRows = 8;         // rows a pass over the coefficients serves
ExpertsPlan make_experts_plan(int64_t T, int E, int k, int I, int O, int deg, bool bf16, bool wbf16);

struct ExpertsArgs {
  ExpertsPlan p;
  const void *x, *coeffs, *weights, *dy;
  const int64_t* indices;
  void *y, *dx, *dcoeffs, *dweights;
  char *saved, *ws;
};
void launch_experts_forward(const ExpertsArgs& a, bool keep, hipStream_t st);
// The forward without a backward of few slots (p.stream).
void launch_experts_stream(const ExpertsArgs& a, hipStream_t st);
void launch_experts_backward(const ExpertsArgs& a, hipStream_t st);

// ---- a mixture layer for few rows (ckan_few.hip) ---------------------------------
// Gate, choice, experts and their sum without a backward.
struct FewArgs {
  RouteArgs route;     // rows, experts, choice; the outputs' weights and indices
  int I, O, D, S;      // S: slots, rows top_k
  const void *x, *gate, *coeffs;
  int x_bf16, gate_bf16, coeff_bf16;
  void* y;
  char* ws;
  // the launch's plan (few_plan)
  bool few;            // whether this form takes the call
  bool apart;          // logits by a launch of their own
  bool gated;          // the choice made by the products' launch
  bool by_row;         // the products by k_few_rows
  int runs, chunks, chunk_inputs;
  size_t part_off, ws_bytes;
};
void few_plan(FewArgs* a);
void launch_few(const FewArgs& a, hipStream_t st);
void launch_few_bf16(const FewArgs& a, hipStream_t st);  // the products on bf16 coefficients (ckan_few_bf16.hip)

size_t ortho_workspace_bytes(const OrthoArgs& a);
void launch_ortho(const OrthoArgs& a, void* ws, hipStream_t st);
// Matrices whose smaller side is at most 64 (ckan_ortho_small.hip): its 64 x 64 products in
// one CU's LDS are the limit.  [64, 3920] takes 71 us there, [65, 3920] 181 in fp32 and 134 in
// bf16 by the launches of ckan_ortho.hip.
inline bool ortho_small(int rows, int cols) { return (rows < cols ? rows : cols) <= 64; }
size_t ortho_small_workspace_bytes(const OrthoArgs& a);
void launch_ortho_small(const OrthoArgs& a, void* ws, hipStream_t st);

}  // namespace ckan
