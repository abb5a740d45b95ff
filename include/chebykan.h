/*
 * chebykan.h -- C-ABI of the MI355X (gfx950) ChebyKAN layer hot path.
 *
 * The reference (0xEodum/KAN) is pure Python on torch; this boundary replaces
 * the torch op sequences its ChebyKAN layer executes.  Each entry point names
 * the reference code it stands in for.  No torch or C++ types cross it: plain
 * device pointers, sizes and a hipStream_t passed as void*.
 *
 * Conventions
 *   - All pointers are device pointers unless stated; all launches are
 *     stream-ordered on `stream` (a hipStream_t) and never synchronise the host.
 *   - x, y, dy, dx and t are row-major fp32.  Coefficients C are [in, out, D]
 *     row-major (D = degree + 1), fp32 or bf16, the layout of the reference's
 *     `cheby_coeffs` parameter (kan/layers/chebykan.py:48-51).
 *   - Every call returns a ckan_status; on failure ckan_last_error() returns a
 *     thread-local message.  Argument checks happen on the host before any
 *     launch, so an invalid call launches nothing.
 *   - Workspaces are caller-allocated scratch (split-K partials, re-laid
 *     operands); no call needs them zeroed.  Calls that share one workspace
 *     must not overlap in time.
 */
#ifndef CHEBYKAN_H
#define CHEBYKAN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum ckan_status {
  CKAN_OK = 0,
  CKAN_ERR_INVALID_ARG = 1,   /* bad shape, null pointer, size mismatch  */
  CKAN_ERR_UNSUPPORTED = 2,   /* valid request this build does not serve */
  CKAN_ERR_WORKSPACE = 3,     /* workspace smaller than required          */
  CKAN_ERR_HIP = 4            /* a HIP runtime call or launch failed      */
} ckan_status;

typedef enum ckan_compute {
  CKAN_COMPUTE_FP32 = 0,      /* fp32 results: fp32 MFMA, or fp32 operands as three exact bf16 planes */
  CKAN_COMPUTE_BF16 = 1       /* bf16 MFMA, fp32 accumulate (v_mfma_f32_32x32x16_bf16) */
} ckan_compute;

typedef enum ckan_dtype {
  CKAN_DTYPE_F32 = 0,
  CKAN_DTYPE_BF16 = 1
} ckan_dtype;

/* How the layer maps an input x to the argument t of its basis. */
typedef enum ckan_input_map {
  CKAN_INPUT_TANH = 0,    /* t = tanh(x), the reference's default
                             (kan/basis/chebyshev.py:68-78)                */
  CKAN_INPUT_AFFINE = 1   /* t = in_scale * x + in_shift: the Hermite
                             layer's map of a finite domain onto [-3, 3]
                             (kan/basis/hermite.py:102-112), expressed on
                             [-1, 1] with the basis scale 3               */
} ckan_input_map;

/* Problem descriptor: one ChebyKANLayer(in_dim, out_dim, degree) applied to a
 * batch of `batch` rows (kan/layers/chebykan.py:21-22,64).
 * Degrees 0..16 run on the MFMA kernels in the compute precision.  Degrees
 * 17..1024 (the reference layer takes any degree, kan/layers/chebykan.py:21-51)
 * run on the general kernels (fp32 matrix instructions) in fp32 whatever
 * `compute` asks, with either input map; their packed buffer is C widened to
 * fp32 in its own [in, out, D] layout followed by the basis recurrence block,
 * and they need no workspace (the size queries return 0). */
typedef struct ckan_desc {
  int64_t batch;        /* B: rows of x after x.view(-1, in_dim)          */
  int32_t in_dim;       /* I                                               */
  int32_t out_dim;      /* O                                               */
  int32_t degree;       /* deg (0..1024); D = deg + 1 coefficients per (i, o) */
  int32_t compute;      /* ckan_compute                                    */
  int32_t coeff_dtype;  /* ckan_dtype of C passed to ckan_pack_coeffs      */
  int32_t input_map;    /* ckan_input_map (0: tanh)                        */
  float in_scale;       /* CKAN_INPUT_AFFINE: t = in_scale * x + in_shift  */
  float in_shift;       /* (both 0 with CKAN_INPUT_TANH)                   */
} ckan_desc;

/* ---- sizes (host only, no device work) ---------------------------------- */

/* Bytes of the packed-coefficient buffer written by ckan_pack_coeffs. */
size_t ckan_packed_bytes(const ckan_desc* desc);
/* Elements (fp32) of the tanh cache written by ckan_forward and read by
 * ckan_backward: tanh(x) as [B, in_pad] with zero padding columns. */
size_t ckan_tcache_elems(const ckan_desc* desc);
/* Bytes of forward / backward workspace. */
size_t ckan_fwd_workspace_bytes(const ckan_desc* desc);
size_t ckan_bwd_workspace_bytes(const ckan_desc* desc, int need_dx, int need_dcoeffs);

/* Zero-fill a workspace on `stream` with a fill kernel (no hipMemset).  No
 * entry point requires it; kept for callers that want defined contents. */
int ckan_workspace_init(void* ws, size_t ws_bytes, void* stream);

/* ---- layer operators ---------------------------------------------------- */

/* Re-lays C [in, out, D] out into the MFMA operand layouts used by the
 * forward and input-gradient contractions, in the compute precision, and the
 * per-output bias sum_i C[i, o, 0] (the T_0 = 1 term).
 * Replaces: the coefficient permute/reshape/clone inside
 * torch.einsum('bid,iod->bo') (kan/basis/chebyshev.py:101). */
int ckan_pack_coeffs(const ckan_desc* desc, const void* coeffs, void* packed, void* stream);

/* y[b, o] = sum_{i, d} T_d(tanh x[b, i]) C[i, o, d]; also writes t = tanh(x)
 * into t_cache (ckan_tcache_elems floats) for the backward.
 * Replaces: ChebyshevBasis.forward (kan/basis/chebyshev.py:80-101): tanh
 * (:78), closed-form basis (:130-145) and the einsum (:101). */
int ckan_forward(const ckan_desc* desc, const float* x, const void* packed, float* y,
                 float* t_cache, void* ws, size_t ws_bytes, void* stream);

/* ckan_pack_coeffs (or, with a non-NULL basis spec, ckan_pack_coeffs_basis,
 * below) followed by ckan_forward, in fewer launches: the tanh of x is
 * computed by the pack launch itself where the layout allows, and the
 * per-output bias sum is reduced by the forward GEMM where it can.  Same
 * arguments, results and packed-buffer contents as the two calls.
 * Replaces: the layer forward as the reference runs it on every call, the
 * einsum's coefficient re-layout included (kan/layers/chebykan.py:64-67,
 * kan/basis/chebyshev.py:78,92-101). */
struct ckan_basis_spec;
int ckan_pack_forward(const ckan_desc* desc, const struct ckan_basis_spec* spec,
                      const void* coeffs, void* packed, const float* x, float* y, float* t_cache,
                      void* ws, size_t ws_bytes, void* stream);

/* ckan_forward without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, serving loops and
 * harnesses that forbid hipMalloc).  No counterpart in the reference.  The
 * split-K partials of the small-batch paths go to a fixed device array of
 * CKAN_NOALLOC_SCRATCH_BYTES, one per GPU, held until the process ends; the
 * call allocates nothing (no hipMalloc / hipFree).  Shapes whose
 * ckan_fwd_workspace_bytes exceeds that size return CKAN_ERR_WORKSPACE and
 * launch nothing.  Every call on one GPU shares that GPU's array, so calls that
 * overlap in time on one GPU (e.g. on two streams) race; calls in one stream
 * order are safe.  Results are identical to ckan_forward's. */
#define CKAN_NOALLOC_SCRATCH_BYTES ((size_t)16 << 20)
int ckan_forward_noalloc(const ckan_desc* desc, const float* x, const void* packed, float* y,
                         float* t_cache, void* stream);

/* Gradients of the forward for upstream gradient dy [B, out]:
 *   dx[b, i]    = (1 - t^2) sum_{o, d} dy[b, o] C[i, o, d] d U_{d-1}(t)   (dx may be NULL)
 *   dC[i, o, d] = sum_b T_d(t[b, i]) dy[b, o]                            (dcoeffs may be NULL)
 * With accumulate != 0, dC is added to the existing contents of dcoeffs
 * (torch AccumulateGrad semantics); otherwise it is overwritten.  packed may
 * be NULL when dx is NULL, except above degree 16, where it also carries the
 * basis recurrence that dC needs.
 * Replaces: torch autograd through kan/basis/chebyshev.py:78,101,136-145
 * (BmmBackward0 x2, CosBackward0, MulBackward0, AcosBackward0, TanhBackward0).
 * Divergence: for |x| >= 9.0108, where fp32 tanh(x) == +-1, the reference
 * yields NaN in dx (acos'(+-1) = -inf); this returns the finite analytic value. */
int ckan_backward(const ckan_desc* desc, const float* t_cache, const void* packed,
                  const float* dy, float* dx, float* dcoeffs, int accumulate,
                  void* ws, size_t ws_bytes, void* stream);

/* ---- fp64 path ------------------------------------------------------------
 * The reference layer computes in fp64 when its parameter is fp64
 * (kan/layers/chebykan.py:48-51 after .double(); kan/basis/chebyshev.py:78-101
 * then runs in fp64).  These entry points run that case in fp64 end to end
 * (fp64 matrix instructions).  x, coeffs [in, out, D], y, t_cache [B, in],
 * dy, dx and dcoeffs are fp64; desc->compute and desc->coeff_dtype must be 0.
 * No packing and no workspace: coeffs are read in their own layout.
 * Same formulas, NULL rules and accumulate semantics as ckan_forward /
 * ckan_backward, and the same finite value at tanh saturation (|x| >= 19.06
 * in fp64). */
int ckan_forward_f64(const ckan_desc* desc, const double* x, const double* coeffs, double* y,
                     double* t_cache, void* stream);
int ckan_backward_f64(const ckan_desc* desc, const double* t_cache, const double* coeffs,
                      const double* dy, double* dx, double* dcoeffs, int accumulate, void* stream);

/* The fp64 path for a layer of another polynomial family (ckan_basis_spec,
 * below): the Jacobi and Hermite layers after .double(), whose reference
 * computes their bases in fp64 (kan/basis/jacobi.py:96-117,159-188,
 * kan/basis/hermite.py:118-139,158-233).  The basis P_n(s tanh x) is evaluated
 * by the family's three-term recurrence in fp64 (no change of basis, whose
 * matrix entries reach 1e10 for Hermite), from a recurrence block that
 * ckan_write_recurrence_f64 writes into a caller-owned device buffer of
 * ckan_recurrence_bytes_f64(spec) bytes (8-byte aligned) once per spec;
 * the forward and backward then read it (spec->degree must equal
 * desc->degree: the library cannot check the buffer's contents).  dcoeffs is
 * the family coefficients' gradient.  The tanh input map only. */
size_t ckan_recurrence_bytes_f64(const struct ckan_basis_spec* spec);
int ckan_write_recurrence_f64(const struct ckan_basis_spec* spec, double* rec, void* stream);
int ckan_forward_f64_basis(const ckan_desc* desc, const double* rec, const double* x,
                           const double* coeffs, double* y, double* t_cache, void* stream);
int ckan_backward_f64_basis(const ckan_desc* desc, const double* rec, const double* t_cache,
                            const double* coeffs, const double* dy, double* dx, double* dcoeffs,
                            int accumulate, void* stream);

/* ---- other polynomial bases through the same kernels ---------------------
 * A layer whose basis is a three-term-recurrence family P_0..P_deg evaluated
 * at s * tanh(x) is the ChebyKAN layer with coefficients C' = C M, where
 *   P_n(s u) = sum_k M[n, k] T_k(u)      (M lower triangular, exact),
 * and its coefficient gradient is dC = dC' M^T; the input gradient is the
 * ChebyKAN layer's with C'.  So ckan_pack_coeffs_basis + ckan_forward +
 * ckan_backward (into dC') + ckan_coeff_grad_from_chebyshev run such a layer
 * (ckan_backward_basis: the last two in one call).
 * Above degree 16 (the general kernels) the packed buffer carries the
 * family's recurrence instead of C M: the kernels evaluate P_n(s u) by the
 * recurrence and differentiate it, ckan_backward's dC is already the family
 * coefficients' gradient and ckan_coeff_grad_from_chebyshev is the identity
 * (a copy, an accumulation, or nothing in place), so the same four calls
 * serve every degree.
 * Families and the reference code each replaces:
 *   JACOBI     P_n^(alpha,beta), alpha, beta > -1, s = 1: JacobiBasis
 *              (kan/basis/jacobi.py:84-117,147-188), JacobiKANLayer
 *              (kan/layers/jacobikan.py:26-77)
 *   HERMITE    physicists' H_n; HermiteKANLayer's default input map is
 *              s = 3 (kan/basis/hermite.py:85-116,158-193)
 *   HERMITE_E  probabilists' He_n, s = 3 (kan/basis/hermite.py:195-233)
 *   CHEBYSHEV  T_n (M = identity)
 */
typedef enum ckan_basis_family {
  CKAN_BASIS_CHEBYSHEV = 0,
  CKAN_BASIS_JACOBI = 1,
  CKAN_BASIS_HERMITE = 2,
  CKAN_BASIS_HERMITE_E = 3
} ckan_basis_family;

typedef struct ckan_basis_spec {
  int32_t family;   /* ckan_basis_family                                      */
  int32_t degree;   /* 0..1024 (0..16 for ckan_basis_to_chebyshev and the
                       derivative entry points); equal to desc->degree where a
                       desc is passed too */
  double alpha;     /* Jacobi parameters (> -1); ignored by the other families */
  double beta;
  double scale;     /* s: the basis is evaluated at s * tanh(x) (finite)       */
} ckan_basis_spec;

/* Host only: M as (degree+1)^2 doubles, M[n * (degree+1) + k]. */
int ckan_basis_to_chebyshev(const ckan_basis_spec* spec, double* M);
/* ckan_pack_coeffs of C' = C M, for C in the family's basis (fp32 or bf16 per
 * desc->coeff_dtype).  M is built on the host and passed by value.  Above
 * degree 16: C widened to fp32 and the family's recurrence block. */
int ckan_pack_coeffs_basis(const ckan_desc* desc, const ckan_basis_spec* spec, const void* coeffs,
                           void* packed, void* stream);
/* dcoeffs[i, o, n] (+)= sum_k dcheb[i, o, k] M[n, k] (fp32 [in, out, D]);
 * dcheb may equal dcoeffs when accumulate == 0 (in place).  Above degree 16,
 * dcoeffs (+)= dcheb (ckan_backward's output is already in the family basis). */
int ckan_coeff_grad_from_chebyshev(const ckan_desc* desc, const ckan_basis_spec* spec,
                                   const float* dcheb, float* dcoeffs, int accumulate, void* stream);
/* ckan_backward (accumulate = 0) followed by ckan_coeff_grad_from_chebyshev
 * in place, in one call: dcoeffs receives the family coefficients' gradient
 * (stored), dx the input gradient, the workspace as for ckan_backward.  Where
 * one pipelined dC launch writes the whole gradient, it applies M^T to each
 * row before its stores (no second pass over dC); otherwise the map runs as
 * its own launch.  The results are the same bits either way.
 * Replaces: torch autograd through kan/basis/jacobi.py:95-116 and
 * kan/basis/hermite.py:118-139 (the einsum's backward in the family basis). */
int ckan_backward_basis(const ckan_desc* desc, const ckan_basis_spec* spec, const float* t_cache,
                        const void* packed, const float* dy, float* dx, float* dcoeffs, void* ws,
                        size_t ws_bytes, void* stream);
/* out[q, n] = P_n(t[q]), n = 0..degree (<= 1024), by the family's recurrence
 * (the reference's basis_functions of an already-normalised input; s unused). */
int ckan_family_basis(const ckan_basis_spec* spec, const float* t, int64_t n, float* out,
                      void* stream);
/* dt[q] = sum_n g[q, n] P_n'(t[q]): backward of ckan_family_basis. */
int ckan_family_basis_backward(const ckan_basis_spec* spec, const float* t, const float* g,
                               int64_t n, float* dt, void* stream);

/* ---- derivatives with respect to the input --------------------------------
 * Each univariate function of a layer, f(x) = sum_n C[i, o, n] P_n(s tanh x)
 * (spec NULL: the ChebyKAN layer's T_n(tanh x)), has an order-k derivative in
 * x that is again a Chebyshev series in t = tanh x, of degree degree + k:
 *   d^k f / dx^k = sum_j Ck[i, o, j] T_j(t),   Ck = C R,   R = M L^k,
 * with M the family's change of basis and L : p -> (1 - t^2) p'(t) (exact in
 * the T basis).  Under the affine input map of desc (t = a x + b, the Hermite
 * layer's finite domain) L : p -> a p'(t) instead, the series one degree
 * lower (Ck keeps degree + 1 + k columns, the last 2k zero).  Requires fp32
 * coefficients and degree + k <= 16 for a family basis or the affine map,
 * degree + k <= 256 for the Chebyshev one under tanh (above 16 the device
 * applies L row by row in place of the matrix R).
 * Replaces KANLayer.compute_derivatives / jacobian (kan/layers/base.py:102-141)
 * and ChebyshevBasis.derivative (kan/basis/chebyshev.py:174-267).  Divergence:
 * the reference's derivative coefficients are wrong for n >= 3, omit the
 * tanh chain factor and its jacobian adds the other inputs' derivatives at 0;
 * these return the exact derivatives with respect to x. */
/* R (fp64, row-major [degree + 1][degree + 1 + order]) of the tanh map; host only. */
int ckan_derivative_matrix(const ckan_basis_spec* spec, int32_t degree, int32_t order, double* R);
/* out [in, out, degree + 1 + order] = coeffs [in, out, degree + 1] R; a
 * ChebyKAN forward of degree desc->degree + order with `out` then gives
 * sum_i d^k f_{i,o} / dx^k (x_i), the layer's compute_derivatives(x, k). */
int ckan_derivative_coeffs(const ckan_desc* desc, const ckan_basis_spec* spec, int32_t order,
                           const float* coeffs, float* out, void* stream);
/* dcoeffs [in, out, degree + 1] = dout_grad [in, out, degree + 1 + order] R^T
 * (the gradient of ckan_derivative_coeffs). */
int ckan_derivative_coeffs_backward(const ckan_desc* desc, const ckan_basis_spec* spec,
                                    int32_t order, const float* dout_grad, float* dcoeffs,
                                    void* stream);
/* jac [batch, out, in]: jac[b, o, i] = d y[b, o] / d x[b, i] for x [batch, in]
 * and fp32 coeffs; the workspace holds the order-1 coefficients re-laid out. */
size_t ckan_jacobian_workspace_bytes(const ckan_desc* desc);
int ckan_jacobian(const ckan_desc* desc, const ckan_basis_spec* spec, const float* x,
                  const float* coeffs, float* jac, void* ws, size_t ws_bytes, void* stream);

/* out[n, d] = T_d(t[n]) for d = 0..degree (fp32).  Replaces
 * ChebyshevBasis.basis_functions (kan/basis/chebyshev.py:103-172). */
int ckan_basis(const float* t, int64_t n, int32_t degree, float* out, void* stream);
/* d_t[n] = sum_d g[n, d] d U_{d-1}(t[n]): backward of ckan_basis. */
int ckan_basis_backward(const float* t, const float* g, int64_t n, int32_t degree,
                        float* dt, void* stream);

/* ---- optimizers (in place, fp32) ---------------------------------------- */

/* p -= lr * (g + weight_decay * p).  Replaces torch.optim.SGD.step without
 * momentum (torch/optim/sgd.py, used by configs 2 and 4). */
int ckan_sgd_step(float* p, const float* g, int64_t n, float lr, float weight_decay,
                  void* stream);

/* Adam in torch's single-tensor order (torch/optim/adam.py; README.md:59,66):
 *   g' = g + wd p;  m = lerp(m, g', 1 - b1);  v = b2 v + (1 - b2) g'^2;
 *   p -= (lr / (1 - b1^step)) * m / (sqrt(v) / sqrt(1 - b2^step) + eps).
 * `step` is the step count after increment (1 on the first call). */
int ckan_adam_step(float* p, const float* g, float* m, float* v, int64_t n, int64_t step,
                   double lr, double beta1, double beta2, double eps, double weight_decay,
                   void* stream);

/* ---- mixture of experts: routing -------------------------------------------- */
/* Rows of logits choose top_k of `experts` experts each.
 *   s = softmax(l) or sigmoid(l);  key = s + bias (bias may be NULL).
 *   An expert with logit -inf or NaN is not eligible: s = 0.  A logit of +inf counts as
 *   the largest finite one.  One with a key of NaN or -inf (by its bias) is never chosen
 *   either, but its score stays what it is and counts in a softmax's sum.
 *   groups > 1: the experts are `groups` equal runs; a group's value is the sum of
 *   its two largest keys (a missing or ineligible second counts 0), and only the
 *   top_groups groups of largest value stay.
 *   The top_k largest keys among them are chosen, in falling order.  Equal keys
 *   or values: the lowest index first.
 *   weights = scale * s_j / (sum of the chosen s + 1e-20) with renormalize,
 *   scale * s_j without.  The bias moves the choice only, not the weights.
 * A row with fewer than top_k eligible experts fills up with index -1, weight 0.
 * No counterpart in the reference (its models are single layers and stacks). */
typedef enum ckan_score {
  CKAN_SCORE_SOFTMAX = 0,
  CKAN_SCORE_SIGMOID = 1
} ckan_score;

typedef struct ckan_route_desc {
  int64_t rows;         /* 0..2^26 - 1                                    */
  int64_t logits_ld;    /* elements from a row of logits to the next      */
  int32_t experts;      /* 1..512                                         */
  int32_t top_k;        /* 1..64, at most the experts of top_groups groups */
  int32_t score;        /* ckan_score                                     */
  int32_t groups;       /* 1..64, divides experts                         */
  int32_t top_groups;   /* 1..groups                                      */
  int32_t renormalize;  /* 0 or 1                                         */
  int32_t dtype;        /* ckan_dtype of logits and dlogits               */
  float scale;
} ckan_route_desc;

/* weights [rows, top_k] fp32, indices [rows, top_k]; scores in fp32. */
int ckan_route(const ckan_route_desc* desc, const void* logits, const float* bias, float* weights,
               int64_t* indices, void* stream);
/* dlogits [rows, experts] (dense rows, in the logits' dtype) from dweights
 * [rows, top_k]; `indices` are ckan_route's.  No gradient goes through the choice. */
int ckan_route_backward(const ckan_route_desc* desc, const void* logits, const int64_t* indices,
                        const float* dweights, void* dlogits, void* stream);

/* ---- mixture of experts: the experts' products -------------------------------------- */
/* y[t] = sum_j w[t, j] f_e(x[t]) with e = indices[t, j] and expert e's ChebyKAN layer
 *   f_e(x)[o] = sum_{i, d} T_d(tanh x_i) C[e, i, o, d]   (kan/layers/chebykan.py:64-67).
 * x [rows, in], y [rows, out], coeffs [experts, in, out, degree + 1] in `dtype`,
 * weights [rows, top_k] in `wdtype`, indices int64 [rows, top_k].  A slot whose index
 * lies outside [0, experts) has no expert: it adds nothing and its weight's
 * gradient is 0.  A row may name an expert twice.
 * fp32 tensors are computed on two fp16 planes an operand (22 bits), bf16 ones on
 * one (11 bits); sums, tanh and the basis recurrence are in fp32.  The planes are scaled
 * by powers of two.  Coefficients by the largest of their expert: down to 2^-13 of it
 * they keep 22 bits, smaller ones an error of 2^-35 of it.  Gradients w dy by the largest
 * of their row for dx, and by the largest of the expert's rows for dcoeffs, where rows
 * are summed (down to 2^-16 of it 22 bits, smaller ones an error of 2^-38 of it).
 * `saved` (ckan_experts_saved_bytes) carries the sorted slots, tanh values, expert
 * outputs and packed coefficients from the forward to its backward; NULL where no
 * backward follows.  Buffers need 16-byte alignment. */
typedef struct ckan_experts_desc {
  int64_t rows;      /* >= 0; rows * top_k at most 2^26, rows * dims 2^33 */
  int32_t experts;   /* 1..512                                     */
  int32_t top_k;     /* 1..64                                      */
  int32_t in_dim;    /* 1..65536                                   */
  int32_t out_dim;   /* 1..65536                                   */
  int32_t degree;    /* 1..16                                      */
  int32_t dtype;     /* ckan_dtype of x, coeffs, y, dy, dx, dcoeffs */
  int32_t wdtype;    /* ckan_dtype of weights and dweights         */
} ckan_experts_desc;

size_t ckan_experts_saved_bytes(const ckan_experts_desc* desc);
/* Workspace of the forward (backward == 0; without_saved != 0 when saved is NULL) or the backward. */
size_t ckan_experts_workspace_bytes(const ckan_experts_desc* desc, int backward, int without_saved);
int ckan_experts_forward(const ckan_experts_desc* desc, const void* x, const void* coeffs, const int64_t* indices,
                         const void* weights, void* y, void* saved, void* ws, size_t ws_bytes, void* stream);
/* dx [rows, in], dcoeffs (as coeffs; zero for experts without rows), dweights
 * [rows, top_k] from dy [rows, out]; each may be NULL. */
int ckan_experts_backward(const ckan_experts_desc* desc, const int64_t* indices, const void* weights, void* saved,
                          const void* dy, void* dx, void* dcoeffs, void* dweights, void* ws, size_t ws_bytes,
                          void* stream);

/* ---- a whole mixture layer for few rows ---------------------------------------------- */
/* logits = x gate^T, ckan_route's choice and weights on them, and ckan_experts_forward's
 * sum, without a backward, for as few rows as the experts' coefficients are streamed for
 * (ckan_mixture_few: at most 1024 slots, fewer than 64 an expert on average, and of many fp32
 * coefficients of degree 9 and more at most 8 rows of 64 slots or at least 8 slots an expert).
 * The logits are summed in 64 bits and rounded once to fp32, so that the choice does not hang on an order
 * of sums.  x [rows, in] and y have x_dtype, gate [experts, in] and coeffs [experts, in, out,
 * degree + 1] a dtype each;
 * bias fp32 [experts] or NULL; weights fp32 and indices [rows, top_k] are outputs.  Buffers need
 * 16-byte alignment. */
typedef struct ckan_mixture_desc {
  int64_t rows;
  int32_t experts, top_k, in_dim, out_dim, degree;      /* as ckan_experts_desc's */
  int32_t score, groups, top_groups, renormalize;       /* as ckan_route_desc's   */
  int32_t x_dtype, gate_dtype, coeff_dtype;
  float scale;
} ckan_mixture_desc;
int ckan_mixture_few(const ckan_mixture_desc* desc);  /* 1: ckan_mixture_forward takes it */
size_t ckan_mixture_workspace_bytes(const ckan_mixture_desc* desc);
int ckan_mixture_forward(const ckan_mixture_desc* desc, const void* x, const void* gate, const void* coeffs,
                         const float* bias, void* y, float* weights, int64_t* indices, void* ws, size_t ws_bytes,
                         void* stream);

/* ---- norms around a residual block ------------------------------------------------ */
/*   u = drop(post(y)),  out = x + scale gate u,  h = next(out)
 * over rows of `dim` values, post and next being (v - mean) r w + b with
 * r = 1 / sqrt(mean((v - mean)^2) + eps), mean taken as 0 in the RMS form.  A NULL
 * post_weight or next_weight leaves that norm (and h) out, a NULL gate is 1 (gate_rows then
 * says nothing), a NULL y leaves only h = next(x).  gate is [dim] or, with gate_rows, [rows, dim].
 * x, out, dout and dx have x_dtype, y, h, dh and dy have y_dtype; parameters, row gates
 * and their gradients have a dtype each.  Rows are contiguous, `*_ld` elements apart (out, h and
 * the gradients dense).  Arithmetic in fp32, results rounded once; h comes from out
 * before its rounding.
 * Dropout (dropout > 0) as ckan_dropout's, on rows and columns of y. */
typedef enum ckan_norm {
  CKAN_NORM_RMS = 0,
  CKAN_NORM_LAYER = 1
} ckan_norm;

typedef struct ckan_residual_desc {
  int64_t rows;        /* 0..2^32 - 1                                        */
  int64_t x_ld, y_ld, gate_ld;
  int32_t dim;         /* 1..2^20                                            */
  int32_t x_dtype, y_dtype;
  int32_t gate_dtype, post_weight_dtype, post_bias_dtype, next_weight_dtype, next_bias_dtype;
  int32_t norm;        /* ckan_norm                                          */
  int32_t gate_rows;   /* 0 or 1                                             */
  float eps, scale;
  double dropout;      /* 0..1                                               */
} ckan_residual_desc;

typedef struct ckan_residual_buffers {
  const void *x, *y, *gate, *post_weight, *post_bias, *next_weight, *next_bias;
  const int64_t* dropout_state;  /* as ckan_dropout's                         */
  void *out, *h;                 /* written by the forward                     */
  void* stats;                   /* written by a forward that a backward follows (else NULL), read by it */
  const void *dout, *dh;         /* gradients of out and h; NULL is zero       */
  void *dx, *dy, *dgate, *dpost_weight, *dpost_bias, *dnext_weight, *dnext_bias;  /* NULL: not wanted */
  int64_t dout_ld, dh_ld;
  uint64_t dropout_seed, dropout_offset;  /* as ckan_dropout_desc's; a backward takes the forward's from stats */
} ckan_residual_buffers;

size_t ckan_residual_stats_bytes(const ckan_residual_desc* desc);
size_t ckan_residual_workspace_bytes(const ckan_residual_desc* desc);
int ckan_residual_forward(const ckan_residual_desc* desc, const ckan_residual_buffers* buffers, void* stream);
/* Needs the forward's inputs and stats as they were; sums over rows run in a fixed order. */
int ckan_residual_backward(const ckan_residual_desc* desc, const ckan_residual_buffers* buffers, void* ws,
                           size_t ws_bytes, void* stream);

/* ---- dropout -------------------------------------------------------------------------- */
/* y[r, c] = keep(r, c) x[r, c] / (1 - p).  The 32-bit number of an element is made of two
 * 16-bit halves, the high one from Philox 4x32-10 on the counter (c / 8, r, call) under the
 * seed, half c % 8 of its four words; the low one likewise from the counter with its top
 * bit set; the element is kept where the number reaches round(p 2^32).  (seed, call): the
 * given ones, or with `state` (int64[2] on the device) state[0] and state[1] + offset; calls
 * count modulo 2^63.  `used` (int64[2], or NULL) receives them: a gradient is the same call
 * on dy with `used` as its state. */
typedef struct ckan_dropout_desc {
  int64_t rows;      /* 0..2^32 - 1                        */
  int64_t dim;       /* 1..2^34; contiguous within a row   */
  int64_t x_ld;      /* elements from a row to the next    */
  double p;          /* 0..1                               */
  uint64_t seed, offset;
  int32_t dtype;     /* ckan_dtype of x and y              */
} ckan_dropout_desc;
int ckan_dropout(const ckan_dropout_desc* desc, const int64_t* state, const void* x, void* y, int64_t* used,
                 void* stream);

/* ---- log probabilities -------------------------------------------------------------- */
/* Of rows of logits [rows, classes]: logp[r] = log softmax(logits[r])[targets[r]] (0 where the
 * target lies outside [0, classes): such a row has none), entropy[r], and with top > 0
 * the top likeliest classes' log probabilities and indices [rows, top], equal logits by the lower
 * index.  A logit of -inf has no probability and is not among the likeliest (index -1,
 * log probability -inf fill up); a row of nothing else has logp -inf, entropy 0 and no gradient.
 * NaN or +inf in a row gives NaN.  Sums in fp32, the largest logit's share apart, so that rows
 * that are sure of one class keep their relative precision. */
typedef struct ckan_log_probs_desc {
  int64_t rows;      /* 0..2^31 - 1                        */
  int64_t logits_ld; /* elements from a row to the next    */
  int32_t classes;   /* 1..2^30                            */
  int32_t top;       /* 0..64, at most classes             */
  int32_t dtype;     /* ckan_dtype of logits and dlogits   */
} ckan_log_probs_desc;
size_t ckan_log_probs_workspace_bytes(const ckan_log_probs_desc* desc);
/* stats: fp32 [rows, 3], or NULL where no backward follows. */
int ckan_log_probs(const ckan_log_probs_desc* desc, const void* logits, const int64_t* targets, float* logp,
                   float* entropy, float* top_logp, int64_t* top_indices, float* stats, void* ws, size_t ws_bytes,
                   void* stream);
/* dlogits (dense rows) from the gradients of logp and entropy (fp32 [rows]; NULL is zero). */
int ckan_log_probs_backward(const ckan_log_probs_desc* desc, const void* logits, const int64_t* targets,
                            const float* stats, const float* dlogp, const float* dentropy, void* dlogits, void* stream);

/* ---- orthogonalised updates ---------------------------------------------------- */
/* Newton-Schulz orthogonalisation of a batch of matrices G [rows, cols]:
 *   X = G / (|G|_F + eps), then `steps` times
 *   X = a X + (b A + c A^2) X with A = X X^T (X^T X for rows > cols).
 * Products run on two fp16 planes an operand (22 bits) with fp32 sums, those of a side of
 * at most 64 in fp64; the norm is summed in fp64.  bf16 matrices take as many steps in powers of X X^T as keep
 * the error that this adds below 2^-9, their own rounding.  |b A + c A^2| and |a + b A + c A^2|
 * have to stay below 15 for singular values in [0, 1] over all steps (checked on
 * the host).
 * Element (r, col) of matrix i lies at i batch_stride + r row_stride +
 * (col / inner) outer_stride + (col % inner) inner_stride elements; inner divides
 * cols, and the strides have to make each matrix dense: row-major, column-major or, with
 * inner > 1, [cols / inner, rows, inner].  The matrices of a batch must not overlap.  An
 * ordinary matrix has inner = 1 and its column stride in outer_stride.  A
 * ChebyKAN layer's coefficients [in, out, D] as [out, in D], the matrix by which
 * the basis values act on the outputs, have inner = D, row_stride = D,
 * outer_stride = out D, inner_stride = 1.  Replaces nothing in the reference, whose
 * training loop uses torch's optimizers (README.md:59-69). */
typedef struct ckan_ortho_desc {
  int64_t batch_stride, row_stride, outer_stride, inner_stride;
  int32_t batch;       /* 0..65535                                       */
  int32_t rows, cols;  /* >= 1; the smaller at most 16384                */
  int32_t inner;       /* >= 1, divides cols                             */
  int32_t steps;       /* 0..100                                         */
  int32_t dtype;       /* ckan_dtype of in and out; fp32 for the Muon step */
  float a, b, c, eps;  /* eps >= 0                                       */
} ckan_ortho_desc;

size_t ckan_orthogonalize_workspace_bytes(const ckan_ortho_desc* desc);
/* out = the orthogonalised in; both in the descriptor's layout (they may be the same). */
int ckan_orthogonalize(const ckan_ortho_desc* desc, const void* in, void* out, void* ws, size_t ws_bytes,
                       void* stream);
/* One step of Muon on parameters p with gradient g and momentum buf (fp32, all in
 * the descriptor's layout, p and buf updated in place):
 *   buf = momentum buf + (1 - momentum) g
 *   u = nesterov ? (1 - momentum) g + momentum buf : buf
 *   p = (1 - lr weight_decay) p - lr scale O(u),   O the orthogonalisation above. */
int ckan_muon_step(const ckan_ortho_desc* desc, float* p, const float* g, float* buf, float lr, float momentum,
                   float weight_decay, float scale, int nesterov, void* ws, size_t ws_bytes, void* stream);

/* ---- resident multi-layer executor ---------------------------------------- */
/* A stack of ChebyKAN layers (KANSequential, kan/layers/base.py:144-166)
 * trained in place on one GPU: the executor owns fp32 master coefficients,
 * their packed operands, activations, tanh caches, gradients, optimizer state
 * and workspaces, allocated once at creation.  One ckan_exec_step runs
 * forward, the loss and its gradient, backward and the optimizer update for
 * every layer, the work of one iteration of the reference's training loop
 * (README.md:61-69) over a KANSequential. */

typedef struct ckan_exec ckan_exec;  /* opaque */

typedef enum ckan_loss {
  CKAN_LOSS_MSE = 0,  /* torch.nn.MSELoss(): mean over all B x out elements   */
  CKAN_LOSS_CE = 1    /* torch.nn.CrossEntropyLoss(): mean over B; int64 labels */
} ckan_loss;

typedef enum ckan_optimizer {
  CKAN_OPT_SGD = 0,   /* torch.optim.SGD (no momentum)  */
  CKAN_OPT_ADAM = 1   /* torch.optim.Adam (no amsgrad)  */
} ckan_optimizer;

typedef struct ckan_exec_config {
  int32_t n_layers;        /* >= 1                                          */
  const int32_t* widths;   /* host array, n_layers + 1 entries              */
  const int32_t* degrees;  /* host array, n_layers entries                  */
  int64_t batch;           /* rows per step (fixed for the executor)        */
  int32_t compute;         /* ckan_compute                                  */
  int32_t loss;            /* ckan_loss                                     */
  int32_t optimizer;       /* ckan_optimizer                                */
  int32_t use_graph;       /* replay each step as a captured HIP graph      */
  float lr, beta1, beta2, eps, weight_decay;
  int32_t flags;           /* ckan_exec_flags, 0 for the defaults           */
} ckan_exec_config;

typedef enum ckan_exec_flags {
  /* A stack whose step is at most 2^18 multiply-adds (e.g. the README's
   * ChebyKANLayer(1, 1, 8) on 100 points) runs each step as one launch of a
   * single-workgroup kernel instead of the per-layer kernel sequence; this
   * flag keeps the kernel sequence for such stacks too. */
  CKAN_EXEC_NO_FUSED_SMALL = 1,
  /* A two-layer cross-entropy stack of small layers (e.g. 784 -> 64 -> 10)
   * keeps its packed operands current from the step's dC launch, which
   * writes them from the updated coefficients, so its steps run no pack
   * launch; this flag packs at every step instead (the same bits). */
  CKAN_EXEC_PACK_EACH_STEP = 2
} ckan_exec_flags;

/* Allocates every device buffer; coefficients start at zero (set them with
 * ckan_exec_set_coeffs).  `stream` orders the initialisation. */
int ckan_exec_create(const ckan_exec_config* cfg, ckan_exec** out, void* stream);
/* ckan_exec_create for a KANSequential whose layers may be JacobiKANLayer
 * (kan/layers/jacobikan.py:64-78) or HermiteKANLayer
 * (kan/layers/hermitekan.py:68-82).  `bases` holds n_layers basis specs (host
 * array; spec.degree must equal degrees[l]; a Chebyshev spec of scale 1 is the
 * plain ChebyKAN layer), NULL for a stack of ChebyKAN layers.  `affine` (host
 * array of 2 * n_layers floats, or NULL) gives layer l the input map
 * t = affine[2l] * x + affine[2l+1] (CKAN_INPUT_AFFINE: the Hermite layer's
 * finite domain) in place of tanh; (0, 0) keeps tanh.  A layer's
 * coefficients (ckan_exec_set/get_coeffs, Adam state) are those of its own
 * basis.  Family layers up to degree 16 train through the change of basis
 * into Chebyshev coefficients (gradient mapped back by the transpose before
 * the optimizer step); above it, on the family's recurrence. */
int ckan_exec_create_basis(const ckan_exec_config* cfg, const struct ckan_basis_spec* bases,
                           const float* affine, ckan_exec** out, void* stream);
int ckan_exec_destroy(ckan_exec* ex);
/* Device-to-device copy of one layer's fp32 master coefficients [in, out, D]. */
int ckan_exec_set_coeffs(ckan_exec* ex, int32_t layer, const float* src, void* stream);
int ckan_exec_get_coeffs(ckan_exec* ex, int32_t layer, float* dst, void* stream);
/* Adam moments of one layer (fp32, [in, out, D] each) and the step count,
 * for checkpoint/resume; SGD has none (returns CKAN_ERR_UNSUPPORTED). */
int ckan_exec_get_adam_state(ckan_exec* ex, int32_t layer, float* m, float* v,
                             int64_t* step, void* stream);
int ckan_exec_set_adam_state(ckan_exec* ex, int32_t layer, const float* m, const float* v,
                             int64_t step, void* stream);
/* One training step on x [batch, widths[0]] (fp32, device) and target:
 * fp32 [batch, widths[n]] for MSE or int64 [batch] class indices for CE.
 * Writes the step's loss (fp32 scalar, device) to loss_out when non-NULL.
 * CE labels must lie in [0, widths[n]): there is no ignore_index, every row
 * counts in the mean, and the kernels do not check the labels (an
 * out-of-range label reads nothing out of bounds but leaves the loss and its
 * gradient without that row's target term).  The Python wrapper rejects such
 * labels before the launch, as torch.nn.CrossEntropyLoss would. */
int ckan_exec_step(ckan_exec* ex, const float* x, const void* target, float* loss_out,
                   void* stream);
/* `nsteps` training steps on the same x and target (the reference loop's
 * full-batch epochs, README.md:61-69), issued from the library without a
 * return to the caller between steps; step k's loss goes to losses[k] (fp32,
 * device, nsteps entries) when losses is non-NULL.  Runs eagerly (no graph). */
int ckan_exec_steps(ckan_exec* ex, const float* x, const void* target, int64_t nsteps,
                    float* losses, void* stream);
/* Forward only: y [batch, widths[n]] (fp32, device). */
int ckan_exec_forward(ckan_exec* ex, const float* x, float* y, void* stream);

/* ---- diagnostics --------------------------------------------------------- */

const char* ckan_last_error(void);
const char* ckan_version(void);
/* Per-kernel HIP-event timing on the launch stream (off by default). */
int ckan_profile_enable(int on);
/* Writes "name count total_ms\n" lines (synchronises on the recorded events)
 * and clears the records.  Returns the number of bytes needed. */
size_t ckan_profile_report(char* buf, size_t len);

#ifdef __cplusplus
}
#endif

#endif /* CHEBYKAN_H */
