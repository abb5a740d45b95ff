// Matrix products on fp16 planes: the tile core shared by the mixture-of-experts
// and orthogonalisation kernels.
//
// An fp32 value x, scaled by a power of two into fp16's range, is held as the
// sum of NP fp16 planes: h = fp16(x), l = fp16(x - h).  Two planes keep 22 bits,
// and a product takes the three plane products h h + h l + l h in fp32
// accumulators (l l is below 2^-22 of it): three instructions where six of bf16
// planes give the same error, 2-3e-6 after five Newton-Schulz steps where plain
// fp32 products give 2-3e-6 too.  One plane keeps 11 bits, three more than bf16,
// at the bf16 rate: the form for operands that are bf16 already, or whose
// results are rounded to bf16.
//
// Operands are stored fragment-major for v_mfma_f32_32x32x16_f16: for a block of
// 32 rows and 16 consecutive k, NP planes of 64 lanes x 8 values (1 KiB), lane l
// holding row l % 32 and k = 8 (l / 32) + 0..7:
//   byte(rb, kb, plane, lane) = ((rb * KB + kb) * NP + plane) * 1024 + lane * 16.
// A stage of several k-blocks of one row block is one contiguous run, copied to
// LDS as it lies; a fragment is read back with one conflict-free 16-byte read a
// lane.  Rows past the matrix may hold anything (they give results that are not
// stored); k past the matrix holds zeros in both operands.
#pragma once

#include "ckan_common.hpp"

namespace ckan {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4_t;

constexpr int kPlaneBytes = 1024;

// A value in a register that the compiler does not see through.  The planes need
// it: h = fp16(a b) and l = fp16(a b - h) from one expression may be contracted
// differently (h in a mixed-precision multiply that rounds once, a b in l twice),
// and then h + l misses the value by an fp16 ulp of h.
__device__ __forceinline__ float opaque(float v) {
  asm("" : "+v"(v));
  return v;
}

// The 8 values of a lane in planes (round to nearest even each).
template <int NP> struct Planes8 { typedef f16x8_t part; f16x8_t p[NP]; };
template <int NP>
__device__ __forceinline__ Planes8<NP> to_planes8(const float* v) {
  Planes8<NP> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = NP == 2 ? opaque(v[j]) : v[j];
    const _Float16 h = (_Float16)x;
    f.p[0][j] = h;
    if constexpr (NP == 2) f.p[1][j] = (_Float16)(x - (float)h);
  }
  return f;
}
template <int NP> struct Planes4 { typedef f16x4_t part; f16x4_t p[NP]; };
template <int NP>
__device__ __forceinline__ Planes4<NP> to_planes4(const float* v) {
  Planes4<NP> f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x = NP == 2 ? opaque(v[j]) : v[j];
    const _Float16 h = (_Float16)x;
    f.p[0][j] = h;
    if constexpr (NP == 2) f.p[1][j] = (_Float16)(x - (float)h);
  }
  return f;
}

__device__ __forceinline__ f32x16_t mfma16(f16x8_t a, f16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// acc[m][n] += a[m] b[n] for FM x FN fragments of one k-block; the small plane
// products first.  With NC = 3 accumulators each of the three plane products has its
// own: a wave of one fragment would otherwise wait for each instruction's result.
template <int NA, int NB, int FM, int FN, int NC = 1>
__device__ __forceinline__ void mfma_planes(const f16x8_t (&a)[FM][NA], const f16x8_t (&b)[FN][NB],
                                            f32x16_t (&acc)[NC * FM][FN]) {
  if constexpr (NA == 2) {
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n) acc[m][n] = mfma16(a[m][1], b[n][0], acc[m][n]);
  }
  constexpr int k1 = NC == 3 ? FM : 0, k2 = NC == 3 ? 2 * FM : 0;
  if constexpr (NB == 2) {
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int n = 0; n < FN; ++n) acc[k1 + m][n] = mfma16(a[m][0], b[n][1], acc[k1 + m][n]);
  }
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) acc[k2 + m][n] = mfma16(a[m][0], b[n][0], acc[k2 + m][n]);
}

__device__ __forceinline__ f16x8_t lds_frag(const char* base, int lane) {
  return *reinterpret_cast<const f16x8_t*>(base + lane * 16);
}

// The LDS address that a copy takes for a generic pointer into shared memory.
__device__ __forceinline__ uint32_t lds_address(char* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)p;
}
// A 16-byte-per-lane copy from per-lane addresses: lane l's 16 bytes at src land at
// LDS byte lds + 16 l (lds wave-uniform); counted in vmcnt, like dma16s.
__device__ __forceinline__ void dma16v(const void* src, uint32_t lds) {
  const uint32_t l = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(l) : "memory", "m0");
}
// The address of row block r of an operand whose row blocks lie `pitch` bytes apart.
struct RowBlocks {
  const char* base;
  size_t pitch;
  __device__ const char* operator()(int r) const { return base + r * pitch; }
};

// Waits until at most N of the wave's vector memory operations are in flight.
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// One block's tile of C = A B^T over stored operands: WM x WN waves, each FM x FN
// fragments of 32 x 32; A tile of WM FM row blocks, B tile of WN FN.  Stages of
// KS k-blocks go through a ring of NBUF LDS buffers by direct copies, NBUF - 1
// stages ahead, one barrier a stage.  WK > 1: that many groups of waves take a share
// of each stage's k-blocks and leave their sums to the caller.
template <int NA, int NB, int WM, int WN, int FM, int FN, int KS, int NBUF, int NC = 1, int WK = 1>
struct NtTile {
  static constexpr int kWaves = WM * WN * WK, kStageBlocks = KS;
  static_assert(KS % WK == 0, "k-blocks divide among the groups");
  static constexpr int kRA = WM * FM, kRB = WN * FN;
  static constexpr int kChunksA = kRA * KS * NA, kChunks = kChunksA + kRB * KS * NB;
  static constexpr int kStageBytes = kChunks * kPlaneBytes;
  static constexpr int kLdsBytes = NBUF * kStageBytes;
  static_assert(kChunks % kWaves == 0, "copies divide among the waves");
  static constexpr int kPer = kChunks / kWaves;  // copies a wave and stage

  // Copies stage kb.. of both operands: the 1 KiB chunks in LDS order, chunk c by
  // wave c % kWaves (row block, then k-block and plane, both contiguous in memory).
  // A(r) and B(r) give the address of the tile's r-th row block.
  template <typename SrcA, typename SrcB>
  __device__ static void copy(const SrcA& A, const SrcB& B, int kb, uint32_t lds, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = i * kWaves + wave;
      const char* src;
      if (c < kChunksA) {
        src = A(c / (KS * NA)) + ((size_t)kb * NA + c % (KS * NA)) * kPlaneBytes;
      } else {
        const int d = c - kChunksA;
        src = B(d / (KS * NB)) + ((size_t)kb * NB + d % (KS * NB)) * kPlaneBytes;
      }
      dma16s(src, lane * 16, lds + c * kPlaneBytes);
    }
  }

  __device__ static void compute(const char* buf, int wm, int wn, int wk, int lane, f32x16_t (&acc)[NC * FM][FN]) {
    const char* a = buf + wm * FM * KS * NA * kPlaneBytes;
    const char* b = buf + (kChunksA + wn * FN * KS * NB) * kPlaneBytes;
#pragma unroll
    for (int u = 0; u < KS / WK; ++u) {
      const int k = wk * (KS / WK) + u;
      f16x8_t fa[FM][NA], fb[FN][NB];
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int p = 0; p < NA; ++p) fa[m][p] = lds_frag(a + ((m * KS + k) * NA + p) * kPlaneBytes, lane);
#pragma unroll
      for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int p = 0; p < NB; ++p) fb[n][p] = lds_frag(b + ((n * KS + k) * NB + p) * kPlaneBytes, lane);
      mfma_planes<NA, NB, FM, FN, NC>(fa, fb, acc);
    }
  }

  // acc += the product over the nst stages from k-block kb0 on.  A and B give the
  // addresses of the tile's row blocks.  Ends with every wave past its last LDS
  // read.
  template <typename SrcA, typename SrcB>
  __device__ static void run(const SrcA& A, const SrcB& B, int kb0, int nst, char* lds,
                             f32x16_t (&acc)[NC * FM][FN]) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wk = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
    const uint32_t l0 = lds_address(lds);
#pragma unroll
    for (int s = 0; s < NBUF - 1; ++s)
      if (s < nst) copy(A, B, kb0 + s * KS, l0 + s * kStageBytes, wave, lane);
    int cur = 0;
    for (int s = 0; s < nst; ++s) {
      // stage s has landed when only the later stages' copies are in flight
      const int later = nst - 1 - s < NBUF - 2 ? nst - 1 - s : NBUF - 2;
      if (NBUF > 2 && later == NBUF - 2)
        wait_vm<kPer * (NBUF - 2)>();
      else
        wait_vm<0>();
      wait_lds();
      block_barrier();
      const int nxt = s + NBUF - 1;
      if (nxt < nst) {
        int at = cur + NBUF - 1;
        if (at >= NBUF) at -= NBUF;
        copy(A, B, kb0 + nxt * KS, l0 + at * kStageBytes, wave, lane);
      }
      compute(lds + cur * kStageBytes, wm, wn, wk, lane, acc);
      if (++cur == NBUF) cur = 0;
    }
    wait_lds();
    block_barrier();
  }
};

}  // namespace ckan
