// Launch interface of the residual-block, dropout, log-probability and few-row
// mixture kernels, and the device helpers that they share.
#pragma once

#include <float.h>

#include "ckan_kernels.hpp"

namespace ckan {

// ---- rows in chunks of eight values -------------------------------------------
// A row of any length and alignment is read in chunks of eight consecutive values:
// whole chunks by unaligned vector accesses (16 bytes of bf16, 32 of fp32; the
// target's memory mode allows them at any element), a row's last, partial one by
// elements, so that nothing past a row's end is touched.
constexpr int kChunk = 8;

struct __attribute__((packed)) RawBf16 { u32x4_t v; };
struct __attribute__((packed)) RawF32 { u32x4_t v[2]; };
template <typename T> struct RawOf;
template <> struct RawOf<__bf16> { typedef RawBf16 type; };
template <> struct RawOf<float> { typedef RawF32 type; };

__device__ __forceinline__ void unpack8(const RawBf16& r, float (&f)[kChunk]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(r.v[i] << 16);
    f[2 * i + 1] = __uint_as_float(r.v[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const RawF32& r, float (&f)[kChunk]) {
#pragma unroll
  for (int i = 0; i < kChunk; ++i) f[i] = __uint_as_float(r.v[i >> 2][i & 3]);
}

// `left` values of the row remain from p on (at least one); those past it read as 0.
template <typename T>
__device__ __forceinline__ typename RawOf<T>::type load_raw8(const T* p, int64_t left) {
  typename RawOf<T>::type r;
  if (left >= kChunk) {
    r = *(const typename RawOf<T>::type*)p;
  } else {
    union { typename RawOf<T>::type raw; T e[kChunk]; } u;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) u.e[i] = i < left ? p[i] : (T)0.0f;
    r = u.raw;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t left, float (&f)[kChunk]) {
  unpack8(load_raw8(p, left), f);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t left, const float (&f)[kChunk]) {
  union { typename RawOf<T>::type raw; T e[kChunk]; } u;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) u.e[i] = (T)f[i];
  if (left >= kChunk) {
    *(typename RawOf<T>::type*)p = u.raw;
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (i < left) p[i] = u.e[i];
  }
}

// The same without elementwise reads, for rows of at least eight values: a row's partial chunk in one
// access too, reaching past the row's end where `spare` values follow it, and beginning `back` values
// early where they do not. settle8 puts its values right.
__device__ __forceinline__ int back_of(int left, int64_t spare) {
  return left < kChunk && left + spare < kChunk ? (int)(kChunk - left - spare) : 0;
}
// `tail`, uniform: rows have a partial chunk.
template <typename T>
__device__ __forceinline__ typename RawOf<T>::type load_near8(const T* row, int at, int left, int64_t spare, bool tail) {
  typename RawOf<T>::type r = {};
  if (tail && spare < kChunk - 1) at -= back_of(left, spare);
  if (left > 0) r = *(const typename RawOf<T>::type*)(row + at);
  return r;
}
__device__ __forceinline__ void zero_past(int left, float (&f)[kChunk]) {
#pragma unroll
  for (int i = 0; i < kChunk; ++i) f[i] = i < left ? f[i] : 0.0f;
}

__device__ __forceinline__ void settle8(int left, int64_t spare, float (&f)[kChunk]) {
  if (spare < kChunk - 1) {  // the tensor's last row
    const int back = left > 0 ? back_of(left, spare) : 0;
#pragma unroll
    for (int w = 4; w; w >>= 1)
#pragma unroll
      for (int i = 0; i < kChunk; ++i) f[i] = back & w ? (i + w < kChunk ? f[i + w < kChunk ? i + w : i] : 0.0f) : f[i];
  }
  zero_past(left, f);
}

// The sum over a group of L lanes (8, 16, 32 or 64, aligned), in each of them: butterflies
// on the vector ALU, so every lane has the same bits.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  v = dpp_add<0xb1>(v);   // lanes 1, 0, 3, 2
  v = dpp_add<0x4e>(v);   // lanes 2, 3, 0, 1
  v = dpp_add<0x141>(v);  // the mirror of 8
  if constexpr (L >= 16) v = dpp_add<0x140>(v);  // the mirror of 16
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// A tensor whose type is known at run time (parameters, row gates).
struct AnyPtr {
  const void* p;
  int bf16;
};
__device__ __forceinline__ void load8(const AnyPtr& a, int64_t at, int64_t left, float (&f)[kChunk]) {
  if (a.bf16)
    load8((const __bf16*)a.p + at, left, f);
  else
    load8((const float*)a.p + at, left, f);
}

// ---- dropout's generator ---------------------------------------------------------
// Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as
// easy as 1, 2, 3", 2011), keyed by the seed, on the counter (column / 8, row, call):
// four words are 16 bits for each of a chunk's eight values.  An element is kept where
// its 32-bit number reaches p 2^32.  Its high half decides all but one case in 2^16: only
// where that half equals the threshold's is the stream of the low halves (the counter's
// top bit) drawn, so the mask has the resolution of 32 bits for little more than the
// cost of 16.
struct DropArgs {
  const int64_t* state;  // (seed, offset) on the device, or NULL: (seed, offset) below
  uint64_t seed, offset; // offset is added to the state's
  uint32_t high, low;    // round(p 2^32) = high 2^16 + low
  uint32_t cut;          // what kept() compares with: high, at least 1
  float scale;           // 1 / (1 - p)
  int on, none;          // none: p 2^32 rounds to 2^32, nothing is kept
};

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}
__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
    c[0] = xor3((uint32_t)(b >> 32), c[1], k0);
    c[2] = xor3((uint32_t)(a >> 32), c[3], k1);
    c[1] = (uint32_t)b;
    c[3] = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// Seed and call of a launch: uniform, read once a thread.
struct DropKey {
  uint32_t k0, k1, call0, call1;
};
__device__ __forceinline__ DropKey drop_key(const DropArgs& d) {
  uint64_t seed = d.seed, call = d.offset;
  if (d.state) {
    seed = (uint64_t)d.state[0];
    call += (uint64_t)d.state[1];
  }
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)call, (uint32_t)(call >> 32) & 0x7fffffffu};
}

// A chunk's eight numbers, 16 bits each, settled such that an element is kept where its
// number reaches DropArgs::cut: 0 where the low halves decided against it.
struct DropWords {
  uint32_t w[kChunk / 2];
  __device__ __forceinline__ bool kept(int i, const DropArgs& d) const {
    return (i & 1 ? w[i >> 1] : w[i >> 1] << 16) >= d.cut << 16;
  }
};
__device__ __forceinline__ DropWords drop_words(const DropArgs& d, const DropKey& k, uint32_t row, uint32_t chunk) {
  DropWords r;
  uint32_t c[4] = {chunk, row, k.call0, k.call1};
  philox(c, k.k0, k.k1);
  // halves that equal the threshold's: those that are 0 in x. (x - 0x10001) & ~x & 0x80008000 marks
  // the words that have one (and with them perhaps another half)
  uint32_t any = 0;
  const uint32_t twice = d.high << 16 | d.high;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.w[i] = c[i];
    const uint32_t x = c[i] ^ twice;
    any |= (x - 0x10001u) & ~x & 0x80008000u;
  }
  if (d.high == 0 || d.none)
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = d.none ? 0u : 0xffffffffu;
  if (d.low && any && !d.none) {  // the low halves decide
    uint32_t e[4] = {chunk, row, k.call0, k.call1 | 0x80000000u};
    philox(e, k.k0, k.k1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((c[i] & 0xffffu) == d.high && (e[i] & 0xffffu) < d.low) r.w[i] &= 0xffff0000u;
      if (c[i] >> 16 == d.high && e[i] >> 16 < d.low) r.w[i] &= 0xffffu;
    }
  }
  return r;
}

constexpr int64_t kDropMaxRows = (int64_t)1 << 32, kDropMaxDim = (int64_t)1 << 34;

struct DropoutArgs {
  const void* x;
  void* y;
  int64_t rows, dim, ld;
  int bf16;
  DropArgs drop;
  int64_t* used;  // (seed, offset) as this launch read them, or NULL
};
void launch_dropout(const DropoutArgs& a, hipStream_t st);

// ---- norms around a residual block (ckan_residual.hip) -----------------------------
// out = x + scale gate drop(post(y)) and h = next(out); post and next are norms of the
// rows.  Without y: h = next(x).
struct ResidualArgs {
  int64_t rows, x_ld, y_ld, gate_ld, dout_ld, dh_ld;
  int dim;
  int x_bf16, y_bf16;  // the stream's type (x, out, dout, dx), the branch's (y, h, dh, dy)
  int layer;           // norms with the mean taken out
  int gate_rows;       // gate is [rows, dim] (else [dim])
  float eps, scale;
  DropArgs drop;
  const void *x, *y;
  AnyPtr gate, post_w, post_b, next_w, next_b;  // p NULL: absent
  void *out, *h;
  float* stats;        // [rows, 4]: post's mean and factor, next's mean and factor; then (seed, offset)
  const void *dout, *dh;
  void *dx, *dy, *dgate, *dpost_w, *dpost_b, *dnext_w, *dnext_b;  // NULL: not wanted
  float* ws;
};
constexpr int kResMaxDim = 1 << 20;
size_t residual_workspace_bytes(const ResidualArgs& a);
void launch_residual_forward(const ResidualArgs& a, hipStream_t st);
void launch_residual_backward(const ResidualArgs& a, hipStream_t st);

// ---- log probabilities (ckan_logprobs.hip) ------------------------------------------
constexpr int kLogpMaxTop = 64;
struct LogpArgs {
  const void* logits;  // [rows, classes], row pitch ld
  const int64_t* targets;
  int64_t rows, ld;
  int classes, top, bf16;
  float *logp, *entropy, *top_logp;
  int64_t* top_idx;
  float* stats;        // [rows, 3]: shift, log of the sum, entropy; NULL where no backward follows
  const float *dlogp, *dentropy;  // NULL: zero
  void* dlogits;
  char* ws;
  int parts, part_len; // a long row's parts (set by the launch)
  size_t keys_off;
};
size_t logprobs_workspace_bytes(const LogpArgs& a);
void launch_logprobs(const LogpArgs& a, hipStream_t st);
void launch_logprobs_backward(const LogpArgs& a, hipStream_t st);

}  // namespace ckan
