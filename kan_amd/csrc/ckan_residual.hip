// Norms around a residual block (ckan_residual_forward, ckan_residual_backward):
//
//   u = drop(post(y)),  out = x + scale gate u,  h = next(out)
//
// with post and next a row's (v - mean) r w + b, r = 1 / sqrt(mean((v - mean)^2) + eps)
// (mean 0 in the rms form), and either of them absent.  Backward, with o^ = (out - mean) r
// and y^ likewise:
//
//   g = dh w_next,  dx = dout + r (g - o^ mean(g o^) - mean(g)),     dw_next = sum dh o^
//   dgate = scale dx u,  e = drop(scale gate dx),                    dw_post = sum e y^
//   dy = r (e w_post - y^ mean(e w_post y^) - mean(e w_post))
//
// out is made again from x and y, unrounded, so that no gradient sees its rounding: the
// same bytes as reading out.  Sums over a row and over rows are in fp32, in a fixed order.
//
// Bound by the bytes: every tensor once, a row in the registers of a team of lanes between its sums (65536 x 512
// in fp32, layer norms with biases and a gate a row: forward 130 us, backward 206, both 5.2 TB/s, the rate of a large
// copy; 32768 x 1024 in bf16 60 and 98 us, 4.4 and 4.1 TB/s, by instructions too). Rows above 8192 values, a forward with
// five parameters from 8153 on, and rows below 8 values are read again for every sum (2048 x 16384 in fp32: forward 170 to 178
// us, backward 318 + 118; 65536 x 4, a block a row and one thread of it at work: 343 and 591 + 434).
#include <type_traits>

#include "ckan_block.hpp"

namespace ckan {
namespace {

constexpr int kStats = 4;  // floats a row keeps for the backward

// ---- any width: a block a row, the row read again for every sum ------------------

constexpr int kAnyThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int w = 32; w; w >>= 1) v += __shfl_xor(v, w);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

struct RowStats {
  float m1, r1, m2, r2;
};

// One chunk of a row: u (after dropout), y^ and out's unrounded value.
template <typename TX, typename TY>
__device__ __forceinline__ DropWords chunk_values(const ResidualArgs& a, const DropKey& key, int64_t row, int c,
                                                 const RowStats& st, float (&yh)[kChunk], float (&u)[kChunk],
                                                 float (&gate)[kChunk], float (&o)[kChunk]) {
  const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
  load8((const TX*)a.x + row * a.x_ld + at, left, o);
  DropWords keep = {};
  if (!a.y) return keep;
  load8((const TY*)a.y + row * a.y_ld + at, left, yh);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) u[i] = yh[i];
  if (a.post_w.p) {
    float w[kChunk], b[kChunk] = {};
    load8(a.post_w, at, left, w);
    if (a.post_b.p) load8(a.post_b, at, left, b);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      yh[i] = i < left ? (yh[i] - st.m1) * st.r1 : 0.0f;
      u[i] = fmaf(yh[i], w[i], b[i]);
    }
  }
  if (a.drop.on) {
    keep = drop_words(a.drop, key, (uint32_t)row, (uint32_t)c);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) u[i] = keep.kept(i, a.drop) ? u[i] * a.drop.scale : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) gate[i] = 1.0f;
  if (a.gate.p) load8(a.gate, (a.gate_rows ? row * a.gate_ld : 0) + at, left, gate);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    gate[i] *= a.scale;
    o[i] = fmaf(gate[i], u[i], o[i]);
  }
  return keep;
}

template <typename TX, typename TY>
__global__ __launch_bounds__(kAnyThreads) void k_residual_any(ResidualArgs a) {
  __shared__ float red[kAnyThreads / 64];
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const int chunks = (a.dim + kChunk - 1) / kChunk, tid = threadIdx.x;
  const float inv = 1.0f / (float)a.dim;
  if (a.stats && a.drop.on && blockIdx.x == 0 && tid == 0) {
    int64_t* used = (int64_t*)(a.stats + a.rows * kStats);
    used[0] = a.drop.state ? a.drop.state[0] : (int64_t)a.drop.seed;
    used[1] = (int64_t)(((uint64_t)key.call1 << 32) | key.call0);
  }
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    RowStats st = {};
    float yh[kChunk], u[kChunk], gate[kChunk], o[kChunk];
    if (a.y && a.post_w.p) {
      for (int pass = a.layer ? 0 : 1; pass < 2; ++pass) {
        float sum = 0.0f;
        for (int c = tid; c < chunks; c += kAnyThreads) {
          const int64_t left = a.dim - (int64_t)c * kChunk;
          load8((const TY*)a.y + row * a.y_ld + (int64_t)c * kChunk, left, yh);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            const float d = i < left ? yh[i] - st.m1 : 0.0f;
            sum += pass ? d * d : d;
          }
        }
        sum = block_sum(sum, red) * inv;
        if (pass)
          st.r1 = 1.0f / sqrtf(sum + a.eps);
        else
          st.m1 = sum;
      }
    }
    if (a.next_w.p) {
      for (int pass = a.layer ? 0 : 1; pass < 2; ++pass) {
        float sum = 0.0f;
        for (int c = tid; c < chunks; c += kAnyThreads) {
          const int64_t left = a.dim - (int64_t)c * kChunk;
          chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            const float d = i < left ? o[i] - st.m2 : 0.0f;
            sum += pass ? d * d : d;
          }
        }
        sum = block_sum(sum, red) * inv;
        if (pass)
          st.r2 = 1.0f / sqrtf(sum + a.eps);
        else
          st.m2 = sum;
      }
    }
    for (int c = tid; c < chunks; c += kAnyThreads) {
      const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
      chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
      if (a.out) store8((TX*)a.out + row * a.dim + at, left, o);
      if (a.next_w.p) {
        float w[kChunk], b[kChunk] = {};
        load8(a.next_w, at, left, w);
        if (a.next_b.p) load8(a.next_b, at, left, b);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) o[i] = fmaf((o[i] - st.m2) * st.r2, w[i], b[i]);
        store8((TY*)a.h + row * a.dim + at, left, o);
      }
    }
    if (a.stats && tid == 0) {
      float* s = a.stats + row * kStats;
      s[0] = st.m1;
      s[1] = st.r1;
      s[2] = st.m2;
      s[3] = st.r2;
    }
  }
}

// A chunk's gradients: dx, e (the gradient of post's result) and o^.
struct RowMeans {
  float go, g, ey, e;  // mean(g o^), mean(g), mean(e w y^), mean(e w)
};

template <typename TX, typename TY>
__device__ __forceinline__ void chunk_dx(const ResidualArgs& a, int64_t row, int c, const RowStats& st, const RowMeans& mean,
                                         const float (&o)[kChunk], float (&oh)[kChunk], float (&dh)[kChunk],
                                         float (&dx)[kChunk]) {
  const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) oh[i] = dh[i] = dx[i] = 0.0f;
  if (a.dout) load8((const TX*)a.dout + row * a.dout_ld + at, left, dx);
  if (a.next_w.p && a.dh) {
    float w[kChunk];
    load8((const TY*)a.dh + row * a.dh_ld + at, left, dh);
    load8(a.next_w, at, left, w);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      oh[i] = i < left ? (o[i] - st.m2) * st.r2 : 0.0f;
      dx[i] += st.r2 * (dh[i] * w[i] - oh[i] * mean.go - mean.g);
    }
  }
}

// dx, dy and a row gate's gradient; the row's means to the workspace for the sums over rows.
template <typename TX, typename TY>
__global__ __launch_bounds__(kAnyThreads) void k_residual_any_dx(ResidualArgs a) {
  __shared__ float red[kAnyThreads / 64];
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const int chunks = (a.dim + kChunk - 1) / kChunk, tid = threadIdx.x;
  const float inv = 1.0f / (float)a.dim;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* s = a.stats + row * kStats;
    const RowStats st = {s[0], s[1], s[2], s[3]};
    RowMeans mean = {};
    float yh[kChunk], u[kChunk], gate[kChunk], o[kChunk], oh[kChunk], dh[kChunk], dx[kChunk], w[kChunk];
    if (a.next_w.p && a.dh) {
      float go = 0.0f, g = 0.0f;
      for (int c = tid; c < chunks; c += kAnyThreads) {
        chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
        chunk_dx<TX, TY>(a, row, c, st, mean, o, oh, dh, dx);
        load8(a.next_w, (int64_t)c * kChunk, a.dim - (int64_t)c * kChunk, w);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          go = fmaf(dh[i] * w[i], oh[i], go);
          g = fmaf(dh[i], w[i], g);
        }
      }
      mean.go = block_sum(go, red) * inv;
      if (a.layer) mean.g = block_sum(g, red) * inv;
    }
    const bool post = a.y && a.post_w.p;
    for (int pass = post && a.dy ? 0 : 1; pass < 2; ++pass) {
      float ey = 0.0f, e = 0.0f;
      for (int c = tid; c < chunks; c += kAnyThreads) {
        const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
        const DropWords keep = chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
        chunk_dx<TX, TY>(a, row, c, st, mean, o, oh, dh, dx);
        if (pass && a.dx) store8((TX*)a.dx + row * a.dim + at, left, dx);
        if (!a.y) continue;
        if (pass && a.gate_rows && a.dgate) {
          float dg[kChunk];
#pragma unroll
          for (int i = 0; i < kChunk; ++i) dg[i] = a.scale * dx[i] * u[i];
          if (a.gate.bf16)
            store8((__bf16*)a.dgate + row * a.dim + at, left, dg);
          else
            store8((float*)a.dgate + row * a.dim + at, left, dg);
        }
        if (post) load8(a.post_w, at, left, w);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          float v = gate[i] * dx[i];
          if (a.drop.on) v = keep.kept(i, a.drop) ? v * a.drop.scale : 0.0f;
          if (post) {
            v *= w[i];
            ey = fmaf(v, yh[i], ey);
            e += v;
            v = st.r1 * (v - yh[i] * mean.ey - mean.e);
          }
          dx[i] = v;
        }
        if (pass && a.dy) store8((TY*)a.dy + row * a.dim + at, left, dx);
      }
      if (!pass) {
        mean.ey = block_sum(ey, red) * inv;
        if (a.layer) mean.e = block_sum(e, red) * inv;
      }
    }
    if (tid == 0) {
      a.ws[row * 2] = mean.go;
      a.ws[row * 2 + 1] = mean.g;
    }
  }
}

// Sums over rows of the parameters' gradients: a thread a column chunk, the rows of its slab one
// after another; partial sums [slab, 5, dim].
constexpr int kSums = 5;  // dpost_w, dpost_b, dgate, dnext_w, dnext_b
constexpr int kAnySlabs = 256;

template <typename TX, typename TY>
__global__ __launch_bounds__(kAnyThreads) void k_residual_any_sums(ResidualArgs a, float* part) {
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const int c = blockIdx.x * kAnyThreads + threadIdx.x;
  const int64_t at = (int64_t)c * kChunk, left = a.dim - at;
  if (left <= 0) return;
  const int64_t per = (a.rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
  float s[kSums][kChunk] = {};
  for (int64_t row = r0; row < r1; ++row) {
    const float* q = a.stats + row * kStats;
    const RowStats st = {q[0], q[1], q[2], q[3]};
    RowMeans mean = {};
    mean.go = a.ws[row * 2];
    mean.g = a.ws[row * 2 + 1];
    float yh[kChunk], u[kChunk], gate[kChunk], o[kChunk], oh[kChunk], dh[kChunk], dx[kChunk];
    const DropWords keep = chunk_values<TX, TY>(a, key, row, c, st, yh, u, gate, o);
    chunk_dx<TX, TY>(a, row, c, st, mean, o, oh, dh, dx);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      s[3][i] = fmaf(dh[i], oh[i], s[3][i]);
      s[4][i] += dh[i];
      if (!a.y) continue;
      s[2][i] = fmaf(a.scale * dx[i], u[i], s[2][i]);
      float v = gate[i] * dx[i];
      if (a.drop.on) v = keep.kept(i, a.drop) ? v * a.drop.scale : 0.0f;
      s[0][i] = fmaf(v, yh[i], s[0][i]);
      s[1][i] += v;
    }
  }
  float* p = part + (int64_t)blockIdx.y * kSums * a.dim + at;
#pragma unroll
  for (int k = 0; k < kSums; ++k) store8(p + (int64_t)k * a.dim, left, s[k]);
}

// The parts of one parameter's sums: 64 columns a block, a wave every 16th part, each in
// order, then the waves in order.
__global__ __launch_bounds__(1024) void k_residual_sums(ResidualArgs a, const float* part, int parts) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.y;
  void* outs[kSums] = {a.dpost_w, a.dpost_b, a.gate_rows ? nullptr : a.dgate, a.dnext_w, a.dnext_b};
  const int types[kSums] = {a.post_w.bf16, a.post_b.bf16, a.gate.bf16, a.next_w.bf16, a.next_b.bf16};
  void* out = outs[k];
  if (!out) return;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (col < a.dim) {
#pragma unroll 16
    for (int s = wave; s < parts; s += 16) v += part[((int64_t)s * kSums + k) * a.dim + col];
  }
  red[wave][lane] = v;
  __syncthreads();
  if (wave || col >= a.dim) return;
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) v += red[w][lane];
  if (types[k])
    ((__bf16*)out)[col] = (__bf16)v;
  else
    ((float*)out)[col] = v;
}

// ---- up to kTeamMaxDim values: a row in the registers of a team of lanes --------------
//
// A team of LANES lanes holds a row, N chunks a lane; a block holds several teams and its
// rows stride over the batch, so that the parameters stay in LDS, and in the backward the sums over
// rows in registers. Every value of a row is read once, the next row's while this one is
// worked on.
template <int LANES, int N, int BLOCK>
struct Team {
  static constexpr int kTeams = BLOCK / LANES;
  static constexpr int kWaves = LANES > 64 ? LANES / 64 : 1;
  int team, lane, turn;
  float* red;  // [2][BLOCK / 64][2]
  __device__ Team(float* lds) : team(threadIdx.x / LANES), lane(threadIdx.x % LANES), turn(0), red(lds) {
    if constexpr (LANES >= 64) team = __builtin_amdgcn_readfirstlane(team);  // rows are a wave's: scalar
  }
  // Sums over the team, in every lane; all teams of the block call it together. Two
  // buffers in turn: a wave writes one again only after the barrier of the sum between, which its
  // readers reach when they have read it.
  template <int K>
  __device__ __forceinline__ void sum(float (&v)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lanes_sum<(LANES < 64 ? LANES : 64)>(v[k]);
    if constexpr (LANES > 64) {
      float* r = red + turn * (BLOCK / 64) * 2;
      turn ^= 1;
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) r[wave * 2 + k] = v[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) t += r[(team * kWaves + w) * 2 + k];
        v[k] = t;
      }
    }
  }
};

// A row's values of one tensor as they were read.
template <typename T, int N>
struct RowRaw {
  typename RawOf<T>::type v[N];
  template <int LANES>
  __device__ __forceinline__ void load(const T* base, int64_t row, int64_t ld, const ResidualArgs& a, int lane) {
    const T* p = base + row * ld;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = (n * LANES + lane) * kChunk;
      v[n] = load_near8(p, at, a.dim - at, (a.rows - 1 - row) * ld, a.dim & (kChunk - 1));
    }
  }
};
// The same of a tensor whose type is known at run time.
template <int N>
struct RowAny {
  u32x4_t v[N][2];
  template <int LANES>
  __device__ __forceinline__ void load(const AnyPtr& t, int64_t row, int64_t ld, const ResidualArgs& a, int lane) {
    const int64_t spare = (a.rows - 1 - row) * ld;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = (n * LANES + lane) * kChunk, left = a.dim - at;
      if (t.bf16) {
        v[n][0] = load_near8((const __bf16*)t.p + row * ld, at, left, spare, a.dim & (kChunk - 1)).v;
      } else {
        const RawF32 r = load_near8((const float*)t.p + row * ld, at, left, spare, a.dim & (kChunk - 1));
        v[n][0] = r.v[0];
        v[n][1] = r.v[1];
      }
    }
  }
  __device__ __forceinline__ void unpack(int n, int bf16, float (&f)[kChunk]) const {
    if (bf16) {
      unpack8(RawBf16{v[n][0]}, f);
    } else {
      RawF32 r;
      r.v[0] = v[n][0];
      r.v[1] = v[n][1];
      unpack8(r, f);
    }
  }
};

// The parameters as every row of a block reads them: in LDS, a lane's eight values of a chunk as two
// reads of 16 bytes at neighbouring lanes' neighbouring addresses; 0 past the row's end. In registers
// they would take the room of one to two waves a SIMD.
enum Param { kPostW, kPostB, kGate, kNextW, kNextB, kParams };
//
// A parameter takes two runs of 16 bytes a chunk: a chunk for every lane of the team, or, PACKED, the
// row's chunks and one of zeros for the lanes past it, which lets five parameters of up to 8152 values
// fit into 159.5 KiB (and costs the backward registers that it does not have).
template <int LANES, int N, bool PACKED>
struct ParamTable {
  float* lds;
  int lane, chunks;
  __device__ ParamTable(float* at, int l, int dim)
      : lds(at), lane(l), chunks(PACKED ? (dim + kChunk - 1) / kChunk + 1 : LANES * N) {}
  __device__ __forceinline__ static AnyPtr source(const ResidualArgs& a, int k) {
    switch (k) {
      case kPostW: return a.post_w;
      case kPostB: return a.post_b;
      case kGate: return AnyPtr{a.gate_rows ? nullptr : a.gate.p, a.gate.bf16};
      case kNextW: return a.next_w;
      default: return a.next_b;
    }
  }
  // Every thread of the block calls it, and a barrier follows.
  __device__ __forceinline__ void fill(const ResidualArgs& a, int params) {
    int slot = 0;
    for (int k = 0; k < params; ++k) {
      const AnyPtr src = source(a, k);
      if (!src.p) continue;
      for (int c = threadIdx.x; c < chunks; c += blockDim.x) {
        float f[kChunk] = {};
        if (c * kChunk < a.dim) load8(src, (int64_t)c * kChunk, a.dim - (int64_t)c * kChunk, f);
        f32x4_t* to = PACKED ? (f32x4_t*)lds + slot * 2 * chunks + c
                             : (f32x4_t*)(lds + slot * LANES * N * kChunk + c / LANES * LANES * kChunk) + c % LANES;
        to[0] = f32x4_t{f[0], f[1], f[2], f[3]};
        to[PACKED ? chunks : LANES] = f32x4_t{f[4], f[5], f[6], f[7]};
      }
      ++slot;
    }
  }
  // Where parameter k lies, once it is known to be there.
  __device__ __forceinline__ const float* at(const ResidualArgs& a, int k) const {
    int slot = 0;
    for (int q = 0; q < k; ++q) slot += source(a, q).p != nullptr;
    return lds + slot * (PACKED ? chunks : LANES * N) * kChunk;
  }
  __device__ __forceinline__ void get(const float* p, int n, float (&f)[kChunk]) const {
    f32x4_t lo, hi;
    if constexpr (PACKED) {
      const int own = n * LANES + lane, c = own < chunks ? own : chunks - 1;
      lo = ((const f32x4_t*)p)[c];
      hi = ((const f32x4_t*)p)[chunks + c];
    } else {
      const f32x4_t* from = (const f32x4_t*)(p + n * LANES * kChunk) + lane;
      lo = from[0];
      hi = from[LANES];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = lo[i];
      f[4 + i] = hi[i];
    }
  }
};

// The gate of a row's chunk, times scale.
template <int LANES, int N, bool PACKED>
__device__ __forceinline__ void gate_values(const ResidualArgs& a, const ParamTable<LANES, N, PACKED>& par, const float* pg, const RowAny<N>& rows,
                                            int64_t row, int n, float (&g)[kChunk]) {
  if (a.gate_rows) {
    rows.unpack(n, a.gate.bf16, g);
    if (a.dim & (kChunk - 1)) settle8(a.dim - (n * LANES + par.lane) * kChunk, (a.rows - 1 - row) * a.gate_ld, g);
  } else if (a.gate.p) {
    par.get(pg, n, g);
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) g[i] = 1.0f;
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) g[i] *= a.scale;
}

// The factor of a row's values less their mean. Lanes hold 0 past a row's end, which become -mean r and there meet
// parameters of 0: NaN where that overflows. It does so only where every value is the mean exactly (another one
// would differ by 2^-24 of it, and r be at most 2^24 sqrt(dim) / mean), and any factor gives their 0: with 0, places past the end are 0
// too. One comparison a row: a select a value made 2048 and 4096 values in bf16 8 % slower (55.5 -> 60.6 us).
__device__ __forceinline__ float value_factor(float mean, float r) {
  return fabsf(mean * r) == INFINITY && r != INFINITY ? 0.0f : r;
}

// u (after dropout), y^ in y's place; the mask of the chunk.
template <int LANES, int N, bool PACKED>
__device__ __forceinline__ DropWords branch_values(const ResidualArgs& a, const DropKey& key, const ParamTable<LANES, N, PACKED>& par,
                                                  const float* pw, const float* pb, int64_t row, int n, float m1, float r1,
                                                  float (&y)[kChunk], float (&u)[kChunk]) {
#pragma unroll
  for (int i = 0; i < kChunk; ++i) u[i] = y[i];
  if (a.post_w.p) {
    float w[kChunk], b[kChunk] = {};
    par.get(pw, n, w);
    if (a.post_b.p) par.get(pb, n, b);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      y[i] = (y[i] - m1) * r1;
      u[i] = fmaf(y[i], w[i], b[i]);
    }
  }
  DropWords keep = {};
  if (a.drop.on) {
    keep = drop_words(a.drop, key, (uint32_t)row, (uint32_t)(n * LANES + par.lane));
#pragma unroll
    for (int i = 0; i < kChunk; ++i) u[i] = keep.kept(i, a.drop) ? u[i] * a.drop.scale : 0.0f;
  }
  return keep;
}

// The mean (layer norms) and 1 / root mean square of a row's values, which are 0 past its end.
template <int N, int LANES, typename TEAM>
__device__ __forceinline__ void row_stats(TEAM& team, const ResidualArgs& a, const float (&v)[N][kChunk], float inv,
                                          float& mean, float& r) {
  float s[1] = {0.0f};
  mean = 0.0f;
  if (a.layer) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kChunk; ++i) s[0] += v[n][i];
    team.sum(s);
    mean = s[0] * inv;
    s[0] = 0.0f;
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int left = a.dim - (n * LANES + team.lane) * kChunk;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const float d = i < left ? v[n][i] - mean : 0.0f;
      s[0] = fmaf(d, d, s[0]);
    }
  }
  team.sum(s);
  r = 1.0f / sqrtf(fmaf(s[0], inv, a.eps));
}

template <typename TX, typename TY, int LANES, int N, int BLOCK>
__global__ __launch_bounds__(BLOCK, 4) void k_residual_rows(ResidualArgs a) {
  extern __shared__ __align__(16) float lds[];
  __shared__ float red[2 * BLOCK / 64 * 2];
  Team<LANES, N, BLOCK> team(red);
  const int lane = team.lane;
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  if (a.stats && a.drop.on && blockIdx.x == 0 && threadIdx.x == 0) {
    int64_t* used = (int64_t*)(a.stats + a.rows * kStats);
    used[0] = a.drop.state ? a.drop.state[0] : (int64_t)a.drop.seed;
    used[1] = (int64_t)(((uint64_t)key.call1 << 32) | key.call0);
  }
  const float inv = 1.0f / (float)a.dim;
  const int64_t step = (int64_t)gridDim.x * team.kTeams;
  int64_t row = (int64_t)blockIdx.x * team.kTeams + team.team;
  RowRaw<TX, N> xr;
  RowRaw<TY, N> yr;
  RowAny<N> gr;
  const auto fetch = [&](int64_t r) {
    if (r >= a.rows) return;
    xr.template load<LANES>((const TX*)a.x, r, a.x_ld, a, lane);
    if (a.y) yr.template load<LANES>((const TY*)a.y, r, a.y_ld, a, lane);
    if (a.gate_rows) gr.template load<LANES>(a.gate, r, a.gate_ld, a, lane);
  };
  fetch(row);
  ParamTable<LANES, N, (LANES == 1024)> par(lds, lane, a.dim);
  par.fill(a, kParams);
  __syncthreads();
  const float *pw = par.at(a, kPostW), *pb = par.at(a, kPostB), *pg = par.at(a, kGate), *nw = par.at(a, kNextW),
              *nb = par.at(a, kNextB);
  // every team of the block takes as many turns as its first: the sums' barriers are the block's
  for (int64_t first = (int64_t)blockIdx.x * team.kTeams; first < a.rows; first += step, row += step) {
    const bool active = row < a.rows;
    float x[N][kChunk], y[N][kChunk];
    RowAny<N> gate = gr;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      unpack8(xr.v[n], x[n]);
      if (a.y) unpack8(yr.v[n], y[n]);
      if (a.dim & (kChunk - 1)) {
        const int left = a.dim - (n * LANES + lane) * kChunk;
        const int64_t after = a.rows - 1 - row;
        settle8(left, after * a.x_ld, x[n]);
        if (a.y) settle8(left, after * a.y_ld, y[n]);
      }
    }
    fetch(row + step);
    float m1 = 0.0f, r1 = 0.0f, m2 = 0.0f, r2 = 0.0f;
    if (a.y) {
      if (a.post_w.p) row_stats<N, LANES>(team, a, y, inv, m1, r1);
      const float f1 = value_factor(m1, r1);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float u[kChunk], g[kChunk];
        branch_values(a, key, par, pw, pb, row, n, m1, f1, y[n], u);
        gate_values(a, par, pg, gate, row, n, g);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) x[n][i] = fmaf(g[i], u[i], x[n][i]);
        const int at = (n * LANES + lane) * kChunk;
        if (active && at < a.dim) store8((TX*)a.out + row * a.dim + at, a.dim - at, x[n]);
      }
    }
    if (a.next_w.p) {
      row_stats<N, LANES>(team, a, x, inv, m2, r2);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float w[kChunk], b[kChunk] = {};
        par.get(nw, n, w);
        if (a.next_b.p) par.get(nb, n, b);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) x[n][i] = fmaf((x[n][i] - m2) * r2, w[i], b[i]);
        const int at = (n * LANES + lane) * kChunk;
        if (active && at < a.dim) store8((TY*)a.h + row * a.dim + at, a.dim - at, x[n]);
      }
    }
    if (a.stats && active && lane == 0) *(f32x4_t*)(a.stats + row * kStats) = f32x4_t{m1, r1, m2, r2};
  }
}

// Waves a SIMD that the backward's registers leave room for. The five sums over rows take 8 N registers each whether a call
// has them all or not, and some forms keep values in scratch for it: of 4097 to 8192 values (512 lanes, N = 2) 304 to 384 bytes a lane, in
// bf16 of 64 to 512 lanes 16 to 72, with a bf16 stream and an fp32 branch of 512 lanes 40, in fp32 of 512 lanes 24.
__host__ __device__ constexpr int backward_waves(int lanes, int n) { return lanes < 64 || n > 1 ? 2 : 3; }

// Its sums over rows a block leaves as a part of each, [block, 5, dim].
template <typename TX, typename TY, int LANES, int N, int BLOCK>
__global__ __launch_bounds__(BLOCK, backward_waves(LANES, N)) void k_residual_rows_backward(ResidualArgs a, int sums) {
  // the next row's values on their way, where the registers have room for them
  constexpr bool kAhead = LANES < 64 || (N == 1 && sizeof(TX) + sizeof(TY) == 4);
  extern __shared__ __align__(16) float lds[];
  __shared__ float red[2 * BLOCK / 64 * 2];
  Team<LANES, N, BLOCK> team(red);
  const int lane = team.lane;
  const DropKey key = a.drop.on ? drop_key(a.drop) : DropKey{};
  const float inv = 1.0f / (float)a.dim;
  const int64_t step = (int64_t)gridDim.x * team.kTeams;
  int64_t row = (int64_t)blockIdx.x * team.kTeams + team.team;
  RowRaw<TX, N> xr, dor;
  RowRaw<TY, N> yr, dhr;
  RowAny<N> gr;
  f32x4_t st;
  const bool next = a.next_w.p && a.dh, post = a.post_w.p;
  const auto fetch = [&](int64_t r) {
    if (r >= a.rows) {  // zeros, which add nothing to the sums
      st = f32x4_t{};
      xr = RowRaw<TX, N>{};
      yr = RowRaw<TY, N>{};
      gr = RowAny<N>{};
      dor = RowRaw<TX, N>{};
      dhr = RowRaw<TY, N>{};
      return;
    }
    st = *(const f32x4_t*)(a.stats + r * kStats);
    xr.template load<LANES>((const TX*)a.x, r, a.x_ld, a, lane);
    if (a.y) yr.template load<LANES>((const TY*)a.y, r, a.y_ld, a, lane);
    if (a.gate_rows) gr.template load<LANES>(a.gate, r, a.gate_ld, a, lane);
    if (a.dout) dor.template load<LANES>((const TX*)a.dout, r, a.dout_ld, a, lane);
    if (a.dh) dhr.template load<LANES>((const TY*)a.dh, r, a.dh_ld, a, lane);
  };
  if (kAhead) fetch(row);
  ParamTable<LANES, N, false> par(lds, lane, a.dim);
  par.fill(a, kNextB);  // next's bias has no part in it
  __syncthreads();
  const float *pw = par.at(a, kPostW), *pb = par.at(a, kPostB), *pg = par.at(a, kGate), *nw = par.at(a, kNextW);
  float acc[kSums][N][kChunk] = {};
  for (int64_t first = (int64_t)blockIdx.x * team.kTeams; first < a.rows; first += step, row += step) {
    const bool active = row < a.rows;
    if (!kAhead) fetch(row);
    float x[N][kChunk], y[N][kChunk], u[N][kChunk] = {}, dx[N][kChunk];
    RowRaw<TY, N> dh = dhr;
    RowAny<N> gate = gr;
    DropWords keep[N];
    const float m1 = st[0], r1 = st[1], m2 = st[2], r2 = st[3], f1 = value_factor(m1, r1), f2 = value_factor(m2, r2);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      unpack8(xr.v[n], x[n]);
      if (a.y) unpack8(yr.v[n], y[n]);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) dx[n][i] = 0.0f;
      if (a.dout) unpack8(dor.v[n], dx[n]);
      if (a.dim & (kChunk - 1)) {
        const int left = a.dim - (n * LANES + lane) * kChunk;
        const int64_t after = a.rows - 1 - row;
        settle8(left, after * a.x_ld, x[n]);
        if (a.y) settle8(left, after * a.y_ld, y[n]);
        if (a.dout) settle8(left, after * a.dout_ld, dx[n]);
      }
    }
    if (kAhead) fetch(row + step);
    if (a.y)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float g[kChunk];
        keep[n] = branch_values(a, key, par, pw, pb, row, n, m1, f1, y[n], u[n]);
        gate_values(a, par, pg, gate, row, n, g);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) x[n][i] = fmaf(g[i], u[n][i], x[n][i]);
      }
    if (next) {
      // x becomes o^; g = dh w
      float s[2] = {0.0f, 0.0f}, g[N][kChunk];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float d[kChunk];
        unpack8(dh.v[n], d);
        if (a.dim & (kChunk - 1)) settle8(a.dim - (n * LANES + lane) * kChunk, (a.rows - 1 - row) * a.dh_ld, d);
        par.get(nw, n, g[n]);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          x[n][i] = (x[n][i] - m2) * f2;
          acc[3][n][i] = fmaf(d[i], x[n][i], acc[3][n][i]);
          g[n][i] *= d[i];
          s[0] = fmaf(g[n][i], x[n][i], s[0]);
        }
        if (sums & 16)
#pragma unroll
          for (int i = 0; i < kChunk; ++i) acc[4][n][i] += d[i];
        if (a.layer)
#pragma unroll
          for (int i = 0; i < kChunk; ++i) s[1] += g[n][i];
      }
      team.sum(s);
      const float go = s[0] * inv, gm = a.layer ? s[1] * inv : 0.0f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < kChunk; ++i) dx[n][i] = fmaf(r2, g[n][i] - fmaf(x[n][i], go, gm), dx[n][i]);
    }
    if (a.dx && active)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int at = (n * LANES + lane) * kChunk;
        if (at < a.dim) store8((TX*)a.dx + row * a.dim + at, a.dim - at, dx[n]);
      }
    if (!a.y) continue;
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (a.gate.p) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) u[n][i] *= a.scale * dx[n][i];
        if (!a.gate_rows) {
#pragma unroll
          for (int i = 0; i < kChunk; ++i) acc[2][n][i] += u[n][i];
        } else if (a.dgate) {
          const int at = (n * LANES + lane) * kChunk;
          if (active && at < a.dim) {
            if (a.gate.bf16)
              store8((__bf16*)a.dgate + row * a.dim + at, a.dim - at, u[n]);
            else
              store8((float*)a.dgate + row * a.dim + at, a.dim - at, u[n]);
          }
        }
      }
      float g[kChunk];
      gate_values(a, par, pg, gate, row, n, g);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) dx[n][i] *= g[i];
      if (a.drop.on)
#pragma unroll
        for (int i = 0; i < kChunk; ++i) dx[n][i] = keep[n].kept(i, a.drop) ? dx[n][i] * a.drop.scale : 0.0f;
      if (post) {
        float w[kChunk];
        par.get(pw, n, w);
        if (sums & 2)
#pragma unroll
          for (int i = 0; i < kChunk; ++i) acc[1][n][i] += dx[n][i];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          acc[0][n][i] = fmaf(dx[n][i], y[n][i], acc[0][n][i]);
          dx[n][i] *= w[i];
          s[0] = fmaf(dx[n][i], y[n][i], s[0]);
        }
        if (a.layer)
#pragma unroll
          for (int i = 0; i < kChunk; ++i) s[1] += dx[n][i];
      }
    }
    if (!a.dy) continue;
    if (post) {
      team.sum(s);
      const float ey = s[0] * inv, em = a.layer ? s[1] * inv : 0.0f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < kChunk; ++i) dx[n][i] = r1 * (dx[n][i] - fmaf(y[n][i], ey, em));
    }
    if (active)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int at = (n * LANES + lane) * kChunk;
        if (at < a.dim) store8((TY*)a.dy + row * a.dim + at, a.dim - at, dx[n]);
      }
  }
  if (!sums) return;
  // the teams' sums, in order, to this block's part
  float* part = a.ws + (int64_t)blockIdx.x * kSums * a.dim;
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    if (!(sums >> k & 1)) continue;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kChunk; ++i) lds[(team.team * LANES + lane) * kChunk + i] = acc[k][n][i];
      __syncthreads();
      for (int c = threadIdx.x; c < LANES * kChunk; c += BLOCK) {
        float v = 0.0f;
#pragma unroll
        for (int t = 0; t < team.kTeams; ++t) v += lds[t * LANES * kChunk + c];
        const int col = n * LANES * kChunk + c;
        if (col < a.dim) part[(int64_t)k * a.dim + col] = v;
      }
    }
  }
}

// Row slabs of the sums at any width.
int any_slabs(const ResidualArgs& a) {
  const int64_t wide = ceil_div(a.dim, kChunk * kAnyThreads);
  int64_t slabs = ceil_div(4 * kNumCUs, wide);
  if (slabs > kAnySlabs) slabs = kAnySlabs;
  if (slabs > a.rows) slabs = a.rows;
  return (int)slabs;
}

// The parameters' sums that are wanted, as bits.
int sum_bits(const ResidualArgs& a) {
  return (a.dpost_w ? 1 : 0) | (a.dpost_b ? 2 : 0) | (a.dgate && !a.gate_rows ? 4 : 0) | (a.dnext_w ? 8 : 0) | (a.dnext_b ? 16 : 0);
}

constexpr int kTeamMaxDim = 8192;
constexpr int kLdsBytes = 160 * 1024 - 512;  // less the sums' words

// The parameters that a launch holds in LDS (the backward all but next's bias).
int held(const ResidualArgs& a, bool backward) {
  return (a.post_w.p ? 1 : 0) + (a.post_b.p ? 1 : 0) + (a.gate.p && !a.gate_rows ? 1 : 0) + (a.next_w.p ? 1 : 0) +
         (a.next_b.p && !backward ? 1 : 0);
}
// LDS bytes of a launch of teams; the backward's hold its blocks' sums at the end.
int team_lds(const ResidualArgs& a, bool backward, int lanes, int n, int block) {
  const int chunks = !backward && lanes == 1024 ? (int)ceil_div(a.dim, kChunk) + 1 : lanes * n;
  const int params = held(a, backward) * chunks * kChunk * 4, tile = backward ? block * kChunk * 4 : 0;
  return params > tile ? params : tile;
}

// Blocks of a launch of teams: as many as the chip holds at once (their waves by registers,
// `waves` a SIMD, and their LDS), fewer where rows run out.
int64_t team_blocks(const ResidualArgs& a, int teams, int block, int waves, int lds) {
  int per_cu = waves * 256 / block;
  while (per_cu > 1 && per_cu * (lds + 512) > kLdsBytes) --per_cu;
  if (per_cu < 1) per_cu = 1;
  const int64_t all = ceil_div(a.rows, teams), most = (int64_t)per_cu * kNumCUs;
  return all < most ? all : most;
}
// The forward's, which leave no sums: four times as many in fp32 where their teams keep four rows each. A
// chip of blocks that begin and end apart spreads reads and writes better than one that runs in step (65536 x
// 512 111 -> 103 us, 131072 x 256 111 -> 105); in bf16, with half of the bytes a row, filling the parameters
// costs more (56.8 -> 58.6), with fewer rows too (8192 x 1000 16.0 -> 22.9), and of a wider row's parameters (8192 x
// 4096 101.9 -> 103.7).
template <typename TX, typename TY>
int64_t forward_blocks(const ResidualArgs& a, int teams, int block, int lds) {
  const int64_t blocks = team_blocks(a, teams, block, 4, lds);
  return sizeof(TX) + sizeof(TY) == 8 && block == 256 && a.rows >= 16 * teams * blocks ? 4 * blocks : blocks;
}
constexpr int kPartBlocks = 4;  // at most a CU: each leaves a part of every sum

// The team of a width: a chunk a lane, so that a row is one batch of loads, up to eight rows a wave and 16 waves a
// row. WIDE is that of the widest rows: in the backward half as many lanes, whose 256
// registers hold two chunks and their sums, but for what goes to scratch (4096 x 8192 212 to 224 us in fp32 and 132 to 142 in
// bf16; 1024 lanes of 128 registers 291 and 175).
#define CKAN_TEAM(dim, F, WIDE)                 \
  do {                                          \
    if ((dim) <= 64) { F(8, 1, 256) }           \
    else if ((dim) <= 128) { F(16, 1, 256) }    \
    else if ((dim) <= 256) { F(32, 1, 256) }    \
    else if ((dim) <= 512) { F(64, 1, 256) }    \
    else if ((dim) <= 1024) { F(128, 1, 256) }  \
    else if ((dim) <= 2048) { F(256, 1, 256) }  \
    else if ((dim) <= 4096) { F(512, 1, 512) }  \
    else { WIDE }                               \
  } while (0)

template <typename K>
void launch_team(K kernel, const ResidualArgs& a, int64_t blocks, int block, int lds, hipStream_t st, std::atomic<uint32_t>& done,
                 int sums = -1) {
  ensure_lds_limit((const void*)kernel, kLdsBytes, done);
  if constexpr (std::is_invocable_v<K, ResidualArgs, int>)
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(block), lds, st, a, sums);
  else
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(block), lds, st, a);
}

// Whether the teams' form takes a call: its width, and the parameters' room.
bool by_teams(const ResidualArgs& a, bool backward) {
  if (a.dim > kTeamMaxDim || a.dim < kChunk) return false;
  return a.dim <= 4096 || team_lds(a, backward, 1024, 1, 1024) <= kLdsBytes;
}

template <typename TX, typename TY>
void forward_typed(const ResidualArgs& a, hipStream_t st) {
  if (by_teams(a, false)) {
#define CKAN_FORWARD(L, NN, B)                                                                           \
  static std::atomic<uint32_t> done;                                                                     \
  const int lds = team_lds(a, false, L, NN, B);                                                          \
  launch_team(k_residual_rows<TX, TY, L, NN, B>, a, forward_blocks<TX, TY>(a, B / L, B, lds), B, lds, st, done); \
  return;
    CKAN_TEAM(a.dim, CKAN_FORWARD, CKAN_FORWARD(1024, 1, 1024));
#undef CKAN_FORWARD
  }
  const int64_t blocks = a.rows < 8 * kNumCUs ? a.rows : 8 * kNumCUs;
  hipLaunchKernelGGL((k_residual_any<TX, TY>), dim3((unsigned)blocks), dim3(kAnyThreads), 0, st, a);
}

template <typename TX, typename TY>
void backward_typed(const ResidualArgs& a, hipStream_t st) {
  const int sums = sum_bits(a);
  const dim3 sum_grid((unsigned)ceil_div(a.dim, 64), kSums);
  if (by_teams(a, true)) {
    int64_t blocks = 0;
#define CKAN_BACKWARD(L, NN, B)                                                                          \
  static std::atomic<uint32_t> done;                                                                     \
  const int lds = team_lds(a, true, L, NN, B);                                                           \
  blocks = team_blocks(a, B / L, B, backward_waves(L, NN), lds);                                             \
  launch_team(k_residual_rows_backward<TX, TY, L, NN, B>, a, blocks, B, lds, st, done, sums);
    CKAN_TEAM(a.dim, CKAN_BACKWARD, CKAN_BACKWARD(512, 2, 512));
#undef CKAN_BACKWARD
    if (sums) hipLaunchKernelGGL(k_residual_sums, sum_grid, dim3(1024), 0, st, a, a.ws, (int)blocks);
    return;
  }
  const int64_t blocks = a.rows < 8 * kNumCUs ? a.rows : 8 * kNumCUs;
  hipLaunchKernelGGL((k_residual_any_dx<TX, TY>), dim3((unsigned)blocks), dim3(kAnyThreads), 0, st, a);
  if (!sums) return;
  const int slabs = any_slabs(a);
  float* part = a.ws + round_up(a.rows * 2, 4);
  hipLaunchKernelGGL((k_residual_any_sums<TX, TY>), dim3((unsigned)ceil_div(a.dim, kChunk * kAnyThreads), (unsigned)slabs),
                     dim3(kAnyThreads), 0, st, a, part);
  hipLaunchKernelGGL(k_residual_sums, sum_grid, dim3(1024), 0, st, a, part, slabs);
}

}  // namespace

size_t residual_workspace_bytes(const ResidualArgs& a) {
  // either form's: which one runs hangs on the parameters too
  int64_t parts = any_slabs(a);
  if (a.dim <= kTeamMaxDim) {
    const int64_t most = (int64_t)kPartBlocks * kNumCUs, blocks = a.rows < most ? a.rows : most;
    if (blocks > parts) parts = blocks;
  }
  return align256((round_up(a.rows * 2, 4) + parts * kSums * a.dim) * sizeof(float));
}

void launch_residual_forward(const ResidualArgs& a, hipStream_t st) {
  if (a.x_bf16)
    a.y_bf16 ? forward_typed<__bf16, __bf16>(a, st) : forward_typed<__bf16, float>(a, st);
  else
    a.y_bf16 ? forward_typed<float, __bf16>(a, st) : forward_typed<float, float>(a, st);
}

void launch_residual_backward(const ResidualArgs& a, hipStream_t st) {
  if (a.x_bf16)
    a.y_bf16 ? backward_typed<__bf16, __bf16>(a, st) : backward_typed<__bf16, float>(a, st);
  else
    a.y_bf16 ? backward_typed<float, __bf16>(a, st) : backward_typed<float, float>(a, st);
}

}  // namespace ckan
