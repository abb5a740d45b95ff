// Log probabilities of given classes, entropies and the likeliest classes of rows of
// logits (ckan_log_probs), and the gradient (ckan_log_probs_backward).
//
// One pass over a row keeps four numbers: the largest logit m so far, how many equal it
// (n), the sum s of e = exp(l - m) over the others and a = sum e (l - m).  They give
//   log Z - m = log n + log1p(s / n),   log p_t = (l_t - m) - (log Z - m),
//   H = -sum p log p = (log Z - m) - a / (n + s).
// The largest apart from the rest keeps both exact in rows that are sure of one class,
// where 1 + s would round to 1.  A logit of -inf has no probability; with d = l - m held
// above kFar its products stay 0 instead of 0 inf.  The gradient of a row is
//   dl_j = dlogp (delta_jt - p_j) - dH p_j (log p_j + H).
//
// Bound by the bytes of the logits, read once (the likeliest classes' few chunks twice), the backward reading and
// writing them once. Four tensors in turn: 4000 rows of 50001 classes in bf16 78 to 86 us (4.7 to 5.1 TB/s) without and 87 with five
// likeliest classes, backward 161 to 170 (4.7 to 5.0); in training steps, where it follows a backward that has just written 400
// MB, the forward takes 117 to 119 (3.4). 65536 x 1000 in fp32 63 and 92 us (4.2 and 5.7 TB/s), in bf16 48 and 53 (2.7 and
// 5.0). One row of 131072 is two launches of a few microseconds each: parts of the row, and their join.
#include "ckan_block.hpp"
#include "ckan_mix.hpp"

namespace ckan {
namespace {

constexpr float kFar = -200.0f;  // exp(kFar) is 0 in fp32
constexpr float kLog2e = 1.44269504088896341f;

struct RowSum {
  float m, n, s, a;
};
__device__ __forceinline__ RowSum empty_sum() { return {-FLT_MAX, 0.0f, 0.0f, 0.0f}; }

// exp(d) in two instructions: off by |d| 2^-24 or so, which sums weighted by it do not see.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }
// A probability that is a result's own factor: as exact as its type.
__device__ __forceinline__ float prob_of(float d, float) { return expf(d); }
__device__ __forceinline__ float prob_of(float d, __bf16) { return exp_of(d); }

// The sums with their largest moved up to m (NaN logits never move it, but leave s NaN).
__device__ __forceinline__ void raise(RowSum& r, float m) {
  const float d = r.m - m, c = exp_of(d);
  const float all = r.n + r.s;
  const bool same = r.m == m;
  r.a = same ? r.a : c * fmaf(all, fmaxf(d, kFar), r.a);
  r.s = same ? r.s : c * all;
  r.n = same ? r.n : 0.0f;
  r.m = m;
}
__device__ __forceinline__ RowSum merged(RowSum x, RowSum y) {
  const float m = fmaxf(x.m, y.m);
  raise(x, m);
  raise(y, m);
  return {m, x.n + y.n, x.s + y.s, x.a + y.a};
}
template <int N>
__device__ __forceinline__ void add_logits(RowSum& r, const float (&l)[N]) {
  float m = r.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, l[i]);
  raise(r, m);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = l[i] - m, e = exp_of(d);
    const bool top = l[i] == m;
    r.n += top ? 1.0f : 0.0f;
    r.s += top ? 0.0f : e;
    r.a = fmaf(e, fmaxf(d, kFar), r.a);
  }
}

// What a row's sums say: its shift, log of the sum and entropy.
struct RowResult {
  float m, logs, entropy;
  bool empty;
};
__device__ __forceinline__ RowResult row_result(const RowSum& r) {
  RowResult q;
  q.empty = r.n == 0.0f && r.s == 0.0f;  // nothing above -inf (a NaN leaves s NaN)
  q.m = r.m;
  q.logs = q.empty ? INFINITY : logf(r.n) + log1pf(r.s / r.n);
  if ((r.n == 0.0f && !q.empty) || r.m == INFINITY) q.logs = NAN;  // NaN alone, or +inf
  q.entropy = q.empty ? 0.0f : q.logs - r.a / (r.n + r.s);
  return q;
}

// ---- the likeliest classes ---------------------------------------------------------
// A logit's place in the order: larger first, equal ones by the lower index; 0 for what
// is never chosen (-inf, NaN).
__device__ __forceinline__ uint64_t top_key(float l, uint32_t index) {
  if (!(l > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(l + 0.0f);  // -0 and 0 are equal
  return (uint64_t)(b ^ (b >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int w = 32; w; w >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, w);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ void write_row(const LogpArgs& a, int64_t row, const RowResult& r) {
  const int64_t t = a.targets[row];
  float logp = 0.0f;
  if (t >= 0 && t < a.classes) {
    const float l = a.bf16 ? (float)((const __bf16*)a.logits)[row * a.ld + t] : ((const float*)a.logits)[row * a.ld + t];
    logp = r.empty ? -INFINITY : (l - r.m) - r.logs;
  }
  a.logp[row] = logp;
  a.entropy[row] = r.entropy;
  if (a.stats) {
    a.stats[row * 3] = r.m;
    a.stats[row * 3 + 1] = r.logs;
    a.stats[row * 3 + 2] = r.entropy;
  }
}
__device__ __forceinline__ void write_top(const LogpArgs& a, int64_t row, int j, uint64_t key, const RowResult& r) {
  a.top_logp[row * a.top + j] = key ? (key_logit(key) - r.m) - r.logs : -INFINITY;
  a.top_idx[row * a.top + j] = key ? (int64_t)key_index(key) : -1;
}

constexpr int kThreads = 256;
// 16384 rows, one tensor again and again, by a team and by a block: 3000 classes in fp32 59.5 and 61 us, with five likeliest 71
// and 92, with twenty 111 and 129; 4096 classes in bf16 60.9 and 67.9, 70 and 85, 111 and 116. Only 4096 classes in fp32 without
// any are better by a block (75.9 and 64.2; with five 82.6 and 94.5). Four tensors in turn by a team: 74, 87 and 120 (3000 in
// fp32), 59, 73 and 114 (4096 in bf16).
constexpr int kTeamMaxClasses = 4096;

// ---- up to kTeamMaxClasses: a row in the registers of a team of lanes ----------------
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)));
}
// The largest over a group of L lanes, in each of them (as lanes_sum).
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
  v = dpp_max<0xb1>(v);
  v = dpp_max<0x4e>(v);
  v = dpp_max<0x141>(v);
  if constexpr (L >= 16) v = dpp_max<0x140>(v);
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// One team a row: LANES lanes hold N chunks each. Lane j of the team holds columns j N 8 on, so
// that the lowest column among equal logits is the lowest lane's lowest. The likeliest classes come
// in `top` rounds of the team's largest.
template <typename T, int LANES, int N>
__global__ __launch_bounds__(kThreads) void k_logprobs_team(LogpArgs a) {
  const int lane = threadIdx.x % LANES, in_wave = threadIdx.x & 63;
  const int64_t step = (int64_t)gridDim.x * (kThreads / LANES);
  // all teams of a wave take the same turns: lanes of rows past the end work on the last row
  for (int64_t first = (int64_t)blockIdx.x * (kThreads / LANES); first < a.rows; first += step) {
    const int64_t mine = first + threadIdx.x / LANES, row = mine < a.rows ? mine : a.rows - 1;
    const T* l = (const T*)a.logits + row * a.ld;
    float v[N * kChunk];
    const int64_t spare = (a.rows - 1 - row) * a.ld;
    typename RawOf<T>::type raw[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = (lane * N + n) * kChunk, left = a.classes - at;
      raw[n] = a.classes >= kChunk ? load_near8(l, at, left, spare, a.classes & (kChunk - 1)) : load_raw8(l + at, (int64_t)left);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int left = a.classes - (lane * N + n) * kChunk;
      float f[kChunk];
      unpack8(raw[n], f);
      if (a.classes >= kChunk && (a.classes & (kChunk - 1))) settle8(left, spare, f);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) v[n * kChunk + i] = i < left ? f[i] : -INFINITY;
    }
    RowSum r = empty_sum();
#pragma unroll
    for (int i = 0; i < N * kChunk; ++i) r.m = fmaxf(r.m, v[i]);
    r.m = lanes_max<LANES>(r.m);
#pragma unroll
    for (int i = 0; i < N * kChunk; ++i) {
      const float d = v[i] - r.m, e = exp_of(d);
      const bool top = v[i] == r.m;
      r.n += top ? 1.0f : 0.0f;
      r.s += top ? 0.0f : e;
      r.a = fmaf(e, fmaxf(d, kFar), r.a);
    }
    r.n = lanes_sum<LANES>(r.n);
    r.s = lanes_sum<LANES>(r.s);
    r.a = lanes_sum<LANES>(r.a);
    const RowResult q = row_result(r);
    const bool write = mine < a.rows;
    if (lane == 0 && write) write_row(a, row, q);
    if (!a.top) continue;
    float largest[N];  // of each chunk
#pragma unroll
    for (int n = 0; n < N; ++n) {
      largest[n] = v[n * kChunk];
#pragma unroll
      for (int i = 1; i < kChunk; ++i) largest[n] = fmaxf(largest[n], v[n * kChunk + i]);
    }
    for (int j = 0; j < a.top; ++j) {
      float own = largest[0];
#pragma unroll
      for (int n = 1; n < N; ++n) own = fmaxf(own, largest[n]);
      const float best = lanes_max<LANES>(own);
      const unsigned long long has = __ballot(own == best && best > -INFINITY) >> (in_wave & ~(LANES - 1));
      const unsigned long long team = LANES == 64 ? has : has & ((1ull << (LANES & 63)) - 1);
      const int from = team ? __ffsll(team) - 1 : -1;
      // the lane's first chunk that holds it, a scalar where a wave has one row
      int chunk = N - 1;
#pragma unroll
      for (int n = N - 2; n >= 0; --n) chunk = largest[n] == best ? n : chunk;
      if constexpr (N > 1) chunk = __builtin_amdgcn_readlane(chunk, from < 0 ? 0 : __builtin_amdgcn_readfirstlane(from));
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (n != chunk || lane != from) continue;
        float* w = v + n * kChunk;
        int at = kChunk - 1;
#pragma unroll
        for (int i = kChunk - 2; i >= 0; --i) at = w[i] == best ? i : at;
        largest[n] = -INFINITY;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          w[i] = i == at ? -INFINITY : w[i];
          largest[n] = fmaxf(largest[n], w[i]);
        }
        if (write) {
          a.top_logp[row * a.top + j] = (best - q.m) - q.logs;
          a.top_idx[row * a.top + j] = ((int64_t)lane * N + n) * kChunk + at;
        }
      }
      if (from < 0 && lane == 0 && write) write_top(a, row, j, 0, q);
    }
  }
}

// ---- longer rows: a block a row, or a part of one ------------------------------------
constexpr int kMaxParts = 32;
constexpr int kPartMin = 4096;        // logits a part is worth
constexpr int kCandidates = 1024;
constexpr int kWaves = kThreads / 64;

// Lanes whose condition holds count up in thread order: the thread's place, and the total.
__device__ __forceinline__ int block_place(bool mine, int* counts, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned long long has = __ballot(mine);
  if (lane == 0) counts[wave] = __popcll(has);
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? counts[w] : 0;
    total += counts[w];
  }
  __syncthreads();
  return before + __popcll(has & ((1ull << lane) - 1));
}

// How many of n keys in LDS are larger than key; they lie at 16 bytes, a key of 0 behind an odd count.
__device__ __forceinline__ int rank_among(const uint64_t* keys, int n, uint64_t key) {
  int rank = 0;
#pragma unroll 4
  for (int o = 0; o < n; o += 2) {
    const u32x4_t two = *(const u32x4_t*)(keys + o);
    rank += ((uint64_t)two[1] << 32 | two[0]) > key;
    rank += ((uint64_t)two[3] << 32 | two[2]) > key;
  }
  return rank;
}

struct TopShared {
  float most[kThreads];
  int list[kThreads], counts[kWaves];
  int found, bound;
  float threshold;
  __align__(16) uint64_t keys[kCandidates + 2];
  uint64_t best[kWaves];
};

// The `top` largest keys of a block's logits [c0, c1) of a row, each handed to out(j, key) once (key
// 0 where there is none). `most` is the thread's largest logit (-inf: none) and `seen` the
// column of the chunk that first held it; chunk i of thread t lies at begin + (i kThreads + t) 8,
// and a thread may hold columns outside of them (`edge` on, `edges` of them: thread t has
// edge + t).
//
// At least `top` threads have a largest of at least the top-th largest among the threads' largest, so
// the logits from this threshold on hold the answer, and hardly more than it: those of the few
// threads that reach it are read again, by the whole block. Of logits equal to the
// threshold only columns up to a bound count, that of the first `top` threads that hold it, so that rows of equal
// logits give few candidates too. The candidates' ranks among each other are their places. Where
// they are too many after all, `top` rounds over the row find the answer.
template <typename T, typename F>
__device__ __forceinline__ void block_top(const T* l, int top, int begin, int chunks, int edge0, int edges0, int edge1, int edges1,
                                          int c0, int c1, float most, int seen, TopShared& sh, const F& out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  sh.most[tid] = most;
  if (tid == 0) {
    sh.found = 0;
    sh.bound = -1;
  }
  __syncthreads();
  if (wave == 0) {
    float v[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v[w] = sh.most[w * 64 + lane];
    float best = INFINITY;
    for (int j = 0; j < top && best > -INFINITY; ++j) {
      float own = v[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) own = fmaxf(own, v[w]);
      best = wave_max(own);
      if (lane == __ffsll((unsigned long long)__ballot(own == best)) - 1) {
        bool gone = false;  // one of them
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const bool here = !gone && v[w] == best;
          v[w] = here ? -INFINITY : v[w];
          gone = gone || here;
        }
      }
    }
    if (lane == 0) sh.threshold = best;
  }
  __syncthreads();
  const float threshold = sh.threshold;  // -inf: fewer than `top` threads hold any
  int total, reach;
  const int order = block_place(most == threshold && most > -INFINITY, sh.counts, total);
  if (most == threshold && most > -INFINITY && order < top) atomicMax(&sh.bound, seen + kChunk - 1);
  const int place = block_place(most >= threshold && most > -INFINITY, sh.counts, reach);
  if (most >= threshold && most > -INFINITY) sh.list[place] = tid;
  __syncthreads();
  const int bound = total >= top ? sh.bound : c1;
  const auto offer = [&](float v, int c) {
    if ((v > threshold || (v == threshold && c <= bound)) && v > -INFINITY) {
      const int at = atomicAdd(&sh.found, 1);
      if (at < kCandidates) sh.keys[at] = top_key(v, c);
    }
  };
  const int turns = (chunks + kThreads - 1) / kThreads;
  for (int p = tid; p < reach * turns; p += kThreads) {
    const int i = p / reach, t = sh.list[p - i * reach], q = i * kThreads + t;
    if (q >= chunks) continue;
    float f[kChunk];
    load8(l + begin + q * kChunk, (int64_t)kChunk, f);
#pragma unroll
    for (int e = 0; e < kChunk; ++e) offer(f[e], begin + q * kChunk + e);
  }
  if (tid < edges0) offer((float)l[edge0 + tid], edge0 + tid);
  if (tid < edges1) offer((float)l[edge1 + tid], edge1 + tid);
  __syncthreads();
  const int found = sh.found;
  if (found <= kCandidates) {
    if (found & 1) {
      if (tid == 0) sh.keys[found] = 0;
      __syncthreads();
    }
    for (int i = tid; i < found; i += kThreads) {
      const uint64_t key = sh.keys[i];
      const int rank = rank_among(sh.keys, found, key);
      if (rank < top) out(rank, key);
    }
    for (int j = found + tid; j < top; j += kThreads) out(j, 0);
    __syncthreads();
    return;
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < top; ++j) {
    uint64_t mine = 0;
    for (int c = c0 + tid; c < c1; c += kThreads) {
      const uint64_t k = top_key((float)l[c], c);
      mine = k < last && k > mine ? k : mine;
    }
    mine = wave_max64(mine);
    __syncthreads();
    if (lane == 0) sh.best[wave] = mine;
    __syncthreads();
    last = sh.best[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) last = sh.best[w] > last ? sh.best[w] : last;
    if (tid == 0) out(j, last);
  }
  __syncthreads();
}

__device__ __forceinline__ RowSum block_sums(RowSum r, RowSum* sums) {
  const float m = wave_max(r.m);
  raise(r, m);
  r = {m, lanes_sum<64>(r.n), lanes_sum<64>(r.s), lanes_sum<64>(r.a)};
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = r;
  __syncthreads();
  r = sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = merged(r, sums[w]);
  return r;
}

// The parts of a row: their sums and largest keys, for k_logprobs_join.
__device__ __forceinline__ RowSum* part_sums(const LogpArgs& a, int64_t row) { return (RowSum*)a.ws + row * a.parts; }
__device__ __forceinline__ uint64_t* part_keys(const LogpArgs& a, int64_t row) {
  return (uint64_t*)(a.ws + a.keys_off) + row * a.parts * a.top;
}

template <typename T>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 6 : 1) void k_logprobs_block(LogpArgs a) {
  __shared__ RowSum sums[kWaves];
  __shared__ TopShared sh;
  const int tid = threadIdx.x, part = blockIdx.y;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* l = (const T*)a.logits + row * a.ld;
    const int c0 = part * a.part_len, c1 = a.classes - c0 < a.part_len ? a.classes : c0 + a.part_len;
    // chunks at 16-byte addresses (unaligned ones cost up to half of the bandwidth); what lies before
    // and after them goes one by one to the first threads
    const int off = (int)(((uintptr_t)(l + c0) & 15) / sizeof(T)), per16 = 16 / (int)sizeof(T);
    int head = off ? per16 - off : 0;
    if (head > c1 - c0) head = c1 - c0;
    const int begin = c0 + head, chunks = (c1 - begin) / kChunk, tail = begin + chunks * kChunk;
    // r.m is the wave's: a chunk of the wave with nothing as large, all but a few, needs no comparison
    // with it and no rescaling (4000 rows of 50001 classes in bf16: 98 -> 84 us)
    RowSum r = empty_sum();
    float edge = -INFINITY, edge2 = -INFINITY;
    if (tid < head) edge = (float)l[c0 + tid];
    if (tid < c1 - tail) edge2 = (float)l[tail + tid];
    int seen = 0;
    float most = -INFINITY;
    const T* p = l + begin;
    constexpr int kAhead = 2;  // chunks on their way
    typename RawOf<T>::type raw[kAhead];
    const auto fetch = [&](int q, typename RawOf<T>::type& to) {
      if (q < chunks) to = *(const typename RawOf<T>::type*)__builtin_assume_aligned(p + (int64_t)q * kChunk, 16);
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) fetch(u * kThreads + tid, raw[u]);
    for (int q0 = 0; q0 < chunks; q0 += kAhead * kThreads)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int q = q0 + u * kThreads + tid;
      if (q0 + u * kThreads >= chunks) break;
      float v[kChunk];
      unpack8(raw[u], v);
      if (q >= chunks) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) v[i] = -INFINITY;
      }
      fetch(q + kAhead * kThreads, raw[u]);
      float top = v[0];
#pragma unroll
      for (int i = 1; i < kChunk; ++i) top = fmaxf(top, v[i]);
      if (__any(top >= r.m)) {
        raise(r, wave_max(fmaxf(top, r.m)));
        add_logits(r, v);
      } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          const float d = v[i] - r.m, e = exp_of(d);
          r.s += e;
          r.a = fmaf(e, fmaxf(d, kFar), r.a);
        }
      }
      seen = top > most ? begin + q * kChunk : seen;
      most = fmaxf(most, top);
    }
    {
      const float v[2] = {edge, edge2};
      add_logits(r, v);
    }
    r = block_sums(r, sums);
    if (a.parts > 1) {
      if (tid == 0) part_sums(a, row)[part] = r;
      if (a.top) {
        uint64_t* keys = part_keys(a, row) + part * a.top;
        block_top(l, a.top, begin, chunks, c0, head, tail, c1 - tail, c0, c1, most, seen, sh,
                  [&](int j, uint64_t key) { keys[j] = key; });
      }
    } else {
      const RowResult q = row_result(r);
      if (tid == 0) write_row(a, row, q);
      if (a.top)
        block_top(l, a.top, begin, chunks, c0, head, tail, c1 - tail, c0, c1, most, seen, sh,
                  [&](int j, uint64_t key) { write_top(a, row, j, key, q); });
    }
    __syncthreads();
  }
}

// A row's result from its parts. Their keys lie in falling order; with c = ceil(top / parts)
// and n = ceil(top / c), n parts have c keys each from the n-th largest of the parts' c-th keys
// on, top in all: keys below it are not among the likeliest.
__global__ __launch_bounds__(kThreads) void k_logprobs_join(LogpArgs a) {
  __shared__ __align__(16) uint64_t keys[kMaxParts * kLogpMaxTop + 2], cth[kMaxParts];
  __shared__ RowSum sums;
  __shared__ uint64_t floor;
  __shared__ int found;
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint64_t* from = part_keys(a, row);
    const int c = a.top ? (a.top + a.parts - 1) / a.parts : 1, n = (a.top + c - 1) / c;
    uint64_t mine = 0;
    if (tid < 64) {
      RowSum r = tid < a.parts ? part_sums(a, row)[tid] : empty_sum();
      if (a.top && tid < kMaxParts) cth[tid] = mine = tid < a.parts ? from[tid * a.top + c - 1] : 0;
      const float m = wave_max(r.m);
      raise(r, m);
      r = {m, lanes_sum<64>(r.n), lanes_sum<64>(r.s), lanes_sum<64>(r.a)};
      if (tid == 0) {
        sums = r;
        found = 0;
        floor = 1;  // keys of 0 are none
      }
    }
    __syncthreads();
    const RowResult q = row_result(sums);
    if (tid == 0) write_row(a, row, q);
    if (a.top) {
      if (mine && rank_among(cth, kMaxParts, mine) == n - 1) floor = mine;
      __syncthreads();
      for (int i = tid; i < a.parts * a.top; i += kThreads) {
        const uint64_t k = from[i];
        if (k >= floor) keys[atomicAdd(&found, 1)] = k;
      }
      __syncthreads();
      const int count = found;
      if (tid == 0) keys[count] = 0;
      __syncthreads();
      for (int i = tid; i < count; i += kThreads) {
        const uint64_t key = keys[i];
        const int rank = rank_among(keys, count, key);
        if (rank < a.top) write_top(a, row, rank, key, q);
      }
      for (int j = count + tid; j < a.top; j += kThreads) write_top(a, row, j, 0, q);
    }
    __syncthreads();
  }
}

// ---- gradient ------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprobs_backward(LogpArgs a) {
  const int64_t chunks = ((int64_t)a.classes + kChunk - 1) / kChunk;
  for (int64_t row = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row < a.rows; row += (int64_t)gridDim.y * blockDim.y) {
    const float m = a.stats[row * 3], logs = a.stats[row * 3 + 1], H = a.stats[row * 3 + 2];
    const int64_t t = a.targets[row];
    // a row without any class has no gradient
    const bool has = t >= 0 && t < a.classes && logs != INFINITY;
    const float g = has && a.dlogp ? a.dlogp[row] : 0.0f, dH = a.dentropy ? a.dentropy[row] : 0.0f;
    const T* l = (const T*)a.logits + row * a.ld;
    T* out = (T*)a.dlogits + row * (int64_t)a.classes;
    for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < chunks; c += (int64_t)gridDim.x * blockDim.x) {
      float v[kChunk];
      const int64_t at = c * kChunk, left = a.classes - at;
      load8(l + at, left, v);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const float lp = (v[i] - m) - logs, p = prob_of(lp, T());
        v[i] = -p * fmaf(dH, fmaxf(lp, kFar) + H, g);
        // 1 - p without its cancellation near p = 1
        if (has && at + i == t) v[i] = -fmaf(p * dH, fmaxf(lp, kFar) + H, g * expm1f(lp));
      }
      store8(out + at, left, v);
    }
  }
}


// Parts of a row: one where rows fill the chip, else as many as leave kPartMin logits each
// or two blocks a CU.
void logprobs_plan(LogpArgs& a) {
  a.parts = 1;
  if (a.classes > kTeamMaxClasses && a.rows < 2 * kNumCUs) {
    int64_t parts = ceil_div(a.classes, kPartMin);
    if (parts > ceil_div(2 * kNumCUs, a.rows)) parts = ceil_div(2 * kNumCUs, a.rows);
    a.parts = (int)(parts < kMaxParts ? parts : kMaxParts);
  }
  // whole chunks, so that parts begin at one alignment
  a.part_len = (int)round_up(ceil_div(a.classes, a.parts), kChunk);
  a.parts = (int)ceil_div(a.classes, a.part_len);
  a.keys_off = align256((size_t)a.rows * a.parts * sizeof(RowSum));
}

template <typename T>
void forward_typed(const LogpArgs& a, hipStream_t st) {
  if (a.classes <= kTeamMaxClasses) {
#define CKAN_LOGP_TEAM(L, NN)                                                                                       \
  if (a.classes <= L * NN * kChunk) {                                                                               \
    const int64_t blocks = ceil_div(a.rows, kThreads / L);                                                          \
    hipLaunchKernelGGL((k_logprobs_team<T, L, NN>), dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)),         \
                       dim3(kThreads), 0, st, a);                                                                   \
    return;                                                                                                         \
  }
    CKAN_LOGP_TEAM(8, 1) CKAN_LOGP_TEAM(16, 1) CKAN_LOGP_TEAM(32, 1) CKAN_LOGP_TEAM(64, 1) CKAN_LOGP_TEAM(64, 2)
    CKAN_LOGP_TEAM(64, 4) CKAN_LOGP_TEAM(64, 8)
#undef CKAN_LOGP_TEAM
  }
  const unsigned rows = (unsigned)(a.rows < (1 << 20) ? a.rows : 1 << 20);
  hipLaunchKernelGGL((k_logprobs_block<T>), dim3(rows, (unsigned)a.parts), dim3(kThreads), 0, st, a);
  if (a.parts > 1) hipLaunchKernelGGL(k_logprobs_join, dim3(rows), dim3(kThreads), 0, st, a);
}

}  // namespace

size_t logprobs_workspace_bytes(const LogpArgs& a) {
  LogpArgs b = a;
  logprobs_plan(b);
  return b.parts > 1 ? align256(b.keys_off + (size_t)b.rows * b.parts * b.top * sizeof(uint64_t)) : 0;
}

void launch_logprobs(const LogpArgs& args, hipStream_t st) {
  LogpArgs a = args;
  logprobs_plan(a);
  if (a.bf16)
    forward_typed<__bf16>(a, st);
  else
    forward_typed<float>(a, st);
}

void launch_logprobs_backward(const LogpArgs& a, hipStream_t st) {
  const int64_t chunks = ceil_div(a.classes, kChunk);
  int lanes = kThreads;
  while (lanes > 1 && lanes / 2 >= chunks) lanes /= 2;
  const dim3 block(lanes, kThreads / lanes);
  const int64_t gx = ceil_div(chunks, lanes), gy = ceil_div(a.rows, block.y);
  const dim3 grid((unsigned)(gx < 4096 ? gx : 4096), (unsigned)(gy < 65535 ? gy : 65535));
  if (a.bf16)
    hipLaunchKernelGGL((k_logprobs_backward<__bf16>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((k_logprobs_backward<float>), grid, block, 0, st, a);
}

}  // namespace ckan
