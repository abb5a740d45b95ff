// Dropout from a counter-based generator (ckan_dropout): y = keep x / (1 - p).
//
// The mask is a function of seed, call, row and column (ckan_block.hpp) and never
// stored: the gradient is the same launch on dy.  Bound by the bytes: 65536 x 512 in bf16 25 to 27 us,
// 5.0 to 5.3 TB/s, the generator's 16 bits a value hidden behind them.
#include "ckan_block.hpp"

namespace ckan {
namespace {

// A thread takes one chunk of eight values a round; blockDim = (lanes of a row, rows).
template <typename T>
__global__ __launch_bounds__(256) void k_dropout(DropoutArgs a) {
  const DropKey key = drop_key(a.drop);
  const int64_t chunks = (a.dim + kChunk - 1) / kChunk;
  if (a.used && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && threadIdx.y == 0) {
    a.used[0] = a.drop.state ? a.drop.state[0] : (int64_t)a.drop.seed;
    a.used[1] = (int64_t)(((uint64_t)key.call1 << 32) | key.call0);
  }
  for (int64_t row = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row < a.rows; row += (int64_t)gridDim.y * blockDim.y) {
    const T* x = (const T*)a.x + row * a.ld;
    T* y = (T*)a.y + row * a.dim;
    for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < chunks; c += (int64_t)gridDim.x * blockDim.x) {
      float v[kChunk];
      load8(x + c * kChunk, a.dim - c * kChunk, v);
      const DropWords keep = drop_words(a.drop, key, (uint32_t)row, (uint32_t)c);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) v[i] = keep.kept(i, a.drop) ? v[i] * a.drop.scale : 0.0f;
      store8(y + c * kChunk, a.dim - c * kChunk, v);
    }
  }
}

}  // namespace

void launch_dropout(const DropoutArgs& a, hipStream_t st) {
  const int64_t chunks = ceil_div(a.dim, kChunk);
  int lanes = 256;
  while (lanes > 1 && lanes / 2 >= chunks) lanes /= 2;
  const dim3 block(lanes, 256 / lanes);
  const int64_t gy = ceil_div(a.rows, block.y), gx = ceil_div(chunks, lanes);
  const dim3 grid((unsigned)(gx < 65536 ? gx : 65536), (unsigned)(gy < 65535 ? gy : 65535));
  if (a.bf16)
    hipLaunchKernelGGL((k_dropout<__bf16>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((k_dropout<float>), grid, block, 0, st, a);
}

}  // namespace ckan
