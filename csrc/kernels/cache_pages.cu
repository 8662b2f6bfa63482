// cache_pages.cu - moving what a paged cache holds: copies of whole pages
// (fork, defragment) and the accepted path of a drafted tree.  Both move bytes
// and are bound by memory; every layer's K and V go in one launch.
#include <cuda_runtime.h>

#include <cstdint>

#include "paged.h"

namespace rab {

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kCopyChunk = kCopyThreads * kCopyUnroll * 16;  // bytes of one block

// grid: (chunks of a page, pairs, layers * {K, V}).  The pairs travel in the
// kernel's parameters, so a launch needs no copy of the lists to the GPU first.
__global__ void __launch_bounds__(kCopyThreads)
    page_copy_kernel(const __grid_constant__ PageCopyParams p) {
  const int pair = blockIdx.y;
  const int layer = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  uint8_t* base = is_v ? p.v + layer * p.v_layer : p.k + layer * p.k_layer;
  const int64_t page = is_v ? p.v_page : p.k_page;
  const uint4* src = reinterpret_cast<const uint4*>(base + p.src[pair] * page);
  uint4* dst = reinterpret_cast<uint4*>(base + p.dst[pair] * page);
  const int64_t n = p.page_bytes >> 4;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  uint4 x[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (i0 + u * kCopyThreads < n) x[u] = __ldcs(src + i0 + u * kCopyThreads);
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (i0 + u * kCopyThreads < n) dst[i0 + u * kCopyThreads] = x[u];
}

constexpr int kPathThreads = 128;
constexpr int kPathBatch = 8;

// grid: (request, layer * {K, V}).  A thread owns 16-byte columns of a token's
// [heads, dim] row and walks the path in order.  Places increase, so what step
// i writes (place i) lies before every place a later step reads (path[j] >= j
// > i): the walk is safe in place without a second buffer.
__global__ void __launch_bounds__(kPathThreads) path_kernel(const __grid_constant__ PathParams p) {
  const int b = blockIdx.x;
  const int layer = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  const int n = p.path_lens[b];
  if (n <= 0) return;
  const int64_t ctx = p.ctx[b];
  const int* path = p.path + b * p.path_stride;
  const int* table = p.table + b * p.table_stride;
  const int64_t last = static_cast<int64_t>(p.table_w) * p.page_size;
  __shared__ int bad;
  if (threadIdx.x == 0) bad = n > p.path_w || ctx < 0 ? 1 : 0;
  __syncthreads();
  // the whole path is checked before anything moves
  if (!bad) {
    for (int i = threadIdx.x; i < n; i += kPathThreads) {
      const int64_t at = path[i];
      if (at < i || (i > 0 && at <= path[i - 1]) || ctx + at >= last) {
        bad = 1;
      } else {
        const int s = table[(ctx + at) / p.page_size], d = table[(ctx + i) / p.page_size];
        if (s < 0 || s >= p.num_pages || d < 0 || d >= p.num_pages) bad = 2;
      }
    }
  }
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0 && blockIdx.y == 0)
      st_record(p.status, kStatusBadArgs, bad == 1 ? kBadPath : kBadPage, b);
    return;
  }
  uint8_t* base = is_v ? p.v + layer * p.v_layer : p.k + layer * p.k_layer;
  const int64_t page = is_v ? p.v_page : p.k_page;
  const int64_t head_bytes = static_cast<int64_t>(p.page_size) * p.row_bytes;
  const int per_row = p.row_bytes >> 4;
  for (int c = threadIdx.x; c < p.heads * per_row; c += kPathThreads) {
    uint8_t* col = base + (c / per_row) * head_bytes + (c % per_row) * 16;
    auto place = [&](int64_t at) {
      const int64_t e = at / p.page_size;
      return col + table[e] * page + (at - e * p.page_size) * p.row_bytes;
    };
    for (int i = 0; i < n; i += kPathBatch) {
      uint4 x[kPathBatch];
#pragma unroll
      for (int u = 0; u < kPathBatch; ++u)
        if (i + u < n && path[i + u] != i + u)
          x[u] = *reinterpret_cast<const uint4*>(place(ctx + path[i + u]));
#pragma unroll
      for (int u = 0; u < kPathBatch; ++u)
        if (i + u < n && path[i + u] != i + u) *reinterpret_cast<uint4*>(place(ctx + i + u)) = x[u];
    }
  }
}

}  // namespace

int page_copy_launch(const PageCopyParams& p, cudaStream_t stream) {
  if (p.n == 0 || p.layers == 0 || p.page_bytes == 0) return 0;
  const dim3 grid(static_cast<unsigned>((p.page_bytes + kCopyChunk - 1) / kCopyChunk), p.n,
                  2 * p.layers);
  page_copy_kernel<<<grid, kCopyThreads, 0, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

int path_compact_launch(const PathParams& p, cudaStream_t stream) {
  if (p.batch == 0 || p.layers == 0 || p.path_w == 0) return 0;
  path_kernel<<<dim3(p.batch, 2 * p.layers), kPathThreads, 0, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace rab
