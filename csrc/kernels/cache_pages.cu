// cache_pages.cu - moving what a paged cache holds: copies of whole pages
// (fork, defragment) and the accepted path of a drafted tree.  Both move bytes
// and are bound by memory; every layer's K and V go in one launch.
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.h"
#include "paged.h"

namespace rab {

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kCopyChunk = kCopyThreads * kCopyUnroll * 16;  // bytes of one block

// grid: (chunks of a page, source pages, layers * {K, V}).  The pairs travel in
// the kernel's parameters, so a launch needs no copy of the lists to the GPU
// first, and are grouped by source: a page that goes to several places is read once.
template <int kPairs>
__global__ void __launch_bounds__(kCopyThreads)
    page_copy_kernel(const __grid_constant__ PageCopyParams<kPairs> p) {
  const int s = blockIdx.y;
  const int layer = blockIdx.z >> 1;
  const bool is_v = blockIdx.z & 1;
  uint8_t* base = is_v ? p.v + layer * p.v_layer : p.k + layer * p.k_layer;
  const int64_t page = is_v ? p.v_page : p.k_page;
  const int64_t n = p.page_bytes >> 4;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  const uint4* src = reinterpret_cast<const uint4*>(base + p.src[s] * page) + i0;
  uint4 x[kCopyUnroll];
  let_successor_start();
  wait_for_predecessor();
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (i0 + u * kCopyThreads < n) x[u] = __ldcs(src + u * kCopyThreads);
  for (int j = p.first[s]; j < p.first[s + 1]; ++j) {
    uint4* dst = reinterpret_cast<uint4*>(base + p.dst[j] * page) + i0;
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
      if (i0 + u * kCopyThreads < n) dst[u * kCopyThreads] = x[u];
  }
}

constexpr int kPathThreads = 128;
constexpr int kPathBatch = 8;
constexpr int kPathSteps = 64;  // steps whose places a block holds at a time

// grid: (request, layer * {K, V}).  A thread owns 16-byte columns of a token's
// [heads, dim] row and walks the path in order.  Places increase, so what step
// i writes (place i) lies before every place a later step reads (path[j] >= j
// > i): the walk is safe in place without a second buffer.  The steps' byte
// offsets are formed once per block, eight loads are in flight per thread.  Bound
// by DRAM at its grain: a token's row of one head is 128 to 512 bytes alone in its
// page.  128 paths of 9 in 64 tokens, 16 layers of 8 heads x 128 fp16: 24.7 us, 117
// MB at 4.8 TB/s; two to nine loads in flight, 64 to 256 threads and twice the
// blocks per SM all measured 25 to 29 us.
__global__ void __launch_bounds__(kPathThreads) path_kernel(const __grid_constant__ PathParams p) {
  __shared__ int64_t s_from[kPathSteps], s_to[kPathSteps];
  __shared__ int s_bad;
  const int b = blockIdx.x;
  const int layer = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  let_successor_start();
  wait_for_predecessor();
  const int n = p.path_lens[b];
  if (n <= 0) return;
  const int ctx = p.ctx[b];
  const int* path = p.path + b * p.path_stride;
  const int* table = p.table + b * p.table_stride;
  const int64_t last = static_cast<int64_t>(p.table_w) * p.page_size;
  const int64_t page_stride = is_v ? p.v_page : p.k_page;
  if (threadIdx.x == 0) s_bad = n > p.path_w || ctx < 0 ? kBadPath : 0;
  __syncthreads();
  // the whole path is checked before anything moves
  if (s_bad == 0) {
    for (int i = threadIdx.x; i < n; i += kPathThreads) {
      const int at = path[i];
      if (at < i || (i > 0 && at <= path[i - 1]) || static_cast<int64_t>(ctx) + at >= last) {
        s_bad = kBadPath;
      } else {
        const uint32_t page = p.page_size;
        const int s = table[(static_cast<uint32_t>(ctx) + at) / page];
        const int d = table[(static_cast<uint32_t>(ctx) + i) / page];
        if (s < 0 || s >= p.num_pages || d < 0 || d >= p.num_pages) s_bad = kBadPage;
      }
    }
  }
  __syncthreads();
  if (s_bad != 0) {
    if (threadIdx.x == 0 && blockIdx.y == 0) st_record(p.status, kStatusBadArgs, s_bad, b);
    return;
  }
  uint8_t* base = is_v ? p.v + layer * p.v_layer : p.k + layer * p.k_layer;
  const int64_t head_bytes = static_cast<int64_t>(p.page_size) * p.row_bytes;
  const int per_row = p.row_bytes >> 4;
  for (int i0 = 0; i0 < n; i0 += kPathSteps) {
    const int steps = min(n - i0, kPathSteps);
    if (i0 > 0) __syncthreads();
    for (int i = threadIdx.x; i < 2 * steps; i += kPathThreads) {
      const int step = i0 + (i >> 1);
      const uint32_t at = static_cast<uint32_t>(ctx) + ((i & 1) ? step : path[step]);
      const uint32_t e = at / static_cast<uint32_t>(p.page_size);
      const int64_t off = table[e] * page_stride +
                          static_cast<int64_t>(at - e * p.page_size) * p.row_bytes;
      ((i & 1) ? s_to : s_from)[i >> 1] = off;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.heads * per_row; c += kPathThreads) {
      const int head = c / per_row;
      uint8_t* col = base + head * head_bytes + (c - head * per_row) * 16;
      for (int i = 0; i < steps; i += kPathBatch) {
        uint4 x[kPathBatch];
#pragma unroll
        for (int u = 0; u < kPathBatch; ++u)
          if (i + u < steps && s_from[i + u] != s_to[i + u])
            x[u] = *reinterpret_cast<const uint4*>(col + s_from[i + u]);
#pragma unroll
        for (int u = 0; u < kPathBatch; ++u)
          if (i + u < steps && s_from[i + u] != s_to[i + u])
            *reinterpret_cast<uint4*>(col + s_to[i + u]) = x[u];
      }
    }
  }
}

template <int kPairs>
int copy_run(const PageCopyParams<kPairs>& p, cudaStream_t stream) {
  if (p.n_src == 0 || p.layers == 0 || p.page_bytes == 0) return 0;
  const dim3 grid(static_cast<unsigned>((p.page_bytes + kCopyChunk - 1) / kCopyChunk), p.n_src,
                  2 * p.layers);
  return launch_overlapped(page_copy_kernel<kPairs>, grid, kCopyThreads, 0, stream, &p);
}

}  // namespace

int page_copy_launch(const PageCopyParams<kFewPairs>& p, cudaStream_t stream) {
  return copy_run(p, stream);
}
int page_copy_launch(const PageCopyParams<kManyPairs>& p, cudaStream_t stream) {
  return copy_run(p, stream);
}

int path_compact_launch(const PathParams& p, cudaStream_t stream) {
  if (p.batch == 0 || p.layers == 0 || p.path_w == 0) return 0;
  return launch_overlapped(path_kernel, dim3(p.batch, 2 * p.layers), kPathThreads, 0, stream, &p);
}

}  // namespace rab
