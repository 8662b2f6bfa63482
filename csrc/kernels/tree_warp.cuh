// tree_warp.cuh - frame of the paged-attention kernels whose warps do a tile's
// products with mma.sync and keep scores, weights and outputs in registers:
// tree_f32.cu (fp32) and tree_few.cu (bf16 and fp16, few rows).
//
// Warp 8 walks the pieces of the CTA's share (tree_sched.cuh) and brings tiles of K and
// V by TMA into a ring; warps 0-7 take shares of a tile's keys, with kSplit = 2 of half
// the unit's rows each, and their results are joined at a piece's end.  A kernel's
// configuration C says: kD, kBytes (of an element), kRows, kTile (keys), kStages, kHalf
// and kStage (bytes of K, of K and V), kSplit, kGroups (of eight rows, a warp's), kOwn
// and kOwnRow (floats of a warp's outputs, between two rows), and where each part of
// shared memory lies.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.h"
#include "paged.h"
#include "sm100.cuh"
#include "tree_sched.cuh"

namespace rab {
namespace tree_detail {

constexpr int kWarps = 8;  // that compute
constexpr int kItems = 4;  // queue of pieces
constexpr float kLn2f = 0.69314718055994530942f;

template <typename T>
__device__ __forceinline__ T cast_out(float x);
template <>
__device__ __forceinline__ float cast_out<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 cast_out<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half cast_out<__half>(float x) {
  return __float2half_rn(x);
}

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }

__device__ __forceinline__ void store4(float* to, const float4& o) {
  *reinterpret_cast<float4*>(to) = o;
}
template <typename T>
__device__ __forceinline__ void store4(T* to, const float4& o) {
  alignas(8) T v[4] = {cast_out<T>(o.x), cast_out<T>(o.y), cast_out<T>(o.z), cast_out<T>(o.w)};
  *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(v);
}

// Columns [k0, k1) of a result that this thread has just written take what was left
// out of V among the new tokens of the piece, for the keys that token t sees.
template <typename T>
__device__ __noinline__ void add_left_out(const TreeParams& p, const Piece& c, int t, int tile,
                                          int k0, int k1, int dim, float* rec, T* dst) {
  const int* table = p.table + static_cast<int64_t>(c.request) * p.table_stride;
  const int lo = max(c.ctx, c.tile_begin * tile), hi = min(c.keys, c.tile_end * tile);
  for (int key = lo; key < hi; ++key) {
    const int rel = key - c.ctx;
    const bool sees =
        p.mask == nullptr
            ? rel <= t
            : (rel >> 5) < p.mask_w &&
                  ((p.mask[static_cast<int64_t>(c.first + t) * p.mask_stride + (rel >> 5)] >>
                    (rel & 31)) &
                   1u);
    const int page = table[key >> p.page_shift];
    if (!sees || page < 0 || page >= p.num_pages) continue;
    const T* src = static_cast<const T*>(p.v) + page * p.v_page +
                       (static_cast<int64_t>(c.head_kv) * p.page_size + (key & (p.page_size - 1))) * dim;
    for (int k = k0; k < k1; ++k) {
      const float v = as_float(src[k]);
      if (isfinite(v)) continue;
      if (rec != nullptr) rec[(k & ~3) * c.rows + (k & 3)] += v;
      else dst[k] = cast_out<T>(as_float(dst[k]) + v);
    }
  }
}

// the barriers and the queue of a block
template <typename C>
struct WarpBlock {
  uint8_t* smem;
  __device__ __forceinline__ uint64_t* bars() const {
    return reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  }
  __device__ __forceinline__ uint64_t* full(int i) const { return bars() + i; }
  __device__ __forceinline__ uint64_t* empty(int i) const { return bars() + C::kStages + i; }
  __device__ __forceinline__ uint64_t* item_full(int w) const {
    return bars() + 2 * C::kStages + w % kItems;
  }
  __device__ __forceinline__ uint64_t* item_empty(int w) const {
    return item_full(w) + kItems;
  }
  __device__ __forceinline__ uint64_t* joined() const {
    return bars() + 2 * C::kStages + 2 * kItems;
  }
  __device__ __forceinline__ uint64_t* released() const { return joined() + 1; }
  __device__ __forceinline__ Piece* item(int w) const {
    return reinterpret_cast<Piece*>(smem + C::kItemOff + (w % kItems) * 48);
  }
  // [2], by the piece's parity
  __device__ __forceinline__ volatile int* dirty() const {
    return reinterpret_cast<int*>(smem + C::kDirtyOff);
  }
  __device__ __forceinline__ float* own(int warp) const {
    return reinterpret_cast<float*>(smem + C::kOwnOff) + warp * C::kOwn;
  }
  // maximum and sum of row r of warp u
  __device__ __forceinline__ float2& ml(int u, int r) const {
    return reinterpret_cast<float2*>(smem + C::kMlOff)[u * (C::kGroups * 8) + r];
  }
};

// Every thread of the block, first of all: false when the block cannot work.
template <typename C>
__device__ __forceinline__ bool start_block(const TreeParams& p, const WarpBlock<C>& blk) {
  using namespace sm100;
  if ((smem_u32(blk.smem) & 1023u) != 0) {  // the swizzle counts from 1024-byte boundaries
    wait_for_predecessor();
    if (threadIdx.x == 0) {
      p.meta[blockIdx.x * kMetaInts] = 0;
      st_record(p.status, kStatusBadArgs, kSiteNone);
    }
    return false;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(blk.full(i), 1);
      mbar_init(blk.empty(i), kWarps);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(blk.item_full(i), 1);
      mbar_init(blk.item_empty(i), kWarps);
    }
    mbar_init(blk.joined(), kWarps);
    mbar_init(blk.released(), kWarps);
    blk.dirty()[0] = blk.dirty()[1] = 0;
    fence_barrier_init();
  }
  let_successor_start();
  __syncthreads();
  wait_for_predecessor();
  return true;
}

// One warp: walks the pieces and loads their tiles.
template <typename C>
__device__ __forceinline__ void walk_and_load(const TreeParams& p, const CUtensorMap& tmK,
                                              const CUtensorMap& tmV, const WarpBlock<C>& blk) {
  using namespace sm100;
  constexpr int kTile = C::kTile, kRows = C::kRows;
  constexpr int kSegCols = 128 / C::kBytes, kSegs = C::kD / kSegCols;  // 128 bytes of columns
  const int lane = lane_id();
  DeviceStatus* st = p.status;
  const uint64_t tmo = p.timeout_ns;
  if (lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  Range range;
  Start first;
  const int walker = find_range<kTile, kRows>(p, &range, &first);
  Walk<kTile, kRows> walk;
  if (lane == walker) {
    p.meta[blockIdx.x * kMetaInts] = 0;  // by the lane that may set it later
    walk.start(p, range, first);
  }
  const int rows_box = min(p.page_size, kTile);
  const int boxes = kTile / rows_box * kSegs;
  int n = 0;  // tiles loaded
  bool ok = true;
  for (int w = 0; ok; ++w) {
    if (w >= kItems)
      ok = __all_sync(0xffffffffu, mbar_wait(blk.item_empty(w),
                                             (w / kItems - 1) & 1, st, kSiteItemQueue, tmo));
    if (!ok) break;
    Piece* slot = blk.item(w);
    if (lane == walker) {
      Piece c;
      if (walk.next(p, range, &c)) {
        if (walk.merges) write_meta(p, c, true, walk.merge_c0);
      } else {
        c.request = -1;
      }
      *slot = c;
    }
    __syncwarp();
    const Piece c = *slot;
    if (lane == 0) mbar_arrive(blk.item_full(w));
    if (c.request < 0) break;
    const int* table = p.table + static_cast<int64_t>(c.request) * p.table_stride;
    const int last_entry = (c.keys - 1) >> p.page_shift;
    for (int tile = c.tile_begin; tile < c.tile_end; ++tile) {
      // this lane's box: page, rows within the tile, 128-byte segment
      const int seg = lane % kSegs, part = lane / kSegs;
      int page = p.num_pages, token = 0;
      if (lane < boxes) {
        const int key = tile * kTile + part * rows_box;
        const int entry = key >> p.page_shift;
        token = key & (p.page_size - 1);
        if (entry <= last_entry) {  // behind it: a coordinate past the pool loads zeros
          page = table[entry];
          if (page < 0 || page >= p.num_pages) {
            if (seg == 0) st_record(st, kStatusBadArgs, kBadPage, static_cast<uint32_t>(page));
            page = p.num_pages;
          }
        }
      }
      const int stage = n % C::kStages;
      ok = __all_sync(0xffffffffu, mbar_wait(blk.empty(stage), ((n / C::kStages) & 1) ^ 1, st,
                                             kSiteKEmpty, tmo));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(blk.full(stage), C::kStage);
      __syncwarp();
      if (lane < boxes) {
        uint8_t* dst = blk.smem + stage * C::kStage + seg * (kTile * 128) + part * rows_box * 128;
        tma_load_4d(dst, &tmK, blk.full(stage), seg * kSegCols, token, c.head_kv, page);
        tma_load_4d(dst + C::kHalf, &tmV, blk.full(stage), seg * kSegCols, token, c.head_kv, page);
      }
      ++n;
    }
  }
  // the loads in flight land before the block gives its memory back
  for (int i = 0; i < C::kStages && i < n; ++i) {
    const int k = n - 1 - i;
    mbar_wait(blk.full(k % C::kStages), (k / C::kStages) & 1, nullptr, kSiteKFull, 100000000ull);
  }
}

// A computing warp's share of a piece's results, from the outputs, maxima and sums that
// the warps have left in shared memory.
template <typename C, typename T>
__device__ __forceinline__ void write_results(const TreeParams& p, const WarpBlock<C>& blk,
                                              const Piece& c, int w) {
  using namespace sm100;
  constexpr int D = C::kD, kRows = C::kRows, kKeyWarps = kWarps / C::kSplit;
  const int warp = warp_id(), lane = lane_id();
  // four columns of a row at a time
  for (int x = warp * 32 + lane; x < c.rows * (D / 4); x += kWarps * 32) {
    const int r = x / (D / 4), x4 = x % (D / 4);
    const int u0 = r / (8 * C::kGroups) * kKeyWarps, r_w = r % (8 * C::kGroups);
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kKeyWarps; ++u) top = fmaxf(top, blk.ml(u0 + u, r_w).x);
    const float use = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < kKeyWarps; ++u) {
      const float2 ml = blk.ml(u0 + u, r_w);
      const float f = ex2_approx(ml.x - use);
      const float4 a =
          *reinterpret_cast<const float4*>(blk.own(u0 + u) + r_w * C::kOwnRow + x4 * 4);
      sum += f * ml.y;
      o.x += f * a.x;
      o.y += f * a.y;
      o.z += f * a.z;
      o.w += f * a.w;
    }
    const int row = c.row0 + r, tok = row / p.group;
    const int h = c.head_kv * p.group + row - tok * p.group;
    const float inv = c.record >= 0 ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);
    // a record is [dim / 4][rows][4], the rows of the unit side by side
    float* rec = c.record >= 0
                     ? p.rec_acc + static_cast<int64_t>(c.record) * (kRows * D) + r * 4
                     : nullptr;
    T* out = static_cast<T*>(p.out) + static_cast<int64_t>(c.first + tok) * p.out_t +
                 static_cast<int64_t>(h) * p.out_h;
    o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (rec != nullptr) *reinterpret_cast<float4*>(rec + x4 * 4 * c.rows) = o;
    else store4(out + x4 * 4, o);
    if (blk.dirty()[w & 1] == w + 1)
      add_left_out<T>(p, c, tok, C::kTile, x4 * 4, x4 * 4 + 4, D, rec, out);
    if (x4 == 0) {
      if (c.record >= 0) {
        p.rec_m[c.record * kRows + r] = top;
        p.rec_l[c.record * kRows + r] = sum;
      } else if (p.lse != nullptr) {
        p.lse[static_cast<int64_t>(c.first + tok) * p.heads + h] =
            sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2f;
      }
    }
  }
}

// launches a kernel of this frame; its shared memory is allowed once per device
template <typename C, typename Kernel>
int launch_warp_kernel(Kernel* kernel, bool (&done)[64], const TreeParams& p, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t err =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (err != cudaSuccess) return static_cast<int>(err);
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  const CUtensorMap k = pool_map(p, p.k, p.k_page, C::kBytes, C::kTile);
  const CUtensorMap v = pool_map(p, p.v, p.v_page, C::kBytes, C::kTile);
  return launch_overlapped(kernel, dim3(p.grid), C::kThreads, C::kSmem, stream, &p, &k, &v);
}

}  // namespace tree_detail
}  // namespace rab
