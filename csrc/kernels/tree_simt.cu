// tree_simt.cu - attention of new tokens over a paged cache on the CUDA cores
// (fp32), the merge of split units for every element type, and the masks of
// drafted trees.
//
// Row (token t, head h) of a request with ctx cached tokens sees key j when
// j < ctx, or when j is new token j - ctx and the mask has that bit (without a
// mask: j - ctx <= t):
//   o = sum_j exp(s_j - m) v_j / l,  s_j = scale q . k_j,  l = sum_j exp(s_j - m)
// with the running maximum m and the sums in fp32.  A row that sees nothing
// gives 0 and lse = -inf.
//
// A CTA of four warps takes 8 rows of one kv head over its share of the keys
// (tree_sched.cuh).  64 keys of K and V at a time arrive by 16-byte asynchronous
// copies, one tile ahead of the arithmetic.  Each warp takes 16 of the keys: two
// halves of 16 lanes form the scores of four rows each, then the lanes turn to
// columns for the product with V.  Every warp keeps its own running maximum,
// sum and 8 x dim outputs in registers, so the tile needs no exchange between
// warps; they are joined once per piece.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "paged.h"
#include "sm100.cuh"
#include "tree_sched.cuh"

namespace rab {

using namespace tree_detail;

namespace {

constexpr int kSimtThreads = 128;
constexpr int kSimtTile = 64;
constexpr int kSimtRows = 8;
constexpr float kLn2f = 0.69314718055994530942f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;  // 0: the 16 bytes are zeroed, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}

__device__ __forceinline__ float4 ld4(const float* p) {
  return *reinterpret_cast<const float4*>(p);
}
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

template <int D>
struct SimtCfg {
  static constexpr int kKRow = D + 4;  // K rows shifted by 16 bytes: lanes of 8 keys hit all banks
  static constexpr int kKBytes = kSimtTile * kKRow * 4;
  static constexpr int kVBytes = kSimtTile * D * 4;
  static constexpr int kStage = kKBytes + kVBytes;
  static constexpr int kQRow = D + 4;
  static constexpr int kQBytes = kSimtRows * kQRow * 4;
  static constexpr int kPBytes = 4 * kSimtRows * 16 * 4;
  static constexpr int kJoinBytes = 4 * kSimtRows * D * 4;  // over the stages, once per piece
  static constexpr int kStages = 2 * kStage > kJoinBytes ? 2 * kStage : kJoinBytes;
  static constexpr int kSmem = kStages + kQBytes + kPBytes;
};

template <int D>
__global__ void __launch_bounds__(kSimtThreads)
    tree_simt_kernel(const __grid_constant__ TreeParams p) {
  using C = SimtCfg<D>;
  constexpr int kCols = D / 32;
  extern __shared__ __align__(16) uint8_t smem[];
  float* sQ = reinterpret_cast<float*>(smem + C::kStages);
  float* sP = reinterpret_cast<float*>(smem + C::kStages + C::kQBytes);
  float* sJoin = reinterpret_cast<float*>(smem);
  __shared__ int s_sums[kSimtThreads / 32];
  __shared__ Start s_start;
  __shared__ Piece s_piece;
  __shared__ int s_have, s_merges, s_c0;
  __shared__ float s_m[4][kSimtRows], s_l[4][kSimtRows], s_alpha[4][kSimtRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const Range range = find_range<kSimtTile, kSimtRows, kSimtThreads>(p, s_sums, &s_start);
  Walk<kSimtTile, kSimtRows> walk;
  if (tid == 0) {
    walk.start(p, range, s_start);
    p.meta[blockIdx.x * kMetaInts] = 0;
  }
  while (true) {
    if (tid == 0) {
      s_have = walk.next(p, range, &s_piece);
      s_merges = s_have && walk.merges;
      s_c0 = walk.merge_c0;
    }
    __syncthreads();
    if (!s_have) break;
    const Piece c = s_piece;
    const float* kb = static_cast<const float*>(p.k) + static_cast<int64_t>(c.head_kv) * p.page_size * D;
    const float* vb = static_cast<const float*>(p.v) + static_cast<int64_t>(c.head_kv) * p.page_size * D;
    const int* table = p.table + static_cast<int64_t>(c.request) * p.table_stride;

    // queries, scaled to base-2 exponents
    for (int i = tid; i < kSimtRows * (D / 4); i += kSimtThreads) {
      const int r = i / (D / 4), x = (i % (D / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < c.rows) {
        const int row = c.row0 + r, t = row / p.group, h = c.head_kv * p.group + row % p.group;
        v = ld4(static_cast<const float*>(p.q) + (c.first + t) * p.q_t + h * p.q_h + x);
        v.x *= p.scale_log2;
        v.y *= p.scale_log2;
        v.z *= p.scale_log2;
        v.w *= p.scale_log2;
      }
      *reinterpret_cast<float4*>(sQ + r * C::kQRow + x) = v;
    }
    auto load = [&](int tile, int stage) {
      constexpr int kChunks = D * 4 / 16;
      const uint32_t sk = sm100::smem_u32(smem) + stage * C::kStage;
      const uint32_t sv = sk + C::kKBytes;
#pragma unroll 4
      for (int i = tid; i < kSimtTile * kChunks; i += kSimtThreads) {
        const int r = i / kChunks, x = i % kChunks;
        const int j = tile * kSimtTile + r;
        bool ok = j < c.keys;
        int64_t page = 0;
        int off = 0;
        if (ok) {
          const int e = j / p.page_size;
          off = j - e * p.page_size;
          page = table[e];
          if (page < 0 || page >= p.num_pages) {  // read as zeros, reported
            if (x == 0) st_record(p.status, kStatusBadArgs, kBadPage, static_cast<uint32_t>(page));
            ok = false;
            page = 0;
          }
        }
        const int at = off * D + x * 4;
        cp_async16(sk + r * C::kKRow * 4 + x * 16, kb + page * p.k_page + at, ok);
        cp_async16(sv + r * D * 4 + x * 16, vb + page * p.v_page + at, ok);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float acc[kSimtRows][kCols];
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r)
#pragma unroll
      for (int x = 0; x < kCols; ++x) acc[r][x] = 0.f;
    float m[4], l[4];  // rows 4 * (lane / 16) + i; l is this lane's share
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.f;
    const int half = lane >> 4, key = lane & 15;

    load(c.tile_begin, 0);
    for (int tile = c.tile_begin; tile < c.tile_end; ++tile) {
      const int stage = (tile - c.tile_begin) & 1;
      if (tile + 1 < c.tile_end) {
        load(tile + 1, stage ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
      __syncthreads();
      const float* sk = reinterpret_cast<const float*>(smem + stage * C::kStage);
      const float* sv = reinterpret_cast<const float*>(smem + stage * C::kStage + C::kKBytes);
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      const float* krow = sk + (warp * 16 + key) * C::kKRow;
      const float* qrow = sQ + half * 4 * C::kQRow;
#pragma unroll 8
      for (int x = 0; x < D; x += 4) {
        const float4 kv = ld4(krow + x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 qv = *reinterpret_cast<const float4*>(qrow + i * C::kQRow + x);
          s[i] = fmaf(qv.x, kv.x, s[i]);
          s[i] = fmaf(qv.y, kv.y, s[i]);
          s[i] = fmaf(qv.z, kv.z, s[i]);
          s[i] = fmaf(qv.w, kv.w, s[i]);
        }
      }
      const int j = tile * kSimtTile + warp * 16 + key;
      const bool tail = (tile + 1) * kSimtTile > c.ctx;  // new tokens, or past the end
      if (tail && j >= c.ctx) {
        const int rel = j - c.ctx;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = c.row0 + half * 4 + i;
          bool sees = j < c.keys && half * 4 + i < c.rows;
          if (sees) {
            const int t = row / p.group;
            sees = p.mask == nullptr
                       ? rel <= t
                       : (rel >> 5) < p.mask_w &&
                             ((p.mask[(c.first + t) * p.mask_stride + (rel >> 5)] >> (rel & 31)) &
                              1u);
          }
          if (!sees) s[i] = -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float mx = s[i];
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float mn = fmaxf(m[i], mx);
        const float use = mn == -INFINITY ? 0.f : mn;
        const float alpha = sm100::ex2_approx(m[i] - use);  // m = -inf: 0
        m[i] = mn;
        const float e = sm100::ex2_approx(s[i] - use);
        l[i] = l[i] * alpha + e;
        sP[(warp * kSimtRows + half * 4 + i) * 16 + key] = e;
        if (key == 0) s_alpha[warp][half * 4 + i] = alpha;
      }
      __syncwarp();
#pragma unroll
      for (int r = 0; r < kSimtRows; ++r) {
        const float a = s_alpha[warp][r];
#pragma unroll
        for (int x = 0; x < kCols; ++x) acc[r][x] *= a;
      }
      const float* vcol = sv + warp * 16 * D + lane * kCols;
#pragma unroll
      for (int k4 = 0; k4 < 16; k4 += 4) {
        float v[4][kCols];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int x = 0; x < kCols; ++x) v[u][x] = vcol[(k4 + u) * D + x];
#pragma unroll
        for (int r = 0; r < kSimtRows; ++r) {
          const float4 pr = *reinterpret_cast<const float4*>(sP + (warp * kSimtRows + r) * 16 + k4);
          const float pv[4] = {pr.x, pr.y, pr.z, pr.w};
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int x = 0; x < kCols; ++x) {
              // among the new tokens a row does not take what it does not see: not even a NaN
              if (!tail || pv[u] != 0.f) acc[r][x] = fmaf(pv[u], v[u][x], acc[r][x]);
            }
        }
      }
      __syncthreads();  // the stage may be loaded again
    }

    // join the warps
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int d = 8; d >= 1; d >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
      if (key == 0) {
        s_m[warp][half * 4 + i] = m[i];
        s_l[warp][half * 4 + i] = l[i];
      }
    }
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r)
#pragma unroll
      for (int x = 0; x < kCols; ++x) sJoin[(warp * kSimtRows + r) * D + lane * kCols + x] = acc[r][x];
    __syncthreads();
    for (int i = tid; i < kSimtRows * D; i += kSimtThreads) {
      const int r = i / D, x = i % D;
      if (r >= c.rows) break;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, s_m[w][r]);
      float sum = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = top == -INFINITY ? 1.f : sm100::ex2_approx(s_m[w][r] - top);
        sum += f * s_l[w][r];
        o += f * sJoin[(w * kSimtRows + r) * D + x];
      }
      if (c.record >= 0) {
        const int64_t rr = static_cast<int64_t>(c.record) * kSimtRows + r;
        // a record is [dim / 4][rows][4], the rows of the unit side by side
        p.rec_acc[static_cast<int64_t>(c.record) * (kSimtRows * D) + ((x >> 2) * c.rows + r) * 4 +
                  (x & 3)] = o;
        if (x == 0) {
          p.rec_m[rr] = top;
          p.rec_l[rr] = sum;
        }
      } else {
        const int row = c.row0 + r, t = row / p.group, h = c.head_kv * p.group + row % p.group;
        static_cast<float*>(p.out)[static_cast<int64_t>(c.first + t) * p.out_t +
                                   static_cast<int64_t>(h) * p.out_h + x] =
            sum == 0.f ? 0.f : o / sum;
        if (x == 0 && p.lse != nullptr)
          p.lse[static_cast<int64_t>(c.first + t) * p.heads + h] =
              sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2f;
      }
    }
    if (tid == 0 && s_merges) write_meta(p, c, true, s_c0);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Merge: the blocks (c, y) join the records of the unit that CTA c ended.  A
// thread owns four columns of a row; a record is [dim / 4][rows][4], so the
// threads of a warp read side by side whatever the number of rows.  Bound by
// latency: eight records' maxima, sums and outputs are in flight at once, and
// with more than eight (long contexts, few rows) the block's four warps share the
// records of the same 32 elements and join theirs through shared memory.  The
// launch overlaps the attention kernel's end (griddepcontrol.wait holds it until
// every record is written).
// ---------------------------------------------------------------------------
constexpr int kMergeThreads = 128;

struct Joined {
  float top, sum;
  float4 o;
};

__device__ __forceinline__ void join_into(Joined& a, float m, float l, const float4& o) {
  const float top = fmaxf(a.top, m);
  const float use = top == -INFINITY ? 0.f : top;
  const float f = sm100::ex2_approx(a.top - use), g = sm100::ex2_approx(m - use);
  a.top = top;
  a.sum = f * a.sum + g * l;
  a.o.x = f * a.o.x + g * o.x;
  a.o.y = f * a.o.y + g * o.y;
  a.o.z = f * a.o.z + g * o.z;
  a.o.w = f * a.o.w + g * o.w;
}

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads)
    tree_merge_kernel(const __grid_constant__ TreeParams p, int rows_per_unit) {
  __shared__ Joined s_join[3][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 m0 = *reinterpret_cast<const int4*>(p.meta + blockIdx.x * kMetaInts);
  const int2 m1 = *reinterpret_cast<const int2*>(p.meta + blockIdx.x * kMetaInts + 4);
  if (m0.x == 0) return;
  const int c0 = m0.y, head_kv = m0.z, row0 = m0.w, rows = m1.x, first = m1.y;
  const int n = blockIdx.x - c0 + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool share = n > 8;
  const int i_first = share ? warp : 0, i_step = share ? 4 : 1;
  const int elems = rows * (D / 4), per_block = share ? 32 : kMergeThreads;
  for (int e0 = blockIdx.y * per_block; e0 < elems; e0 += gridDim.y * per_block) {
    const int e = min(e0 + (share ? lane : static_cast<int>(threadIdx.x)), elems - 1);
    const bool mine = e0 + (share ? lane : static_cast<int>(threadIdx.x)) < elems;
    const int x4 = e / rows, r = e - x4 * rows;
    Joined a{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int i0 = i_first; i0 < n; i0 += 8 * i_step) {
      float m[8], l[8];
      float4 o[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        // the first record is the last piece of CTA c0, the others the first of each
        const int i = i0 + u * i_step, k = 2 * (c0 + i) + (i == 0 ? 1 : 0);
        if (i < n) {
          m[u] = p.rec_m[k * rows_per_unit + r];
          l[u] = p.rec_l[k * rows_per_unit + r];
          o[u] = *reinterpret_cast<const float4*>(
              p.rec_acc + static_cast<int64_t>(k) * rows_per_unit * D + e * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i0 + u * i_step < n) join_into(a, m[u], l[u], o[u]);
    }
    if (share) {
      if (warp > 0) s_join[warp - 1][lane] = a;
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 0; w < 3; ++w) {
          const Joined b = s_join[w][lane];
          join_into(a, b.top, b.sum, b.o);
        }
      }
      __syncthreads();
      if (warp > 0) continue;
    }
    if (!mine) continue;
    const float inv = a.sum == 0.f ? 0.f : 1.f / a.sum;
    const int row = row0 + r, t = row / p.group, h = head_kv * p.group + row - t * p.group;
    T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(first + t) * p.out_t +
             static_cast<int64_t>(h) * p.out_h + x4 * 4;
    alignas(16) T v[4] = {cast_out<T>(a.o.x * inv), cast_out<T>(a.o.y * inv),
                          cast_out<T>(a.o.z * inv), cast_out<T>(a.o.w * inv)};
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
    else
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
    if (x4 == 0 && p.lse != nullptr)
      p.lse[static_cast<int64_t>(first + t) * p.heads + h] =
          a.sum == 0.f ? -INFINITY : (a.top + log2f(a.sum)) * kLn2f;
  }
}

template <int D>
int run_simt(const TreeParams& p, cudaStream_t stream) {
  using C = SimtCfg<D>;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t err = cudaFuncSetAttribute(
        tree_simt_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (err != cudaSuccess) return static_cast<int>(err);
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  tree_simt_kernel<D><<<p.grid, kSimtThreads, C::kSmem, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D>
int run_merge(const TreeParams& p, int rows_per_unit, int merge_rows, cudaStream_t stream) {
  cudaLaunchAttribute overlap;
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // a block per 128 elements of the largest unit, up to 64; blocks without a unit leave at once
  const int blocks = (merge_rows * (D / 4) + kMergeThreads - 1) / kMergeThreads;
  cfg.gridDim = dim3(p.grid, blocks < 64 ? blocks : 64);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cfg.attrs = &overlap;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, tree_merge_kernel<T, D>, p, rows_per_unit));
}

// ---------------------------------------------------------------------------
// masks
// ---------------------------------------------------------------------------
__global__ void tree_mask_kernel(const int* parents, const int* cu, int batch, int uniform,
                                 int total, uint32_t* mask, int mask_w, int* depth,
                                 DeviceStatus* status) {
  const int token = blockIdx.x * blockDim.x + threadIdx.x;
  if (token >= total) return;
  int first, end;
  if (cu == nullptr) {
    first = token / uniform * uniform;
    end = first + uniform;
  } else {
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= token) lo = mid;
      else hi = mid;
    }
    first = cu[lo];
    end = cu[lo + 1];
  }
  if (token < first || token >= end || first < 0) return;  // behind the last request
  uint32_t* row = mask + static_cast<int64_t>(token) * mask_w;
  for (int w = 0; w < mask_w; ++w) row[w] = 0u;
  int at = token - first, d = -1;
  // a parent lies before its child, so the walk ends
  while (at >= 0) {
    if ((at >> 5) < mask_w) row[at >> 5] |= 1u << (at & 31);
    ++d;
    const int up = parents[first + at];
    if (up >= at || up < -1) {
      st_record(status, kStatusBadArgs, kBadParent, static_cast<uint32_t>(first + at));
      break;
    }
    at = up;
  }
  depth[token] = d;
}

__global__ void pack_mask_kernel(const uint8_t* in, int64_t in_t, int total, int cols,
                                 uint32_t* mask, int mask_w) {
  const int64_t i = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  if (i >= static_cast<int64_t>(total) * mask_w) return;  // whole warps
  const int row = static_cast<int>(i / mask_w), w = static_cast<int>(i % mask_w);
  const int col = w * 32 + (threadIdx.x & 31);
  const uint32_t bits =
      __ballot_sync(0xffffffffu, col < cols && in[row * in_t + col] != 0);
  if ((threadIdx.x & 31) == 0) mask[i] = bits;
}

}  // namespace

TreePlan tree_plan(Elem elem, const TreeParams& p, int max_q, int sms) {
  TreePlan plan;
  if (elem == Elem::kF32) {
    plan.rows_per_unit = kSimtRows;
    const int smem = p.dim == 64 ? SimtCfg<64>::kSmem : SimtCfg<128>::kSmem;
    plan.grid = sms * ((227 * 1024) / (smem + 2048));
  } else {
    // one row tile keeps two key tiles in the air per CTA and suits what reading
    // the cache bounds; from the second row tile on, both share every key tile
    plan.rows_per_unit = static_cast<int64_t>(max_q) * p.group > 128 ? 256 : 128;
    plan.grid = sms;
  }
  // rows of the largest unit that can occur (max_q is a hint: the merge loops)
  const int64_t most = static_cast<int64_t>(max_q) * p.group;
  plan.merge_rows = static_cast<int>(most < plan.rows_per_unit ? most : plan.rows_per_unit);
  const size_t rows = static_cast<size_t>(2) * plan.grid * plan.rows_per_unit;
  plan.acc_floats = rows * p.dim;
  plan.ml_floats = 2 * rows;
  plan.meta_ints = static_cast<size_t>(plan.grid) * kMetaInts;
  return plan;
}

int tree_launch(Elem elem, const TreeParams& p, const TreePlan& plan, cudaStream_t stream) {
  const int rows = plan.rows_per_unit;
  int err;
  if (elem == Elem::kF32)
    err = p.dim == 64 ? run_simt<64>(p, stream) : run_simt<128>(p, stream);
  else
    err = tree_sm100_launch(elem, p, rows, stream);
  if (err != 0) return err;
  switch (elem) {
    case Elem::kBF16:
      return p.dim == 64 ? run_merge<__nv_bfloat16, 64>(p, rows, plan.merge_rows, stream)
                         : run_merge<__nv_bfloat16, 128>(p, rows, plan.merge_rows, stream);
    case Elem::kF16:
      return p.dim == 64 ? run_merge<__half, 64>(p, rows, plan.merge_rows, stream)
                         : run_merge<__half, 128>(p, rows, plan.merge_rows, stream);
    default:
      return p.dim == 64 ? run_merge<float, 64>(p, rows, plan.merge_rows, stream)
                         : run_merge<float, 128>(p, rows, plan.merge_rows, stream);
  }
}

int tree_mask_launch(const int* parents, const int* cu, int batch, int uniform, int total,
                     uint32_t* mask, int mask_w, int* depth, DeviceStatus* status,
                     cudaStream_t stream) {
  if (total == 0) return 0;
  tree_mask_kernel<<<(total + 127) / 128, 128, 0, stream>>>(parents, cu, batch, uniform, total,
                                                             mask, mask_w, depth, status);
  return static_cast<int>(cudaGetLastError());
}

int pack_mask_launch(const uint8_t* in, int64_t in_t, int total, int cols, uint32_t* mask,
                     int mask_w, cudaStream_t stream) {
  const int64_t warps = static_cast<int64_t>(total) * mask_w;
  if (warps == 0) return 0;
  pack_mask_kernel<<<static_cast<unsigned>((warps * 32 + 255) / 256), 256, 0, stream>>>(
      in, in_t, total, cols, mask, mask_w);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace rab
