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
// One CTA per SM takes its even share of the work (tree_sched.cuh), 8 rows of a kv
// head at a time: at 8 rows the 2 x 8 x dim products of a key take the CUDA cores
// about half the time its 8 x dim bytes take from memory, so a decoding step stays
// bound by reading the cache (more rows read it again, from L2 where it fits).
// Warp 8 walks the pieces and brings tiles of 64 KB (K and V of 128 keys at dim 64,
// 64 keys at dim 128) by TMA into a ring of three.  Warps 0-7 take an eighth of a
// tile's keys each: lanes are keys while scores form (the 128-byte swizzle spreads
// eight keys' words over all banks), then columns for the product with V.  Every
// warp keeps its own running maximum, sum and 8 x dim outputs in registers; they
// are joined once per piece.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.h"
#include "paged.h"
#include "sm100.cuh"
#include "tmap.h"
#include "tree_sched.cuh"

namespace rab {

using namespace tree_detail;

namespace {

constexpr int kSimtThreads = 288;
constexpr int kSimtRows = 8;
constexpr int kSimtWarps = 8;   // that compute
constexpr int kSimtStages = 3;
constexpr int kSimtItems = 4;   // queue of pieces
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

template <int D>
struct SimtCfg {
  static constexpr int kTile = 8192 / D;       // keys: 32 KB of K
  static constexpr int kKeys = kTile / kSimtWarps;  // of a warp: 16 or 8
  static constexpr int kGroups = 32 / kKeys;   // groups of lanes, each with its rows
  static constexpr int kGroupRows = kSimtRows / kGroups;
  static constexpr int kHalf = kTile * D * 4;  // bytes of K (or V) of a tile
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kOwn = kSimtRows * D;   // floats of a warp: its queries, then its outputs
  static constexpr int kPOff = kSimtStages * kStage + kSimtWarps * kOwn * 4;
  static constexpr int kPBytes = kSimtRows * kKeys * 4;  // of a warp: weights; at a piece's end float2 [rows]
  static constexpr int kAlphaOff = kPOff + kSimtWarps * kPBytes;
  static constexpr int kItemOff = kAlphaOff + kSimtWarps * kSimtRows * 4;
  static constexpr int kBarOff = kItemOff + kSimtItems * 48;
  static constexpr int kBars = 2 * kSimtStages + 2 * kSimtItems + 2;
  static constexpr int kSmem = kBarOff + kBars * 8;
  static_assert(kSmem <= 232448 && kBarOff % 8 == 0, "shared memory");
};

// byte offset of element `col` of row `key` in a tile of [dim / 32][keys][32 floats],
// 16-byte chunks swizzled by the row within 128 bytes
template <int D>
__device__ __forceinline__ int tile_at(int key, int col) {
  return (col >> 5) * (SimtCfg<D>::kTile * 128) + key * 128 + ((((col >> 2) & 7) ^ (key & 7)) << 4) +
         (col & 3) * 4;
}

template <int D>
__global__ void __launch_bounds__(kSimtThreads, 1)
    tree_simt_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV) {
  using C = SimtCfg<D>;
  using namespace sm100;
  constexpr int kTile = C::kTile, kKeys = C::kKeys, kGR = C::kGroupRows;
  constexpr int kCols = D / 32;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + kSimtStages;
  uint64_t* item_full = empty + kSimtStages;
  uint64_t* item_empty = item_full + kSimtItems;
  uint64_t* joined = item_empty + kSimtItems;
  uint64_t* released = joined + 1;
  auto item_slot = [&](int w) {
    return reinterpret_cast<Piece*>(smem + C::kItemOff + (w % kSimtItems) * 48);
  };
  const int warp = warp_id(), lane = lane_id();
  DeviceStatus* st = p.status;
  const uint64_t tmo = p.timeout_ns;
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzle counts from 1024-byte boundaries
    wait_for_predecessor();
    if (threadIdx.x == 0) {
      p.meta[blockIdx.x * kMetaInts] = 0;
      st_record(st, kStatusBadArgs, kSiteNone);
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSimtStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kSimtWarps);
    }
    for (int i = 0; i < kSimtItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kSimtWarps);
    }
    mbar_init(joined, kSimtWarps);
    mbar_init(released, kSimtWarps);
    fence_barrier_init();
  }
  let_successor_start();
  __syncthreads();
  wait_for_predecessor();

  if (warp == kSimtWarps) {
    // -------------------------------------------------------- pieces and loads
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      p.meta[blockIdx.x * kMetaInts] = 0;
    }
    Range range;
    Start first;
    const int walker = find_range<kTile, kSimtRows>(p, &range, &first);
    Walk<kTile, kSimtRows> walk;
    if (lane == walker) walk.start(p, range, first);
    const int rows_box = min(p.page_size, kTile);
    const int boxes = kTile / rows_box * (D / 32);
    int n = 0;  // tiles loaded
    bool ok = true;
    for (int w = 0; ok; ++w) {
      if (w >= kSimtItems)
        ok = __all_sync(0xffffffffu, mbar_wait(&item_empty[w % kSimtItems],
                                               (w / kSimtItems - 1) & 1, st, kSiteItemQueue, tmo));
      if (!ok) break;
      Piece* slot = item_slot(w);
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
      if (lane == 0) mbar_arrive(&item_full[w % kSimtItems]);
      if (c.request < 0) break;
      const int* table = p.table + static_cast<int64_t>(c.request) * p.table_stride;
      const int last_entry = (c.keys - 1) >> p.page_shift;
      for (int tile = c.tile_begin; tile < c.tile_end; ++tile) {
        // this lane's box: page, rows within the tile, 32-column segment
        const int seg = lane % (D / 32), part = lane / (D / 32);
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
        const int stage = n % kSimtStages;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], ((n / kSimtStages) & 1) ^ 1, st,
                                               kSiteKEmpty, tmo));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], C::kStage);
        __syncwarp();
        if (lane < boxes) {
          uint8_t* dst = smem + stage * C::kStage + seg * (kTile * 128) + part * rows_box * 128;
          tma_load_4d(dst, &tmK, &full[stage], seg * 32, token, c.head_kv, page);
          tma_load_4d(dst + C::kHalf, &tmV, &full[stage], seg * 32, token, c.head_kv, page);
        }
        ++n;
      }
    }
    // the loads in flight land before the block gives its memory back
    for (int i = 0; i < kSimtStages && i < n; ++i) {
      const int k = n - 1 - i;
      mbar_wait(&full[k % kSimtStages], (k / kSimtStages) & 1, nullptr, kSiteKFull, 100000000ull);
    }
    return;
  }

  // ------------------------------------------------------------------ arithmetic
  float* own = reinterpret_cast<float*>(smem + kSimtStages * C::kStage) + warp * C::kOwn;
  float* s_p = reinterpret_cast<float*>(smem + C::kPOff) + warp * kSimtRows * kKeys;
  auto s_ml = [&](int u, int r) -> float2& {  // maximum and sum of warp u's row r
    return reinterpret_cast<float2*>(smem + C::kPOff + u * C::kPBytes)[r];
  };
  float* s_alpha = reinterpret_cast<float*>(smem + C::kAlphaOff) + warp * kSimtRows;
  const int key = lane % kKeys, row0 = lane / kKeys * kGR;  // this lane's key and first row
  const int turn = lane / kKeys * 4;
  int n = 0;  // tiles taken
  bool ok = true;
  for (int w = 0; ok; ++w) {
    ok = __all_sync(0xffffffffu, mbar_wait(&item_full[w % kSimtItems], (w / kSimtItems) & 1, st,
                                           kSiteItemQueue, tmo));
    if (!ok) break;
    const Piece c = *item_slot(w);
    if (c.request < 0) break;
    // the piece before has been read out of every warp's outputs
    if (w > 0)
      ok = __all_sync(0xffffffffu, mbar_wait(released, (w - 1) & 1, st, kSiteOReady, tmo));
    if (!ok) break;
    // queries, scaled to base-2 exponents; a copy for each warp
    for (int i = lane; i < kSimtRows * (D / 4); i += 32) {
      const int r = i / (D / 4), x = (i % (D / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < c.rows) {
        const int row = c.row0 + r, t = row / p.group, h = c.head_kv * p.group + row - t * p.group;
        v = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) +
                                             static_cast<int64_t>(c.first + t) * p.q_t +
                                             static_cast<int64_t>(h) * p.q_h + x);
        v.x *= p.scale_log2;
        v.y *= p.scale_log2;
        v.z *= p.scale_log2;
        v.w *= p.scale_log2;
      }
      // the groups of lanes read different rows at once: from different banks
      *reinterpret_cast<float4*>(own + r * D + (x ^ (r / kGR * 4))) = v;
    }
    __syncwarp();
    float acc[kSimtRows][kCols];
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r)
#pragma unroll
      for (int x = 0; x < kCols; ++x) acc[r][x] = 0.f;
    float m[kGR], l[kGR];  // rows row0 + i; l is this lane's share
#pragma unroll
    for (int i = 0; i < kGR; ++i) m[i] = -INFINITY, l[i] = 0.f;

    for (int tile = c.tile_begin; tile < c.tile_end; ++tile, ++n) {
      const int stage = n % kSimtStages;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], (n / kSimtStages) & 1, st, kSiteKFull,
                                             tmo));
      if (!ok) break;
      const uint8_t* sk = smem + stage * C::kStage;
      const uint8_t* sv = sk + C::kHalf;
      const int k_in = warp * kKeys + key;  // within the tile
      float s[kGR];
#pragma unroll
      for (int i = 0; i < kGR; ++i) s[i] = 0.f;
#pragma unroll 8
      for (int x = 0; x < D; x += 4) {
        const float4 kv = *reinterpret_cast<const float4*>(sk + tile_at<D>(k_in, x));
#pragma unroll
        for (int i = 0; i < kGR; ++i) {
          const float4 qv = *reinterpret_cast<const float4*>(own + (row0 + i) * D + (x ^ turn));
          s[i] = fmaf(qv.x, kv.x, s[i]);
          s[i] = fmaf(qv.y, kv.y, s[i]);
          s[i] = fmaf(qv.z, kv.z, s[i]);
          s[i] = fmaf(qv.w, kv.w, s[i]);
        }
      }
      const int j = tile * kTile + k_in;
      const bool tail = (tile + 1) * kTile > c.ctx;  // new tokens, or past the end
      if (tail && j >= c.ctx) {
        const int rel = j - c.ctx;
#pragma unroll
        for (int i = 0; i < kGR; ++i) {
          bool sees = j < c.keys && row0 + i < c.rows;
          if (sees) {
            const int t = (c.row0 + row0 + i) / p.group;
            sees = p.mask == nullptr
                       ? rel <= t
                       : (rel >> 5) < p.mask_w &&
                             ((p.mask[static_cast<int64_t>(c.first + t) * p.mask_stride +
                                      (rel >> 5)] >>
                               (rel & 31)) &
                              1u);
          }
          if (!sees) s[i] = -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < kGR; ++i) {
        float mx = s[i];
#pragma unroll
        for (int d = kKeys / 2; d >= 1; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float mn = fmaxf(m[i], mx);
        const float use = mn == -INFINITY ? 0.f : mn;
        const float alpha = ex2_approx(m[i] - use);  // m = -inf: 0
        m[i] = mn;
        const float e = ex2_approx(s[i] - use);
        l[i] = l[i] * alpha + e;
        s_p[(row0 + i) * kKeys + key] = e;
        if (key == 0) s_alpha[row0 + i] = alpha;
      }
      __syncwarp();
#pragma unroll
      for (int r = 0; r < kSimtRows; ++r) {
        const float a = s_alpha[r];
#pragma unroll
        for (int x = 0; x < kCols; ++x) acc[r][x] *= a;
      }
#pragma unroll
      for (int k4 = 0; k4 < kKeys; k4 += 4) {
        float v[4][kCols];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint8_t* at = sv + tile_at<D>(warp * kKeys + k4 + u, lane * kCols);
          if constexpr (kCols == 4)
            *reinterpret_cast<float4*>(v[u]) = *reinterpret_cast<const float4*>(at);
          else
            *reinterpret_cast<float2*>(v[u]) = *reinterpret_cast<const float2*>(at);
        }
#pragma unroll
        for (int r = 0; r < kSimtRows; ++r) {
          const float4 pr = *reinterpret_cast<const float4*>(s_p + r * kKeys + k4);
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
      __syncwarp();  // s_p and the stage have been read
      if (lane == 0) mbar_arrive(&empty[stage]);
    }
    if (!ok) break;

    // join the warps: outputs over the queries, which are no longer needed
#pragma unroll
    for (int i = 0; i < kGR; ++i) {
#pragma unroll
      for (int d = kKeys / 2; d >= 1; d >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
      if (key == 0) s_ml(warp, row0 + i) = make_float2(m[i], l[i]);
    }
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r)
#pragma unroll
      for (int x = 0; x < kCols; ++x) own[r * D + lane * kCols + x] = acc[r][x];
    __syncwarp();
    if (lane == 0) mbar_arrive(joined);
    ok = __all_sync(0xffffffffu, mbar_wait(joined, w & 1, st, kSiteOReady, tmo));
    if (!ok) break;
    const float* all = reinterpret_cast<const float*>(smem + kSimtStages * C::kStage);
    // row `warp` of the eight, four columns at a time
    if (warp < c.rows) {
      const int r = warp;
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < kSimtWarps; ++u) top = fmaxf(top, s_ml(u, r).x);
      const float use = top == -INFINITY ? 0.f : top;
      float sum = 0.f, f[kSimtWarps];
#pragma unroll
      for (int u = 0; u < kSimtWarps; ++u) {
        const float2 ml = s_ml(u, r);
        f[u] = ex2_approx(ml.x - use);
        sum += f[u] * ml.y;
      }
      const int row = c.row0 + r, t = row / p.group, h = c.head_kv * p.group + row - t * p.group;
      const float inv = c.record >= 0 ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);
      if (lane < D / 4) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < kSimtWarps; ++u) {
          const float4 a = *reinterpret_cast<const float4*>(all + u * C::kOwn + r * D + lane * 4);
          o.x += f[u] * a.x;
          o.y += f[u] * a.y;
          o.z += f[u] * a.z;
          o.w += f[u] * a.w;
        }
        o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        // a record is [dim / 4][rows][4], the rows of the unit side by side
        float* dst = c.record >= 0
                         ? p.rec_acc + static_cast<int64_t>(c.record) * (kSimtRows * D) +
                               (lane * c.rows + r) * 4
                         : static_cast<float*>(p.out) + static_cast<int64_t>(c.first + t) * p.out_t +
                               static_cast<int64_t>(h) * p.out_h + lane * 4;
        *reinterpret_cast<float4*>(dst) = o;
      }
      if (lane == 0) {
        if (c.record >= 0) {
          p.rec_m[c.record * kSimtRows + r] = top;
          p.rec_l[c.record * kSimtRows + r] = sum;
        } else if (p.lse != nullptr) {
          p.lse[static_cast<int64_t>(c.first + t) * p.heads + h] =
              sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2f;
        }
      }
    }
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(released);
      mbar_arrive(&item_empty[w % kSimtItems]);
    }
  }
}

// ---------------------------------------------------------------------------
// Merge: the blocks (c, y) join the records of the unit that CTA c ended.  A
// thread owns four columns of a row; a record is [dim / 4][rows][4], so the
// threads of a warp read side by side whatever the number of rows.  Bound by
// latency: four records' maxima, sums and outputs are in flight per thread, and
// with more than eight records (long contexts, few rows) the block's warps share
// those of the same 32 elements and join theirs through shared memory.
// ---------------------------------------------------------------------------
constexpr int kMergeThreads = 256;
constexpr int kMergeWarps = kMergeThreads / 32;
constexpr int kMergeBatch = 4;  // records in flight per thread

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
__global__ void __launch_bounds__(kMergeThreads, 4)
    tree_merge_kernel(const __grid_constant__ TreeParams p, int rows_per_unit) {
  __shared__ Joined s_join[kMergeWarps - 1][32];
  let_successor_start();
  wait_for_predecessor();
  const int4 m0 = *reinterpret_cast<const int4*>(p.meta + blockIdx.x * kMetaInts);
  const int2 m1 = *reinterpret_cast<const int2*>(p.meta + blockIdx.x * kMetaInts + 4);
  if (m0.x == 0) return;
  const int c0 = m0.y, head_kv = m0.z, row0 = m0.w, rows = m1.x, first = m1.y;
  const int n = blockIdx.x - c0 + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool share = n > 8;
  const int i_first = share ? warp : 0, i_step = share ? kMergeWarps : 1;
  const int elems = rows * (D / 4), per_block = share ? 32 : kMergeThreads;
  for (int e0 = blockIdx.y * per_block; e0 < elems; e0 += gridDim.y * per_block) {
    const int e = min(e0 + (share ? lane : static_cast<int>(threadIdx.x)), elems - 1);
    const bool mine = e0 + (share ? lane : static_cast<int>(threadIdx.x)) < elems;
    const int x4 = e / rows, r = e - x4 * rows;
    Joined a{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int i0 = i_first; i0 < n; i0 += kMergeBatch * i_step) {
      float m[kMergeBatch], l[kMergeBatch];
      float4 o[kMergeBatch];
#pragma unroll
      for (int u = 0; u < kMergeBatch; ++u) {
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
      for (int u = 0; u < kMergeBatch; ++u)
        if (i0 + u * i_step < n) join_into(a, m[u], l[u], o[u]);
    }
    if (share) {
      if (warp > 0) s_join[warp - 1][lane] = a;
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 0; w < kMergeWarps - 1; ++w) {
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
  auto pool_map = [&](const void* base, int64_t page_stride) {
    const uint64_t page = p.page_size;
    uint64_t dims[4] = {D, page, static_cast<uint64_t>(p.heads_kv),
                        static_cast<uint64_t>(p.num_pages)};
    uint64_t strides[3] = {D * 4, page * D * 4, static_cast<uint64_t>(page_stride) * 4};
    uint32_t box[4] = {32, static_cast<uint32_t>(p.page_size < C::kTile ? p.page_size : C::kTile),
                       1, 1};
    return make_tmap(base, TmapDtype::kF32, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  const CUtensorMap k = pool_map(p.k, p.k_page), v = pool_map(p.v, p.v_page);
  return launch_overlapped(tree_simt_kernel<D>, dim3(p.grid), kSimtThreads, C::kSmem, stream, &p,
                           &k, &v);
}

template <typename T, int D>
int run_merge(const TreeParams& p, int rows_per_unit, int merge_rows, cudaStream_t stream) {
  // blocks of a unit: about one wave of them over the GPU, each loops; blocks
  // without a unit leave at once
  const int blocks = (merge_rows * (D / 4) + 31) / 32;
  return launch_overlapped(tree_merge_kernel<T, D>, dim3(p.grid, blocks < 8 ? blocks : 8),
                           kMergeThreads, 0, stream, &p, &rows_per_unit);
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
  } else {
    // one row tile keeps two key tiles in the air per CTA and suits what reading
    // the cache bounds; from the second row tile on, both share every key tile
    plan.rows_per_unit = static_cast<int64_t>(max_q) * p.group > 128 ? 256 : 128;
  }
  plan.grid = sms;
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
