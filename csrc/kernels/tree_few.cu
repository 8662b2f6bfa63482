// tree_few.cu - attention of new tokens over a paged cache in bf16 and fp16 for up to
// 32 rows per kv head: decoding steps and small trees (tree_sm100.cu takes more).
//
// Reading the cache bounds this work, so products on the small tensor instructions are
// enough, and they save what the large ones cost a short piece: their scores, weights
// and outputs pass between warps through TMEM, one tile after the other.  Here a warp
// keeps its rows' maximum, sum and outputs in registers from the scores to the result.
//
// Products are 16 x 8 x 16.  Scores: rows are keys, columns query rows, the sum runs
// over dim.  Outputs: rows are columns of V, the sum runs over keys; the weights leave
// the scores' registers as the other operand through an 8 x 8 transposition between
// lanes.  K and V are read by ldmatrix, whose eight 16-byte rows meet the swizzled
// tile's banks once.
//
// Keys no row may see: the score is replaced by -inf, so K may hold anything; V is
// cleaned in the registers of tiles that hold new tokens or the cache's end, and what
// is not finite among the new tokens is added at the end to the rows that see it.
#include "tree_warp.cuh"

namespace rab {

using namespace tree_detail;

namespace {

template <int D, int kRowsT>
struct FewCfg {
  static constexpr int kD = D, kBytes = 2, kRows = kRowsT;
  static constexpr int kThreads = 288;
  // sixteen keys to a warp; with more than eight rows the two halves of the warps take
  // the two halves of the rows
  static constexpr int kSplit = kRows > 8 ? 2 : 1;
  static constexpr int kGroups = kRows / 8 / kSplit;
  static constexpr int kTile = 16 * kWarps / kSplit;
  static constexpr int kHalf = kTile * D * 2;
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kOwnRow = D + 4;  // rows 2t and 2t + 1 of four lanes: no bank twice
  static constexpr int kOwn = kGroups * 8 * kOwnRow;
  static constexpr int kOwnBytes = kWarps * kOwn * 4;
  static constexpr int kRest = kWarps * kGroups * 8 * 8 + kItems * 48 + 256;
  static constexpr int kFit = (232448 - kOwnBytes - kRest) / kStage;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kOwnOff = kStages * kStage;
  static constexpr int kMlOff = kOwnOff + kOwnBytes;  // float2 [warps][own rows]
  static constexpr int kItemOff = kMlOff + kWarps * kGroups * 8 * 8;
  static constexpr int kBarOff = kItemOff + kItems * 48;
  static constexpr int kBars = 2 * kStages + 2 * kItems + 2;
  static constexpr int kDirtyOff = kBarOff + kBars * 8;  // int [2]
  static constexpr int kSmem = kDirtyOff + 8;
  static_assert(kSmem <= 232448 && kBarOff % 8 == 0 && kStages >= 2, "shared memory");
};

template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static constexpr uint32_t kExp = 0x7f80u;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return sm100::pack_bf16x2(lo, hi);
  }
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
};
template <>
struct Half<__half> {
  static constexpr uint32_t kExp = 0x7c00u;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
};

// four 8 x 8 blocks whose rows lanes 0-7, 8-15, 16-23 and 24-31 point at
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// A computing warp.  Lane = 4 g + t; its scores are those of keys g and g + 8 (of the
// warp's 16) for query rows 2t and 2t + 1 of a group, its outputs columns 16 b + g and
// + 8 of the same rows.
template <typename T, int D, int kRows>
__device__ __forceinline__ void few_compute(const TreeParams& p,
                                            const WarpBlock<FewCfg<D, kRows>>& blk) {
  using C = FewCfg<D, kRows>;
  using H = Half<T>;
  using namespace sm100;
  constexpr int kTile = C::kTile, G = C::kGroups;
  constexpr int kKeyWarps = kWarps / C::kSplit;
  const int warp = warp_id(), lane = lane_id();
  DeviceStatus* st = p.status;
  const uint64_t tmo = p.timeout_ns;
  const int g = lane >> 2, t = lane & 3;
  const int key0 = warp % kKeyWarps * 16;        // this warp's first key of a tile
  const int row_w = warp / kKeyWarps * (8 * G);  // and its first row of the unit
  float* own = blk.own(warp);
  // where this lane points for K (keys 0-7, 8-15, then the next 8 columns) and V (keys
  // 0-7 of two 8-column blocks, then keys 8-15), by the place of 16 columns in 64
  const uint32_t ring = smem_u32(blk.smem);
  const uint32_t k_at = ring + (key0 + (lane & 15)) * 128;
  const uint32_t v_at = ring + C::kHalf + (key0 + (lane & 7) + 8 * (lane >> 4)) * 128;
  uint32_t k_col[4], v_col[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    k_col[b] = static_cast<uint32_t>((2 * b + (lane >> 4)) ^ (lane & 7)) << 4;
    v_col[b] = static_cast<uint32_t>((2 * b + ((lane >> 3) & 1)) ^ (lane & 7)) << 4;
  }

  uint32_t q[G][D / 16][2];  // columns 16 b + 2t, + 1 and + 8, + 9 of row g of a group
  Piece c;
  // waits for piece w and asks for its queries, which are due at its first product
  auto fetch = [&](int w) -> bool {
    if (!__all_sync(0xffffffffu, mbar_wait(blk.item_full(w), (w / kItems) & 1, st,
                                           kSiteItemQueue, tmo)))
      return false;
    c = *blk.item(w);
    if (c.request < 0) return true;
#pragma unroll
    for (int u = 0; u < G; ++u) {
      const int row = c.row0 + min(row_w + 8 * u + g, c.rows - 1), tok = row / p.group;
      const int h = c.head_kv * p.group + row - tok * p.group;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          static_cast<const T*>(p.q) + static_cast<int64_t>(c.first + tok) * p.q_t +
          static_cast<int64_t>(h) * p.q_h + 2 * t);
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        q[u][b][0] = src[8 * b];
        q[u][b][1] = src[8 * b + 4];
      }
    }
    return true;
  };

  int n = 0;  // tiles taken
  bool ok = fetch(0);
  for (int w = 0; ok && c.request >= 0; ++w) {
    float acc[G][D / 16][4];
    float m[G][2], l[G][2];  // rows 2t + i; l is this lane's share
#pragma unroll
    for (int u = 0; u < G; ++u) {
#pragma unroll
      for (int b = 0; b < D / 16; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[u][b][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[u][i] = -INFINITY;
        l[u][i] = 0.f;
      }
    }
    bool dirty = false;

    for (int tile = c.tile_begin; tile < c.tile_end; ++tile, ++n) {
      const int stage = n % C::kStages;
      ok = __all_sync(0xffffffffu, mbar_wait(blk.full(stage), (n / C::kStages) & 1, st,
                                             kSiteKFull, tmo));
      if (!ok) break;
      // even and odd steps are summed apart, so that products do not wait for one another
      float s2[2][G][4] = {};
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        uint32_t a[4];
        ldsm4(a, k_at + stage * C::kStage + (b >> 2) * (kTile * 128) + k_col[b & 3]);
#pragma unroll
        for (int u = 0; u < G; ++u) H::mma(s2[b & 1][u], a, q[u][b]);
      }
      const int j0 = tile * kTile + key0;
      const bool tail = (tile + 1) * kTile > c.ctx;  // new tokens, or past the end
      uint32_t wt[G][2];  // weights of keys 2t, 2t + 1 and + 8, + 9 for row g
      float alpha[G][2];
      bool moved = false;
#pragma unroll
      for (int u = 0; u < G; ++u) {
        float s[4];  // [2 (key / 8) + row]
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = (s2[0][u][i] + s2[1][u][i]) * p.scale_log2;
        if (tail) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = row_w + 8 * u + 2 * t + i;
            const int tok = (c.row0 + r) / p.group;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = j0 + g + 8 * x, rel = j - c.ctx;
              if (rel < 0) continue;
              bool sees = j < c.keys && r < c.rows;
              if (sees)
                sees = p.mask == nullptr
                           ? rel <= tok
                           : (rel >> 5) < p.mask_w &&
                                 ((p.mask[static_cast<int64_t>(c.first + tok) * p.mask_stride +
                                          (rel >> 5)] >>
                                   (rel & 31)) &
                                  1u);
              if (!sees) s[2 * x + i] = -INFINITY;
            }
          }
        }
        float e[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(s[i], s[2 + i]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m[u][i], mx);
          const float use = mn == -INFINITY ? 0.f : mn;
          alpha[u][i] = ex2_approx(m[u][i] - use);  // m = -inf: 0
          moved |= mn != m[u][i];
          m[u][i] = mn;
          e[i] = ex2_approx(s[i] - use);
          e[2 + i] = ex2_approx(s[2 + i] - use);
          l[u][i] = l[u][i] * alpha[u][i] + (e[i] + e[2 + i]);  // the weights unrounded
        }
        wt[u][0] = transpose8(H::pack(e[0], e[1]));
        wt[u][1] = transpose8(H::pack(e[2], e[3]));
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int u = 0; u < G; ++u)
#pragma unroll
          for (int b = 0; b < D / 16; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[u][b][i] *= alpha[u][i & 1];
      }
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        uint32_t a[4];  // columns g and g + 8 of keys 2t, 2t + 1, then of keys 8 later
        ldsm4_t(a, v_at + stage * C::kStage + (b >> 2) * (kTile * 128) + v_col[b & 3]);
        if (tail) {
          // rows past the end count for nothing, whatever they hold; what is not finite
          // among the new tokens is left out here and added at the end
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int hlf = 0; hlf < 2; ++hlf) {
              const int j = j0 + 8 * (x >> 1) + 2 * t + hlf;
              const uint32_t bits = hlf ? 0xffff0000u : 0x0000ffffu;
              const uint32_t ex = hlf ? H::kExp << 16 : H::kExp;
              const bool past = j >= c.keys, bad = (a[x] & ex) == ex;
              if (j >= c.ctx && (past || bad)) {
                dirty |= !past;
                a[x] &= ~bits;
              }
            }
        }
#pragma unroll
        for (int u = 0; u < G; ++u) H::mma(acc[u][b], a, wt[u]);
      }
      __syncwarp();  // the stage has been read
      if (lane == 0) mbar_arrive(blk.empty(stage));
    }
    if (!ok) break;

    // the next piece's queries come while the warps join this one
    const Piece done = c;
    ok = fetch(w + 1);
    if (!ok) break;
    if (w > 0) {  // the piece before has been read out of every warp's outputs
      ok = __all_sync(0xffffffffu, mbar_wait(blk.released(), (w - 1) & 1, st, kSiteOReady, tmo));
      if (!ok) break;
    }
    if (dirty) blk.dirty()[w & 1] = w + 1;
#pragma unroll
    for (int u = 0; u < G; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[u][i] += __shfl_xor_sync(0xffffffffu, l[u][i], d);
        if (g == 0) blk.ml(warp, 8 * u + 2 * t + i) = make_float2(m[u][i], l[u][i]);
#pragma unroll
        for (int b = 0; b < D / 16; ++b)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            own[(8 * u + 2 * t + i) * C::kOwnRow + 16 * b + 8 * x + g] = acc[u][b][2 * x + i];
      }
    __syncwarp();
    if (lane == 0) mbar_arrive(blk.joined());
    ok = __all_sync(0xffffffffu, mbar_wait(blk.joined(), w & 1, st, kSiteOReady, tmo));
    if (!ok) break;
    write_results<C, T>(p, blk, done, w);
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(blk.released());
      mbar_arrive(blk.item_empty(w));
    }
  }
}

template <typename T, int D, int kRows>
__global__ void __launch_bounds__(FewCfg<D, kRows>::kThreads, 1)
    tree_few_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV) {
  using C = FewCfg<D, kRows>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const WarpBlock<C> blk{smem};
  if (!start_block<C>(p, blk)) return;
  if (sm100::warp_id() == kWarps)
    walk_and_load<C>(p, tmK, tmV, blk);
  else
    few_compute<T, D, kRows>(p, blk);
}

template <typename T, int D, int kRows>
int run(const TreeParams& p, cudaStream_t stream) {
  static bool done[64] = {};
  return launch_warp_kernel<FewCfg<D, kRows>>(tree_few_kernel<T, D, kRows>, done, p, stream);
}

template <typename T, int D>
int run_rows(const TreeParams& p, int rows, cudaStream_t stream) {
  return rows == 8    ? run<T, D, 8>(p, stream)
         : rows == 16 ? run<T, D, 16>(p, stream)
                      : run<T, D, 32>(p, stream);
}

}  // namespace

int tree_few_launch(Elem elem, const TreeParams& p, int rows_per_unit, cudaStream_t stream) {
  if (elem == Elem::kBF16)
    return p.dim == 64 ? run_rows<__nv_bfloat16, 64>(p, rows_per_unit, stream)
                       : run_rows<__nv_bfloat16, 128>(p, rows_per_unit, stream);
  return p.dim == 64 ? run_rows<__half, 64>(p, rows_per_unit, stream)
                     : run_rows<__half, 128>(p, rows_per_unit, stream);
}

}  // namespace rab
