// tree_few.cu - attention of new tokens over a paged cache in bf16 and fp16 for up to
// 16 rows per kv head: decoding steps and small trees (tree_sm100.cu takes more).
//
// The mathematics is tree_f32.cu's; weights are rounded to the element type for their
// product with V and summed unrounded.  Reading the cache bounds this work, so products
// on the small tensor instructions are enough, and they save what the large ones cost a
// short piece: their scores, weights and outputs pass between warps through TMEM, one
// tile after the other (a piece of one tile: 9200 cycles, here 5500).  A warp keeps its
// rows' maximum, sum and outputs in registers from the scores to the result.
//
// us here and with tree_sm100.cu, 8 kv heads:
//   rows, dim     4 x 32000     64 x 100-3000   24 x 10-300
//    8,  64      50.8 / 64.9    44.5 / 74.4     14 / 17
//   16,  64      54.1 / 64.6    51.5 / 74.4     12 / 17
//    8, 128      87.3 / 89.8    75.5 / 84.9     13 / 18
//   16, 128      89.4 / 90.2    77.2 / 85.6     15 / 18
// (floors 40 / 31 us of bytes at dim 64, 80 / 62 at dim 128).  32 rows in this form are
// bound by the products: 68 / 65 and 115 / 91 us over 4 x 32000.
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
  static_assert(kRowsT == 8 || kRowsT == 16, "rows of a unit");
  static constexpr int kD = D, kBytes = 2, kRows = kRowsT;
  static constexpr int kThreads = 288;
  // with more than eight rows the two halves of the warps take the two halves of the rows
  static constexpr int kSplit = kRows > 8 ? 2 : 1;
  static constexpr int kGroups = kRows / 8 / kSplit;
  static constexpr int kTile = 128;  // 64 with 16 rows: 61 instead of 53 us at dim 64
  static constexpr int kBlocks = kTile * kSplit / (16 * kWarps);  // of sixteen keys, a warp's
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
  static constexpr float kLift = 0.f;
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
  // Weights are formed 2^7 times larger: fp16 holds nothing below 2^-25, and a quarter
  // million keys of such weights add up to a percent.  The sums and the merge carry the
  // factor in the maximum, lowered by it.  Below half of 16, so that the lowered maximum
  // of scores past 2^24, where fp32 counts in steps of 2 to 16, leaves weights of 2^8 at most.
  static constexpr float kLift = 7.f;
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
  constexpr int kTile = C::kTile, G = C::kGroups, KB = C::kBlocks;
  constexpr int kKeyWarps = kWarps / C::kSplit;
  const int warp = warp_id(), lane = lane_id();
  DeviceStatus* st = p.status;
  const uint64_t tmo = p.timeout_ns;
  const int g = lane >> 2, t = lane & 3;
  const int key0 = warp % kKeyWarps * (16 * KB);        // this warp's first key of a tile
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
  int tok_g[G];              // that row's token
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
      tok_g[u] = tok;
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
      const int j0 = tile * kTile + key0;
      if (j0 >= c.keys) {  // no key for this warp
        if (lane == 0) mbar_arrive(blk.empty(stage));
        continue;
      }
      const bool tail = j0 + 16 * KB > c.ctx;  // this warp has new tokens, or keys past the end
      // even and odd steps are summed apart, so that products do not wait for one another
      float s2[2][KB][G][4] = {};
#pragma unroll
      for (int b = 0; b < D / 16; ++b)
#pragma unroll
        for (int y = 0; y < KB; ++y) {
          uint32_t a[4];
          ldsm4(a, k_at + stage * C::kStage + y * 2048 + (b >> 2) * (kTile * 128) + k_col[b & 3]);
#pragma unroll
          for (int u = 0; u < G; ++u) H::mma(s2[b & 1][y][u], a, q[u][b]);
        }
      uint32_t wt[G][KB][2];  // weights of keys 2t, 2t + 1 and + 8, + 9 for row g
      float alpha[G][2];
      bool moved = false;
#pragma unroll
      for (int u = 0; u < G; ++u) {
        float s[2 * KB][2];  // keys g + 8 x, rows 2t + i
#pragma unroll
        for (int x = 0; x < 2 * KB; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = 2 * (x & 1) + i;
            s[x][i] = (s2[0][x >> 1][u][at] + s2[1][x >> 1][u][at]) * p.scale_log2;
          }
        if (tail) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int tok = __shfl_sync(0xffffffffu, tok_g[u], 4 * (2 * t + i));
            const bool row = row_w + 8 * u + 2 * t + i < c.rows;
            const uint32_t* words =
                p.mask + static_cast<int64_t>(c.first + tok) * p.mask_stride;
#pragma unroll
            for (int x = 0; x < 2 * KB; ++x) {
              const int j = j0 + g + 8 * x, rel = j - c.ctx;
              bool sees = row && j < c.keys;
              if (p.mask == nullptr)
                sees &= rel <= tok;
              else if (sees && rel >= 0)
                sees = (rel >> 5) < p.mask_w && ((words[rel >> 5] >> (rel & 31)) & 1u);
              if (!sees) s[x][i] = -INFINITY;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = s[0][i];
#pragma unroll
          for (int x = 1; x < 2 * KB; ++x) mx = fmaxf(mx, s[x][i]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m[u][i], mx - H::kLift);
          const float use = mn == -INFINITY ? 0.f : mn;
          alpha[u][i] = ex2_approx(m[u][i] - use);  // m = -inf: 0
          moved |= mn != m[u][i];
          m[u][i] = mn;
          float sum = 0.f;  // of the weights unrounded
#pragma unroll
          for (int x = 0; x < 2 * KB; ++x) {
            s[x][i] = ex2_approx(s[x][i] - use);
            sum += s[x][i];
          }
          l[u][i] = l[u][i] * alpha[u][i] + sum;
        }
#pragma unroll
        for (int x = 0; x < 2 * KB; ++x)
          wt[u][x >> 1][x & 1] = transpose8(H::pack(s[x][0], s[x][1]));
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
      for (int y = 0; y < KB; ++y) {
        const int jb = j0 + 16 * y;
        const bool clean = jb + 16 > c.ctx;
        // Rows past the end count for nothing, whatever they hold; what is not finite
        // among the new tokens is left out here and added at the end.  By halves of a
        // register, keys 2t and 2t + 1, and + 8 in the second:
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu}, fresh[2] = {};
        if (clean) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = jb + 8 * (x >> 1) + 2 * t + (x & 1);
            const uint32_t bits = x & 1 ? 0xffff0000u : 0x0000ffffu;
            if (j >= c.keys) keep[x >> 1] &= ~bits;
            if (j >= c.ctx) fresh[x >> 1] |= bits & (H::kExp * 0x10001u);
          }
        }
#pragma unroll
        for (int b = 0; b < D / 16; ++b) {
          uint32_t a[4];  // columns g and g + 8 of keys 2t, 2t + 1, then of keys 8 later
          ldsm4_t(a, v_at + stage * C::kStage + y * 2048 + (b >> 2) * (kTile * 128) + v_col[b & 3]);
          if (clean) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              a[x] &= keep[x >> 1];
              // an exponent of ones and its lowest bit carry into the sign's place
              const uint32_t hit =
                  ((a[x] & fresh[x >> 1]) + (H::kExp & -H::kExp) * 0x10001u) & 0x80008000u;
              a[x] &= ~((hit >> 15) * 0xffffu);
              dirty |= hit != 0u;
            }
          }
#pragma unroll
          for (int u = 0; u < G; ++u) H::mma(acc[u][b], a, wt[u][y]);
        }
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
  return rows == 8 ? run<T, D, 8>(p, stream) : run<T, D, 16>(p, stream);
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
