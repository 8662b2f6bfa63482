// tree_f32.cu - attention of new tokens over a paged cache in fp32, the merge of
// split units for every element type, and the masks of drafted trees.
//
// Row (token t, head h) of a request with ctx cached tokens sees key j when
// j < ctx, or when j is new token j - ctx and the mask has that bit (without a
// mask: j - ctx <= t):
//   o = sum_j exp(s_j - m) v_j / l,  s_j = scale q . k_j,  l = sum_j exp(s_j - m)
// with the running maximum m and the sums in fp32.  A row that sees nothing
// gives 0 and lse = -inf.
//
// One CTA per SM takes its even share of the work (tree_sched.cuh), 8, 16 or 32 rows of
// a kv head at a time: the widths of one, two or four small tensor-core products, whose
// other side is keys (scores) or columns of V (outputs).  A decoding step so reads the
// cache once at fp32-level accuracy and stays bound by that.  Products are 3xTF32:
// x = hi + lo, hi rounded to 11 bits, and hi*hi + lo*hi + hi*lo; what is left out is
// 2^-22 of a product.
//
// Warp 8 walks the pieces and brings tiles of 64 KB (K and V of 128 keys at dim 64,
// 64 keys at dim 128) by TMA into a ring.  Warps 0-7 take shares of a tile's keys (and,
// of many rows at dim 128, a half of the rows) with their own running maximum, sum and
// outputs in registers, joined once per piece.  Inside a product the order of the summed
// index is free: it is chosen so that every read of K, V and the weights is 8 or 16
// bytes wide and the lanes of one pass meet different banks.
//
// Up to eight rows (f32_narrow) the split queries stay in registers and the ring has
// three stages; more (f32_wide) read them from shared memory, use each split of K and V
// two or four times, and are bound by the tensor core: 17 cycles per product of a
// scheduler, 16 being its rate.  us with units of 8 / 16 / 32 rows, 8 kv heads:
//   rows of a kv head:      8          16            32           2000 (causal chunk)
//   8000 keys, dim 64    14/-/-   19 / 17 / 23   30 / - / 25   1324 / - / 726
//   8000 keys, dim 128   24/-/-   40 / 30 / 37   67 / - / 41   3003 / - / 1474
//   4 x 32000, dim 128            367 / 275 / 371   804 / - / 365
// hence 8, 16 or 32 by the rows of the longest request.
//
// 3 trees over 4096 to 16384 keys, 8 heads x 64 (126 MB, 19 us at the copy rate): 32
// us with the merge, against 39 us with the products on the CUDA cores, which issue
// three times the instructions.
#include "tree_warp.cuh"

namespace rab {

using namespace tree_detail;

namespace {

template <int D, int kRowsT>
struct F32Cfg {
  static constexpr int kD = D, kBytes = 4, kRows = kRowsT;
  static constexpr bool kWide = kRows > 8;
  // whole warpgroups where they pass registers to the computing warps
  static constexpr int kThreads = kWide ? 384 : 288;
  static constexpr int kStages = kWide ? 2 : 3;
  static constexpr int kTile = 8192 / D;  // keys: 32 KB of K
  static constexpr int kHalf = kTile * D * 4;  // bytes of K (or V) of a tile
  static constexpr int kStage = 2 * kHalf;
  // a warp's keys: 16, or 8 (half a product's height) with eight rows of dim 128; more
  // rows of dim 128 go to the two halves of the warps instead
  static constexpr int kSplit = kWide ? kWarps * 16 / kTile : 1;
  static constexpr int kKeys = kTile * kSplit / kWarps;
  static constexpr int kGroups = kRows / 8 / kSplit;  // of eight rows, a warp's
  // floats of a warp: weights [row][key] in the tiles, [row][dim] outputs at a piece's end
  static constexpr int kOwnRow = D;
  static constexpr int kOwn = kGroups * 8 * D;
  static constexpr int kPRow = kKeys + 4;  // between the weights of two rows
  static constexpr int kOwnOff = kStages * kStage;
  // split queries, [row / 8][dim / 16][hi, lo][lane] fragments; eight rows stay in registers
  static constexpr int kQOff = kOwnOff + kWarps * kOwn * 4;
  static constexpr int kQGroup = D / 16 * 1024;  // bytes of eight rows
  static constexpr int kMlOff = kQOff + (kWide ? kRows / 8 * kQGroup : 0);  // float2 [warps][own rows]
  static constexpr int kItemOff = kMlOff + kWarps * kGroups * 8 * 8;
  static constexpr int kBarOff = kItemOff + kItems * 48;
  static constexpr int kBars = 2 * kStages + 2 * kItems + 2;
  static constexpr int kDirtyOff = kBarOff + kBars * 8;  // int [2]
  static constexpr int kSmem = kDirtyOff + 8;
  static_assert(kSmem <= 232448 && kBarOff % 8 == 0, "shared memory");
  static_assert(!kWide || (kKeys == 16 && kGroups >= 1), "rows of a unit");
};

// byte offset of element `col` of row `key` in a tile of [dim / 32][keys][32 floats],
// 16-byte chunks swizzled by the row within 128 bytes
template <int D>
__device__ __forceinline__ int tile_at(int key, int col) {
  return (col >> 5) * (8192 / D * 128) + key * 128 + ((((col >> 2) & 7) ^ (key & 7)) << 4) +
         (col & 3) * 4;
}

// x = hi + lo for a 3xTF32 product, hi the nearest of 11 bits: rounded, lo has either
// sign, and the product lo * lo that is left out does not add up (cut off, it is
// always positive).  An infinity stays in hi, where its product has the right sign; the
// products of lo are summed apart and mean nothing beside it (`whole_score`).
__device__ __forceinline__ void split3x(float x, float& hi, float& lo) {
  const float top = __uint_as_float(sm100::f32_to_tf32(x));
  lo = x - top;
  hi = top;
}

// The same of V, whose products run into one sum: hi stays finite and lo carries an
// infinity, so that only its product with a weight's hi, which is positive, is infinite.
// Costs the split an instruction more: 500 tokens over 8000 keys of 128 take 1474 us, and
// 1570 with K split so as well.
__device__ __forceinline__ void split3x_v(float x, float& hi, float& lo) {
  uint32_t top;
  asm("cvt.rna.satfinite.tf32.f32 %0, %1;" : "=r"(top) : "f"(x));
  hi = __uint_as_float(top);
  lo = x - hi;
}

// a score from its leading products and the small ones
__device__ __forceinline__ float whole_score(float hi, float lo) {
  return hi + (isfinite(lo) ? lo : 0.f);
}

// c += a * b, one 16 x 8 x 8 product of 11-bit operands
__device__ __forceinline__ void mma_tf32(float* c, const float* a, const float* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
        "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b[0])), "r"(__float_as_uint(b[1])));
}

// c + c_lo += a * b at fp32 level.  The tensor core cuts its sums off instead of
// rounding them, so c is a short sum (a tile's), added up in fp32 outside: the results
// of 16384 keys are off by 2.8e-7 relative to 64 bits, and by 1.6e-6 with one long sum.
__device__ __forceinline__ void mma_3x(float* c, float* c_lo, const float* a, const float* a_lo,
                                       const float* b, const float* b_lo) {
  mma_tf32(c_lo, a_lo, b);
  mma_tf32(c_lo, a, b_lo);
  mma_tf32(c, a, b);
}

// A computing warp, eight rows to a unit.
// Fragments of a 16 x 8 x 8 product: lane = 4 g + t.  Scores: rows are keys, columns
// query rows, the summed index is dim; this lane's sums are keys g and g + 8 (of the
// warp's, in the order key_of) of query rows 2t and 2t + 1.  Outputs: rows are columns
// of V, the summed index is keys; this lane's are dims 32 h + 4 g + 0..3 of query rows
// 2t and 2t + 1.
template <int D>
__device__ __forceinline__ void f32_narrow(const TreeParams& p, const WarpBlock<F32Cfg<D, 8>>& blk) {
  using C = F32Cfg<D, 8>;
  using namespace sm100;
  constexpr int kTile = C::kTile, kKeys = C::kKeys;
  const int warp = warp_id(), lane = lane_id();
  DeviceStatus* st = p.status;
  const uint64_t tmo = p.timeout_ns;
  float* own = blk.own(warp);
  float* s_p = own;
  const int g = lane >> 2, t = lane & 3;
  // rows g and g + 1 of one pass lie four keys apart: their swizzled words meet no bank twice
  const int key_g = (g >> 1) + 4 * (g & 1);
  int n = 0;  // tiles taken
  bool ok = true;
  for (int w = 0; ok; ++w) {
    ok = __all_sync(0xffffffffu, mbar_wait(blk.item_full(w), (w / kItems) & 1, st,
                                           kSiteItemQueue, tmo));
    if (!ok) break;
    const Piece c = *blk.item(w);
    if (c.request < 0) break;
    // queries of row g, scaled to base-2 exponents; dim 16 b + 4 t + 0..3 is summed at
    // places t, t + 4 of step 2 b and t, t + 4 of step 2 b + 1
    float q_hi[D / 8][2], q_lo[D / 8][2];
    {
      const int row = c.row0 + min(g, c.rows - 1), tok = row / p.group;
      const int h = c.head_kv * p.group + row - tok * p.group;
      const float* src = static_cast<const float*>(p.q) +
                         static_cast<int64_t>(c.first + tok) * p.q_t +
                         static_cast<int64_t>(h) * p.q_h + 4 * t;
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        const float4 v = *reinterpret_cast<const float4*>(src + 16 * b);
        q_hi[2 * b][0] = v.x * p.scale_log2;
        q_hi[2 * b][1] = v.y * p.scale_log2;
        q_hi[2 * b + 1][0] = v.z * p.scale_log2;
        q_hi[2 * b + 1][1] = v.w * p.scale_log2;
      }
#pragma unroll
      for (int b = 0; b < D / 8; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) split3x(q_hi[b][i], q_hi[b][i], q_lo[b][i]);
    }
    if (w > 0) {  // the piece before has been read out of every warp's outputs
      ok = __all_sync(0xffffffffu, mbar_wait(blk.released(), (w - 1) & 1, st, kSiteOReady, tmo));
      if (!ok) break;
    }
    float acc[D / 16][4];  // [4 h + i]: dims 64 h + 32 e + 4 g + i of rows 2t + r at 2 e + r
#pragma unroll
    for (int b = 0; b < D / 16; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[b][i] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows 2t + i; l is this lane's share
    bool dirty = false;

    for (int tile = c.tile_begin; tile < c.tile_end; ++tile, ++n) {
      const int stage = n % C::kStages;
      ok = __all_sync(0xffffffffu, mbar_wait(blk.full(stage), (n / C::kStages) & 1, st, kSiteKFull,
                                             tmo));
      if (!ok) break;
      const int j0 = tile * kTile + warp * kKeys;
      if (j0 >= c.keys) {  // no key for this warp
        if (lane == 0) mbar_arrive(blk.empty(stage));
        continue;
      }
      const bool tail = j0 + kKeys > c.ctx;  // this warp has new tokens, or keys past the end
      const uint8_t* sk = blk.smem + stage * C::kStage;
      const uint8_t* sv = sk + C::kHalf;
      // even and odd steps are summed apart, so that products do not wait for one
      // another, and so are the small products (below)
      float s2[2][4] = {}, s_lo[4] = {};
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        float k_hi[2][4], k_lo[2][4];  // of the steps 2 b and 2 b + 1
#pragma unroll
        for (int hlf = 0; hlf < 2; ++hlf) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (hlf == 0 || kKeys == 16)  // with eight keys the lower rows stay empty
            v = *reinterpret_cast<const float4*>(
                sk + tile_at<D>(warp * kKeys + key_g + 8 * hlf, 16 * b + 4 * t));
          k_hi[0][hlf] = v.x;
          k_hi[0][2 + hlf] = v.y;
          k_hi[1][hlf] = v.z;
          k_hi[1][2 + hlf] = v.w;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) split3x(k_hi[e][i], k_hi[e][i], k_lo[e][i]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          mma_3x(s2[e], s_lo, k_hi[e], k_lo[e], q_hi[2 * b + e], q_lo[2 * b + e]);
      }
      constexpr int kMine = kKeys / 8;  // keys of this lane
      float s[kMine][2];
#pragma unroll
      for (int u = 0; u < kMine; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          s[u][i] = whole_score(s2[0][2 * u + i] + s2[1][2 * u + i], s_lo[2 * u + i]);
      if (tail) {
#pragma unroll
        for (int u = 0; u < kMine; ++u) {
          const int j = j0 + key_g + 8 * u, rel = j - c.ctx;
          if (rel < 0) continue;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 2 * t + i;
            bool sees = j < c.keys && r < c.rows;
            if (sees) {
              const int tok = (c.row0 + r) / p.group;
              sees = p.mask == nullptr
                         ? rel <= tok
                         : (rel >> 5) < p.mask_w &&
                               ((p.mask[static_cast<int64_t>(c.first + tok) * p.mask_stride +
                                        (rel >> 5)] >>
                                 (rel & 31)) &
                                1u);
            }
            if (!sees) s[u][i] = -INFINITY;
          }
        }
      }
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = s[0][i];
        if constexpr (kMine == 2) mx = fmaxf(mx, s[1][i]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float mn = fmaxf(m[i], mx);
        const float use = mn == -INFINITY ? 0.f : mn;
        alpha[i] = ex2_approx(m[i] - use);  // m = -inf: 0
        m[i] = mn;
        l[i] *= alpha[i];
#pragma unroll
        for (int u = 0; u < kMine; ++u) {
          const float e = ex2_approx(s[u][i] - use);
          l[i] += e;
          s_p[(2 * t + i) * C::kPRow + key_g + 8 * u] = e;
        }
      }
      __syncwarp();
      float part[D / 16][4];  // this tile's, laid out as acc
#pragma unroll
      for (int b = 0; b < D / 16; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[b][i] = 0.f;
#pragma unroll
      for (int step = 0; step < kKeys / 8; ++step) {
        // keys 8 step + 2t and + 1 are summed at places t and t + 4
        const float2 w2 =
            *reinterpret_cast<const float2*>(s_p + g * C::kPRow + 8 * step + 2 * t);
        float w_hi[2], w_lo[2];
        split3x(w2.x, w_hi[0], w_lo[0]);
        split3x(w2.y, w_hi[1], w_lo[1]);
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          float v[2][2][4];  // [key][columns 64 h + 32 e + 4 g ..]
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int k = warp * kKeys + 8 * step + 2 * t + u;
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<float4*>(v[u][e]) =
                  *reinterpret_cast<const float4*>(sv + tile_at<D>(k, 64 * h + 32 * e + 4 * g));
            if (tail) {
              // rows past the end count for nothing, whatever they hold; what is not
              // finite among the new tokens is left out here and added at the end
              const int rel = tile * kTile + k - c.ctx;
              if (rel >= 0) {
                const bool past = tile * kTile + k >= c.keys;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    dirty |= !past && !isfinite(v[u][e][i]);
                    if (past || !isfinite(v[u][e][i])) v[u][e][i] = 0.f;
                  }
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a[4], a_lo[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) split3x_v(v[x >> 1][x & 1][i], a[x], a_lo[x]);
            mma_3x(part[4 * h + i], part[4 * h + i], a, a_lo, w_hi, w_lo);
          }
        }
      }
      __syncwarp();  // s_p and the stage have been read
      if (lane == 0) mbar_arrive(blk.empty(stage));
#pragma unroll
      for (int b = 0; b < D / 16; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[b][i] = fmaf(acc[b][i], alpha[i & 1], part[b][i]);
    }
    if (!ok) break;

    // join the warps
    if (dirty) blk.dirty()[w & 1] = w + 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
      if (g == 0) blk.ml(warp, 2 * t + i) = make_float2(m[i], l[i]);
    }
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float4*>(own + (2 * t + i) * D + 64 * h + 32 * e + 4 * g) =
              make_float4(acc[4 * h][2 * e + i], acc[4 * h + 1][2 * e + i],
                          acc[4 * h + 2][2 * e + i], acc[4 * h + 3][2 * e + i]);
    __syncwarp();
    if (lane == 0) mbar_arrive(blk.joined());
    ok = __all_sync(0xffffffffu, mbar_wait(blk.joined(), w & 1, st, kSiteOReady, tmo));
    if (!ok) break;
    write_results<C, float>(p, blk, c, w);
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(blk.released());
      mbar_arrive(blk.item_empty(w));
    }
  }
}

// A computing warp, 16 or 32 rows to a unit: the fragments of f32_narrow, with every
// split of K and V used for the warp's kGroups groups of eight rows.  Warp u takes the
// groups of the unit from (u / key warps) * kGroups on.
template <int D, int kRows>
__device__ __forceinline__ void f32_wide(const TreeParams& p,
                                         const WarpBlock<F32Cfg<D, kRows>>& blk) {
  using C = F32Cfg<D, kRows>;
  using namespace sm100;
  constexpr int kTile = C::kTile, kKeys = C::kKeys, G = C::kGroups;
  constexpr int kKeyWarps = kWarps / C::kSplit;
  const int warp = warp_id(), lane = lane_id();
  DeviceStatus* st = p.status;
  const uint64_t tmo = p.timeout_ns;
  float* own = blk.own(warp);
  float* s_p = own;
  const int g = lane >> 2, t = lane & 3;
  const int key_g = (g >> 1) + 4 * (g & 1);
  const int key0 = warp % kKeyWarps * kKeys;      // this warp's first key of a tile
  const int row_w = warp / kKeyWarps * (8 * G);   // and its first row of the unit
  int n = 0;  // tiles taken
  bool ok = true;
  for (int w = 0; ok; ++w) {
    ok = __all_sync(0xffffffffu,
                    mbar_wait(blk.item_full(w), (w / kItems) & 1, st, kSiteItemQueue, tmo));
    if (!ok) break;
    const Piece c = *blk.item(w);
    if (c.request < 0) break;
    // The warps split the unit's queries, scaled to base-2 exponents: this one the 16
    // columns b of every eight rows.  Every warp has left the piece before (`joined`).
    for (int b = warp; b < D / 16; b += kWarps) {
#pragma unroll
      for (int u = 0; u < kRows / 8; ++u) {
        const int row = c.row0 + min(8 * u + g, c.rows - 1), tok = row / p.group;
        const int h = c.head_kv * p.group + row - tok * p.group;
        const float4 v = *reinterpret_cast<const float4*>(
            static_cast<const float*>(p.q) + static_cast<int64_t>(c.first + tok) * p.q_t +
            static_cast<int64_t>(h) * p.q_h + 16 * b + 4 * t);
        float4 hi, lo;
        split3x(v.x * p.scale_log2, hi.x, lo.x);
        split3x(v.y * p.scale_log2, hi.y, lo.y);
        split3x(v.z * p.scale_log2, hi.z, lo.z);
        split3x(v.w * p.scale_log2, hi.w, lo.w);
        float4* dst =
            reinterpret_cast<float4*>(blk.smem + C::kQOff + u * C::kQGroup + b * 1024) + lane;
        dst[0] = hi;
        dst[32] = lo;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(blk.released());
    // the queries are there, and the piece before has been read out of every warp's outputs
    ok = __all_sync(0xffffffffu, mbar_wait(blk.released(), w & 1, st, kSiteOReady, tmo));
    if (!ok) break;
    float acc[G][D / 16][4];
    float m[G][2], l[G][2];
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
      const bool tail = j0 + kKeys > c.ctx;  // this warp has new tokens, or keys past the end
      const uint8_t* sk = blk.smem + stage * C::kStage;
      const uint8_t* sv = sk + C::kHalf;
      const float4* sq =
          reinterpret_cast<const float4*>(blk.smem + C::kQOff + row_w / 8 * C::kQGroup) + lane;
      float s[G][4] = {}, s_lo[G][4] = {};
#pragma unroll
      for (int b = 0; b < D / 16; ++b) {
        float k_hi[2][4], k_lo[2][4];
#pragma unroll
        for (int hlf = 0; hlf < 2; ++hlf) {
          const float4 v = *reinterpret_cast<const float4*>(
              sk + tile_at<D>(key0 + key_g + 8 * hlf, 16 * b + 4 * t));
          split3x(v.x, k_hi[0][hlf], k_lo[0][hlf]);
          split3x(v.y, k_hi[0][2 + hlf], k_lo[0][2 + hlf]);
          split3x(v.z, k_hi[1][hlf], k_lo[1][hlf]);
          split3x(v.w, k_hi[1][2 + hlf], k_lo[1][2 + hlf]);
        }
        float4 hi[G], lo[G];
#pragma unroll
        for (int u = 0; u < G; ++u) {
          hi[u] = sq[u * (C::kQGroup / 16) + b * 64];
          lo[u] = sq[u * (C::kQGroup / 16) + b * 64 + 32];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int u = 0; u < G; ++u) mma_tf32(s_lo[u], k_lo[e], e == 0 ? &hi[u].x : &hi[u].z);
#pragma unroll
          for (int u = 0; u < G; ++u) mma_tf32(s[u], k_hi[e], e == 0 ? &hi[u].x : &hi[u].z);
#pragma unroll
          for (int u = 0; u < G; ++u) mma_tf32(s_lo[u], k_hi[e], e == 0 ? &lo[u].x : &lo[u].z);
        }
      }
      float alpha[G][2];
#pragma unroll
      for (int u = 0; u < G; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = whole_score(s[u][i], s_lo[u][i]);  // [2 key + row]
        if (tail) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = row_w + 8 * u + 2 * t + i;
            const int tok = (c.row0 + r) / p.group;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int j = j0 + key_g + 8 * x, rel = j - c.ctx;
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
              if (!sees) s[u][2 * x + i] = -INFINITY;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(s[u][i], s[u][2 + i]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float mn = fmaxf(m[u][i], mx);
          const float use = mn == -INFINITY ? 0.f : mn;
          alpha[u][i] = ex2_approx(m[u][i] - use);  // m = -inf: 0
          m[u][i] = mn;
          l[u][i] *= alpha[u][i];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float e = ex2_approx(s[u][2 * x + i] - use);
            l[u][i] += e;
            s_p[(8 * u + 2 * t + i) * C::kPRow + key_g + 8 * x] = e;
          }
        }
      }
      __syncwarp();
      // keys 8 step + 2t and + 1 are summed at places t and t + 4 of a step
      float w_hi[2][G][2], w_lo[2][G][2];
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int u = 0; u < G; ++u) {
          const float2 w2 = *reinterpret_cast<const float2*>(s_p + (8 * u + g) * C::kPRow +
                                                             8 * step + 2 * t);
          split3x(w2.x, w_hi[step][u][0], w_lo[step][u][0]);
          split3x(w2.y, w_hi[step][u][1], w_lo[step][u][1]);
        }
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        float v[2][2][2][4];  // [step][key][columns 64 h + 32 e + 4 g ..]
#pragma unroll
        for (int step = 0; step < 2; ++step)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int k = key0 + 8 * step + 2 * t + x;
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<float4*>(v[step][x][e]) =
                  *reinterpret_cast<const float4*>(sv + tile_at<D>(k, 64 * h + 32 * e + 4 * g));
            if (tail) {
              // rows past the end count for nothing, whatever they hold; what is not
              // finite among the new tokens is left out here and added at the end
              const int rel = tile * kTile + k - c.ctx;
              if (rel >= 0) {
                const bool past = tile * kTile + k >= c.keys;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    dirty |= !past && !isfinite(v[step][x][e][i]);
                    if (past || !isfinite(v[step][x][e][i])) v[step][x][e][i] = 0.f;
                  }
              }
            }
          }
        // four sums at once, so that products do not wait for one another
        constexpr int kI = G >= 4 ? 1 : 4 / G;
#pragma unroll
        for (int i0 = 0; i0 < 4; i0 += kI) {
          float part[kI][G][4] = {};
#pragma unroll
          for (int step = 0; step < 2; ++step) {
            float a[kI][4], a_lo[kI][4];
#pragma unroll
            for (int i = 0; i < kI; ++i)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                split3x_v(v[step][x >> 1][x & 1][i0 + i], a[i][x], a_lo[i][x]);
#pragma unroll
            for (int i = 0; i < kI; ++i)
#pragma unroll
              for (int u = 0; u < G; ++u) mma_tf32(part[i][u], a_lo[i], w_hi[step][u]);
#pragma unroll
            for (int i = 0; i < kI; ++i)
#pragma unroll
              for (int u = 0; u < G; ++u) mma_tf32(part[i][u], a[i], w_lo[step][u]);
#pragma unroll
            for (int i = 0; i < kI; ++i)
#pragma unroll
              for (int u = 0; u < G; ++u) mma_tf32(part[i][u], a[i], w_hi[step][u]);
          }
#pragma unroll
          for (int i = 0; i < kI; ++i)
#pragma unroll
            for (int u = 0; u < G; ++u)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                acc[u][4 * h + i0 + i][x] =
                    fmaf(acc[u][4 * h + i0 + i][x], alpha[u][x & 1], part[i][u][x]);
        }
      }
      __syncwarp();  // s_p and the stage have been read
      if (lane == 0) mbar_arrive(blk.empty(stage));
    }
    if (!ok) break;

    // join the key warps
    if (dirty) blk.dirty()[w & 1] = w + 1;
#pragma unroll
    for (int u = 0; u < G; ++u) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[u][i] += __shfl_xor_sync(0xffffffffu, l[u][i], d);
        if (g == 0) blk.ml(warp, 8 * u + 2 * t + i) = make_float2(m[u][i], l[u][i]);
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float4*>(own + (8 * u + 2 * t + i) * D + 64 * h + 32 * e + 4 * g) =
                make_float4(acc[u][4 * h][2 * e + i], acc[u][4 * h + 1][2 * e + i],
                            acc[u][4 * h + 2][2 * e + i], acc[u][4 * h + 3][2 * e + i]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(blk.joined());
    ok = __all_sync(0xffffffffu, mbar_wait(blk.joined(), w & 1, st, kSiteOReady, tmo));
    if (!ok) break;
    write_results<C, float>(p, blk, c, w);
    __syncwarp();
    if (lane == 0) mbar_arrive(blk.item_empty(w));
  }
}

template <int D, int kRows>
__global__ void __launch_bounds__(F32Cfg<D, kRows>::kThreads, 1)
    tree_f32_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV) {
  using C = F32Cfg<D, kRows>;
  using namespace sm100;
  extern __shared__ __align__(1024) uint8_t smem[];
  const WarpBlock<C> blk{smem};
  if (!start_block<C>(p, blk)) return;

  if (warp_id() >= kWarps) {
    // the wide sums take 216 registers: 2 x 216 + 72 is the block's 3 x 168
    if constexpr (C::kWide) warpgroup_reg_dec<72>();
    if (warp_id() == kWarps) walk_and_load<C>(p, tmK, tmV, blk);
  } else if constexpr (C::kWide) {
    warpgroup_reg_inc<216>();
    f32_wide<D, kRows>(p, blk);
  } else {
    f32_narrow<D>(p, blk);
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

template <int D, int kRows>
int run_f32(const TreeParams& p, cudaStream_t stream) {
  static bool done[64] = {};
  return launch_warp_kernel<F32Cfg<D, kRows>>(tree_f32_kernel<D, kRows>, done, p, stream);
}

template <int D>
int run_f32_rows(const TreeParams& p, int rows, cudaStream_t stream) {
  return rows == 8    ? run_f32<D, 8>(p, stream)
         : rows == 16 ? run_f32<D, 16>(p, stream)
                      : run_f32<D, 32>(p, stream);
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
  const int64_t rows = static_cast<int64_t>(max_q) * p.group;
  if (elem == Elem::kF32) {
    // the least width that holds the rows: a wider one computes on empty rows, a
    // narrower one reads and splits the cache again (times at the file's head)
    plan.rows_per_unit = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    plan.tile_keys = 8192 / p.dim;
  } else {
    // few rows: tree_few.cu (times at its head); above them, one row tile of the large
    // tensor cores keeps two key tiles in the air per CTA and suits what reading the
    // cache bounds, and from the second row tile on, both share every key tile
    plan.rows_per_unit = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 128 ? 128 : 256;
    plan.tile_keys = 128;
  }
  plan.grid = sms;
  // rows of the largest unit that can occur (max_q is a hint: the merge loops)
  plan.merge_rows = static_cast<int>(rows < plan.rows_per_unit ? rows : plan.rows_per_unit);
  const size_t recs = static_cast<size_t>(2) * plan.grid * plan.rows_per_unit;
  plan.acc_floats = recs * p.dim;
  plan.ml_floats = 2 * recs;
  plan.meta_ints = static_cast<size_t>(plan.grid) * kMetaInts;
  return plan;
}

int tree_launch(Elem elem, const TreeParams& p, const TreePlan& plan, cudaStream_t stream) {
  const int rows = plan.rows_per_unit;
  int err;
  if (elem == Elem::kF32)
    err = p.dim == 64 ? run_f32_rows<64>(p, rows, stream) : run_f32_rows<128>(p, rows, stream);
  else if (rows <= 16)
    err = tree_few_launch(elem, p, rows, stream);
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
