// tree_sm100.cu - attention of new tokens over a paged cache on the tensor
// cores (bf16 and fp16), for B200 (sm_100a).
//
// The rows of a unit are the (new token, query head) pairs that share a kv head,
// token-major, and K and V are read once for all of them (calls of up to 16 rows are
// tree_few.cu's).  Up to 128 rows the work is bound by reading the cache; a tile of 128
// keys (64 KB at dim 128) takes an SM
// about 1.5 us at the measured 6.55 TB/s, while QK, softmax and PV of the tile
// follow one another and take longer than that in a row.  So two chains run side
// by side in one CTA:
//   kTwoRows = 0  (a unit is 128 rows): chain x takes the key tiles of parity x,
//                 with its own scores, maxima, sums and outputs; the two are
//                 joined when the piece ends, as split records are joined.
//   kTwoRows = 1  (a unit is 256 rows): chain x takes row tile x, both use every
//                 key tile, so a tile read once serves 256 rows (work bound by the
//                 tensor cores: chunks of prompts, wide trees).
//
// CTA = 12 warps, persistent over the pieces of its even share (tree_sched.cuh):
//   warp 0      walks the pieces, looks pages up (a lane per page) and issues the
//               TMA loads of K and V, one box per page and 64 columns
//   warp 1      MMA issuer (one thread), TMEM owner
//   warps 2-3   queries: gathered rows, 16-byte asynchronous copies, swizzled
//   warps 4-7   softmax and results of chain 0, warps 8-11 of chain 1
// TMEM: S_0 [0,128) S_1 [128,256) O_0 [256,..) O_1 [384,..); P lies over S.
//
// Keys no row may see: the score is replaced by -inf, so K may hold anything.  V
// enters a product with a weight of zero, which a NaN or infinity would survive,
// so in the tiles that hold new tokens or the end of the cache the softmax warps
// clean V in shared memory first: rows past the end become zeros, and what is not
// finite among the new tokens is taken out and, for the rows that do see it, added
// to the result at the end (a path no sane cache takes).
//
// Weights are rounded to the element type for their product with V, since the tensor
// cores take both operands in one type, and summed unrounded: off by half a step of a
// weight each, 2.2e-3 of the result in bf16 where the last rounding alone is 1.7e-3.
//
// Every wait is bounded; no TMA load uses cluster broadcast.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.h"
#include "paged.h"
#include "sm100.cuh"
#include "tree_sched.cuh"

namespace rab {

using namespace sm100;
using namespace tree_detail;

namespace {

constexpr int kThreads = 384;
constexpr int kN = 128;  // keys of a tile
constexpr int kM = 128;  // rows of a chain
constexpr uint32_t kCols = 512;
constexpr float kRescale = 8.0f;  // the running maximum moves when it grows by 2^8
// fp16 weights are formed 2^7 times larger, at most 2^15 until the maximum moves: fp16
// holds nothing below 2^-25, and many such weights of a long context add up.  7 and not
// more as in tree_few.cu.
constexpr float kLiftF16 = 7.0f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr uint32_t kRegsLaunch = 168;
constexpr uint32_t kRegsLow = 72;
constexpr uint32_t kRegsHigh = 216;
static_assert(128 * kRegsLow + 256 * kRegsHigh <= kRegsLaunch * kThreads,
              "register split exceeds the launch allocation");
constexpr int kItems = 4;  // queue of pieces

template <int D, bool kTwoRows>
struct Cfg {
  static constexpr int kTile = kN * D * 2;  // bytes of a K or V tile
  static constexpr int kQBytes = (kTwoRows ? 2 : 1) * kM * D * 2;
  // K and V tiles take turns in one ring: what is left of 227 KB beside the queries
  static constexpr int kStages = D == 64 ? (kTwoRows ? 10 : 12) : (kTwoRows ? 5 : 6);
  // softmax hands P over in this many parts: with two, the PV products of the first
  // 64 keys start while the second half's exponentials form
  static constexpr int kParts = kTwoRows ? 2 : 1;
  static constexpr int kBars = 2 * kStages + 2 + 2 + 2 + 4 + 2 * kItems + 2;
  static constexpr int kBarOff = kQBytes + kStages * kTile;
  static constexpr int kMlOff = kBarOff + kBars * 8;       // float2 [2][128]
  static constexpr int kItemOff = kMlOff + 2 * kM * 8;     // Piece [kItems]
  static constexpr int kMiscOff = kItemOff + kItems * 48;  // int [4]
  static constexpr int kSmem = kMiscOff + 16;
  static_assert(kMlOff % 8 == 0 && kMiscOff % 8 == 0 && kSmem <= 232448, "shared memory");
  static_assert(sizeof(Piece) <= 48, "piece");
};

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBF16) return pack_bf16x2(lo, hi);
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <bool kBF16>
__device__ __forceinline__ bool not_finite(uint32_t h) {  // the low 16 bits
  constexpr uint32_t e = kBF16 ? 0x7f80u : 0x7c00u;
  return (h & e) == e;
}

template <bool kBF16>
__device__ __forceinline__ float widen(uint32_t h) {
  if constexpr (kBF16) return __uint_as_float(h << 16);
  float f;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.f32.f16 %0, t;\n\t}" : "=f"(f) : "r"(h));
  return f;
}

// The 32 columns of new tokens rel0 .. rel0 + 31 that token t of the request
// sees, as bits; places before the new tokens (rel < 0) are cached and seen.
__device__ __forceinline__ uint32_t seen_bits(const TreeParams& p, const Piece* c, int t,
                                              int rel0) {
  int n = min(c->tokens, c->keys - c->ctx) - rel0;  // columns that hold a key
  uint32_t bits;
  if (p.mask == nullptr) {
    n = min(n, t - rel0 + 1);
    bits = 0xffffffffu;
  } else {
    const uint32_t* row = p.mask + static_cast<int64_t>(c->first + t) * p.mask_stride;
    const int w = rel0 >> 5, sh = rel0 & 31;
    auto word = [&](int i) { return i < 0 ? 0xffffffffu : (i < p.mask_w ? row[i] : 0u); };
    const uint32_t lo = word(w);
    const uint32_t hi = sh ? word(w + 1) : 0u;
    bits = __funnelshift_r(lo, hi, sh);
  }
  if (n <= 0) return 0u;
  return n < 32 ? bits & ((1u << n) - 1u) : bits;
}

// V rows [vr0, vr1) of a tile whose first key is k0, by 128 threads: rows at or
// past `keys` become zeros (up to the end of the last page: behind it TMA wrote
// zeros), and among the new tokens (from ctx on) what is not finite does; true when
// this thread took something out.
template <int D, bool kBF16>
__device__ __noinline__ bool clean_v(uint8_t* tile, int k0, int ctx, int keys, int page_size,
                                     int vr0, int vr1, int tid) {
  constexpr int kPerRow = D / 8;
  bool dirty = false;
  vr0 = max(vr0, ctx - k0);
  vr1 = min(vr1, ((keys + page_size - 1) & ~(page_size - 1)) - k0);
  for (int i = vr0 * kPerRow + tid; i < vr1 * kPerRow; i += 128) {
    const int vr = i / kPerRow, ch = i % kPerRow;
    uint4* at = reinterpret_cast<uint4*>(tile + (ch / 8) * (kN * 128) + vr * 128 + (ch % 8) * 16);
    if (k0 + vr >= keys) {
      *at = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    const uint4 v = *at;
    uint32_t e[4] = {v.x, v.y, v.z, v.w};
    bool hit = false;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (not_finite<kBF16>(e[u])) e[u] &= 0xffff0000u, hit = true;
      if (not_finite<kBF16>(e[u] >> 16)) e[u] &= 0x0000ffffu, hit = true;
    }
    if (hit) {
      *at = make_uint4(e[0], e[1], e[2], e[3]);
      dirty = true;
    }
  }
  return dirty;
}

// Adds what clean_v took out to columns [k0, k1) of a result this thread has
// just written (a record's row, or the output row), for the keys its token sees.
template <bool kBF16>
__device__ __noinline__ void add_taken_out(const TreeParams& p, const Piece* c, int t, int k0,
                                           int k1, int dim, float* rec, uint16_t* dst) {
  const int lo = max(c->ctx, c->tile_begin * kN), hi = min(c->keys, c->tile_end * kN);
  const int* table = p.table + static_cast<int64_t>(c->request) * p.table_stride;
  for (int key = lo; key < hi; ++key) {
    const int rel = key - c->ctx;
    if (!((seen_bits(p, c, t, rel & ~31) >> (rel & 31)) & 1u)) continue;
    const int page = table[key >> p.page_shift];
    if (page < 0 || page >= p.num_pages) continue;
    const uint16_t* src =
        static_cast<const uint16_t*>(p.v) + page * p.v_page +
        (static_cast<int64_t>(c->head_kv) * p.page_size + (key & (p.page_size - 1))) * dim;
    for (int k = k0; k < k1; ++k) {
      if (!not_finite<kBF16>(src[k])) continue;
      const float v = widen<kBF16>(src[k]);
      if (rec != nullptr) {
        rec[(k & ~3) * c->rows + (k & 3)] += v;
      } else {
        dst[k] = static_cast<uint16_t>(pack2<kBF16>(widen<kBF16>(dst[k]) + v, 0.f));
      }
    }
  }
}

template <int D, bool kBF16, bool kTwoRows>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attn_kernel(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV) {
  using C = Cfg<D, kTwoRows>;
  constexpr int NS = C::kStages;
  constexpr int kRows = kTwoRows ? 2 * kM : kM;
  constexpr uint32_t kFmt = kBF16 ? kFmtBF16 : kFmtF16;
  constexpr uint32_t kIdescQK = make_idesc(kFmt, kFmt, kM, kN, kMajorK, kMajorK);
  constexpr uint32_t kIdescPV = make_idesc(kFmt, kFmt, kM, D, kMajorK, kMajorMN);
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + C::kQBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);  // [NS]
  uint64_t* empty = full + NS;                                      // [NS]
  uint64_t* q_full = empty + NS;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_full + 2;  // [2]
  uint64_t* p_full = q_full + 4;  // [2]
  uint64_t* o_final = q_full + 6;
  uint64_t* o_free = q_full + 7;
  uint64_t* joined = q_full + 8;
  uint64_t* drain = q_full + 9;
  uint64_t* item_full = q_full + 10;           // [kItems]
  uint64_t* item_empty = item_full + kItems;   // [kItems]
  uint64_t* p_hi = item_empty + kItems;        // [2], with two parts
  float2* s_ml = reinterpret_cast<float2*>(smem + C::kMlOff);
  int* s_misc = reinterpret_cast<int*>(smem + C::kMiscOff);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_misc);
  volatile int* s_dirty = s_misc + 2;  // [2], by the piece's parity
  auto item_slot = [&](int w) {
    return reinterpret_cast<Piece*>(smem + C::kItemOff + (w % kItems) * 48);
  };

  const uint32_t warp = warp_id();
  DeviceStatus* st = p.status;
  const uint64_t tmo = p.timeout_ns;
  // the swizzle of the tiles counts from 1024-byte boundaries; the block has no
  // other shared memory, so its dynamic part starts on one
  if ((smem_u32(smem) & 1023u) != 0) {
    wait_for_predecessor();
    if (threadIdx.x == 0) {
      p.meta[blockIdx.x * kMetaInts] = 0;
      st_record(st, kStatusBadArgs, kSiteNone);
    }
    return;
  }

  if (threadIdx.x == 64) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 64);
    mbar_init(q_empty, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4);
      mbar_init(&p_hi[x], 4);
    }
    mbar_init(o_final, 1);
    mbar_init(o_free, 8);
    mbar_init(joined, 8);
    mbar_init(drain, 1);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 1 + 2 + 8);  // MMA thread, query warps, softmax warps
    }
    s_dirty[0] = s_dirty[1] = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, kCols);
    tmem_relinquish();
  } else if (warp >= 4) {  // the rows that no query will fill (below, among the queries)
    for (int i = threadIdx.x - 128; i < C::kQBytes / 16; i += kThreads - 128)
      reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  let_successor_start();
  __syncthreads();
  tc_fence_after();
  wait_for_predecessor();
  const uint32_t tmem = *s_tmem;

  if (warp < 4) {
    warpgroup_reg_dec<kRegsLow>();
    if (warp == 0) {
      // ------------------------------------------------------ pieces and loads
      const int lane = lane_id();
      if (lane == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
      }
      Range range;
      Start first;
      const int walker = find_range<kN, kRows>(p, &range, &first);
      Walk<kN, kRows> walk;
      if (lane == walker) {
        p.meta[blockIdx.x * kMetaInts] = 0;  // by the lane that may set it later
        walk.start(p, range, first);
      }
      const int rows_box = min(p.page_size, kN);
      const int boxes = kN / rows_box * (D / 64);
      int n = 0;  // loads issued (K and V tiles)
      bool ok = true;
      for (int w = 0; ok; ++w) {
        if (w >= kItems)
          ok = __all_sync(0xffffffffu, mbar_wait(&item_empty[w % kItems], (w / kItems - 1) & 1, st,
                                                 kSiteItemQueue, tmo));
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
        if (lane == 0) mbar_arrive(&item_full[w % kItems]);
        if (c.request < 0) break;
        const int* table = p.table + static_cast<int64_t>(c.request) * p.table_stride;
        const int last_entry = (c.keys - 1) >> p.page_shift;
        for (int tile = c.tile_begin; tile < c.tile_end && ok; ++tile) {
          // this lane's box: page, rows within the tile, 64-column half
          const int half = lane % (D / 64), part = lane / (D / 64);
          int page = p.num_pages, token = 0;
          if (lane < boxes) {
            const int key = tile * kN + part * rows_box;
            const int entry = key >> p.page_shift;
            token = key & (p.page_size - 1);
            // behind the last key: a page coordinate past the pool loads zeros
            if (entry <= last_entry) {
              page = table[entry];
              if (page < 0 || page >= p.num_pages) {
                if (half == 0) st_record(st, kStatusBadArgs, kBadPage, static_cast<uint32_t>(page));
                page = p.num_pages;
              }
            }
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int stage = n % NS;
            ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], ((n / NS) & 1) ^ 1, st,
                                                   kv ? kSiteVEmpty : kSiteKEmpty, tmo));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[stage], C::kTile);
            __syncwarp();
            if (lane < boxes)
              tma_load_4d(sKV + stage * C::kTile + half * (kN * 128) + part * rows_box * 128,
                          kv ? &tmV : &tmK, &full[stage], half * 64, token, c.head_kv, page);
            ++n;
          }
        }
      }
      // the loads in flight land before the block gives its memory back
      for (int i = 0; i < NS && i < n; ++i) {
        const int k = n - 1 - i;
        mbar_wait(&full[k % NS], (k / NS) & 1, nullptr, kSiteKFull, 100000000ull);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA
      if (elect_one()) {
        int g0 = 0;  // tiles of the pieces before this one
        int px[2] = {0, 0};  // P tiles taken from each chain
        bool ok = true;
        const uint32_t kvb = smem_u32(sKV), qb0 = smem_u32(sQ);
        auto wait_tile = [&](int idx, uint32_t site) {
          return mbar_wait(&full[idx % NS], (idx / NS) & 1, st, site, tmo);
        };
        auto qk = [&](int x, int g, int qtile) {
          const uint32_t kb = kvb + (2 * g % NS) * C::kTile;
          const uint32_t qb = qb0 + qtile * (kM * D * 2);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t sub = ks >> 2, inner = (ks & 3) * 32;
            mma_ss<false>(tmem + x * 128, make_sdesc(qb + sub * (kM * 128) + inner, 16, 1024),
                          make_sdesc(kb + sub * (kN * 128) + inner, 16, 1024), kIdescQK,
                          ks ? 1u : 0u);
          }
          mma_commit(&s_full[x]);
        };
        auto pv = [&](int x, int g, bool first) -> bool {
          const uint32_t vb = kvb + ((2 * g + 1) % NS) * C::kTile;
#pragma unroll
          for (int ks = 0; ks < kN / 16; ++ks) {
            if (C::kParts == 2 && ks == kN / 32) {
              if (!mbar_wait(&p_hi[x], px[x] & 1, st, kSitePFull, tmo)) return false;
              tc_fence_after();
            }
            mma_ts<false>(tmem + 256 + x * 128, tmem + x * 128 + ks * 8,
                          make_sdesc(vb + ks * 2048, kN * 128, 1024), kIdescPV,
                          (first && ks == 0) ? 0u : 1u);
          }
          ++px[x];
          return true;
        };
        auto wait_p = [&](int x) {
          return mbar_wait(&p_full[x], px[x] & 1, st, kSitePFull, tmo);
        };
        for (int w = 0; ok; ++w) {
          ok = mbar_wait(&item_full[w % kItems], (w / kItems) & 1, st, kSiteItemQueue, tmo);
          if (!ok) break;
          const Piece c = *item_slot(w);
          mbar_arrive(&item_empty[w % kItems]);
          if (c.request < 0) break;
          const int n = c.tile_end - c.tile_begin;
          ok = mbar_wait(q_full, w & 1, st, kSiteQFull, tmo);
          if (!ok) break;
          tc_fence_after();
          // the results of the piece before have left the accumulators
          auto wait_o = [&]() {
            return w == 0 || mbar_wait(o_free, (w - 1) & 1, st, kSiteOReady, tmo);
          };
          if constexpr (!kTwoRows) {
            auto next_qk = [&](int j) -> bool {
              if (!wait_tile(2 * (g0 + j), kSiteKFull)) return false;
              tc_fence_after();
              qk(j & 1, g0 + j, 0);
              mma_commit(&empty[2 * (g0 + j) % NS]);
              if (j == n - 1) mma_commit(q_empty);
              return true;
            };
            ok = next_qk(0) && (n < 2 || next_qk(1));
            for (int j = 0; j < n && ok; ++j) {
              const int x = j & 1;
              ok = wait_p(x) && wait_tile(2 * (g0 + j) + 1, kSiteVFull) && (j > 0 || wait_o());
              if (!ok) break;
              tc_fence_after();
              ok = pv(x, g0 + j, j < 2);
              if (!ok) break;
              mma_commit(&empty[(2 * (g0 + j) + 1) % NS]);
              if (j + 2 < n) ok = next_qk(j + 2);
            }
          } else {
            auto do_pv = [&](int x, int j) -> bool {
              if (!wait_p(x)) return false;
              // a tile whose V both chains clean: each has done its half
              if (x == 0 && (c.tile_begin + j + 1) * kN > c.ctx && !wait_p(1)) return false;
              if (x == 0 && !wait_tile(2 * (g0 + j) + 1, kSiteVFull)) return false;
              if (x == 0 && j == 0 && !wait_o()) return false;
              tc_fence_after();
              if (!pv(x, g0 + j, j == 0)) return false;
              if (x == 1) mma_commit(&empty[(2 * (g0 + j) + 1) % NS]);
              return true;
            };
            for (int j = 0; j < n && ok; ++j) {
              ok = wait_tile(2 * (g0 + j), kSiteKFull);
              if (!ok) break;
              tc_fence_after();
              qk(0, g0 + j, 0);
              if (j > 0) {
                ok = do_pv(1, j - 1);
                if (!ok) break;
              }
              qk(1, g0 + j, 1);
              mma_commit(&empty[2 * (g0 + j) % NS]);
              if (j == n - 1) mma_commit(q_empty);
              ok = do_pv(0, j);
            }
            if (ok) ok = do_pv(1, n - 1);
          }
          if (!ok) break;
          mma_commit(o_final);
          g0 += n;
        }
        mma_commit(drain);
        mbar_wait(drain, 0, nullptr, kSiteOReady, 1000000000ull);
      }
    } else {
      // -------------------------------------------------------------- queries
      const int tid = threadIdx.x - 64;
      int filled = 0;  // rows that hold queries of a piece before
      bool ok = true;
      for (int w = 0; ok; ++w) {
        ok = __all_sync(0xffffffffu, mbar_wait(&item_full[w % kItems], (w / kItems) & 1, st,
                                               kSiteItemQueue, tmo));
        if (!ok) break;
        const Piece c = *item_slot(w);
        __syncwarp();
        if (lane_id() == 0) mbar_arrive(&item_empty[w % kItems]);
        if (c.request < 0) break;
        ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (w & 1) ^ 1, st, kSiteQFull, tmo));
        if (!ok) break;
        // Rows behind the unit's last are zeros: an MMA row is its own, but products of
        // zeros draw less power, which bounds the clock (32 trees, row tiles 58 % full:
        // 1455 instead of 1402 MHz and 318 instead of 323 us at the 1000 W cap).
        // A thread copies one 16-byte column of every kStep-th row; token and head move on
        // by additions (a division per copy held the first scores up by 5 us).
        constexpr int kChunks = D / 8, kStep = 64 / kChunks;
        const int x = tid % kChunks;
        const uint32_t qb = smem_u32(sQ) + (x / 8) * (kM * 128);
        auto place = [&](int r) {
          return qb + (r / kM) * (kM * D * 2) + (r % kM) * 128 + (((x % 8) ^ (r & 7)) << 4);
        };
        const int dt = kStep / p.group, dh = kStep - dt * p.group;
        int r = tid / kChunks;
        const int t0 = (c.row0 + r) / p.group;
        int h = c.row0 + r - t0 * p.group;
        const uint16_t* src = static_cast<const uint16_t*>(p.q) +
                              static_cast<int64_t>(c.first + t0) * p.q_t +
                              static_cast<int64_t>(c.head_kv * p.group + h) * p.q_h + x * 8;
        const int64_t step = dt * p.q_t + dh * p.q_h, wrap = p.q_t - p.group * p.q_h;
#pragma unroll 4
        for (; r < c.rows; r += kStep) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place(r)), "l"(src)
                       : "memory");
          src += step;
          h += dh;
          if (h >= p.group) {
            h -= p.group;
            src += wrap;
          }
        }
        for (; r < filled; r += kStep)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(place(r)), "r"(0)
                       : "memory");
        filled = c.rows;
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
    }
  } else {
    warpgroup_reg_inc<kRegsHigh>();
    // -------------------------------------------------------------- softmax
    const int x = (warp - 4) >> 2;
    const int row = (threadIdx.x - 128) & 127;
    const uint32_t lane_base = ((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lane_base + x * 128;
    // a scale of zero or below is applied before the mask and the maximum
    const bool flip = !(p.scale_log2 > 0.f);
    const float sl2 = flip ? 1.f : p.scale_log2;
    int g0 = 0;
    int sx = 0;  // tiles this chain has seen
    bool ok = true;
    for (int w = 0; ok; ++w) {
      ok = __all_sync(0xffffffffu, mbar_wait(&item_full[w % kItems], (w / kItems) & 1, st,
                                             kSiteItemQueue, tmo));
      if (!ok) break;
      // the piece stays in its slot: its fields are read again where they are
      // used rather than kept beside a row of 128 scores
      const Piece* c = item_slot(w);
      if (c->request < 0) break;
      const int n = c->tile_end - c->tile_begin;
      const int old_keys = c->ctx - c->tile_begin * kN;  // of the piece, before the new tokens
      const int r = kTwoRows ? x * kM + row : row;  // row of the unit
      // a warp without rows only keeps the order of things
      const int rows = c->rows;
      const bool active = r - static_cast<int>(lane_id()) < rows;
      const uint32_t o_col = tmem + lane_base + 256 + x * 128;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = kTwoRows ? 0 : x; j < n; j += kTwoRows ? 1 : 2) {
        const bool tail = (j + 1) * kN > old_keys;
        uint32_t bits[4];  // seen columns, looked up while the scores form
        if (tail && active) {
          const int token = min(c->row0 + r, c->row0 + c->rows - 1) / p.group;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            bits[q] = seen_bits(p, c, token, j * kN + 32 * q - old_keys);
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[x], sx & 1, st, kSiteSFull, tmo));
        if (!ok) break;
        ++sx;
        tc_fence_after();
        if (active) {
          uint32_t sr[kN];
#pragma unroll
          for (int k = 0; k < kN; k += 32) tmem_ld32(s_col + k, sr + k);
          tmem_ld_wait();
          if (flip) {
#pragma unroll
            for (int k = 0; k < kN; ++k)
              sr[k] = __float_as_uint(__uint_as_float(sr[k]) * p.scale_log2);
          }
          if (tail) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              // past over where every row sees all: this code is long and seldom run
              if (__all_sync(0xffffffffu, bits[q] == 0xffffffffu)) continue;
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!((bits[q] >> k) & 1u)) sr[32 * q + k] = 0xff800000u;  // -inf
            }
          }
          float pm[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) pm[i] = __uint_as_float(sr[i]);
#pragma unroll
          for (int k = 8; k < kN; k += 2)
            pm[(k >> 1) & 7] =
                fmax3(pm[(k >> 1) & 7], __uint_as_float(sr[k]), __uint_as_float(sr[k + 1]));
          const float mx = fmaxf(fmax3(fmax3(pm[0], pm[1], pm[2]), fmax3(pm[3], pm[4], pm[5]),
                                       pm[6]),
                                 pm[7]) * sl2;
          // by the difference, which is exact where it matters: m_run + 8 would be rounded
          // to steps of 16 for scores past 2^27
          constexpr float kLift = kBF16 ? 0.f : kLiftF16;
          const bool need = mx - m_run > kRescale + kLift;
          float alpha = 1.f;
          if (need) {
            const float top = mx - kLift;
            alpha = m_run == -INFINITY ? 0.f : ex2_approx(m_run - top);
            m_run = top;
            l_run *= alpha;
          }
          // the scores' commit covers this chain's products before them: O is at rest
          if (j > (kTwoRows ? 0 : 1) && __any_sync(0xffffffffu, need)) {
#pragma unroll
            for (int k = 0; k < D; k += 32) {
              uint32_t o[32];
              tmem_ld32(o_col + k, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i)
                o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st32(o_col + k, o);
            }
          }
          // a row of the tile that is none of the unit's gets weights of zero
          const float m_use = r >= rows ? INFINITY : (m_run == -INFINITY ? 0.f : m_run);
          const float2 scale2 = make_float2(sl2, sl2);
          const float2 shift2 = make_float2(-m_use, -m_use);
          float2 ps[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                          make_float2(0.f, 0.f)};
#pragma unroll
          for (int hlf = 0; hlf < 2; ++hlf) {
            uint32_t pk[32];
#pragma unroll
            for (int q = 0; q < 32; ++q) {
              const int i = hlf * 32 + q;
              const float2 y = ffma2(make_float2(__uint_as_float(sr[2 * i]),
                                                 __uint_as_float(sr[2 * i + 1])),
                                     scale2, shift2);
              const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
              ps[q & 3] = fadd2(ps[q & 3], e);  // the sum takes the weights unrounded
              pk[q] = pack2<kBF16>(e.x, e.y);
            }
            tmem_st32(s_col + hlf * 32, pk);
            if (C::kParts == 2 && hlf == 0 && !tail) {
              tmem_st_wait();
              tc_fence_before();
              __syncwarp();
              if (lane_id() == 0) mbar_arrive(&p_full[x]);
            }
          }
          const float2 sum = fadd2(fadd2(ps[0], ps[1]), fadd2(ps[2], ps[3]));
          l_run += sum.x + sum.y;
          tmem_st_wait();
        }
        if (tail) {
          // Clean V before the weights are handed over, whole: by now it has arrived.
          // With two row tiles each chain takes half the rows.
          const int idx = 2 * (g0 + j) + 1;
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&full[idx % NS], (idx / NS) & 1, st, kSiteVFull, tmo));
          if (!ok) break;
          constexpr int kVRows = kTwoRows ? kN / 2 : kN;
          if (clean_v<D, kBF16>(sKV + (idx % NS) * C::kTile, (c->tile_begin + j) * kN, c->ctx,
                                c->keys, p.page_size, kTwoRows ? x * kVRows : 0,
                                kTwoRows ? (x + 1) * kVRows : kVRows, row))
            s_dirty[w & 1] = w + 1;
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane_id() == 0) {
          if (C::kParts == 1 || tail || !active) mbar_arrive(&p_full[x]);
          if (C::kParts == 2) mbar_arrive(&p_hi[x]);
        }
      }
      if (!ok) break;
      // ------------------------------------------------------------ results
      ok = __all_sync(0xffffffffu, mbar_wait(o_final, w & 1, st, kSiteOReady, tmo));
      if (!ok) break;
      tc_fence_after();
      // Behind the wait: the piece's first product with V waited for `o_free` of the piece
      // before, so by now every warp has read that piece's pairs.
      s_ml[x * kM + row] = make_float2(m_run, l_run);
      __syncwarp();
      if (lane_id() == 0) mbar_arrive(joined);
      ok = __all_sync(0xffffffffu, mbar_wait(joined, w & 1, st, kSiteOReady, tmo));
      if (!ok) break;
      if (active) {
        float f0 = 1.f, f1 = 0.f;  // factors of the two chains' outputs
        if constexpr (!kTwoRows) {
          const float2 a = s_ml[row], b = s_ml[kM + row];
          const float top = fmaxf(a.x, b.x);
          if (top != -INFINITY) {
            f0 = ex2_approx(a.x - top);
            f1 = ex2_approx(b.x - top);
          }
          m_run = top;
          l_run = f0 * a.y + f1 * b.y;
        }
        const bool mine = r < rows;
        const int record = c->record;
        const int out_row = c->row0 + r;
        const int t = static_cast<int>(static_cast<uint32_t>(out_row) /
                                       static_cast<uint32_t>(p.group));
        const int h = c->head_kv * p.group + out_row - t * p.group;
        if (record < 0) {
          const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
          f0 *= inv;
          f1 *= inv;
        }
        // a record is [dim / 4][rows][4]: the rows of a warp lie side by side
        float* rec = p.rec_acc + static_cast<int64_t>(record) * (kRows * D) + r * 4;
        uint16_t* dst = static_cast<uint16_t*>(p.out) +
                        static_cast<int64_t>(c->first + t) * p.out_t +
                        static_cast<int64_t>(h) * p.out_h;
        // with two key chains each warpgroup writes half the columns
        constexpr int kSpan = kTwoRows ? D : D / 2;
        const int k_first = kTwoRows ? 0 : x * kSpan;
#pragma unroll 1
        for (int k = k_first; k < k_first + kSpan; k += 32) {
          uint32_t o[32];
          float* v = reinterpret_cast<float*>(o);
          if constexpr (kTwoRows) {
            tmem_ld32(o_col + k, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= f0;
          } else {
            uint32_t o1[32];
            tmem_ld32(tmem + lane_base + 256 + k, o);
            if (n > 1) {
              tmem_ld32(tmem + lane_base + 384 + k, o1);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = v[i] * f0 + __uint_as_float(o1[i]) * f1;
            } else {
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= f0;
            }
          }
          if (!mine) {
            // (the TMEM loads above are warp-collective)
          } else if (record >= 0) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(rec + (k + i) * rows) =
                  make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(dst + k + i) =
                  make_uint4(pack2<kBF16>(v[i], v[i + 1]), pack2<kBF16>(v[i + 2], v[i + 3]),
                             pack2<kBF16>(v[i + 4], v[i + 5]), pack2<kBF16>(v[i + 6], v[i + 7]));
          }
        }
        if (mine && (kTwoRows || x == 0)) {
          if (record >= 0) {
            p.rec_m[record * kRows + r] = m_run;
            p.rec_l[record * kRows + r] = l_run;
          } else if (p.lse != nullptr) {
            p.lse[static_cast<int64_t>(c->first + t) * p.heads + h] =
                l_run == 0.f ? -INFINITY : (m_run + log2f(l_run)) * kLn2;
          }
        }
        if (mine && s_dirty[w & 1] == w + 1)
          add_taken_out<kBF16>(p, c, t, k_first, k_first + kSpan, D,
                               record >= 0 ? rec : nullptr, dst);
      }
      tc_fence_before();
      __syncwarp();
      if (lane_id() == 0) {
        mbar_arrive(o_free);
        mbar_arrive(&item_empty[w % kItems]);
      }
      g0 += n;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

template <int D, bool kBF16, bool kTwoRows>
int launch(const TreeParams& p, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t stream) {
  using C = Cfg<D, kTwoRows>;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t err =
        cudaFuncSetAttribute(tree_attn_kernel<D, kBF16, kTwoRows>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (err != cudaSuccess) return static_cast<int>(err);
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  return launch_overlapped(tree_attn_kernel<D, kBF16, kTwoRows>, dim3(p.grid), kThreads, C::kSmem,
                           stream, &p, &k, &v);
}

}  // namespace

int tree_sm100_launch(Elem elem, const TreeParams& p, int rows_per_unit, cudaStream_t stream) {
  const CUtensorMap k = pool_map(p, p.k, p.k_page, 2, kN), v = pool_map(p, p.v, p.v_page, 2, kN);
  const bool two = rows_per_unit == 256;
  if (elem == Elem::kBF16) {
    if (p.dim == 64)
      return two ? launch<64, true, true>(p, k, v, stream) : launch<64, true, false>(p, k, v, stream);
    return two ? launch<128, true, true>(p, k, v, stream) : launch<128, true, false>(p, k, v, stream);
  }
  if (p.dim == 64)
    return two ? launch<64, false, true>(p, k, v, stream) : launch<64, false, false>(p, k, v, stream);
  return two ? launch<128, false, true>(p, k, v, stream) : launch<128, false, false>(p, k, v, stream);
}

}  // namespace rab
