// tree_sched.cuh - work of the attention over a paged cache, shared out evenly
// on the device.
//
// A unit is (request, kv head, row tile): rows are the (new token, query head
// of the group) pairs of one kv head, token-major, rows_per_unit to a tile.
// Lengths live on the GPU, so every CTA computes the same prefix sum over the
// requests and takes an equal range of the line of all units, on which a unit
// is kUnitCost places long plus one for each of its key tiles; kUnitCost stands
// for what a unit costs whatever its length (its queries, its results).  A
// range cuts units at arbitrary tiles; a piece that is not a whole unit writes
// a split record, and the merge kernel joins them in CTA order, so results do
// not depend on timing.
#pragma once

#include <cuda.h>

#include <cstdint>

#include "paged.h"
#include "tmap.h"

namespace rab {
namespace tree_detail {

constexpr int kUnitCost = 2;
// places below which a further CTA costs more than it takes over; us with 4 / 2 / 1, bf16,
// 8 kv heads of 128: one token over 10 keys 8.3 / 6.0 / 6.0, over 1000 9.4 / 8.4 / 8.6, a
// tree of 30 over 500 17.2 / 14.4 / 15.7, a chunk of 200 25.6 / 21.0 / 21.7
constexpr int kMinShare = 2;
constexpr int kMetaInts = 8;

struct Request {
  int first;   // first packed token
  int tokens;  // new tokens (clamped to what the tensors hold)
  int ctx;     // cached tokens before them, at most the table's room
  int keys;    // keys that exist: ctx + tokens, at most the table's room
};

// Places, rows and keys are 32-bit numbers: the bindings refuse calls whose
// table, rows or line of units could pass 2^31 (64-bit divisions before a CTA's
// first load cost a decoding step a microsecond).
__device__ __forceinline__ Request load_request(const TreeParams& p, int b) {
  Request r;
  const int ctx = p.ctx[b];
  int end;
  if (p.cu == nullptr) {
    r.first = b * p.uniform;
    end = r.first + p.uniform;
  } else {
    const int lo = p.cu[b], hi = p.cu[b + 1];
    r.first = max(0, min(lo, p.total));
    end = max(r.first, min(hi, p.total));
  }
  r.tokens = end - r.first;
  const int room = p.table_w * p.page_size;
  r.ctx = max(0, min(ctx, room));
  r.keys = min(r.ctx + r.tokens, room);
  return r;
}

template <int kRows>
__device__ __forceinline__ int row_tiles(const TreeParams& p, const Request& r) {
  return (r.tokens * p.group + kRows - 1) / kRows;
}

// Key tiles of row tile t: under the causal rule the tile's last token bounds
// them; a mask bounds them by the request's last token.
template <int kTile, int kRows>
__device__ __forceinline__ int unit_tiles(const TreeParams& p, const Request& r, int t) {
  int keys = r.keys;
  if (p.mask == nullptr && (t + 1) * kRows < r.tokens * p.group) {
    const int last = static_cast<int>((static_cast<uint32_t>(t + 1) * kRows - 1) /
                                      static_cast<uint32_t>(p.group));
    keys = min(keys, r.ctx + last + 1);
  }
  return (keys + kTile - 1) / kTile;
}

// places of one kv head of a request
template <int kTile, int kRows>
__device__ __forceinline__ int head_places(const TreeParams& p, const Request& r) {
  const int n = row_tiles<kRows>(p, r);
  if (n == 0) return 0;
  if (p.mask != nullptr || n == 1) return n * (kUnitCost + unit_tiles<kTile, kRows>(p, r, n - 1));
  int s = 0;
  for (int t = 0; t < n; ++t) s += kUnitCost + unit_tiles<kTile, kRows>(p, r, t);
  return s;
}

// One piece of work.
struct Piece {
  int request, head_kv, row0, rows;  // rows [row0, row0 + rows) of the request
  int first, ctx, tokens, keys;      // the request
  int tile_begin, tile_end;
  int record;                        // -1: a whole unit, written as a result
};

// The line of `total` places in `grid` ranges of `share` or, the first `more` of
// them, share + 1 places.
struct Range {
  int total, grid, share, more;
  int begin, end;  // this CTA's
  __device__ __forceinline__ int start(int c) const { return c * share + min(c, more); }
  // the CTA whose range holds place x
  __device__ __forceinline__ int owner(int x) const {
    const int big = more * (share + 1);
    return x < big ? static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(share + 1))
                   : more + static_cast<int>(static_cast<uint32_t>(x - big) /
                                             static_cast<uint32_t>(share));
  }
};

// Where a range begins: the request that holds its first place, that request's
// own first place, and the places of one of its kv heads.
struct Start {
  int at, request, per_head;
  Request r;
};

// One warp executes, on its own: nothing but the piece queue ties the block's other
// warps to it.  Every CTA reaches the same totals.  Returns the lane that holds the
// range's first request (its `start` is the one filled in) and goes on to walk the
// range.  A decoding step waits for this before its first load, so up to 32
// requests take one read and one scan; more are shared out in runs, and the run that
// holds the first is read again.
template <int kTile, int kRows>
__device__ __forceinline__ int find_range(const TreeParams& p, Range* range, Start* start) {
  const int lane = threadIdx.x & 31;
  Range g;
  auto places = [&](int b) {
    if (b >= p.batch) return 0;
    start->request = b;
    start->r = load_request(p, b);
    start->per_head = head_places<kTile, kRows>(p, start->r);
    if (blockIdx.x == 0 && start->r.tokens > 0 &&
        (p.ctx[b] < 0 || start->r.keys - start->r.tokens != p.ctx[b]))
      st_record(p.status, kStatusBadArgs, kBadPosition, b);  // longer than its table
    return start->per_head * p.heads_kv;
  };
  auto scan = [&](int v) {  // inclusive sum over the warp
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    return v;
  };
  // a lane's requests lie side by side: the second reading is of one lane's only
  const int per = (p.batch + 31) >> 5, mine_0 = lane * per;
  int mine = 0, inc;
  if (per == 1) {
    mine = places(lane);
    inc = scan(mine);
  } else {
    int sum = 0;
#pragma unroll 4
    for (int b = mine_0; b < mine_0 + per; ++b) sum += places(b);
    mine = sum;
    inc = scan(sum);
  }
  g.total = __shfl_sync(0xffffffffu, inc, 31);
  const int c = blockIdx.x;
  g.grid = min(max(g.total / kMinShare, 1), p.grid);
  g.share = static_cast<int>(static_cast<uint32_t>(g.total) / static_cast<uint32_t>(g.grid));
  g.more = g.total - g.share * g.grid;
  g.begin = c < g.grid ? g.start(c) : g.total;
  g.end = c < g.grid ? g.start(c + 1) : g.total;
  *range = g;
  if (g.begin >= g.end) return 0;
  int before = 0;
  if (per > 1) {
    const int in = __ffs(__ballot_sync(0xffffffffu, g.begin < inc)) - 1;
    before = __shfl_sync(0xffffffffu, inc - mine, in);
    for (int b0 = in * per;; b0 += 32) {  // ends: the range begins below the total
      mine = places(b0 + lane);
      inc = scan(mine);
      const int all = __shfl_sync(0xffffffffu, inc, 31);
      if (g.begin < before + all) break;
      before += all;
    }
  }
  start->at = before + inc - mine;
  return __ffs(__ballot_sync(0xffffffffu, g.begin < before + inc)) - 1;
}

// Walks the pieces of a CTA's range; one thread uses it, and the block waits for
// its first piece, so `next` moves on from a unit only when it is called again.
template <int kTile, int kRows>
struct Walk {
  int pos, end;        // place reached, end of the range
  int unit_at;         // first place of the current unit
  int request, head, tile;
  int n_tiles;         // row tiles of the request
  int tiles;           // key tiles of the current unit
  Request r;
  int merge_c0;        // set with `merges`: the CTA that holds the first piece of the unit
  bool merges;         // the piece ends a unit that an earlier CTA began

  __device__ __forceinline__ void start(const TreeParams& p, const Range& g, const Start& s) {
    pos = g.begin;
    end = g.end;
    tile = 0;
    if (pos >= end) return;
    request = s.request;
    r = s.r;
    n_tiles = row_tiles<kRows>(p, r);
    head = static_cast<int>(static_cast<uint32_t>(pos - s.at) / static_cast<uint32_t>(s.per_head));
    unit_at = s.at + head * s.per_head;
    if (n_tiles == 1) {
      tiles = s.per_head - kUnitCost;
    } else {
      while (true) {
        tiles = unit_tiles<kTile, kRows>(p, r, tile);
        if (pos < unit_at + kUnitCost + tiles) break;
        unit_at += kUnitCost + tiles;
        ++tile;
      }
    }
  }

  __device__ __forceinline__ void next_unit(const TreeParams& p) {
    unit_at = pos;
    if (++tile == n_tiles) {
      tile = 0;
      if (++head == p.heads_kv) {
        head = 0;
        do {
          r = load_request(p, ++request);
          n_tiles = row_tiles<kRows>(p, r);
        } while (n_tiles == 0);
      }
    }
    tiles = unit_tiles<kTile, kRows>(p, r, tile);
  }

  // the next piece with tiles in it, or false at the range's end
  __device__ __forceinline__ bool next(const TreeParams& p, const Range& g, Piece* c) {
    while (pos < end) {
      if (pos == unit_at + kUnitCost + tiles) next_unit(p);
      const int stop = min(unit_at + kUnitCost + tiles, end);
      const int tb = max(pos - unit_at - kUnitCost, 0), te = max(stop - unit_at - kUnitCost, 0);
      pos = stop;
      if (te <= tb) continue;
      const bool from_start = tb == 0, to_end = te == tiles;
      merges = to_end && !from_start;
      if (merges) merge_c0 = g.owner(unit_at + kUnitCost);
      const int cta = 2 * static_cast<int>(blockIdx.x);
      c->request = request;
      c->head_kv = head;
      c->row0 = tile * kRows;
      c->rows = min(kRows, r.tokens * p.group - tile * kRows);
      c->first = r.first;
      c->ctx = r.ctx;
      c->tokens = r.tokens;
      c->keys = r.keys;
      c->tile_begin = tb;
      c->tile_end = te;
      c->record = from_start ? (to_end ? -1 : cta + 1) : cta;
      return true;
    }
    return false;
  }
};

// what the merge kernel's block c joins; valid == 0: nothing
__device__ __forceinline__ void write_meta(const TreeParams& p, const Piece& c, bool merges,
                                           int c0) {
  int* m = p.meta + blockIdx.x * kMetaInts;
  m[0] = merges ? 1 : 0;
  if (merges) {
    m[1] = c0;
    m[2] = c.head_kv;
    m[3] = c.row0;
    m[4] = c.rows;
    m[5] = c.first;
  }
}

// a pool's tiles: boxes of 128 bytes of columns and a page's rows, at most a tile's
inline CUtensorMap pool_map(const TreeParams& p, const void* base, int64_t page_stride, int bytes,
                            int tile) {
  const uint64_t d = p.dim, page = p.page_size;
  uint64_t dims[4] = {d, page, static_cast<uint64_t>(p.heads_kv),
                      static_cast<uint64_t>(p.num_pages)};
  uint64_t strides[3] = {d * bytes, page * d * bytes, static_cast<uint64_t>(page_stride) * bytes};
  uint32_t box[4] = {static_cast<uint32_t>(128 / bytes),
                     static_cast<uint32_t>(p.page_size < tile ? p.page_size : tile), 1, 1};
  // 16-bit elements are copied, not read, so one type serves bf16 and fp16
  return make_tmap(base, bytes == 4 ? TmapDtype::kF32 : TmapDtype::kBF16, 4, dims, strides, box,
                   CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace tree_detail
}  // namespace rab
