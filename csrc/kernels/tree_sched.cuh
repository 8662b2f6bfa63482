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

#include <cstdint>

#include "paged.h"

namespace rab {
namespace tree_detail {

constexpr int kUnitCost = 2;
constexpr int kMinShare = 4;  // places below which a further CTA costs more than it takes over
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

// Where a range begins: the request that holds its first place, and that
// request's own first place.  One thread finds it and leaves it in shared memory.
struct Start {
  int at;
  int request;
  Request r;
};

// Whole block executes; `sums` holds an int per warp.  Every CTA reaches the same
// totals.  Up to kThreads requests are read once and kept in registers.
template <int kTile, int kRows, int kThreads>
__device__ __forceinline__ Range find_range(const TreeParams& p, int* sums, Start* start) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Range g;
  g.total = 0;
  Request r;
  int mine = 0, lo = 0;
  // one block of kThreads requests: adds up, leaves this thread's in r / mine / lo
  auto block_of = [&](int b0, int before) {
    const int b = b0 + threadIdx.x;
    mine = 0;
    if (b < p.batch) {
      r = load_request(p, b);
      mine = head_places<kTile, kRows>(p, r) * p.heads_kv;
    }
    int inc = mine;  // inclusive sum over the warp
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    int base = before, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int v = sums[w];
      if (w < warp) base += v;
      all += v;
    }
    lo = base + inc - mine;
    if (p.batch > kThreads) __syncthreads();  // `sums` is used again
    return before + all;
  };
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    g.total = block_of(b0, g.total);
    const int b = b0 + threadIdx.x;
    if (blockIdx.x == 0 && mine > 0 && (p.ctx[b] < 0 || r.keys - r.tokens != p.ctx[b]))
      st_record(p.status, kStatusBadArgs, kBadPosition, b);  // longer than its table
  }
  const int c = blockIdx.x;
  g.grid = min(max(g.total / kMinShare, 1), p.grid);
  g.share = static_cast<int>(static_cast<uint32_t>(g.total) / static_cast<uint32_t>(g.grid));
  g.more = g.total - g.share * g.grid;
  g.begin = c < g.grid ? g.start(c) : g.total;
  g.end = c < g.grid ? g.start(c + 1) : g.total;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    if (p.batch > kThreads) before = block_of(b0, before);
    if (mine > 0 && g.begin >= lo && g.begin < lo + mine) {
      start->at = lo;
      start->request = b0 + threadIdx.x;
      start->r = r;
    }
  }
  __syncthreads();
  return g;
}

// Walks the pieces of a CTA's range; one thread uses it.
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
    head = 0;
    tile = 0;
    if (pos >= end) return;
    request = s.request;
    unit_at = s.at;
    r = s.r;
    n_tiles = row_tiles<kRows>(p, r);
    const uint32_t per_head = head_places<kTile, kRows>(p, r);
    head = static_cast<int>(static_cast<uint32_t>(pos - unit_at) / per_head);
    unit_at += head * static_cast<int>(per_head);
    while (true) {
      tiles = unit_tiles<kTile, kRows>(p, r, tile);
      if (pos < unit_at + kUnitCost + tiles) break;
      unit_at += kUnitCost + tiles;
      ++tile;
    }
  }

  // the next piece with tiles in it, or false at the range's end
  __device__ __forceinline__ bool next(const TreeParams& p, const Range& g, Piece* out) {
    while (pos < end) {
      const int unit_end = unit_at + kUnitCost + tiles;
      const int stop = min(unit_end, end);
      Piece c;
      c.tile_begin = max(pos - unit_at - kUnitCost, 0);
      c.tile_end = max(stop - unit_at - kUnitCost, 0);
      c.request = request;
      c.head_kv = head;
      c.row0 = tile * kRows;
      c.rows = min(kRows, r.tokens * p.group - c.row0);
      c.first = r.first;
      c.ctx = r.ctx;
      c.tokens = r.tokens;
      c.keys = r.keys;
      const int cta = 2 * static_cast<int>(blockIdx.x);
      const bool from_start = c.tile_begin == 0, to_end = c.tile_end == tiles;
      c.record = from_start ? (to_end ? -1 : cta + 1) : cta;
      merges = to_end && !from_start;
      if (merges) merge_c0 = g.owner(unit_at + kUnitCost);
      pos = stop;
      if (pos == unit_end) {  // the next unit
        unit_at = unit_end;
        if (++tile == n_tiles) {
          tile = 0;
          if (++head == p.heads_kv) {
            head = 0;
            if (pos < end) {
              do {
                r = load_request(p, ++request);
                n_tiles = row_tiles<kRows>(p, r);
              } while (n_tiles == 0);
            }
          }
        }
        if (pos < end) tiles = unit_tiles<kTile, kRows>(p, r, tile);
      }
      if (c.tile_end > c.tile_begin) {
        *out = c;
        return true;
      }
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

}  // namespace tree_detail
}  // namespace rab
