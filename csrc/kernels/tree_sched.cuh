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

__device__ __forceinline__ Request load_request(const TreeParams& p, int b) {
  Request r;
  int end;
  if (p.cu == nullptr) {
    r.first = b * p.uniform;
    end = r.first + p.uniform;
  } else {
    r.first = max(0, min(p.cu[b], p.total));
    end = max(r.first, min(p.cu[b + 1], p.total));
  }
  r.tokens = end - r.first;
  const int room = p.table_w * p.page_size;  // at most 2^30 (checked by the bindings)
  r.ctx = max(0, min(p.ctx[b], room));
  r.keys = min(r.ctx + r.tokens, room);
  return r;
}

__device__ __forceinline__ int row_tiles(const TreeParams& p, const Request& r, int rows) {
  return static_cast<int>((static_cast<long long>(r.tokens) * p.group + rows - 1) / rows);
}

// Key tiles of row tile t: under the causal rule the tile's last token bounds
// them; a mask bounds them by the request's last token.
template <int kTile>
__device__ __forceinline__ int unit_tiles(const TreeParams& p, const Request& r, int t, int rows) {
  int keys = r.keys;
  if (p.mask == nullptr) {
    const long long last = ((static_cast<long long>(t) + 1) * rows - 1) / p.group;
    if (last < r.tokens) keys = min(keys, r.ctx + static_cast<int>(last) + 1);
  }
  return (keys + kTile - 1) / kTile;
}

// places of one kv head of a request
template <int kTile>
__device__ __forceinline__ long long head_places(const TreeParams& p, const Request& r, int rows) {
  const int n = row_tiles(p, r, rows);
  if (n == 0) return 0;
  if (p.mask != nullptr || n == 1)
    return static_cast<long long>(n) * (kUnitCost + unit_tiles<kTile>(p, r, n - 1, rows));
  long long s = 0;
  for (int t = 0; t < n; ++t) s += kUnitCost + unit_tiles<kTile>(p, r, t, rows);
  return s;
}

// One piece of work.
struct Piece {
  int request, head_kv, row0, rows;  // rows [row0, row0 + rows) of the request
  int first, ctx, tokens, keys;      // the request
  int tile_begin, tile_end;
  int record;                        // -1: a whole unit, written as a result
};

struct Range {
  long long total;  // places in all
  int grid;         // CTAs that share them
  long long begin, end;  // this CTA's
  // the request that holds `begin`, and its first place
  int request;
  long long at;
};

__device__ __forceinline__ long long range_start(long long total, int grid, int c) {
  return total * c / grid;
}
// the CTA whose range holds place x
__device__ __forceinline__ int range_owner(long long total, int grid, long long x) {
  return static_cast<int>(((x + 1) * grid - 1) / total);
}

// Whole block executes; `sums` holds a long long per warp.  Every CTA reaches the same totals.
template <int kTile, int kThreads>
__device__ __forceinline__ Range find_range(const TreeParams& p, int rows, long long* sums,
                                            int* s_request, long long* s_at) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Range g;
  long long total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    long long before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      long long mine = 0;
      if (b < p.batch) {
        const Request r = load_request(p, b);
        if (pass == 0 && blockIdx.x == 0 && r.tokens > 0 &&
            (p.ctx[b] < 0 || r.keys - r.tokens != p.ctx[b]))
          st_record(p.status, kStatusBadArgs, kBadPosition, b);  // longer than its table
        mine = head_places<kTile>(p, r, rows) * p.heads_kv;
      }
      long long inc = mine;  // inclusive sum over the warp
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
      }
      if (lane == 31) sums[warp] = inc;
      __syncthreads();
      long long base = before, all = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) base += sums[w];
        all += sums[w];
      }
      if (pass == 1 && mine > 0) {
        const long long lo = base + inc - mine;
        if (g.begin >= lo && g.begin < lo + mine) {
          *s_request = b;
          *s_at = lo;
        }
      }
      before += all;
      __syncthreads();
      if (pass == 0) total = before;
    }
    if (pass == 0) {
      g.total = total;
      const long long most = total / kMinShare;
      g.grid = static_cast<int>(most < 1 ? 1 : (most < p.grid ? most : p.grid));
      const int c = blockIdx.x;
      g.begin = c < g.grid ? range_start(total, g.grid, c) : total;
      g.end = c < g.grid ? range_start(total, g.grid, c + 1) : total;
    }
  }
  g.request = *s_request;
  g.at = *s_at;
  return g;
}

// Walks the pieces of a CTA's range; one thread uses it.
template <int kTile>
struct Walk {
  long long pos, end;  // place reached, end of the range
  long long unit_at;   // first place of the current unit
  int request, head, tile;
  int n_tiles;         // row tiles of the request
  Request r;
  int merge_c0;        // set with `merges`: the CTA that holds the first piece of the unit
  bool merges;         // the piece ends a unit that an earlier CTA began

  __device__ __forceinline__ void start(const TreeParams& p, const Range& g, int rows) {
    pos = g.begin;
    end = g.end;
    request = g.request;
    unit_at = g.at;
    head = 0;
    tile = 0;
    if (pos >= end) return;
    r = load_request(p, request);
    n_tiles = row_tiles(p, r, rows);
    const long long per_head = head_places<kTile>(p, r, rows);
    head = static_cast<int>((pos - unit_at) / per_head);
    unit_at += head * per_head;
    if (p.mask != nullptr || n_tiles == 1) {
      const int len = kUnitCost + unit_tiles<kTile>(p, r, 0, rows);
      tile = static_cast<int>((pos - unit_at) / len);
      unit_at += static_cast<long long>(tile) * len;
    } else {
      while (true) {
        const int len = kUnitCost + unit_tiles<kTile>(p, r, tile, rows);
        if (pos < unit_at + len) break;
        unit_at += len;
        ++tile;
      }
    }
  }

  // the next piece with tiles in it, or false at the range's end
  __device__ __forceinline__ bool next(const TreeParams& p, const Range& g, int rows, Piece* out) {
    while (pos < end) {
      const int tiles = unit_tiles<kTile>(p, r, tile, rows);
      const long long unit_end = unit_at + kUnitCost + tiles;
      const long long stop = unit_end < end ? unit_end : end;
      const long long tb = pos - unit_at - kUnitCost, te = stop - unit_at - kUnitCost;
      Piece c;
      c.tile_begin = static_cast<int>(tb > 0 ? tb : 0);
      c.tile_end = static_cast<int>(te > 0 ? te : 0);
      c.request = request;
      c.head_kv = head;
      c.row0 = tile * rows;
      c.rows = min(rows, r.tokens * p.group - c.row0);
      c.first = r.first;
      c.ctx = r.ctx;
      c.tokens = r.tokens;
      c.keys = r.keys;
      const int cta = 2 * static_cast<int>(blockIdx.x);
      const bool from_start = c.tile_begin == 0, to_end = c.tile_end == tiles;
      c.record = from_start ? (to_end ? -1 : cta + 1) : cta;
      merges = to_end && !from_start;
      if (merges) merge_c0 = range_owner(g.total, g.grid, unit_at + kUnitCost);
      const bool have = c.tile_end > c.tile_begin || tiles == 0;
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
                n_tiles = row_tiles(p, r, rows);
              } while (n_tiles == 0);
            }
          }
        }
      }
      if (have) {
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
