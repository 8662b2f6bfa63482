// paged.h - parameters and host API of the rotary-position kernels and of the
// paged key/value cache: writing new tokens, copying pages, keeping the
// accepted path of a drafted tree, and attention over the cache.
//
// A cache pool is [pages, heads_kv, page_size, dim] (optionally with a leading
// layer dimension): one head's keys of one page are contiguous, so an
// attention tile of one head reads whole runs of page_size rows.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "status.h"

namespace rab {

enum class Elem : int { kBF16 = 0, kF16 = 1, kF32 = 2 };
inline int elem_bytes(Elem e) { return e == Elem::kF32 ? 4 : 2; }

// ---- rotary positions / append ----
// One tensor of a rotary or append launch.  Strides are in elements.  A dense
// operand writes out + token * out_t + head * out_h; a paged one writes
// out + page * out_t + head * out_h + offset * dim.
struct RopeOperand {
  const void* in;
  void* out;
  int64_t in_t, in_h, out_t, out_h;
  int heads;  // 1 or more
  int rotate;
  int paged;
};

struct RopeParams {
  RopeOperand op[3];
  int n_op;
  int sms;  // of the GPU, for the launch
  int tokens, dim, rotary_dim;
  int interleaved;       // pairs (2p, 2p+1); otherwise (p, p + rotary_dim/2)
  float scale;           // factor on the rotated elements
  float sign;            // +1 forward, -1 inverse rotation
  const void* positions; // int64 or int32 [tokens]; nullptr: the cache position
  int positions64;
  const double* inv_freq;  // [rotary_dim/2]
  // paged operands
  const int* table;      // [batch, table_w] page ids
  int64_t table_stride;
  int table_w, num_pages, page_size;
  const int* ctx;        // [batch] tokens cached before this call
  const int* cu;         // [batch + 1] borders of the packed tokens; nullptr: uniform
  int batch, uniform;    // uniform: tokens per request when cu == nullptr
  DeviceStatus* status;
};

int rope_launch(Elem elem, const RopeParams& p, bool vectors, cudaStream_t stream);

// ---- page copies ----
// The pairs of one launch travel in its parameters; few of them take a small
// block of parameters, which a launch hands over faster.
constexpr int kFewPairs = 32, kManyPairs = 1000;
template <int kPairs>
struct PageCopyParams {
  static constexpr int kMax = kPairs;
  uint8_t* k;
  uint8_t* v;
  int64_t k_layer, k_page, v_layer, v_page;  // byte strides
  int64_t page_bytes;
  int layers, n_src;
  int src[kPairs];        // distinct source pages
  int first[kPairs + 1];  // source s goes to dst[first[s]] .. dst[first[s + 1] - 1]
  int dst[kPairs];
};
int page_copy_launch(const PageCopyParams<kFewPairs>& p, cudaStream_t stream);
int page_copy_launch(const PageCopyParams<kManyPairs>& p, cudaStream_t stream);

// ---- accepted path ----
struct PathParams {
  uint8_t* k;
  uint8_t* v;
  int64_t k_layer, k_page, v_layer, v_page;  // byte strides
  int layers, heads, page_size, row_bytes, num_pages;
  const int* table;
  int64_t table_stride;
  int table_w;
  const int* ctx;
  const int* path;  // [batch, path_w] places among the new tokens, increasing
  int64_t path_stride;
  int path_w;
  const int* path_lens;  // [batch]
  int batch;
  DeviceStatus* status;
};
int path_compact_launch(const PathParams& p, cudaStream_t stream);

// ---- attention over the cache ----
struct TreeParams {
  const void* q;
  int64_t q_t, q_h;  // element strides of a token and a head
  void* out;
  int64_t out_t, out_h;
  float* lse;  // [total, heads] or nullptr
  const void* k;
  const void* v;
  int64_t k_page, v_page;  // element strides of a page
  int num_pages, page_size, page_shift;  // a power of two
  const int* table;
  int64_t table_stride;
  int table_w;
  const int* ctx;
  const int* cu;
  int batch, uniform, total;
  int heads, heads_kv, group, dim;
  const uint32_t* mask;  // [total, mask_w] bits, or nullptr: causal among the new tokens
  int64_t mask_stride;
  int mask_w;
  float scale_log2;
  // split records: record r holds [rows][dim] unnormalised outputs and per row
  // the running maximum (log2 units) and sum
  float* rec_acc;
  float* rec_m;
  float* rec_l;
  int* meta;  // [grid][8]: the unit whose records block c of the merge joins
  int grid;
  DeviceStatus* status;
  uint64_t timeout_ns;
};

struct TreePlan {
  int rows_per_unit;
  int grid;
  int merge_rows;  // rows the merge launch is sized for
  int tile_keys;
  size_t acc_floats, ml_floats, meta_ints;
};

TreePlan tree_plan(Elem elem, const TreeParams& p, int max_q, int sms);
int tree_launch(Elem elem, const TreeParams& p, const TreePlan& plan, cudaStream_t stream);
// the kernels of bf16 and fp16 (tree_launch calls them): 8 or 16 rows per unit, and 128
// or 256
int tree_few_launch(Elem elem, const TreeParams& p, int rows_per_unit, cudaStream_t stream);
int tree_sm100_launch(Elem elem, const TreeParams& p, int rows_per_unit, cudaStream_t stream);

// ancestor bits and depths of drafted trees from parent indices
int tree_mask_launch(const int* parents, const int* cu, int batch, int uniform, int total,
                     uint32_t* mask, int mask_w, int* depth, DeviceStatus* status,
                     cudaStream_t stream);
// bool [total, cols] -> bits
int pack_mask_launch(const uint8_t* in, int64_t in_t, int total, int cols, uint32_t* mask,
                     int mask_w, cudaStream_t stream);

}  // namespace rab
