// paged_bindings.cpp - torch surface of the rotary positions and the paged
// key/value cache.  Every argument is checked here, in one call per operator:
// shapes, types and strides first, then the devices, so a refused call raises a
// RuntimeError before anything is launched.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <numeric>
#include <vector>

#include "bind_util.h"
#include "flash.h"
#include "paged.h"
#include "strfmt.h"

namespace rab {
namespace {

using OptTensor = c10::optional<torch::Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

long long ll(int64_t x) { return static_cast<long long>(x); }

Elem elem_of(const torch::Tensor& t, const char* name) {
  const auto s = t.scalar_type();
  RAB_CHECK(s == torch::kBFloat16 || s == torch::kHalf || s == torch::kFloat32,
            "%s must be bfloat16, float16 or float32", name);
  return s == torch::kBFloat16 ? Elem::kBF16 : (s == torch::kHalf ? Elem::kF16 : Elem::kF32);
}

void check_same(const torch::Tensor& t, const char* name, const torch::Tensor& ref) {
  RAB_CHECK(t.is_cuda(), "%s must be a CUDA tensor", name);
  RAB_CHECK(t.device() == ref.device(), "%s must be on the same GPU as the other tensors", name);
}

void check_int32(const torch::Tensor& t, const char* name, int64_t dims) {
  RAB_CHECK(t.scalar_type() == torch::kInt32, "%s must be int32", name);
  RAB_CHECK(t.dim() == dims, "%s must have %lld dimension(s)", name, ll(dims));
  // (the stride of a single element is any: contiguous() leaves it as it is)
  RAB_CHECK(t.size(dims - 1) <= 1 || t.stride(dims - 1) == 1,
            "%s must be contiguous in its last dimension", name);
}

// [tokens, heads, dim] with adjacent elements of a row
void check_rows(const torch::Tensor& t, const char* name) {
  RAB_CHECK(t.dim() == 3, "%s must be [tokens, heads, dim]", name);
  RAB_CHECK(t.size(2) == 1 || t.stride(2) == 1, "%s must be contiguous in its last dimension", name);
  RAB_CHECK(t.size(0) <= INT32_MAX && t.size(1) <= 65535, "%s is too large", name);
}

// A new contiguous tensor, straight from the caching allocator: torch::empty goes
// through the dispatcher, which costs a short call about a microsecond a tensor.
torch::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

// every row begins on a 16-byte boundary (the stride of a single token or head is none)
bool rows_aligned(const torch::Tensor& t) {
  const int64_t e = t.element_size();
  return aligned16(t.data_ptr()) && (t.size(0) <= 1 || t.stride(0) * e % 16 == 0) &&
         (t.size(1) <= 1 || t.stride(1) * e % 16 == 0);
}

// Strides and sizes in bytes of the dimensions that step through memory.
struct Steps {
  int64_t stride[10], count[10];
  int n = 0;
  void add(const torch::Tensor& t) {
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 1) {
        stride[n] = t.stride(d) * t.element_size();
        count[n++] = t.size(d);
      }
  }
};

// bytes from the first element to the end of the last, over the steps below `limit`
int64_t span_below(const torch::Tensor& t, int64_t limit) {
  Steps s;
  s.add(t);
  int64_t bytes = t.element_size();
  for (int i = 0; i < s.n; ++i)
    if (s.stride[i] < limit) bytes += (s.count[i] - 1) * s.stride[i];
  return bytes;
}

// two elements of `t` may share an address (an expanded tensor, overlapping rows): not a
// place to write to.  Every step must clear what the smaller ones span.
bool overlaps(const torch::Tensor& t) {
  Steps s;
  s.add(t);
  for (int i = 0; i < s.n; ++i) {
    if (s.stride[i] < span_below(t, s.stride[i])) return true;
    for (int j = 0; j < i; ++j)
      if (s.stride[i] == s.stride[j]) return true;
  }
  return false;
}

bool same_view(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.scalar_type() != b.scalar_type() || a.sizes() != b.sizes())
    return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// An address may belong to both.  False for slices that lie between one another, like
// the heads of one projection: where the larger steps of both are multiples of a period,
// what the smaller steps span must lie apart within it.
bool may_share(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t at = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
  if (at >= span_below(a, INT64_MAX) || -at >= span_below(b, INT64_MAX)) return false;
  Steps s;
  s.add(a);
  s.add(b);
  for (int i = 0; i < s.n; ++i) {
    int64_t period = 0;
    for (int j = 0; j < s.n; ++j)
      if (s.stride[j] >= s.stride[i]) period = std::gcd(period, s.stride[j]);
    if (period == 0) continue;
    const int64_t d = (at % period + period) % period;
    if (d >= span_below(a, s.stride[i]) && d + span_below(b, s.stride[i]) <= period) return false;
  }
  return true;
}

void check_apart(const torch::Tensor& written, const char* name, const torch::Tensor& other,
                 const char* other_name) {
  RAB_CHECK(!may_share(written, other), "%s shares memory with %s", name, other_name);
}

// a result may take its own input's place, element by element
void check_result(const torch::Tensor& written, const char* name, const torch::Tensor& in,
                  const char* in_name) {
  if (!same_view(written, in)) check_apart(written, name, in, in_name);
}

// A tensor that a call writes through its pointer: one that takes part in autograd's
// bookkeeping is refused, ...
void check_written(const torch::Tensor& t, const char* name) {
  RAB_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()),
            "%s is written in place and must not require a gradient", name);
}

// ... and any other counts as changed, so that a backward pass which saved it raises
// (inference tensors keep no count)
void mark_written(const torch::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

DeviceStatus* status_of(const OptTensor& status, const torch::Tensor& ref) {
  if (!status.has_value()) return nullptr;
  RAB_CHECK(status->scalar_type() == torch::kInt32 && status->numel() >= 8 &&
                status->is_contiguous(),
            "status must be int32[8]");
  check_same(*status, "status", ref);
  return reinterpret_cast<DeviceStatus*>(status->data_ptr());
}

// ---- rotary ----
void set_frequencies(RopeParams& p, const torch::Tensor& inv_freq, int64_t dim) {
  RAB_CHECK(inv_freq.scalar_type() == torch::kFloat64 && inv_freq.dim() == 1 &&
                inv_freq.is_contiguous(),
            "inv_freq must be a contiguous float64 vector");
  RAB_CHECK(inv_freq.numel() >= 1 && 2 * inv_freq.numel() <= dim,
            "inv_freq holds %lld frequencies; the head dim is %lld", ll(inv_freq.numel()), ll(dim));
  p.inv_freq = static_cast<const double*>(inv_freq.data_ptr());
  p.rotary_dim = static_cast<int>(2 * inv_freq.numel());
}

void set_positions(RopeParams& p, const torch::Tensor& positions, int64_t tokens) {
  const auto s = positions.scalar_type();
  RAB_CHECK(s == torch::kInt64 || s == torch::kInt32, "positions must be int64 or int32");
  RAB_CHECK(positions.dim() == 1 && positions.size(0) == tokens && positions.is_contiguous(),
            "positions must be a contiguous vector of %lld tokens", ll(tokens));
  p.positions = positions.data_ptr();
  p.positions64 = s == torch::kInt64;
}

// vectors of 16 bytes fit the head, the rotated part and its halves or pairs
bool rope_vectors(Elem e, int64_t dim, int rotary_dim) {
  const int64_t v = 16 / elem_bytes(e);
  return dim % v == 0 && rotary_dim % (2 * v) == 0;
}

RopeOperand dense_operand(const torch::Tensor& in, const torch::Tensor& out) {
  RopeOperand o;
  o.in = in.data_ptr();
  o.out = out.data_ptr();
  o.in_t = in.stride(0);
  o.in_h = in.stride(1);
  o.out_t = out.stride(0);
  o.out_h = out.stride(1);
  o.heads = static_cast<int>(in.size(1));
  o.rotate = 1;
  o.paged = 0;
  return o;
}

// The rotation has a gradient for backward passes alone: a tangent would be dropped.
void check_no_tangent(const torch::Tensor& t, const char* name) {
  RAB_CHECK(!t._fw_grad(0).defined(), "%s carries a tangent: forward-mode gradients are not offered",
            name);
}

void check_rope_input(const torch::Tensor& t, const char* name, const torch::Tensor& ref) {
  check_rows(t, name);
  RAB_CHECK(t.scalar_type() == ref.scalar_type(), "%s has another dtype than the first tensor", name);
  RAB_CHECK(t.size(0) == ref.size(0) && t.size(2) == ref.size(2),
            "%s must have the same tokens and head dim as the first tensor", name);
}

void check_rope_output(const torch::Tensor& t, const char* name, const torch::Tensor& in) {
  check_rows(t, name);
  RAB_CHECK(t.scalar_type() == in.scalar_type() && t.sizes() == in.sizes(),
            "%s must have its input's shape and dtype", name);
  RAB_CHECK(!overlaps(t), "%s shares memory between its elements", name);
  check_written(t, name);
}

constexpr int64_t kMaxRopeDim = 512;  // two elements per thread in a block of 256

std::tuple<torch::Tensor, OptTensor> rotary(torch::Tensor q, OptTensor k, torch::Tensor positions,
                                            torch::Tensor inv_freq, bool interleaved, double scale,
                                            bool inverse, OptTensor q_out, OptTensor k_out) {
  check_rows(q, "q");
  const Elem e = elem_of(q, "q");
  RAB_CHECK(q.size(2) <= kMaxRopeDim, "head dim %lld is over %lld", ll(q.size(2)), ll(kMaxRopeDim));
  RopeParams p{};
  p.tokens = static_cast<int>(q.size(0));
  p.dim = static_cast<int>(q.size(2));
  set_frequencies(p, inv_freq, q.size(2));
  set_positions(p, positions, q.size(0));
  RAB_CHECK(std::isfinite(static_cast<float>(scale)), "scale must be finite in fp32");
  if (k) check_rope_input(*k, "k", q);
  RAB_CHECK(k || !k_out, "k_out without k");
  check_no_tangent(q, "q");
  if (k) check_no_tangent(*k, "k");
  if (q_out) check_rope_output(*q_out, "q_out", q);
  if (k_out) check_rope_output(*k_out, "k_out", *k);
  if (q_out) {
    check_result(*q_out, "q_out", q, "q");
    if (k) check_apart(*q_out, "q_out", *k, "k");
    if (k_out) check_apart(*q_out, "q_out", *k_out, "k_out");
  }
  if (k_out) {
    check_result(*k_out, "k_out", *k, "k");
    check_apart(*k_out, "k_out", q, "q");
  }
  RAB_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  check_same(positions, "positions", q);
  check_same(inv_freq, "inv_freq", q);
  if (k) check_same(*k, "k", q);
  if (q_out) check_same(*q_out, "q_out", q);
  if (k_out) check_same(*k_out, "k_out", q);
  const c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor qo = q_out ? *q_out : fresh(q.sizes(), q.scalar_type(), q);
  OptTensor ko = k_out;
  if (k && !ko) ko = fresh(k->sizes(), k->scalar_type(), q);
  p.sms = flash_sm_count();
  p.interleaved = interleaved;
  p.scale = static_cast<float>(scale);
  p.sign = inverse ? -1.f : 1.f;
  // an operand without heads has no rows: the kernels share their threads out by heads
  bool vec = rope_vectors(e, q.size(2), p.rotary_dim);
  if (q.size(1) > 0) {
    p.op[p.n_op++] = dense_operand(q, qo);
    vec = vec && rows_aligned(q) && rows_aligned(qo);
  }
  if (k && k->size(1) > 0) {
    p.op[p.n_op++] = dense_operand(*k, *ko);
    vec = vec && rows_aligned(*k) && rows_aligned(*ko);
  }
  const int err = p.n_op == 0 ? 0 : rope_launch(e, p, vec, cur_stream());
  RAB_CHECK(err == 0, "rotary launch failed: %s", cudaGetErrorString(static_cast<cudaError_t>(err)));
  if (q_out) mark_written(qo);
  if (k_out) mark_written(*ko);
  return {qo, ko};
}

// The rotation as an autograd function.  Its gradient is the transposed rotation, the
// same pass by the negative angle; it goes through the function again, so it has a
// gradient of its own.  In C++, since short training steps are bound by host time: a
// forward call takes 9 us of it, and a backward pass little beside torch's own engine.
class RotaryFunction : public torch::autograd::Function<RotaryFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const torch::Tensor& q, const OptTensor& k,
                                                const torch::Tensor& positions,
                                                const torch::Tensor& inv_freq, bool interleaved,
                                                double scale, bool inverse) {
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["has_k"] = k.has_value();
    auto out = rotary(q, k, positions, inv_freq, interleaved, scale, inverse, c10::nullopt,
                      c10::nullopt);
    if (!k) return {std::get<0>(out)};
    return {std::get<0>(out), *std::get<1>(out)};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool();
    const double scale = ctx->saved_data["scale"].toDouble();
    const bool inverse = !ctx->saved_data["inverse"].toBool();
    const bool has_k = ctx->saved_data["has_k"].toBool();
    // a gradient may be expanded or transposed; the kernel needs adjacent elements
    auto rows = [](const torch::Tensor& t) {
      return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous();
    };
    const bool need_q = ctx->needs_input_grad(0), need_k = has_k && ctx->needs_input_grad(1);
    torch::autograd::variable_list result(7);
    if (need_q && need_k) {
      auto g = apply(rows(grads[0]), OptTensor(rows(grads[1])), saved[0], saved[1], interleaved,
                     scale, inverse);
      result[0] = g[0];
      result[1] = g[1];
    } else if (need_q || need_k) {
      result[need_q ? 0 : 1] = apply(rows(grads[need_q ? 0 : 1]), OptTensor(), saved[0], saved[1],
                                     interleaved, scale, inverse)[0];
    }
    return result;
  }
};

std::tuple<torch::Tensor, OptTensor> rotary_autograd(torch::Tensor q, OptTensor k,
                                                     torch::Tensor positions,
                                                     torch::Tensor inv_freq, bool interleaved,
                                                     double scale, bool inverse) {
  auto out = RotaryFunction::apply(q, k, positions, inv_freq, interleaved, scale, inverse);
  return {out[0], k ? OptTensor(out[1]) : OptTensor()};
}

// ---- pools and tables ----
// k and v pools [.., pages, heads_kv, page_size, dim]; `layers` allows a leading layer dimension
void check_pools(const torch::Tensor& k, const torch::Tensor& v, bool layers) {
  RAB_CHECK(k.dim() == 4 || (layers && k.dim() == 5),
            layers ? "k_pages must be [pages, heads_kv, page_size, dim], or with a leading layer dimension"
                   : "k_pages must be [pages, heads_kv, page_size, dim]");
  RAB_CHECK(v.sizes() == k.sizes(), "v_pages must have k_pages' shape");
  RAB_CHECK(v.scalar_type() == k.scalar_type(), "v_pages must have k_pages' dtype");
  const int64_t d = k.dim();
  const int64_t hk = k.size(d - 3), page = k.size(d - 2), dim = k.size(d - 1);
  RAB_CHECK(k.size(d - 4) >= 1 && k.size(d - 4) <= INT32_MAX && hk >= 1 && hk <= 65535 && page >= 1 && page <= 65536 &&
                dim >= 1 && dim <= 4096,
            "the cache pool has a dimension of zero or too large");
  for (const torch::Tensor* t : {&k, &v}) {
    RAB_CHECK(t->stride(d - 1) == 1 && (page == 1 || t->stride(d - 2) == dim) &&
                  (hk == 1 || t->stride(d - 3) == page * dim),
              "a page ([heads_kv, page_size, dim]) must be contiguous");
    RAB_CHECK(!overlaps(*t), "the cache pool shares memory between its pages");
    RAB_CHECK(dim * t->element_size() % 16 == 0, "a row of the cache must be a multiple of 16 bytes");
    RAB_CHECK(aligned16(t->data_ptr()) && t->stride(d - 4) * t->element_size() % 16 == 0 &&
                  (d == 4 || t->stride(0) * t->element_size() % 16 == 0),
              "the cache pool must be aligned to 16 bytes");
  }
}

struct Requests {
  int batch, uniform;
};

// page table, cached lengths and borders of the packed tokens
Requests check_requests(const torch::Tensor& table, const torch::Tensor& ctx, const OptTensor& cu,
                        int64_t tokens) {
  check_int32(table, "block_table", 2);
  check_int32(ctx, "context_lens", 1);
  const int64_t batch = ctx.size(0);
  RAB_CHECK(batch >= 1, "context_lens is empty");
  RAB_CHECK(table.size(0) == batch, "block_table has %lld rows for %lld requests", ll(table.size(0)),
            ll(batch));
  RAB_CHECK(table.size(1) >= 1 && table.size(1) <= INT32_MAX, "block_table has no columns");
  Requests r{static_cast<int>(batch), 0};
  if (cu) {
    check_int32(*cu, "cu_q", 1);
    RAB_CHECK(cu->size(0) == batch + 1, "cu_q must have %lld entries for %lld requests",
              ll(batch + 1), ll(batch));
  } else {
    RAB_CHECK(tokens % batch == 0,
              "%lld tokens cannot be shared evenly by %lld requests: give cu_q", ll(tokens),
              ll(batch));
    r.uniform = static_cast<int>(tokens / batch);
  }
  return r;
}

void check_requests_device(const torch::Tensor& table, const torch::Tensor& ctx,
                           const OptTensor& cu, const torch::Tensor& ref) {
  check_same(table, "block_table", ref);
  check_same(ctx, "context_lens", ref);
  if (cu) check_same(*cu, "cu_q", ref);
}

// ---- append ----
OptTensor append_kv(torch::Tensor k, torch::Tensor v, torch::Tensor k_pages, torch::Tensor v_pages,
                    torch::Tensor table, torch::Tensor ctx, OptTensor cu, OptTensor positions,
                    OptTensor inv_freq, bool interleaved, double scale, OptTensor q,
                    OptTensor q_out, OptTensor status) {
  check_pools(k_pages, v_pages, false);
  check_written(k_pages, "k_pages");
  check_written(v_pages, "v_pages");
  check_rows(k, "k");
  const Elem e = elem_of(k, "k");
  RAB_CHECK(k.scalar_type() == k_pages.scalar_type(), "k and the cache must share a dtype");
  RAB_CHECK(v.dim() == 3 && v.sizes() == k.sizes(), "v must have k's shape");
  check_rope_input(v, "v", k);
  const int64_t dim = k.size(2);
  RAB_CHECK(k.size(1) == k_pages.size(1) && dim == k_pages.size(3),
            "k must be [tokens, %lld, %lld] for this cache", ll(k_pages.size(1)),
            ll(k_pages.size(3)));
  RAB_CHECK(dim <= kMaxRopeDim, "head dim %lld is over %lld", ll(dim), ll(kMaxRopeDim));
  const Requests r = check_requests(table, ctx, cu, k.size(0));
  RopeParams p{};
  p.tokens = static_cast<int>(k.size(0));
  p.dim = static_cast<int>(dim);
  if (inv_freq) set_frequencies(p, *inv_freq, dim);
  RAB_CHECK(inv_freq || (!positions && !q), "positions and q have no use without inv_freq");
  if (positions) set_positions(p, *positions, k.size(0));
  RAB_CHECK(std::isfinite(static_cast<float>(scale)), "scale must be finite in fp32");
  if (q) check_rope_input(*q, "q", k);
  RAB_CHECK(q || !q_out, "q_out without q");
  check_apart(k_pages, "k_pages", v_pages, "v_pages");
  if (q_out) {
    check_rope_output(*q_out, "q_out", *q);
    check_result(*q_out, "q_out", *q, "q");
    check_apart(*q_out, "q_out", k, "k");
    check_apart(*q_out, "q_out", v, "v");
    check_apart(*q_out, "q_out", k_pages, "k_pages");
    check_apart(*q_out, "q_out", v_pages, "v_pages");
  }
  RAB_CHECK(k.is_cuda(), "k must be a CUDA tensor");
  check_same(v, "v", k);
  check_same(k_pages, "k_pages", k);
  check_same(v_pages, "v_pages", k);
  check_requests_device(table, ctx, cu, k);
  if (inv_freq) check_same(*inv_freq, "inv_freq", k);
  if (positions) check_same(*positions, "positions", k);
  if (q) check_same(*q, "q", k);
  if (q_out) check_same(*q_out, "q_out", k);
  p.status = status_of(status, k);
  const c10::cuda::CUDAGuard guard(k.device());
  bool vec = rope_vectors(e, dim, p.rotary_dim) && rows_aligned(k) && rows_aligned(v);
  OptTensor qo = q_out;
  if (q) {
    if (!qo) qo = fresh(q->sizes(), q->scalar_type(), k);
    if (q->size(1) > 0) {
      p.op[p.n_op++] = dense_operand(*q, *qo);
      vec = vec && rows_aligned(*q) && rows_aligned(*qo);
    }
  }
  const std::pair<const torch::Tensor*, const torch::Tensor*> kv[2] = {{&k, &k_pages},
                                                                       {&v, &v_pages}};
  for (int i = 0; i < 2; ++i) {
    RopeOperand o = dense_operand(*kv[i].first, *kv[i].second);  // page stride, head stride
    o.out_h = k_pages.size(2) * dim;
    o.rotate = i == 0 && inv_freq ? 1 : 0;
    o.paged = 1;
    p.op[p.n_op++] = o;
  }
  p.sms = flash_sm_count();
  p.interleaved = interleaved;
  p.scale = static_cast<float>(scale);
  p.sign = 1.f;
  p.table = static_cast<const int*>(table.data_ptr());
  p.table_stride = table.stride(0);
  p.table_w = static_cast<int>(table.size(1));
  p.num_pages = static_cast<int>(k_pages.size(0));
  p.page_size = static_cast<int>(k_pages.size(2));
  p.ctx = static_cast<const int*>(ctx.data_ptr());
  p.cu = cu ? static_cast<const int*>(cu->data_ptr()) : nullptr;
  p.batch = r.batch;
  p.uniform = r.uniform;
  const int err = rope_launch(e, p, vec, cur_stream());
  RAB_CHECK(err == 0, "append_kv launch failed: %s",
            cudaGetErrorString(static_cast<cudaError_t>(err)));
  mark_written(k_pages);
  mark_written(v_pages);
  if (q_out) mark_written(qo.value());
  return qo;
}

// ---- page copies ----
void copy_pages(torch::Tensor k_pages, torch::Tensor v_pages, torch::Tensor src, torch::Tensor dst) {
  check_pools(k_pages, v_pages, true);
  check_written(k_pages, "k_pages");
  check_written(v_pages, "v_pages");
  check_result(k_pages, "k_pages", v_pages, "v_pages");  // one pool twice is copied alike
  for (const torch::Tensor* t : {&src, &dst})
    RAB_CHECK(!t->is_cuda() && t->dim() == 1 && t->is_contiguous() &&
                  (t->scalar_type() == torch::kInt32 || t->scalar_type() == torch::kInt64),
              "src and dst must be int32 or int64 vectors on the host");
  RAB_CHECK(src.size(0) == dst.size(0), "src names %lld pages, dst %lld", ll(src.size(0)),
            ll(dst.size(0)));
  const int64_t d = k_pages.dim(), pages = k_pages.size(d - 4), n = src.size(0);
  RAB_CHECK(d == 4 || k_pages.size(0) <= 32767, "over 32767 layers");
  auto at = [](const torch::Tensor& t, int64_t i) {
    return t.scalar_type() == torch::kInt32 ? static_cast<int64_t>(static_cast<const int*>(t.data_ptr())[i])
                                            : static_cast<const int64_t*>(t.data_ptr())[i];
  };
  // every page is written once at most, and none that is also read: the copies
  // of a launch run at the same time.  `mark`: a page that is written, or the
  // number of the group of pairs that read it.
  constexpr int kFree = -1, kWritten = -2;
  std::vector<int> mark(static_cast<size_t>(pages), kFree);
  for (int64_t i = 0; i < n; ++i) {
    const int64_t x = at(dst, i);
    RAB_CHECK(x >= 0 && x < pages, "dst[%lld] = %lld is no page of a pool of %lld", ll(i), ll(x),
              ll(pages));
    RAB_CHECK(mark[static_cast<size_t>(x)] == kFree, "page %lld is twice in dst", ll(x));
    mark[static_cast<size_t>(x)] = kWritten;
  }
  std::vector<int> group(static_cast<size_t>(n)), sources, count;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t x = at(src, i);
    RAB_CHECK(x >= 0 && x < pages, "src[%lld] = %lld is no page of a pool of %lld", ll(i), ll(x),
              ll(pages));
    int& m = mark[static_cast<size_t>(x)];
    RAB_CHECK(m != kWritten, "page %lld is both in src and in dst", ll(x));
    if (m == kFree) {
      m = static_cast<int>(sources.size());
      sources.push_back(static_cast<int>(x));
      count.push_back(0);
    }
    group[static_cast<size_t>(i)] = m;
    ++count[static_cast<size_t>(m)];
  }
  // the pairs in the order of their groups
  std::vector<int> place(sources.size() + 1, 0), sorted(static_cast<size_t>(n));
  for (size_t s = 0; s < sources.size(); ++s) place[s + 1] = place[s] + count[s];
  const std::vector<int> begin = place;
  for (int64_t i = 0; i < n; ++i)
    sorted[static_cast<size_t>(place[static_cast<size_t>(group[static_cast<size_t>(i)])]++)] =
        static_cast<int>(at(dst, i));
  RAB_CHECK(k_pages.is_cuda(), "k_pages must be a CUDA tensor");
  check_same(v_pages, "v_pages", k_pages);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  const int64_t es = k_pages.element_size();
  auto launch = [&](auto& p) {
    constexpr int kMax = std::remove_reference_t<decltype(p)>::kMax;
    p.k = static_cast<uint8_t*>(k_pages.data_ptr());
    p.v = static_cast<uint8_t*>(v_pages.data_ptr());
    p.k_page = k_pages.stride(d - 4) * es;
    p.v_page = v_pages.stride(d - 4) * es;
    p.layers = d == 5 ? static_cast<int>(k_pages.size(0)) : 1;
    p.k_layer = d == 5 ? k_pages.stride(0) * es : 0;
    p.v_layer = d == 5 ? v_pages.stride(0) * es : 0;
    p.page_bytes = k_pages.size(d - 3) * k_pages.size(d - 2) * k_pages.size(d - 1) * es;
    size_t s = 0;
    for (int i = 0; i < n; i += kMax) {  // a group cut here reads its page again
      const int end = static_cast<int>(std::min<int64_t>(n, i + kMax));
      p.n_src = 0;
      p.first[0] = 0;
      std::copy(sorted.begin() + i, sorted.begin() + end, p.dst);
      for (; s < sources.size() && begin[s] < end; ++s) {
        p.src[p.n_src] = sources[s];
        p.first[++p.n_src] = std::min(begin[s + 1], end) - i;
        if (begin[s + 1] > end) break;
      }
      const int err = page_copy_launch(p, cur_stream());
      RAB_CHECK(err == 0, "copy_pages launch failed: %s",
                cudaGetErrorString(static_cast<cudaError_t>(err)));
    }
  };
  if (n <= kFewPairs) {
    PageCopyParams<kFewPairs> p;
    launch(p);
  } else {
    PageCopyParams<kManyPairs> p;
    launch(p);
  }
  mark_written(k_pages);
  mark_written(v_pages);
}

// ---- accepted path ----
void compact_path(torch::Tensor k_pages, torch::Tensor v_pages, torch::Tensor table,
                  torch::Tensor ctx, torch::Tensor path, torch::Tensor path_lens, OptTensor status) {
  check_pools(k_pages, v_pages, true);
  check_written(k_pages, "k_pages");
  check_written(v_pages, "v_pages");
  check_apart(k_pages, "k_pages", v_pages, "v_pages");
  const Requests r = check_requests(table, ctx, c10::nullopt, 0);
  check_int32(path, "path", 2);
  check_int32(path_lens, "path_lens", 1);
  RAB_CHECK(path.size(0) == r.batch && path_lens.size(0) == r.batch,
            "path and path_lens must have a row for each of %d requests", r.batch);
  RAB_CHECK(path.size(1) <= INT32_MAX, "path is too wide");
  const int64_t d = k_pages.dim();
  RAB_CHECK(d == 4 || k_pages.size(0) <= 32767, "over 32767 layers");
  RAB_CHECK(k_pages.is_cuda(), "k_pages must be a CUDA tensor");
  check_same(v_pages, "v_pages", k_pages);
  check_requests_device(table, ctx, c10::nullopt, k_pages);
  check_same(path, "path", k_pages);
  check_same(path_lens, "path_lens", k_pages);
  const int64_t es = k_pages.element_size();
  PathParams p{};
  p.status = status_of(status, k_pages);
  p.k = static_cast<uint8_t*>(k_pages.data_ptr());
  p.v = static_cast<uint8_t*>(v_pages.data_ptr());
  p.k_page = k_pages.stride(d - 4) * es;
  p.v_page = v_pages.stride(d - 4) * es;
  p.layers = d == 5 ? static_cast<int>(k_pages.size(0)) : 1;
  p.k_layer = d == 5 ? k_pages.stride(0) * es : 0;
  p.v_layer = d == 5 ? v_pages.stride(0) * es : 0;
  p.heads = static_cast<int>(k_pages.size(d - 3));
  p.page_size = static_cast<int>(k_pages.size(d - 2));
  p.row_bytes = static_cast<int>(k_pages.size(d - 1) * es);
  p.num_pages = static_cast<int>(k_pages.size(d - 4));
  p.table = static_cast<const int*>(table.data_ptr());
  p.table_stride = table.stride(0);
  p.table_w = static_cast<int>(table.size(1));
  p.ctx = static_cast<const int*>(ctx.data_ptr());
  p.path = static_cast<const int*>(path.data_ptr());
  p.path_stride = path.stride(0);
  p.path_w = static_cast<int>(path.size(1));
  p.path_lens = static_cast<const int*>(path_lens.data_ptr());
  p.batch = r.batch;
  const c10::cuda::CUDAGuard guard(k_pages.device());
  const int err = path_compact_launch(p, cur_stream());
  RAB_CHECK(err == 0, "compact_path launch failed: %s",
            cudaGetErrorString(static_cast<cudaError_t>(err)));
  mark_written(k_pages);
  mark_written(v_pages);
}

// ---- attention over the cache ----
std::tuple<torch::Tensor, OptTensor> tree_attention(torch::Tensor q, torch::Tensor k_pages,
                                                    torch::Tensor v_pages, torch::Tensor table,
                                                    torch::Tensor ctx, OptTensor cu,
                                                    c10::optional<int64_t> max_q, OptTensor mask,
                                                    c10::optional<double> scale, bool return_lse,
                                                    OptTensor out, OptTensor status,
                                                    double timeout_s) {
  check_pools(k_pages, v_pages, false);
  check_rows(q, "q");
  const Elem e = elem_of(q, "q");
  RAB_CHECK(q.scalar_type() == k_pages.scalar_type(), "q and the cache must share a dtype");
  const int64_t dim = q.size(2), heads = q.size(1), hk = k_pages.size(1), total = q.size(0);
  RAB_CHECK(dim == 64 || dim == 128, "head_dim must be 64 or 128");
  RAB_CHECK(k_pages.size(3) == dim, "q has head dim %lld, the cache %lld", ll(dim),
            ll(k_pages.size(3)));
  RAB_CHECK(heads >= 1 && heads % hk == 0, "%lld query heads are no multiple of %lld kv heads",
            ll(heads), ll(hk));
  const int64_t page = k_pages.size(2);
  RAB_CHECK(page >= 16 && page <= 256 && (page & (page - 1)) == 0,
            "page size %lld: attention takes 16, 32, 64, 128 or 256", ll(page));
  const Requests r = check_requests(table, ctx, cu, total);
  RAB_CHECK(table.size(1) <= (1 << 30) / page, "block_table has room for over 2^30 tokens");
  const int64_t rows = total * (heads / hk);
  RAB_CHECK(rows <= (1 << 30), "over 2^30 rows of a kv head");
  RAB_CHECK(!max_q || *max_q >= 1, "max_q must be positive");
  if (mask) {
    RAB_CHECK(mask->dim() == 2 && mask->size(0) == total,
              "mask must have a row for each of %lld tokens", ll(total));
    RAB_CHECK(mask->scalar_type() == torch::kBool || mask->scalar_type() == torch::kInt32,
              "mask must be bool, or int32 words of 32 bits");
    RAB_CHECK(mask->size(1) >= 1 && (mask->stride(1) == 1 || mask->size(1) == 1),
              "mask must have columns, contiguous in a row");
    RAB_CHECK(mask->size(1) <= (1 << 24), "mask is too wide");
  }
  const double sc = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(dim));
  const float scale_log2 = static_cast<float>(sc * 1.4426950408889634074);
  RAB_CHECK(std::isfinite(scale_log2), "scale must be finite in fp32");
  if (out) {
    check_rope_output(*out, "out", q);
    RAB_CHECK(rows_aligned(*out), "out must have rows aligned to 16 bytes");
    check_result(*out, "out", q, "q");
    check_apart(*out, "out", k_pages, "k_pages");
    check_apart(*out, "out", v_pages, "v_pages");
  }
  RAB_CHECK(timeout_s > 0 && timeout_s <= 3600, "timeout_s must be in (0, 3600]");
  RAB_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  check_same(k_pages, "k_pages", q);
  check_same(v_pages, "v_pages", q);
  check_requests_device(table, ctx, cu, q);
  if (mask) check_same(*mask, "mask", q);
  if (out) check_same(*out, "out", q);
  TreeParams p{};
  p.status = status_of(status, q);
  const c10::cuda::CUDAGuard guard(q.device());
  // the kernels read q 4 to 16 bytes at a time; contiguous() would hand a contiguous tensor
  // at an odd place back as it is
  if (!rows_aligned(q)) q = q.clone(at::MemoryFormat::Contiguous);
  torch::Tensor o = out ? *out : fresh({total, heads, dim}, q.scalar_type(), q);
  OptTensor lse;
  if (return_lse) lse = fresh({total, heads}, torch::kFloat32, q);
  if (total == 0) return {o, lse};
  const cudaStream_t stream = cur_stream();
  torch::Tensor bits;
  if (mask && mask->scalar_type() == torch::kBool) {
    const int64_t words = (mask->size(1) + 31) / 32;
    bits = fresh({total, words}, torch::kInt32, q);
    const int err = pack_mask_launch(static_cast<const uint8_t*>(mask->data_ptr()), mask->stride(0),
                                     static_cast<int>(total), static_cast<int>(mask->size(1)),
                                     static_cast<uint32_t*>(bits.data_ptr()),
                                     static_cast<int>(words), stream);
    RAB_CHECK(err == 0, "mask packing failed: %s", cudaGetErrorString(static_cast<cudaError_t>(err)));
  } else if (mask) {
    bits = *mask;
  }
  p.q = q.data_ptr();
  p.q_t = q.stride(0);
  p.q_h = q.stride(1);
  p.out = o.data_ptr();
  p.out_t = o.stride(0);
  p.out_h = o.stride(1);
  p.lse = lse ? static_cast<float*>(lse->data_ptr()) : nullptr;
  p.k = k_pages.data_ptr();
  p.v = v_pages.data_ptr();
  p.k_page = k_pages.stride(0);
  p.v_page = v_pages.stride(0);
  p.num_pages = static_cast<int>(k_pages.size(0));
  p.page_size = static_cast<int>(page);
  while ((1 << p.page_shift) < p.page_size) ++p.page_shift;
  p.table = static_cast<const int*>(table.data_ptr());
  p.table_stride = table.stride(0);
  p.table_w = static_cast<int>(table.size(1));
  p.ctx = static_cast<const int*>(ctx.data_ptr());
  p.cu = cu ? static_cast<const int*>(cu->data_ptr()) : nullptr;
  p.batch = r.batch;
  p.uniform = r.uniform;
  p.total = static_cast<int>(total);
  p.heads = static_cast<int>(heads);
  p.heads_kv = static_cast<int>(hk);
  p.group = static_cast<int>(heads / hk);
  p.dim = static_cast<int>(dim);
  if (mask) {
    p.mask = static_cast<const uint32_t*>(bits.data_ptr());
    p.mask_stride = bits.stride(0);
    p.mask_w = static_cast<int>(bits.size(1));
  }
  p.scale_log2 = scale_log2;
  p.timeout_ns = static_cast<uint64_t>(timeout_s * 1e9);
  const int64_t most = max_q ? std::min<int64_t>(*max_q, total) : (cu ? total : r.uniform);
  const TreePlan plan = tree_plan(e, p, static_cast<int>(most), flash_sm_count());
  // the kernels count the places of their line of units in 32 bits
  RAB_CHECK((rows / plan.rows_per_unit + r.batch) * hk <=
                (int64_t{1} << 31) / (table.size(1) * page / plan.tile_keys + 4),
            "too many units of work for one call: split the batch");
  const size_t floats = plan.acc_floats + plan.ml_floats + plan.meta_ints;
  torch::Tensor ws = fresh({static_cast<int64_t>(floats)}, torch::kFloat32, q);
  p.rec_acc = static_cast<float*>(ws.data_ptr());
  p.rec_m = p.rec_acc + plan.acc_floats;
  p.rec_l = p.rec_m + plan.ml_floats / 2;
  p.meta = reinterpret_cast<int*>(p.rec_m + plan.ml_floats);
  p.grid = plan.grid;
  const int err = tree_launch(e, p, plan, stream);
  RAB_CHECK(err == 0, "tree_attention launch failed: %s",
            cudaGetErrorString(static_cast<cudaError_t>(err)));
  if (out) mark_written(o);
  return {o, lse};
}

std::tuple<torch::Tensor, torch::Tensor> tree_mask(torch::Tensor parents, OptTensor cu,
                                                   int64_t batch, int64_t max_q, OptTensor status) {
  check_int32(parents, "parents", 1);
  const int64_t total = parents.size(0);
  RAB_CHECK(max_q >= 1 && max_q <= (1 << 24), "max_q must be positive and below 2^24");
  RAB_CHECK(total <= INT32_MAX, "parents is too long");
  if (cu) {
    check_int32(*cu, "cu_q", 1);
    RAB_CHECK(cu->size(0) >= 2, "cu_q is empty");
    batch = cu->size(0) - 1;
  } else {
    RAB_CHECK(batch >= 1 && total % batch == 0, "%lld tokens cannot be shared evenly by %lld requests",
              ll(total), ll(batch));
  }
  RAB_CHECK(parents.is_cuda(), "parents must be a CUDA tensor");
  if (cu) check_same(*cu, "cu_q", parents);
  DeviceStatus* st = status_of(status, parents);
  const c10::cuda::CUDAGuard guard(parents.device());
  const int64_t words = (max_q + 31) / 32;
  torch::Tensor mask = fresh({total, words}, torch::kInt32, parents);
  torch::Tensor depth = fresh({total}, torch::kInt32, parents);
  const int err = tree_mask_launch(
      static_cast<const int*>(parents.data_ptr()), cu ? static_cast<const int*>(cu->data_ptr()) : nullptr,
      static_cast<int>(batch), cu ? 0 : static_cast<int>(total / batch), static_cast<int>(total),
      static_cast<uint32_t*>(mask.data_ptr()), static_cast<int>(words),
      static_cast<int*>(depth.data_ptr()), st, cur_stream());
  RAB_CHECK(err == 0, "tree_mask launch failed: %s",
            cudaGetErrorString(static_cast<cudaError_t>(err)));
  return {mask, depth};
}

torch::Tensor pack_mask(torch::Tensor mask) {
  RAB_CHECK(mask.scalar_type() == torch::kBool && mask.dim() == 2, "mask must be bool [tokens, columns]");
  RAB_CHECK(mask.size(1) >= 1 && mask.size(1) <= (1 << 24) && mask.size(0) <= INT32_MAX &&
                (mask.stride(1) == 1 || mask.size(1) == 1),
            "mask must have columns, contiguous in a row");
  RAB_CHECK(mask.is_cuda(), "mask must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(mask.device());
  const int64_t words = (mask.size(1) + 31) / 32;
  torch::Tensor bits = fresh({mask.size(0), words}, torch::kInt32, mask);
  const int err = pack_mask_launch(static_cast<const uint8_t*>(mask.data_ptr()), mask.stride(0),
                                   static_cast<int>(mask.size(0)), static_cast<int>(mask.size(1)),
                                   static_cast<uint32_t*>(bits.data_ptr()), static_cast<int>(words),
                                   cur_stream());
  RAB_CHECK(err == 0, "mask packing failed: %s", cudaGetErrorString(static_cast<cudaError_t>(err)));
  return bits;
}

}  // namespace
}  // namespace rab

void register_paged(pybind11::module_& m) {
  m.def("rotary", &rab::rotary, "rotary positions on q and k", py::arg("q"), py::arg("k"),
        py::arg("positions"), py::arg("inv_freq"), py::arg("interleaved") = false,
        py::arg("scale") = 1.0, py::arg("inverse") = false, py::arg("q_out") = c10::nullopt,
        py::arg("k_out") = c10::nullopt);
  m.def("rotary_autograd", &rab::rotary_autograd, "rotary positions with their gradient",
        py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("inv_freq"),
        py::arg("interleaved") = false, py::arg("scale") = 1.0, py::arg("inverse") = false);
  m.def("append_kv", &rab::append_kv, "write new tokens' K and V into a paged cache", py::arg("k"),
        py::arg("v"), py::arg("k_pages"), py::arg("v_pages"), py::arg("block_table"),
        py::arg("context_lens"), py::arg("cu_q") = c10::nullopt,
        py::arg("positions") = c10::nullopt, py::arg("inv_freq") = c10::nullopt,
        py::arg("interleaved") = false, py::arg("scale") = 1.0, py::arg("q") = c10::nullopt,
        py::arg("q_out") = c10::nullopt, py::arg("status") = c10::nullopt);
  m.def("copy_pages", &rab::copy_pages, "copy pages of a cache pool", py::arg("k_pages"),
        py::arg("v_pages"), py::arg("src"), py::arg("dst"));
  m.def("compact_path", &rab::compact_path, "keep the accepted path of drafted trees",
        py::arg("k_pages"), py::arg("v_pages"), py::arg("block_table"), py::arg("context_lens"),
        py::arg("path"), py::arg("path_lens"), py::arg("status") = c10::nullopt);
  m.def("tree_attention", &rab::tree_attention, "attention of new tokens over a paged cache",
        py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("block_table"),
        py::arg("context_lens"), py::arg("cu_q") = c10::nullopt, py::arg("max_q") = c10::nullopt,
        py::arg("mask") = c10::nullopt, py::arg("scale") = c10::nullopt,
        py::arg("return_lse") = false, py::arg("out") = c10::nullopt,
        py::arg("status") = c10::nullopt, py::arg("timeout_s") = 10.0);
  m.def("tree_mask", &rab::tree_mask, "ancestor bits and depths of drafted trees",
        py::arg("parents"), py::arg("cu_q") = c10::nullopt, py::arg("batch") = 1, py::arg("max_q"),
        py::arg("status") = c10::nullopt);
  m.def("pack_mask", &rab::pack_mask, "bool mask -> 32-bit words", py::arg("mask"));
}
