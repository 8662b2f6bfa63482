// rotary.cu - rotary positions on q and k, and the append of new tokens to a
// paged cache (rotated K, V, and q' in one launch).
//
// A pair (x1, x2) of token t turns by the angle a = position * inv_freq[p]:
//   (x1 cos a - x2 sin a, x2 cos a + x1 sin a) * scale
// The gradient is the same rotation by -a.  Positions are whole numbers, so
// the angle is kept in turns as a 64-bit binary fraction: step = inv_freq /
// (2 pi) mod 1 in units of 2^-64, phase = position * step mod 2^64.  The wrap of
// the integer product is the reduction to one turn, exact at any position;
// only the rounding of step (2^-53 relative) grows with it.  sin and cos of
// the top 32 bits follow in fp32 (sincospif).
//
// Bound by memory: every element is read and written once.  A thread owns two
// 16-byte vectors of a row (8 pairs of 2-byte types, 4 of fp32), forms their
// sines and cosines once and then walks a group of heads with all loads of four
// heads in flight; the head group shrinks until the grid fills the GPU.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "paged.h"

namespace rab {

namespace {

constexpr int kRopeThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <>
__device__ __forceinline__ float to_f<__half>(__half x) {
  return __half2float(x);
}
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float x) {
  return __float2half_rn(x);
}

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T x[VEC];
};

// frequency in radians per position -> fraction of a turn per position, 2^-64 units
__device__ __forceinline__ uint64_t phase_step(double inv_freq) {
  double t = inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  t -= floor(t);
  return __double2ull_rn(t * 18446744073709551616.0);
}

template <typename T, int VEC, bool kInter>
__device__ __forceinline__ void rotate(Pack<T, VEC>& a, Pack<T, VEC>& b, const float* cs,
                                       const float* sn) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if constexpr (kInter) {  // the 2 * VEC elements of a | b hold the pairs side by side
      T& e1 = 2 * i < VEC ? a.x[(2 * i) % VEC] : b.x[(2 * i) % VEC];
      T& e2 = 2 * i + 1 < VEC ? a.x[(2 * i + 1) % VEC] : b.x[(2 * i + 1) % VEC];
      const float x1 = to_f(e1), x2 = to_f(e2);
      e1 = from_f<T>(x1 * cs[i] - x2 * sn[i]);
      e2 = from_f<T>(x2 * cs[i] + x1 * sn[i]);
    } else {
      const float x1 = to_f(a.x[i]), x2 = to_f(b.x[i]);
      a.x[i] = from_f<T>(x1 * cs[i] - x2 * sn[i]);
      b.x[i] = from_f<T>(x2 * cs[i] + x1 * sn[i]);
    }
  }
}

// grid.x: token groups; grid.y: head groups of `hc` heads, operand after operand
template <typename T, int VEC, bool kInter>
__global__ void __launch_bounds__(kRopeThreads)
    rope_kernel(const __grid_constant__ RopeParams p, int tasks, int tokens_per_block, int hc) {
  using P = Pack<T, VEC>;
  const int local = threadIdx.x / tasks;
  const int task = threadIdx.x - local * tasks;
  const int token = blockIdx.x * tokens_per_block + local;
  if (local >= tokens_per_block || token >= p.tokens) return;
  int o = 0, g = blockIdx.y;
  while (o + 1 < p.n_op && g >= (p.op[o].heads + hc - 1) / hc) {
    g -= (p.op[o].heads + hc - 1) / hc;
    ++o;
  }
  const RopeOperand& op = p.op[o];
  const int h_end = min(op.heads, (g + 1) * hc);

  // where the token lies in the cache
  int64_t at = 0, dst = static_cast<int64_t>(token) * op.out_t;
  if (p.ctx != nullptr) {
    int b;
    int first;
    if (p.cu == nullptr) {
      b = token / p.uniform;
      first = b * p.uniform;
    } else {
      int lo = 0, hi = p.batch;  // the last request that starts at or before the token
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid] <= token) lo = mid;
        else hi = mid;
      }
      b = lo;
      first = p.cu[b];
      if (token < first || token >= p.cu[b + 1]) return;  // behind the last request
    }
    at = static_cast<int64_t>(p.ctx[b]) + (token - first);
    if (op.paged) {
      const int64_t entry = at / p.page_size;
      if (at < 0 || entry >= p.table_w) {
        if (task == 0 && g == 0) st_record(p.status, kStatusBadArgs, kBadPosition, token);
        return;
      }
      const int page = p.table[static_cast<int64_t>(b) * p.table_stride + entry];
      if (page < 0 || page >= p.num_pages) {
        if (task == 0 && g == 0) st_record(p.status, kStatusBadArgs, kBadPage, page);
        return;
      }
      dst = static_cast<int64_t>(page) * op.out_t + (at - entry * p.page_size) * p.dim;
    }
  }

  const int rot_tasks = op.rotate ? p.rotary_dim / (2 * VEC) : 0;
  const bool rot = task < rot_tasks;
  const int rest = rot_tasks * 2 * VEC;  // first element that passes through
  int ea, eb;
  if (rot && !kInter) {
    ea = task * VEC;
    eb = p.rotary_dim / 2 + task * VEC;
  } else {
    ea = rot ? task * 2 * VEC : rest + (task - rot_tasks) * 2 * VEC;
    eb = ea + VEC;
  }
  if (ea >= p.dim) return;
  const bool two = eb < p.dim;

  float cs[VEC], sn[VEC];
  if (rot) {
    int64_t pos = at;
    if (p.positions != nullptr)
      pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[token]
                          : static_cast<int64_t>(static_cast<const int*>(p.positions)[token]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const uint64_t phase = static_cast<uint64_t>(pos) * phase_step(p.inv_freq[task * VEC + i]);
      const int top = static_cast<int>((phase + 0x80000000ull) >> 32);
      sincospif(static_cast<float>(top) * 0x1p-31f, &sn[i], &cs[i]);
      cs[i] *= p.scale;
      sn[i] *= p.scale * p.sign;
    }
  }

  const T* in = static_cast<const T*>(op.in) + static_cast<int64_t>(token) * op.in_t;
  T* out = static_cast<T*>(op.out) + dst;
  constexpr int kU = 4;
  for (int h = g * hc; h < h_end; h += kU) {
    P a[kU], b[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (h + u < h_end) {
        const T* r = in + static_cast<int64_t>(h + u) * op.in_h;
        a[u] = *reinterpret_cast<const P*>(r + ea);
        if (two) b[u] = *reinterpret_cast<const P*>(r + eb);
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (h + u < h_end) {
        if (rot) rotate<T, VEC, kInter>(a[u], b[u], cs, sn);
        T* w = out + static_cast<int64_t>(h + u) * op.out_h;
        *reinterpret_cast<P*>(w + ea) = a[u];
        if (two) *reinterpret_cast<P*>(w + eb) = b[u];
      }
    }
  }
}

template <typename T, int VEC, bool kInter>
int rope_run(const RopeParams& p, cudaStream_t stream) {
  // a row's tasks: two vectors each; one more when the dims leave a single vector over
  const int tasks = (p.dim + 2 * VEC - 1) / (2 * VEC);
  // rows wider than a block are not offered (the bindings bound dim)
  const int tpb = kRopeThreads / tasks;
  const int gx = (p.tokens + tpb - 1) / tpb;
  int hc = 16, gy = 0;
  // shrink the head group until there are eight blocks per SM: each block
  // repeats its tokens' sines, which is cheap beside idle SMs
  for (; hc >= 1; hc >>= 1) {
    gy = 0;
    for (int i = 0; i < p.n_op; ++i) gy += (p.op[i].heads + hc - 1) / hc;
    if (hc == 1 || static_cast<int64_t>(gx) * gy >= 148 * 8) break;
  }
  rope_kernel<T, VEC, kInter><<<dim3(gx, gy), kRopeThreads, 0, stream>>>(p, tasks, tpb, hc);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int VEC>
int rope_layout(const RopeParams& p, cudaStream_t stream) {
  return p.interleaved ? rope_run<T, VEC, true>(p, stream) : rope_run<T, VEC, false>(p, stream);
}

}  // namespace

int rope_launch(Elem elem, const RopeParams& p, bool vectors, cudaStream_t stream) {
  if (p.tokens == 0) return 0;
  switch (elem) {
    case Elem::kBF16:
      return vectors ? rope_layout<__nv_bfloat16, 8>(p, stream)
                     : rope_layout<__nv_bfloat16, 1>(p, stream);
    case Elem::kF16:
      return vectors ? rope_layout<__half, 8>(p, stream) : rope_layout<__half, 1>(p, stream);
    default:
      return vectors ? rope_layout<float, 4>(p, stream) : rope_layout<float, 1>(p, stream);
  }
}

}  // namespace rab
