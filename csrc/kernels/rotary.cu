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
// Bound by memory: every element is read and written once.  A block takes a few
// tokens and a group of heads: its threads first form the sines and cosines of
// the tokens' pairs once, into shared memory, together with each token's place in
// the cache, and then stream rows past them.  A thread keeps one place in the row
// (two 16-byte vectors: 8 pairs of a 2-byte type, 4 of fp32), so its sines stay in
// the same shared-memory words.  One row per thread and 32 registers, so that eight
// blocks share an SM, beat more rows in flight per thread: 16384 tokens x 40 heads
// x 128 in bf16 take 56 us (6.0 TB/s, 0.91 of the measured copy rate) against 70 to
// 100 us with two to four rows and the registers they need, and 57 us with packed
// fp32 products.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.h"
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

// Where a pair's sine lies among its token's: a thread reads the VEC pairs of its
// task two at a time, and the tasks of a row side by side, so that a warp's
// 16-byte reads meet no bank twice.
template <int VEC>
__device__ __forceinline__ int cs_slot(int pair, int pairs) {
  if constexpr (VEC == 1) return pair;
  const int task = pair / VEC, i = pair % VEC;
  return (i / 2) * 2 * (pairs / VEC) + 2 * task + (i & 1);
}

constexpr int kRopeTokens = kRopeThreads / 32;  // tokens of a block, at most: a warp places one

// The last request that starts at or before the token, by a whole warp: 32
// borders are compared at a time, so 1024 requests take two loads in a row.
__device__ __forceinline__ int find_request(const int* cu, int batch, int token) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + static_cast<int>(threadIdx.x & 31) * step;
    const int n = __popc(__ballot_sync(0xffffffffu, at < hi && cu[at] <= token));
    lo += max(n - 1, 0) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// grid.x: groups of `tb` tokens; grid.y: groups of `hc` heads, operand after operand
template <typename T, int VEC, bool kInter>
__global__ void __launch_bounds__(kRopeThreads, 8)
    rope_kernel(const __grid_constant__ RopeParams p, int tasks, int tb, int hc) {
  using P = Pack<T, VEC>;
  extern __shared__ __align__(16) float2 s_cs[];  // [tb][rotary_dim / 2]
  __shared__ int64_t s_dst[kRopeTokens], s_pos[kRopeTokens];
  __shared__ int s_ok[kRopeTokens];
  let_successor_start();
  int o = 0, g = blockIdx.y;
  while (o + 1 < p.n_op && g >= (p.op[o].heads + hc - 1) / hc) {
    g -= (p.op[o].heads + hc - 1) / hc;
    ++o;
  }
  const RopeOperand& op = p.op[o];
  const int h0 = g * hc, heads = min(op.heads - h0, hc);
  const int token0 = blockIdx.x * tb, tokens = min(tb, p.tokens - token0);
  const int pairs = op.rotate ? p.rotary_dim / 2 : 0;

  // this thread's place in the row; its first row is on its way to L2 meanwhile
  const int rows_step = kRopeThreads / tasks;
  const int task = threadIdx.x % tasks, sub = threadIdx.x / tasks;
  const int rot_tasks = pairs / VEC;
  const bool rot = task < rot_tasks;
  int ea, eb;
  if (rot && !kInter) {
    ea = task * VEC;
    eb = pairs + task * VEC;
  } else {  // pairs side by side, or elements behind the rotated ones
    ea = task * 2 * VEC;
    eb = ea + VEC;
  }
  const bool two = eb < p.dim;
  const T* in = static_cast<const T*>(op.in) + static_cast<int64_t>(token0) * op.in_t +
                static_cast<int64_t>(h0) * op.in_h;
  int row = sub < rows_step ? sub : tokens * heads;
  int t = sub / heads, h = sub - t * heads;
  wait_for_predecessor();
  const int step_t = rows_step / heads, step_h = rows_step - step_t * heads;
  if (row < tokens * heads) {  // holds no registers until it is used
    const T* r = in + static_cast<int64_t>(t) * op.in_t + static_cast<int64_t>(h) * op.in_h;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(r + ea));
    if (two) asm volatile("prefetch.global.L2 [%0];" ::"l"(r + eb));
  }

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < tokens) {  // where the warp's token lies in the cache, and its position
    const int token = token0 + warp;
    int64_t at = 0, dst = static_cast<int64_t>(token) * op.out_t;
    bool ok = true;
    int req = 0;
    if (p.ctx != nullptr)
      req = p.cu == nullptr ? token / p.uniform : find_request(p.cu, p.batch, token);
    if (lane == 0) {
      if (p.ctx != nullptr) {
        int first = req * p.uniform;
        if (p.cu != nullptr) {
          first = p.cu[req];
          ok = token >= first && token < p.cu[req + 1];  // else: behind the last request
        }
        if (ok) at = static_cast<int64_t>(p.ctx[req]) + (token - first);
        if (ok && op.paged) {
          ok = at >= 0 && at < static_cast<int64_t>(p.table_w) * p.page_size;
          if (!ok) {
            if (g == 0) st_record(p.status, kStatusBadArgs, kBadPosition, token);
          } else {
            const uint32_t entry = static_cast<uint32_t>(at) / static_cast<uint32_t>(p.page_size);
            const int page = p.table[static_cast<int64_t>(req) * p.table_stride + entry];
            ok = page >= 0 && page < p.num_pages;
            if (!ok && g == 0) st_record(p.status, kStatusBadArgs, kBadPage, page);
            dst = static_cast<int64_t>(page) * op.out_t +
                  (at - static_cast<int64_t>(entry) * p.page_size) * p.dim;
          }
        }
      }
      if (p.positions != nullptr)
        at = p.positions64 ? static_cast<const int64_t*>(p.positions)[token]
                           : static_cast<int64_t>(static_cast<const int*>(p.positions)[token]);
      s_dst[warp] = dst;
      s_ok[warp] = ok;
      s_pos[warp] = at;
    }
  }
  if (pairs > 0) {
    const int pair = threadIdx.x % pairs, t_step = kRopeThreads / pairs;
    const uint64_t step = phase_step(p.inv_freq[pair]);
    __syncthreads();
    for (int u = threadIdx.x / pairs; u < tokens && threadIdx.x < t_step * pairs; u += t_step) {
      const uint64_t phase = static_cast<uint64_t>(s_pos[u]) * step;
      const int top = static_cast<int>((phase + 0x80000000ull) >> 32);
      float sn, cs;
      sincospif(static_cast<float>(top) * 0x1p-31f, &sn, &cs);
      s_cs[u * pairs + cs_slot<VEC>(pair, pairs)] = make_float2(cs * p.scale, sn * p.scale * p.sign);
    }
  }
  __syncthreads();

  T* out = static_cast<T*>(op.out) + static_cast<int64_t>(h0) * op.out_h;
  while (row < tokens * heads) {
    if (s_ok[t]) {
      const T* r = in + static_cast<int64_t>(t) * op.in_t + static_cast<int64_t>(h) * op.in_h;
      P a = *reinterpret_cast<const P*>(r + ea), b;
      if (two) b = *reinterpret_cast<const P*>(r + eb);
      if (rot) {
        float cs[VEC], sn[VEC];
        const float2* c = s_cs + t * pairs;
        if constexpr (VEC == 1) {
          cs[0] = c[task].x;
          sn[0] = c[task].y;
        } else {
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const float4 v = *reinterpret_cast<const float4*>(c + i * rot_tasks + 2 * task);
            cs[i] = v.x;
            sn[i] = v.y;
            cs[i + 1] = v.z;
            sn[i + 1] = v.w;
          }
        }
        rotate<T, VEC, kInter>(a, b, cs, sn);
      }
      T* w = out + s_dst[t] + static_cast<int64_t>(h) * op.out_h;
      *reinterpret_cast<P*>(w + ea) = a;
      if (two) *reinterpret_cast<P*>(w + eb) = b;
    }
    row += rows_step;
    t += step_t;
    h += step_h;
    if (h >= heads) {
      h -= heads;
      ++t;
    }
  }
}

constexpr int kJointTokens = 64;       // tokens of a block of the kernel below, at most
constexpr int kJointSmem = 32 * 1024;  // and bytes of their cosines and sines

// The same for few heads: a block takes all operands of `tb` tokens, a thread to a
// token while they are placed.
template <typename T, int VEC, bool kInter>
__global__ void __launch_bounds__(kRopeThreads, 8)
    rope_joint_kernel(const __grid_constant__ RopeParams p, int tasks, int tb) {
  using P = Pack<T, VEC>;
  extern __shared__ __align__(16) float2 s_cs[];  // [tb][rotary_dim / 2]
  // a token's place in the pool, and what may be done with it: 1 read, 2 written to the pool
  __shared__ int s_page[kJointTokens], s_in[kJointTokens], s_ok[kJointTokens];
  __shared__ int64_t s_pos[kJointTokens];
  let_successor_start();
  const int token0 = blockIdx.x * tb, tokens = min(tb, p.tokens - token0);
  const int rows_step = kRopeThreads / tasks;
  const int task = threadIdx.x % tasks, sub = threadIdx.x / tasks;
  const int half = p.rotary_dim / 2;
  wait_for_predecessor();
  // where the tokens lie in the cache, and their positions
  if (threadIdx.x < tokens) {
    const int mine = threadIdx.x, token = token0 + mine;
    int req = 0;
    if (p.ctx != nullptr) {
      if (p.cu == nullptr) {
        req = token / p.uniform;
      } else {
        int hi = p.batch;  // the last request that starts at or before the token
        while (hi - req > 1) {
          const int mid = (req + hi) >> 1;
          if (p.cu[mid] <= token) req = mid;
          else hi = mid;
        }
      }
    }
    int64_t at = 0;
    int ok = 3, page = 0, in = 0;
    if (p.ctx != nullptr) {
      int first = req * p.uniform;
      if (p.cu != nullptr) {
        first = p.cu[req];
        if (token < first || token >= p.cu[req + 1]) ok = 0;  // behind the last request
      }
      if (ok) {
        at = static_cast<int64_t>(p.ctx[req]) + (token - first);
        if (at < 0 || at >= static_cast<int64_t>(p.table_w) * p.page_size) {
          ok = 1;
          st_record(p.status, kStatusBadArgs, kBadPosition, token);
        } else {
          const uint32_t entry = static_cast<uint32_t>(at) / static_cast<uint32_t>(p.page_size);
          page = p.table[static_cast<int64_t>(req) * p.table_stride + entry];
          in = static_cast<int>(static_cast<uint32_t>(at) - entry * p.page_size) * p.dim;
          if (page < 0 || page >= p.num_pages) {
            ok = 1;
            st_record(p.status, kStatusBadArgs, kBadPage, page);
          }
        }
      }
    }
    if (p.positions != nullptr)
      at = p.positions64 ? static_cast<const int64_t*>(p.positions)[token]
                         : static_cast<int64_t>(static_cast<const int*>(p.positions)[token]);
    s_page[mine] = page;
    s_in[mine] = in;
    s_ok[mine] = ok;
    s_pos[mine] = at;
  }
  if (half > 0) {
    const int pair = threadIdx.x % half, t_step = kRopeThreads / half;
    const uint64_t step = phase_step(p.inv_freq[pair]);
    __syncthreads();
    for (int u = threadIdx.x / half; u < tokens && threadIdx.x < t_step * half; u += t_step) {
      const uint64_t phase = static_cast<uint64_t>(s_pos[u]) * step;
      const int top = static_cast<int>((phase + 0x80000000ull) >> 32);
      float sn, cs;
      sincospif(static_cast<float>(top) * 0x1p-31f, &sn, &cs);
      s_cs[u * half + cs_slot<VEC>(pair, half)] = make_float2(cs * p.scale, sn * p.scale * p.sign);
    }
  }
  __syncthreads();

  for (int o = 0; o < p.n_op; ++o) {
    const RopeOperand& op = p.op[o];
    const int heads = op.heads;
    const int rot_tasks = op.rotate ? half / VEC : 0;
    const bool rot = task < rot_tasks;
    int ea, eb;
    if (rot && !kInter) {
      ea = task * VEC;
      eb = half + task * VEC;
    } else {  // pairs side by side, or elements behind the rotated ones
      ea = task * 2 * VEC;
      eb = ea + VEC;
    }
    const bool two = eb < p.dim;
    const int need = op.paged ? 2 : 1;
    const T* in = static_cast<const T*>(op.in) + static_cast<int64_t>(token0) * op.in_t;
    T* out = static_cast<T*>(op.out);
    const int step_t = rows_step / heads, step_h = rows_step - step_t * heads;
    int t = sub < rows_step ? sub / heads : tokens, h = sub - sub / heads * heads;
    while (t < tokens) {
      if (s_ok[t] & need) {
        const T* r = in + static_cast<int64_t>(t) * op.in_t + static_cast<int64_t>(h) * op.in_h;
        P a = *reinterpret_cast<const P*>(r + ea), b;
        if (two) b = *reinterpret_cast<const P*>(r + eb);
        if (rot) {
          float cs[VEC], sn[VEC];
          const float2* c = s_cs + t * half;
          if constexpr (VEC == 1) {
            cs[0] = c[task].x;
            sn[0] = c[task].y;
          } else {
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
              const float4 v = *reinterpret_cast<const float4*>(c + i * rot_tasks + 2 * task);
              cs[i] = v.x;
              sn[i] = v.y;
              cs[i + 1] = v.z;
              sn[i + 1] = v.w;
            }
          }
          rotate<T, VEC, kInter>(a, b, cs, sn);
        }
        T* w = out + static_cast<int64_t>(h) * op.out_h +
               (op.paged ? static_cast<int64_t>(s_page[t]) * op.out_t + s_in[t]
                         : static_cast<int64_t>(token0 + t) * op.out_t);
        *reinterpret_cast<P*>(w + ea) = a;
        if (two) *reinterpret_cast<P*>(w + eb) = b;
      }
      t += step_t;
      h += step_h;
      if (h >= heads) {
        h -= heads;
        ++t;
      }
    }
  }
}

template <typename T, int VEC, bool kInter>
int rope_run(const RopeParams& p, cudaStream_t stream) {
  // a row's tasks: two vectors each; one more when the dims leave a single vector over
  const int tasks = (p.dim + 2 * VEC - 1) / (2 * VEC);
  if constexpr (VEC > 1) {
    // Few heads and many tokens: sines formed once for all operands, and enough tokens
    // to a block that its widest operand gives every thread a row.  262144 tokens of
    // one q and one k head x 64 take 40 us, 207 with a block per eight tokens and
    // operand; 16 q and 4 k heads x 64 19 against 23, but 32 and 8 heads x 128 62
    // against 56: many rows want the short loop.
    const int rows_step = kRopeThreads / tasks;
    int most = 1;
    for (int i = 0; i < p.n_op; ++i) most = p.op[i].heads > most ? p.op[i].heads : most;
    if (2 * most < rows_step && p.tokens >= p.sms * 16) {
      int tb = rows_step / most;
      tb = tb < 16 ? 16 : (tb > kJointTokens ? kJointTokens : tb);
      while (tb > 8 && tb * p.rotary_dim * static_cast<int>(sizeof(float)) > kJointSmem) tb >>= 1;
      while (tb > 8 && (p.tokens + tb - 1) / tb < p.sms * 4) tb >>= 1;
      const size_t smem = static_cast<size_t>(tb) * (p.rotary_dim / 2) * sizeof(float2);
      return launch_overlapped(rope_joint_kernel<T, VEC, kInter>, dim3((p.tokens + tb - 1) / tb),
                               kRopeThreads, smem, stream, &p, &tasks, &tb);
    }
  }
  // Tokens of a block: as many as leave eight blocks per SM, down to one (a block
  // forms its sines itself, which is cheap beside idle SMs), whose heads are then
  // cut so that every thread has one row.
  int tb = kRopeTokens, hc = 64, gy = 0;
  while (true) {
    gy = 0;
    for (int i = 0; i < p.n_op; ++i) gy += (p.op[i].heads + hc - 1) / hc;
    if (tb == 1 || static_cast<int64_t>((p.tokens + tb - 1) / tb) * gy >= p.sms * 8) break;
    tb >>= 1;
    if (tb == 1) hc = kRopeThreads / tasks;
  }
  const size_t smem = static_cast<size_t>(tb) * (p.rotary_dim / 2) * sizeof(float2);
  return launch_overlapped(rope_kernel<T, VEC, kInter>, dim3((p.tokens + tb - 1) / tb, gy),
                           kRopeThreads, smem, stream, &p, &tasks, &tb, &hc);
}

template <typename T, int VEC>
int rope_layout(const RopeParams& p, cudaStream_t stream) {
  return p.interleaved ? rope_run<T, VEC, true>(p, stream) : rope_run<T, VEC, false>(p, stream);
}

}  // namespace

int rope_launch(Elem elem, const RopeParams& p, bool vectors, cudaStream_t stream) {
  if (p.tokens == 0) return 0;
  for (int i = 0; i < p.n_op; ++i)
    if (p.op[i].heads < 1) return static_cast<int>(cudaErrorInvalidValue);
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
