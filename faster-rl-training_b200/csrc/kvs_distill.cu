// Distillation from a teacher's top logits, beside the log-prob of one target
// (kvs_logprobs.cu).  Row r has `top` slots (id_j, t_j); a slot is kept when id_j >= 0 and
// t_j > -inf.  With x the student's logits row and T the temperature,
//   p_j  = exp(t_j / T) / sum_kept exp(t_i / T)            (the teacher, over the kept slots)
//   lse  = log sum_v exp(x_v / T)
//   loss = sum_kept p_j (log p_j - (x[id_j] / T - lse))    (0 for a row without kept slots)
//   d loss / d x_v = (exp(x_v / T - lse) - sum_{j: id_j = v} p_j) / T
// Everything is computed in 32 bits (64 for double logits): the running maximum and sum of a
// row, the teacher's softmax and the loss; half-precision logits are widened when they are
// read and a half-precision gradient is rounded once, when it is written.
//
// Bound by HBM: the forward reads each logits row once, the backward reads it once and writes
// the gradient once (nothing is read for a row without kept slots).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kvs_common.cuh"

using namespace kvs;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 1024;

__device__ __forceinline__ float exp_of(float x) { return __expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float exp_full(float x) { return expf(x); }
__device__ __forceinline__ double exp_full(double x) { return exp(x); }
__device__ __forceinline__ float log_full(float x) { return logf(x); }
__device__ __forceinline__ double log_full(double x) { return log(x); }

template <typename A> __device__ __forceinline__ A block_sum(A v, A* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  A r = A(0);
  for (int i = 0; i < kThreads / 32; ++i) r += red[i];
  __syncthreads();
  return r;
}
template <typename A> __device__ __forceinline__ A block_max(A v, A* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const A w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  A r = -INFINITY;
  for (int i = 0; i < kThreads / 32; ++i) r = red[i] > r ? red[i] : r;
  __syncthreads();
  return r;
}

// The teacher's softmax statistics of one row (all threads of the CTA): the largest kept t_j,
// sum exp((t_j - max) / T) over the kept slots, and whether a kept id is past the vocabulary.
template <typename A>
struct Teacher {
  A m, z;
  bool any, bad;
};
template <typename A>
__device__ Teacher<A> teacher_stats(const int64_t* ids, const A* t, int top, int vocab, A inv_temp, A* red) {
  A m = -INFINITY;
  int bad = 0;
  for (int j = threadIdx.x; j < top; j += kThreads) {
    if (ids[j] >= 0 && t[j] > -INFINITY) {
      m = t[j] > m ? t[j] : m;
      bad |= ids[j] >= vocab;
    }
  }
  Teacher<A> r;
  r.m = block_max(m, red);
  r.any = r.m > -INFINITY;
  r.bad = __syncthreads_or(bad) != 0;
  A z = A(0);
  for (int j = threadIdx.x; j < top; j += kThreads)
    if (ids[j] >= 0 && t[j] > -INFINITY) z += exp_full((t[j] - r.m) * inv_temp);
  r.z = block_sum(z, red);
  return r;
}

// one CTA per row
template <typename T, typename A>
__global__ void __launch_bounds__(kThreads)
distill_kernel(const T* __restrict__ logits, int64_t ld, int vocab, const int64_t* __restrict__ ids,
               const A* __restrict__ teacher, int top, A inv_temp, A* __restrict__ loss, A* __restrict__ lse_out) {
  __shared__ A red[kThreads / 32];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  A m = -INFINITY, s = A(0);
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    const A v = to_acc<T>(x[i]) * inv_temp;
    if (v > m) {
      s = s * exp_of(m - v) + A(1);
      m = v;
    } else if (v != -INFINITY) {
      s += exp_of(v - m);
    }
  }
  const A mm = block_max(m, red);
  // a thread that saw only -inf adds nothing (its exponent would be inf - inf)
  const A S = block_sum(m == -INFINITY && s == A(0) ? A(0) : s * exp_full(m - mm), red);
  const A lse = mm + log_full(S);
  const int64_t* id = ids + row * top;
  const A* t = teacher + row * top;
  const Teacher<A> te = teacher_stats(id, t, top, vocab, inv_temp, red);
  A part = A(0);
  if (te.any && !te.bad) {
    const A logz = log_full(te.z);
    for (int j = threadIdx.x; j < top; j += kThreads) {
      if (!(id[j] >= 0 && t[j] > -INFINITY)) continue;
      const A lp = (t[j] - te.m) * inv_temp - logz;
      const A p = exp_full(lp);
      if (p != A(0)) part += p * (lp - (to_acc<T>(x[id[j]]) * inv_temp - lse));
    }
  }
  const A l = block_sum(part, red);
  if (threadIdx.x == 0) {
    loss[row] = te.bad ? A(NAN) : l;
    lse_out[row] = lse;
  }
}

template <typename O, typename A> __device__ __forceinline__ O round_to(A v) {
  if constexpr (std::is_same<O, __nv_bfloat16>::value) return __float2bfloat16_rn((float)v);
  else if constexpr (std::is_same<O, __half>::value) return __float2half_rn((float)v);
  else return (O)v;
}

// one CTA per row; dlogits may be the logits themselves
template <typename T, typename A, typename O>
__global__ void __launch_bounds__(kThreads)
distill_bwd_kernel(const T* logits, int64_t ld, int vocab, const int64_t* __restrict__ ids,
                   const A* __restrict__ teacher, int top, const A* __restrict__ lse_in, const A* __restrict__ grad,
                   A inv_temp, O* dlogits, int64_t ld_out) {
  __shared__ A red[kThreads / 32];
  __shared__ A sp[kMaxTop];
  __shared__ int sid[kMaxTop];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  O* d = dlogits + row * ld_out;
  const int64_t* id = ids + row * top;
  const A* t = teacher + row * top;
  const Teacher<A> te = teacher_stats(id, t, top, vocab, inv_temp, red);
  if (!te.any || te.bad) {
    const O fill = round_to<O, A>(te.bad ? A(NAN) : A(0));
    for (int i = threadIdx.x; i < vocab; i += kThreads) d[i] = fill;
    return;
  }
  const A lse = lse_in[row], g = grad[row] * inv_temp, inv_z = A(1) / te.z;
  for (int j = threadIdx.x; j < top; j += kThreads) {
    const bool keep = id[j] >= 0 && t[j] > -INFINITY;
    sid[j] = keep ? (int)id[j] : -1;
    sp[j] = keep ? exp_full((t[j] - te.m) * inv_temp) * inv_z : A(0);
  }
  __syncthreads();
  // the entries that a slot names, before the row is overwritten: the first slot of an id takes
  // the sum of all its slots, in slot order
  constexpr int PER = kMaxTop / kThreads;
  A val[PER];
  int at[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int j = threadIdx.x + u * kThreads;
    at[u] = j < top ? sid[j] : -1;
    if (at[u] >= 0) {
      A p = A(0);
      for (int i = 0; i < top; ++i) {
        if (sid[i] != at[u]) continue;
        if (i < j) {
          at[u] = -1;
          break;
        }
        p += sp[i];
      }
      if (at[u] >= 0) val[u] = g * (exp_of(to_acc<T>(x[at[u]]) * inv_temp - lse) - p);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < vocab; i += kThreads)
    d[i] = round_to<O, A>(g * exp_of(to_acc<T>(x[i]) * inv_temp - lse));
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (at[u] >= 0) d[at[u]] = round_to<O, A>(val[u]);
}

template <typename T, typename A>
int launch_fwd(const void* logits, int64_t ld, int32_t n_rows, int32_t vocab, const int64_t* ids, const void* teacher,
               int32_t top, double temperature, void* loss, void* lse, cudaStream_t st) {
  distill_kernel<T, A><<<(unsigned)n_rows, kThreads, 0, st>>>(
      static_cast<const T*>(logits), ld, vocab, ids, static_cast<const A*>(teacher), top, (A)(1.0 / temperature),
      static_cast<A*>(loss), static_cast<A*>(lse));
  return launch_rc();
}

template <typename T, typename A, typename O>
int launch_bwd(const void* logits, int64_t ld, int32_t n_rows, int32_t vocab, const int64_t* ids, const void* teacher,
               int32_t top, const void* lse, const void* grad, double temperature, void* dlogits, int64_t ld_out,
               cudaStream_t st) {
  distill_bwd_kernel<T, A, O><<<(unsigned)n_rows, kThreads, 0, st>>>(
      static_cast<const T*>(logits), ld, vocab, ids, static_cast<const A*>(teacher), top,
      static_cast<const A*>(lse), static_cast<const A*>(grad), (A)(1.0 / temperature), static_cast<O*>(dlogits),
      ld_out);
  return launch_rc();
}

// positive and finite, and so is its reciprocal in the arithmetic's type
bool temperature_ok(double t) { return t > 1e-30 && t < 1e30; }

}  // namespace

KVS_API int kvs_distill(const void* logits, int64_t ld, int32_t n_rows, int32_t vocab, const int64_t* ids,
                        const void* teacher, int32_t top, double temperature, int32_t dtype, void* loss, void* lse,
                        kvs_stream_t stream) {
  if (n_rows < 0 || vocab <= 0 || top <= 0 || ld < vocab || !temperature_ok(temperature)) return KVS_E_ARG;
  if (top > kMaxTop) return KVS_E_UNSUPPORTED;
  if (dtype < KVS_F32 || dtype > KVS_F16) return KVS_E_UNSUPPORTED;
  if (n_rows == 0) return KVS_OK;
  if (!logits || !ids || !teacher || !loss || !lse) return KVS_E_ARG;
  const cudaStream_t st = to_cuda(stream);
  switch (dtype) {
    case KVS_F32:
      return launch_fwd<float, float>(logits, ld, n_rows, vocab, ids, teacher, top, temperature, loss, lse, st);
    case KVS_F64:
      return launch_fwd<double, double>(logits, ld, n_rows, vocab, ids, teacher, top, temperature, loss, lse, st);
    case KVS_BF16:
      return launch_fwd<__nv_bfloat16, float>(logits, ld, n_rows, vocab, ids, teacher, top, temperature, loss, lse,
                                              st);
    default:
      return launch_fwd<__half, float>(logits, ld, n_rows, vocab, ids, teacher, top, temperature, loss, lse, st);
  }
}

KVS_API int kvs_distill_backward(const void* logits, int64_t ld, int32_t n_rows, int32_t vocab, const int64_t* ids,
                                 const void* teacher, int32_t top, const void* lse, const void* grad,
                                 double temperature, int32_t dtype, void* dlogits, int64_t ld_out, int32_t out_dtype,
                                 kvs_stream_t stream) {
  if (n_rows < 0 || vocab <= 0 || top <= 0 || ld < vocab || ld_out < vocab || !temperature_ok(temperature))
    return KVS_E_ARG;
  if (top > kMaxTop) return KVS_E_UNSUPPORTED;
  if (dtype < KVS_F32 || dtype > KVS_F16) return KVS_E_UNSUPPORTED;
  const bool half_of_f32 = dtype == KVS_F32 && (out_dtype == KVS_BF16 || out_dtype == KVS_F16);
  if (out_dtype != dtype && !half_of_f32) return KVS_E_UNSUPPORTED;
  if (n_rows == 0) return KVS_OK;
  if (!logits || !ids || !teacher || !lse || !grad || !dlogits) return KVS_E_ARG;
  // in place only element by element: the same rows at the same distance
  if (logits == dlogits && (dtype != out_dtype || ld != ld_out)) return KVS_E_ARG;
  const cudaStream_t st = to_cuda(stream);
#define KVS_DISTILL_BWD(T, A, O) \
  launch_bwd<T, A, O>(logits, ld, n_rows, vocab, ids, teacher, top, lse, grad, temperature, dlogits, ld_out, st)
  switch (dtype) {
    case KVS_F32:
      if (out_dtype == KVS_BF16) return KVS_DISTILL_BWD(float, float, __nv_bfloat16);
      if (out_dtype == KVS_F16) return KVS_DISTILL_BWD(float, float, __half);
      return KVS_DISTILL_BWD(float, float, float);
    case KVS_F64: return KVS_DISTILL_BWD(double, double, double);
    case KVS_BF16: return KVS_DISTILL_BWD(__nv_bfloat16, float, __nv_bfloat16);
    default: return KVS_DISTILL_BWD(__half, float, __half);
  }
#undef KVS_DISTILL_BWD
}
