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
// the gradient once (nothing is read for a row without kept slots).  8192 x 128256 float32, 64 slots:
// loss 610 us (4.2 GB, 6.9 TB/s: a read stream, above a copy's 6.46); 4096 rows with a bf16 gradient:
// loss and gradient 794 us (5.25 GB, 6.6 TB/s).
//
// A group of G threads takes a row (or a segment of one): a whole CTA of 256 usually, a warp for
// short rows, where a CTA's barriers would cost more than the row.  When there are too few rows
// to fill the machine, the CTAs of a row (a cluster in the forward, which joins their maxima and
// sums through distributed shared memory) take contiguous segments of it.
#include <algorithm>
#include <cmath>
#include <cooperative_groups.h>
#include <type_traits>

#include "kvs_common.cuh"
#include "kvs_sm100.cuh"

using namespace kvs;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 1024;
constexpr int kWarpTop = 128;      // slots of a row that a warp takes
constexpr int kMaxSegments = 8;    // CTAs of one row

__device__ __forceinline__ float exp_full(float x) { return expf(x); }
__device__ __forceinline__ double exp_full(double x) { return exp(x); }
__device__ __forceinline__ float log_full(float x) { return logf(x); }
__device__ __forceinline__ double log_full(double x) { return log(x); }
// exp(d / T) with c = log2(e) / T for float, 1 / T for double.  The hardware's 2^x (2^-22 relative;
// results below 2^-126, which no sum or rounded gradient here can tell from 0, become 0).
__device__ __forceinline__ float exp_scaled(float d, float c) { return sm100::ex2_approx(d * c); }
__device__ __forceinline__ double exp_scaled(double d, double c) { return exp(d * c); }

template <int G> __device__ __forceinline__ void group_sync() {
  if constexpr (G == 32) __syncwarp();
  else __syncthreads();
}
struct MaxOp {
  template <typename A> __device__ A operator()(A a, A b) const { return b > a ? b : a; }
};
struct SumOp {
  template <typename A> __device__ A operator()(A a, A b) const { return a + b; }
};
// N values reduced over the group at once (one pair of barriers); `red`: N per warp of the CTA
template <int G, typename Op, typename A, int N> __device__ __forceinline__ void group_reduce(A (&v)[N], A* red) {
  const Op op;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = op(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
  if constexpr (G != 32) {
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) red[(threadIdx.x >> 5) * N + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = red[k];
#pragma unroll
    for (int i = 1; i < G / 32; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = op(v[k], red[i * N + k]);
    __syncthreads();
  }
}

// A thread's slots of a row (PER of them; one where a CTA has a thread for each), in registers: loaded
// before the row is streamed, so that their latency is behind it.  id < 0: empty.
template <typename A, int PER>
struct Slots {
  int64_t id[PER];
  A t[PER];
};
template <int G, typename A, int PER>
__device__ __forceinline__ void load_slots(const int64_t* ids, const A* t, int top, int tid, Slots<A, PER>& s) {
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int j = tid + u * G;
    s.id[u] = -1;
    s.t[u] = -INFINITY;
    if (j < top) {
      s.id[u] = ids[j];
      s.t[u] = t[j];
    }
    if (!(s.t[u] > -INFINITY)) s.id[u] = -1;
  }
}

// 16 bytes of a row
template <typename T> struct alignas(16) Pack {
  static constexpr int n = 16 / sizeof(T);
  T v[n];
};

// elements before the first 16-byte boundary of `p`, at most `n`
template <typename T> __device__ __forceinline__ int head_of(const T* p, int n) {
  const int h = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
  return min(h, n);
}

// the largest of a pack (a NaN is passed over here and caught by the sum)
__device__ __forceinline__ float pack_max(const Pack<float>& q) {
  return fmaxf(fmaxf(q.v[0], q.v[1]), fmaxf(q.v[2], q.v[3]));
}
__device__ __forceinline__ double pack_max(const Pack<double>& q) { return q.v[1] > q.v[0] ? q.v[1] : q.v[0]; }
template <typename T2, typename T> __device__ __forceinline__ float pack_max_half(const Pack<T>& q) {
  const T2* h = reinterpret_cast<const T2*>(&q);
  const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(to_acc<T>(m.x), to_acc<T>(m.y));
}
__device__ __forceinline__ float pack_max(const Pack<__nv_bfloat16>& q) { return pack_max_half<__nv_bfloat162>(q); }
__device__ __forceinline__ float pack_max(const Pack<__half>& q) { return pack_max_half<__half2>(q); }

// s += sum over the pack of exp((x - m) / T); two partial sums, and float's differences, scalings
// and sums two at a time.  (The difference is formed before it is scaled: x / T log2(e) of a logit
// at the type's lowest value would overflow, and its rounding would be that of the large number.)
template <typename T> __device__ __forceinline__ void pack_sum(const Pack<T>& q, float c, float m, float& s0, float& s1) {
#pragma unroll
  for (int k = 0; k < Pack<T>::n; k += 2) {
    float z0, z1;
    sm100::addmul2(z0, z1, to_acc<T>(q.v[k]), to_acc<T>(q.v[k + 1]), -m, -m, c, c);
    sm100::fadd2(s0, s1, sm100::ex2_approx(z0), sm100::ex2_approx(z1));
  }
}
__device__ __forceinline__ void pack_sum(const Pack<double>& q, double c, double m, double& s0, double& s1) {
  s0 += exp_scaled(q.v[0] - m, c);
  s1 += exp_scaled(q.v[1] - m, c);
}

// A thread's share of `n` elements at x: the largest, m (-inf before anything but -inf came), and
// s = sum of exp((x - m) / T).  16-byte loads between the ends, kUnroll of them in flight, one
// rescale of the sum per batch.
template <int G, typename T, typename A>
__device__ void row_lse(const T* x, int n, A c, int tid, A& m, A& s) {
  using P = Pack<T>;
  constexpr int kUnroll = 4;
  auto raise = [&](A xm) {  // the reference for a batch whose largest element is xm
    if (xm > m) {
      s *= exp_scaled(m - xm, c);  // (0 the first time)
      m = xm;
    }
    return m == -INFINITY ? A(0) : m;  // nothing but -inf so far: no inf - inf
  };
  auto one = [&](T e) {
    const A v = to_acc<T>(e), ref = raise(v);
    s += exp_scaled(v - ref, c);
  };
  const int head = head_of(x, n);
  const int packs = (n - head) / P::n;
  const P* xp = reinterpret_cast<const P*>(x + head);
  for (int i0 = tid; i0 < packs; i0 += kUnroll * G) {
    P q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i0 + u * G < packs) *reinterpret_cast<uint4*>(&q[u]) = *reinterpret_cast<const uint4*>(xp + i0 + u * G);
    A bm = pack_max(q[0]);
#pragma unroll
    for (int u = 1; u < kUnroll; ++u)
      if (i0 + u * G < packs) {
        const A pm = pack_max(q[u]);
        bm = pm > bm ? pm : bm;
      }
    const A ref = raise(bm);
    A s0 = A(0), s1 = A(0);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i0 + u * G < packs) pack_sum(q[u], c, ref, s0, s1);
    s += s0 + s1;
  }
  if (tid < head) one(x[tid]);
  const int tail = head + packs * P::n + tid;
  if (tail < n) one(x[tail]);  // fewer than P::n <= G elements
}

// (No __restrict__ on what these kernels read: a kernel that starts before the one before it has ended may not load
// that one's results as read-only data, nor may the compiler move the loads up past the wait as such.)
//
// Grid: rows / (256 / G) CTAs of one row group each, times `segs` CTAs (one cluster) per row.
template <typename T, typename A, int G, int PER>
__global__ void __launch_bounds__(kThreads)
distill_kernel(const T* logits, int64_t ld, int n_rows, int vocab, const int64_t* ids, const A* teacher, int top,
               A inv_temp, A c, int segs, A* loss, A* lse_out) {
  __shared__ A red[3 * (kThreads / 32)];
  __shared__ A part[2];
  sm100::pdl_let_next_start();
  sm100::pdl_wait_for_previous();
  const int tid = threadIdx.x % G;
  const int seg = segs > 1 ? (int)(blockIdx.x % segs) : 0;
  const int64_t row = (int64_t)(blockIdx.x / segs) * (kThreads / G) + threadIdx.x / G;
  if (G == 32 && row >= n_rows) return;
  const T* x = logits + row * ld;
  int beg = 0, len = vocab;
  if (segs > 1) {
    const int per = (vocab + segs - 1) / segs;
    beg = min(seg * per, vocab);
    len = min(per, vocab - beg);
  }
  Slots<A, PER> slot;
  load_slots<G>(ids + row * top, teacher + row * top, seg == 0 ? top : 0, tid, slot);
  A m = -INFINITY, s = A(0);
  row_lse<G, T, A>(x + beg, len, c, tid, m, s);
  T xs[PER];  // the named logits, just streamed
  A bad = A(0), tm = -INFINITY;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    xs[u] = T(0.f);
    if (slot.id[u] >= 0) {
      tm = slot.t[u] > tm ? slot.t[u] : tm;
      if (slot.id[u] < vocab) xs[u] = x[slot.id[u]];
      else bad = A(1);
    }
  }
  A mx[2] = {m, tm};
  group_reduce<G, MaxOp>(mx, red);
  tm = mx[1];
  // a thread that saw nothing but -inf has s == 0 and adds nothing; a NaN stays one
  A sum[3] = {s == A(0) ? A(0) : s * exp_scaled(m - mx[0], c), A(0), bad};
  A e[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    e[u] = slot.id[u] >= 0 ? (slot.t[u] - tm) * inv_temp : A(0);  // log of the weight times their sum
    if (slot.id[u] >= 0) sum[1] += exp_full(e[u]);
  }
  group_reduce<G, SumOp>(sum, red);
  A mm = mx[0], S = sum[0];
  if (segs > 1) {  // join the segments in order; the first CTA of the cluster goes on
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) {
      part[0] = mm;
      part[1] = S;
    }
    cluster.sync();
    if (seg == 0) {  // every thread reads the few pairs: no further exchange
      A all = -INFINITY, tot = A(0);
      for (int i = 0; i < segs; ++i) all = MaxOp()(all, cluster.map_shared_rank(part, i)[0]);
      for (int i = 0; i < segs; ++i) {
        const A* o = cluster.map_shared_rank(part, i);
        if (o[1] != A(0)) tot += o[1] * exp_scaled(o[0] - all, c);
      }
      mm = all;
      S = tot;
    }
    cluster.sync();  // the others' shared memory stays until it is read
    if (seg != 0) return;
  }
  const A logS = log_full(S), lse = mm * inv_temp + logS;
  const A logz = log_full(sum[1]);
  A term[1] = {A(0)};
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (slot.id[u] < 0) continue;
    // log q by the distance to the row's largest: the loss does not change with a shift of the row, and
    // x / T - lse would carry half a step of lse (5e-4 at logits near 1e4)
    const A lp = e[u] - logz, p = exp_full(lp);
    if (p != A(0)) term[0] += p * (lp - ((to_acc<T>(xs[u]) - mm) * inv_temp - logS));
  }
  group_reduce<G, SumOp>(term, red);
  if (tid == 0) {
    loss[row] = sum[2] > A(0) ? A(NAN) : term[0];
    lse_out[row] = lse;
  }
}

template <typename O, typename A> __device__ __forceinline__ O round_to(A v) {
  if constexpr (std::is_same<O, __nv_bfloat16>::value) return __float2bfloat16_rn((float)v);
  else if constexpr (std::is_same<O, __half>::value) return __float2half_rn((float)v);
  else return (O)v;
}

// N values to d, as widely as d's address allows
template <typename O, typename A, int N> __device__ __forceinline__ void put(O* d, const A (&v)[N]) {
  struct alignas(sizeof(O) * N > 16 ? 16 : sizeof(O) * N) Out { O v[N]; } o;
#pragma unroll
  for (int k = 0; k < N; ++k) o.v[k] = round_to<O, A>(v[k]);
  if ((reinterpret_cast<uintptr_t>(d) & (alignof(Out) - 1)) == 0) {
    *reinterpret_cast<Out*>(d) = o;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) d[k] = o.v[k];
  }
}

// dlogits may be the logits themselves.  A CTA writes only its segment, after it has read what it
// needs of it (the entries that slots name).
template <typename T, typename A, typename O, int G, int PER>
__global__ void __launch_bounds__(kThreads)
distill_bwd_kernel(const T* logits, int64_t ld, int n_rows, int vocab, const int64_t* ids, const A* teacher, int top,
                   const A* lse_in, const A* grad, A inv_temp, A c, int segs, O* dlogits, int64_t ld_out) {
  constexpr int TOP = G * PER;  // slots of a row at most
  __shared__ A red[2 * (kThreads / 32)];
  __shared__ A sp_all[kThreads / G][TOP];
  __shared__ int sid_all[kThreads / G][TOP];
  sm100::pdl_let_next_start();
  sm100::pdl_wait_for_previous();
  const int tid = threadIdx.x % G, group = threadIdx.x / G;
  A* sp = sp_all[group];
  int* sid = sid_all[group];
  const int seg = segs > 1 ? (int)(blockIdx.x % segs) : 0;
  const int64_t row = (int64_t)(blockIdx.x / segs) * (kThreads / G) + group;
  if (G == 32 && row >= n_rows) return;
  int beg = 0, len = vocab;
  if (segs > 1) {
    const int per = (vocab + segs - 1) / segs;
    beg = min(seg * per, vocab);
    len = min(per, vocab - beg);
  }
  const T* x = logits + row * ld;
  O* d = dlogits + row * ld_out;
  const A lse = lse_in[row], g = grad[row] * inv_temp;
  // exp(x / T - lse) = exp((x - lse T) / T): the difference is formed before it is scaled
  const A at_one = lse / inv_temp;
  auto prob = [&](T e) { return g * exp_scaled(to_acc<T>(e) - at_one, c); };
  Slots<A, PER> slot;
  load_slots<G>(ids + row * top, teacher + row * top, top, tid, slot);
  T xs[PER];
  A tm[1] = {-INFINITY}, sum[2] = {A(0), A(0)};
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    xs[u] = T(0.f);
    if (slot.id[u] >= vocab) sum[1] = A(1);
    if (slot.id[u] >= beg && slot.id[u] < beg + len) xs[u] = x[slot.id[u]];
    tm[0] = slot.id[u] >= 0 ? MaxOp()(tm[0], slot.t[u]) : tm[0];
  }
  group_reduce<G, MaxOp>(tm, red);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    slot.t[u] = slot.id[u] >= 0 ? exp_full((slot.t[u] - tm[0]) * inv_temp) : A(0);
    sum[0] += slot.t[u];
    const int j = tid + u * G;
    if (j < top) {
      sid[j] = slot.id[u] < 0 ? -1 : (int)slot.id[u];
      sp[j] = slot.t[u];
    }
  }
  group_reduce<G, SumOp>(sum, red);
  if constexpr (G == 32) __syncwarp();
  using P = Pack<T>;
  const int head = head_of(x + beg, len);
  const int packs = (len - head) / P::n;
  const bool bad = sum[1] > A(0);
  if (!(tm[0] > -INFINITY) || bad) {
    const A one = bad ? A(NAN) : A(0);
    A v[P::n];
#pragma unroll
    for (int k = 0; k < P::n; ++k) v[k] = one;
    O* dp = d + beg + head;
    if (tid < head) d[beg + tid] = round_to<O, A>(one);
    for (int i = tid; i < packs; i += G) put<O, A, P::n>(dp + (int64_t)i * P::n, v);
    for (int i = head + packs * P::n + tid; i < len; i += G) d[beg + i] = round_to<O, A>(one);
    return;
  }
  // the first slot of an id takes the sum of all its slots, in slot order.  (Every slot is compared with every
  // other, top^2 / G steps a thread: hidden at 128 slots, not past 256: 4096 x 128256 float32 to a bf16 gradient
  // takes 496 us with 64 slots, 509 with 128, 539 with 256, 760 with 512, 1780 with 1024.)
  const A gz = g / sum[0];
  A val[PER];
  int at[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int j = tid + u * G;
    at[u] = (int)slot.id[u];
    if (slot.id[u] < beg || slot.id[u] >= beg + len) at[u] = -1;
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
      if (at[u] >= 0) val[u] = prob(xs[u]) - gz * p;
    }
  }
  // (every slot's logit was read before the first barrier above)
  {
    constexpr int kUnroll = 4;
    const P* xp = reinterpret_cast<const P*>(x + beg + head);
    O* dp = d + beg + head;
    if (tid < head) d[beg + tid] = round_to<O, A>(prob(x[beg + tid]));
    for (int i = head + packs * P::n + tid; i < len; i += G) d[beg + i] = round_to<O, A>(prob(x[beg + i]));
    for (int i0 = tid; i0 < packs; i0 += kUnroll * G) {
      P q[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i0 + u * G < packs) *reinterpret_cast<uint4*>(&q[u]) = *reinterpret_cast<const uint4*>(xp + i0 + u * G);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i0 + u * G < packs) {
          A v[P::n];
#pragma unroll
          for (int k = 0; k < P::n; ++k) v[k] = prob(q[u].v[k]);
          put<O, A, P::n>(dp + (int64_t)(i0 + u * G) * P::n, v);
        }
    }
  }
  group_sync<G>();
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (at[u] >= 0) d[at[u]] = round_to<O, A>(val[u]);
}

// Short rows go to warps: below this many bytes a row's own work is shorter than a CTA's barriers.
constexpr int kWarpRowBytes = 4096;
template <typename T> bool warp_rows(int vocab, int top) {
  return (int64_t)vocab * (int64_t)sizeof(T) <= kWarpRowBytes && top <= kWarpTop;
}
// CTAs per row: doubled while the rows give the machine less than four CTAs an SM and a segment
// keeps 8 KB (two 16-byte loads a thread)
template <typename T> int segments(int vocab, int n_rows) {
  int s = 1;
  while (s < kMaxSegments && (int64_t)n_rows * s < 4 * 148 && (int64_t)vocab * (int64_t)sizeof(T) / (2 * s) >= 8192)
    s *= 2;
  return s;
}
template <typename A> A log2e_of(double inv_temp) {
  return (A)(std::is_same<A, double>::value ? inv_temp : inv_temp * 1.4426950408889634);
}

template <typename T, typename A>
int launch_fwd(const void* logits, int64_t ld, int32_t n_rows, int32_t vocab, const int64_t* ids, const void* teacher,
               int32_t top, double temperature, void* loss, void* lse, cudaStream_t st) {
  const T* x = static_cast<const T*>(logits);
  const A* t = static_cast<const A*>(teacher);
  const A inv = (A)(1.0 / temperature), c = log2e_of<A>(1.0 / temperature);
  A *l = static_cast<A*>(loss), *e = static_cast<A*>(lse);
  constexpr int R = kThreads / 32;
  if (warp_rows<T>(vocab, top))
    return launch_overlapped(distill_kernel<T, A, 32, kWarpTop / 32>, (n_rows + R - 1) / R, kThreads, 0, st, 0, x, ld,
                             n_rows, vocab, ids, t, top, inv, c, 1, l, e);
  const int segs = segments<T>(vocab, n_rows);
  const auto kernel = top <= kThreads ? distill_kernel<T, A, kThreads, 1> : distill_kernel<T, A, kThreads, kMaxTop / kThreads>;
  return launch_overlapped(kernel, n_rows * segs, kThreads, 0, st, segs > 1 ? segs : 0, x, ld, n_rows, vocab, ids, t,
                           top, inv, c, segs, l, e);
}

template <typename T, typename A, typename O>
int launch_bwd(const void* logits, int64_t ld, int32_t n_rows, int32_t vocab, const int64_t* ids, const void* teacher,
               int32_t top, const void* lse, const void* grad, double temperature, void* dlogits, int64_t ld_out,
               cudaStream_t st) {
  const T* x = static_cast<const T*>(logits);
  const A *t = static_cast<const A*>(teacher), *e = static_cast<const A*>(lse), *g = static_cast<const A*>(grad);
  const A inv = (A)(1.0 / temperature), c = log2e_of<A>(1.0 / temperature);
  O* d = static_cast<O*>(dlogits);
  constexpr int R = kThreads / 32;
  if (warp_rows<T>(vocab, top))
    return launch_overlapped(distill_bwd_kernel<T, A, O, 32, kWarpTop / 32>, (n_rows + R - 1) / R, kThreads, 0, st, 0, x,
                             ld, n_rows, vocab, ids, t, top, e, g, inv, c, 1, d, ld_out);
  const int segs = segments<T>(vocab, n_rows);
  const auto kernel = top <= kThreads ? distill_bwd_kernel<T, A, O, kThreads, 1>
                                      : distill_bwd_kernel<T, A, O, kThreads, kMaxTop / kThreads>;
  return launch_overlapped(kernel, n_rows * segs, kThreads, 0, st, 0, x, ld, n_rows, vocab, ids, t, top, e, g, inv, c,
                           segs, d, ld_out);
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
