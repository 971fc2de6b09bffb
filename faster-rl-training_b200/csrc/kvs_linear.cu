// Matrix products of a decoder layer with their epilogues, and their gradients (the projections
// of model.py:58-63, 74-75 and the gated feed-forward of model.py:78-86), for bf16 / fp16:
//
//   kvs_linear, plain   y = act(x W^T + b) + r                x [M][K], W [N][K], r, y [M][N]
//   kvs_linear, gated   h = act(x Wg^T) * (x Wu^T)            Wg, Wu [N][K]
//   kvs_linear_backward dz = gy act'(z);  dx = dz W,  dW = dz^T x,  db = sum_rows dz
//                       gated: dg = gh u act'(g), du = gh act(g);  dx = dg Wg + du Wu,
//                       dWg = dg^T x,  dWu = du^T x
//
// Every product accumulates in float32 (TMEM); bias, activation, gate product and residual are
// applied to the float32 sums and the result is rounded once.  One rounding lies inside: dz / dg /
// du, operands of the tensor cores, have the activations' type (half a step, 2^-9 relative for
// bf16).  The pre-activations kept for the backward (`pre`) are float32, or, where the caller
// prefers half the memory to another rounding of that size, of the activations' type.
//
// pair_gemm_kernel: units of 256 rows x 256 columns of the result, computed by a pair of CTAs
// (a 2-CTA cluster) with M = 256 tcgen05 MMAs (cta_group::2).  Each CTA stages its 128 rows of
// A and its 128 rows of B per 64-wide K block by TMA, the even CTA issues the MMAs, and each
// CTA's TMEM receives 128 result rows x 256 columns.  An operand is read as it lies: "K-major"
// when the reduced index is its inner one (x and W in the forward, dz in dx), "MN-major" when it
// is the outer one (W in dx, dz and x in dW), so no operand is ever transposed in memory.  The
// gated form takes 128 gate columns and the 128 up columns of the same index as one unit: the
// even CTA stages rows of Wg and the odd one rows of Wu, and a thread of the epilogue finds
// g and u of one output in the same TMEM lane.
//
// Roles per CTA (384 threads): warp 0 lane 0 = TMA producer (6-stage ring of 32 KB), warp 1 =
// TMEM allocation and, in the even CTA, the MMA issuer; warps 4..11 = epilogue.  TMEM holds two
// 256-column accumulators, so the epilogue of one unit overlaps the MMAs of the next.  Persistent
// grid: pair p takes units p, p + P, ...  Every wait is bounded; after one that ran out the
// outputs of the units concerned are NaN.
//
// Where whole units would leave pairs idle (fewer units than pairs, or a last round that is not
// full) the last units are cut along the reduced index into equal runs of K blocks, one per pair,
// in unit order.  A pair that comes into a unit in its middle does that part first and leaves the
// float32 sums in scratch; the pair that holds the unit's beginning does it last, so the others'
// sums are there when it needs them, adds them in order and finishes the unit.  Parts wait only for
// pairs of lower block indexes, which were scheduled before, and a part that is waited for never
// waits itself.
//
// Bound by the tensor cores: 4096 x 14336 gated x 4096 takes 590 us alone (1631 TFLOP/s, what the
// library product of 8192^3 reaches; the tensor pipe is active 93 % of the time), 8192 x 4096 x 4096
// 199 us with its residual (1381).  In long loops the power cap lowers the clock: 1395 there.  Reduced
// indexes over about 8192 also wait for HBM, where the pairs of a round are too far apart for L2.
#include "kvs_common.cuh"
#include "kvs_sm100.cuh"

#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
#include <mutex>
#include <type_traits>

using namespace kvs;
using namespace kvs::sm100;

namespace {

// ------------------------------------------------------------------ element-wise helpers
// 1 / (1 + e^-z), by t = e^-|z| <= 1 on either side: t becomes subnormal and 0 below z = -87.3, where e^-z passes
// 2^126 and an approximate quotient by it would be 0 already (silu(-88) = -5.3e-37 is a normal bf16 number)
__device__ __forceinline__ float sigmoid_f(float z) {
  const float t = __expf(-fabsf(z));
  return __fdividef(z < 0.f ? t : 1.f, 1.f + t);  // (good to an ulp or two; a NaN stays one)
}

// The normal distribution function F(z) and e = exp(-z^2 / 2).  For z <= 0, F(z) = e t P(t) with t = 1 / (1 + 0.3 |z|):
// the tail divided by e is smooth in t (the form of Abramowitz and Stegun 7.1.26).  P is of degree 7, fitted here to the
// smallest largest relative error over |z| <= 14, 1.5e-7 (iteratively reweighted least squares, Lawson 1961), so the
// tail is good to a few float32 roundings of itself: z F(z) is within 2e-6 of its value to z = -6 (8e-6 at -13, from the
// exponent's rounding), where 0.5 z (1 + erff) cancels; for z > 0, 1 - F is that good and F(z) a rounding off.
// 4096 x 4096 x 1024 with gelu takes 38.8 us, with erff 43; gated 4096 x 14336 x 4096 611, with 7.1.26 itself, which is
// three multiply-adds shorter and 0.3 % off in the tail, 606.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float t = __fdividef(1.f, fmaf(0.3f, fabsf(z), 1.f));
  e = ex2_approx(-0.72134752044448170f * z * z);
  float q = fmaf(0.03567476044f, t, -0.157203025f);
  q = fmaf(q, t, 0.2063534069f);
  q = fmaf(q, t, -0.05368355283f);
  q = fmaf(q, t, 0.1285615785f);
  q = fmaf(q, t, 0.09991350659f);
  q = fmaf(q, t, 0.1207539537f);
  q = fmaf(q, t, 0.1196292990f);
  q = __fmul_rn(q, t * e);
  return z > 0.f ? 1.f - q : q;
}

// (the last product is kept out of a multiply-add with the residual, so that every path rounds alike)
__device__ __forceinline__ float act_f(float z, int act) {
  if (act == KVS_ACT_RELU) return z <= 0.f ? 0.f : z;  // a NaN stays one
  if (act == KVS_ACT_SILU) return __fmul_rn(z, sigmoid_f(z));
  if (act == KVS_ACT_GELU) {
    float e;
    return __fmul_rn(z, normal_cdf(z, e));
  }
  return z;
}

// act(z) and act'(z)
__device__ __forceinline__ void act_grad_f(float z, int act, float& a, float& da) {
  if (act == KVS_ACT_RELU) {
    a = z <= 0.f ? 0.f : z;
    da = z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  } else if (act == KVS_ACT_SILU) {
    const float s = sigmoid_f(z);
    a = z * s;
    da = s * (1.f + z * (1.f - s));
  } else if (act == KVS_ACT_GELU) {
    float e;
    const float c = normal_cdf(z, e);
    a = z * c;
    da = c + z * 0.39894228040143268f * e;
  } else {
    a = z;
    da = 1.f;
  }
}

// `f` with the activation as a compile-time constant (chosen inside a loop it would be evaluated
// in every form for every element)
template <typename F> __device__ __forceinline__ void with_act_code(int act, F f) {
  if (act == KVS_ACT_SILU) f(std::integral_constant<int, KVS_ACT_SILU>());
  else if (act == KVS_ACT_GELU) f(std::integral_constant<int, KVS_ACT_GELU>());
  else if (act == KVS_ACT_RELU) f(std::integral_constant<int, KVS_ACT_RELU>());
  else f(std::integral_constant<int, KVS_ACT_NONE>());
}

template <typename T> struct alignas(sizeof(T) * 4) Vec4 { T v[4]; };
template <typename T> struct alignas(16) Vec8 { T v[8]; };

// four consecutive elements in one access
template <typename T> __device__ __forceinline__ float4 load4(const T* p) {
  const Vec4<T> q = *reinterpret_cast<const Vec4<T>*>(p);
  return make_float4(to_acc<T>(q.v[0]), to_acc<T>(q.v[1]), to_acc<T>(q.v[2]), to_acc<T>(q.v[3]));
}
// two floats rounded to nearest into one register
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T> __device__ __forceinline__ void store4(T* p, float4 f) {
  if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float4*>(p) = f;
  else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(f.x, f.y), pack2<T>(f.z, f.w));
}
// the first n of four elements; one access when `vec` (n is 4 then)
template <typename T> __device__ __forceinline__ float4 load_n(const T* p, int n, bool vec) {
  if (vec) return load4(p);
  float4 r = make_float4(to_acc<T>(p[0]), 0.f, 0.f, 0.f);
  if (n > 1) r.y = to_acc<T>(p[1]);
  if (n > 2) r.z = to_acc<T>(p[2]);
  if (n > 3) r.w = to_acc<T>(p[3]);
  return r;
}
template <typename T> __device__ __forceinline__ void store_n(T* p, float4 f, int n, bool vec) {
  if (vec) {
    store4(p, f);
    return;
  }
  p[0] = from_acc<T>(f.x);
  if (n > 1) p[1] = from_acc<T>(f.y);
  if (n > 2) p[2] = from_acc<T>(f.z);
  if (n > 3) p[3] = from_acc<T>(f.w);
}
// ------------------------------------------------------------------ pair GEMM
constexpr int BM = 128;  // result rows per CTA (256 per pair)
constexpr int BK = 64;   // reduced elements per stage
constexpr int TILE_BYTES = 128 * BK * 2;     // 16 KB, either major
constexpr int HALF_TILE = TILE_BYTES / 2;    // MN-major: 64 MN elements x 64 K rows
constexpr int EPI_WARPS = 8;  // two per TMEM lane quadrant, each half of the columns
constexpr int NT = 128 + 32 * EPI_WARPS;
constexpr int RING_BYTES = 6 * 2 * TILE_BYTES;  // 6 stages of a 256-column unit, 8 of a 128-column one
constexpr int MAX_STAGES = 8;
constexpr int OFF_STAGING = RING_BYTES;  // per epilogue warp 32 rows x 32 float32
constexpr int STAGING_BYTES = EPI_WARPS * 32 * 32 * 4;
constexpr int OFF_BAR = OFF_STAGING + STAGING_BYTES;
enum { B_FULL = 0, B_EMPTY = MAX_STAGES, B_ACCF = 2 * MAX_STAGES, B_ACCE = 2 * MAX_STAGES + 2,
       B_FINAL = 2 * MAX_STAGES + 4, NBAR = 2 * MAX_STAGES + 5 };
constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
constexpr int PAIR_SMEM = OFF_MISC + 16 + 1024;  // + alignment slack
static_assert(PAIR_SMEM <= 232448, "pair GEMM shared memory");

struct PairParams {
  int M, N;        // rows and columns of one result (gated: N columns of h)
  int n_kb;        // K blocks of one operand pair
  int k_parts;     // 2: the sum runs over (a0, b0), then (a1, b1)
  int mb, nb;      // units per result: row blocks, column blocks
  int m_parts;     // 2: two results, (a0, b0) -> out0 and (a1, b0) -> out1
  int group;       // row blocks whose columns are walked together (operand reuse in L2)
  int n_units;
  int whole;       // units done whole; the others' K blocks are dealt out to cut_pairs pairs
  int cut_pairs;
  int act;
  int vec;         // N is a multiple of 8 and out, res, pre and bias suit 16-byte accesses and TMA
  int pre_f32;     // pre is float32 (else of the activations' type)
  void* out0;
  void* out1;
  const void* bias;
  const void* res;
  void* pre;
  int64_t ld_out, ld_res, ld_pre;
  float* sums;                // [cut_pairs][2 CTAs][8 warps][4 chunks][8][32 lanes][4]: parts' float32 sums
  unsigned long long* ready;  // [cut_pairs][2][8]: flag words (flag_give / flag_take) of those sums
  unsigned long long token;   // of this launch; never that of another
};

constexpr int SUMS_PER_WARP = 32 * 128;  // floats

// What a pair does, one after the other: K blocks k0 .. k1 of unit u.
struct Part {
  int u, k0, k1;
};
__device__ __forceinline__ int64_t cut_begin(const PairParams& p, int kb_all, int pair) {
  return (int64_t)(p.n_units - p.whole) * kb_all * pair / p.cut_pairs;
}
// the i-th part of a pair; false past the last
__device__ __forceinline__ bool part_of(const PairParams& p, int kb_all, int pair, int n_pairs, int i, Part& s) {
  const int64_t u = pair + (int64_t)i * n_pairs;
  if (u < p.whole) {
    s = {(int)u, 0, kb_all};
    return true;
  }
  if (pair >= p.cut_pairs) return false;
  if (pair < p.whole) i -= (p.whole - 1 - pair) / n_pairs + 1;
  const int64_t beg = cut_begin(p, kb_all, pair), end = cut_begin(p, kb_all, pair + 1);
  const int64_t first = beg / kb_all + i;  // among the cut units
  s.u = p.whole + (int)first;
  s.k0 = i == 0 ? (int)(beg - first * kb_all) : 0;
  s.k1 = (int)min((int64_t)kb_all, end - first * kb_all);
  return s.k0 < s.k1;
}

// Polls, of about 4 us, that a wait for the sums of a run of K blocks may take: the default bound, and 1 us for each
// block, which takes 0.3 (2^24 blocks, the most that a product has, take longer than the default bound where one pair
// has them all: a product without scratch, or on fewer SMs than a whole B200's)
__device__ __forceinline__ uint32_t run_polls(int blocks) { return 400000u + (uint32_t)blocks / 4; }

// unit -> (result, row block, column block): `group` row blocks x all columns at a time, so that
// the units in flight read few rows of A and few rows of B
__device__ __forceinline__ void unit_of(const PairParams& p, int u, int& part, int& mb, int& nb) {
  const int rows = p.mb * p.m_parts;
  const int per = p.group * p.nb;
  const int g = u / per, first = g * p.group;
  const int size = min(p.group, rows - first);
  const int in = u - g * per;
  nb = in / size;
  const int r = first + in - nb * size;
  part = r >= p.mb;
  mb = part ? r - p.mb : r;
}

template <typename T> __host__ __device__ constexpr uint32_t idesc_of(int M, int N, int a_mn, int b_mn) {
  return (std::is_same<T, __half>::value ? idesc_f16(M, N, b_mn) : idesc_bf16(M, N, b_mn)) | ((uint32_t)a_mn << 15);
}

template <bool MN> __device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  return MN ? desc_mnmajor_sw128(saddr, HALF_TILE) : desc_kmajor_sw128(saddr);
}

// ROWS rows (MN index from `row` on) x 64 reduced elements (block kb) of an operand into `dst`
template <bool MN, int ROWS>
__device__ __forceinline__ void load_tile_pair(uint8_t* dst, const CUtensorMap* map, int kb, int row, uint32_t bar) {
  if (MN) {  // map: inner index MN, outer K
    tma_load_2d_pair(dst, map, row, kb * BK, bar);
    if (ROWS > 64) tma_load_2d_pair(dst + HALF_TILE, map, row + 64, kb * BK, bar);
  } else {
    tma_load_2d_pair(dst, map, kb * BK, row, bar);
  }
}

// what the epilogue does with an accumulator: store it, the plain product's whole epilogue, or the
// gate's product
enum { EPI_STORE = 0, EPI_LINEAR = 1, EPI_GATED = 2 };

template <typename T, bool A_MN, bool B_MN, int EPI, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NT, 1)
pair_gemm_kernel(const __grid_constant__ CUtensorMap tm_a0, const __grid_constant__ CUtensorMap tm_a1,
                 const __grid_constant__ CUtensorMap tm_b0, const __grid_constant__ CUtensorMap tm_b1,
                 const __grid_constant__ CUtensorMap tm_o0, const __grid_constant__ CUtensorMap tm_o1,
                 const __grid_constant__ CUtensorMap tm_pre, const PairParams p) {
  constexpr bool GATED = EPI == EPI_GATED;
  constexpr int B_BYTES = BN / 2 * BK * 2;  // a CTA's share of B
  constexpr int STAGE_BYTES = TILE_BYTES + B_BYTES;
  constexpr int STAGES = RING_BYTES / STAGE_BYTES;
  static_assert(STAGES <= MAX_STAGES, "ring");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_MISC + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();  // 0: the even CTA, which issues the MMAs
  // (in reverse, so that a part waits for CTAs that were scheduled before its own)
  const int n_pairs = (int)(gridDim.x >> 1), pair = n_pairs - 1 - (int)(blockIdx.x >> 1);

  if (tid == 0) {
    for (int i = 0; i < NBAR; ++i) mbar_init(&bar[i], i == B_ACCE || i == B_ACCE + 1 ? 2 * EPI_WARPS : 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barrier inits and the TMEM allocation visible to both CTAs
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int kb_all = p.n_kb * p.k_parts;
  pdl_let_next_start();
  pdl_wait_for_previous();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------------- producer
      bool ok = true;
      int it = 0;
      Part s;
      for (int i = 0; ok && part_of(p, kb_all, pair, n_pairs, i, s); ++i) {
        int part, mb, nb;
        unit_of(p, s.u, part, mb, nb);
        const int row = mb * 2 * BM + (int)rank * BM;
        const int col = GATED ? nb * (BN / 2) : nb * BN + (int)rank * (BN / 2);
        for (int k = s.k0; k < s.k1; ++k, ++it) {
          const int slot = it % STAGES;
          if (it >= STAGES && !mbar_wait_fast(&bar[B_EMPTY + slot], ((it / STAGES) - 1) & 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t full = mapa_shared(&bar[B_FULL + slot], 0);
          if (rank == 0) mbar_arrive_expect_tx(&bar[B_FULL + slot], 2 * STAGE_BYTES);
          uint8_t* st = smem + slot * STAGE_BYTES;
          const bool second = k >= p.n_kb;  // of two K parts
          const int kb = second ? k - p.n_kb : k;
          load_tile_pair<A_MN, BM>(st, part || second ? &tm_a1 : &tm_a0, kb, row, full);
          load_tile_pair<B_MN, BN / 2>(st + TILE_BYTES, second || (GATED && rank) ? &tm_b1 : &tm_b0, kb, col, full);
        }
      }
      if (!ok) *abort_flag = 1;
      // every copy of the pair has landed before either CTA may leave (they all complete on the
      // even CTA's barriers, and the CTAs leave together); bounded, and immediate unless aborting
      if (rank == 0)
        for (int j = max(0, it - STAGES); j < it; ++j)
          mbar_wait(&bar[B_FULL + j % STAGES], (j / STAGES) & 1, nullptr, ok ? 400000 : 20000);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------------------------------------------------------- MMA issuer (even CTA)
      constexpr uint32_t IDESC = idesc_of<T>(2 * BM, BN, A_MN, B_MN);
      constexpr uint32_t AS = A_MN ? 128 : 2, BS = B_MN ? 128 : 2;  // one K16 step: 2 KB / 32 B (>> 4)
      const uint32_t base = smem_addr(smem);
      bool ok = true;
      int it = 0;
      Part part;
      for (int ui = 0; ok && part_of(p, kb_all, pair, n_pairs, ui, part); ++ui) {
        const int ab = ui & 1;
        if (ui >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait_fast(&bar[B_ACCE + ab], ((ui >> 1) - 1) & 1, abort_flag));
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t d = tmem + ab * BN;
        for (int k = part.k0; k < part.k1; ++k, ++it) {
          const int s = it % STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait_fast(&bar[B_FULL + s], (it / STAGES) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = operand_desc<A_MN>(base + s * STAGE_BYTES);
          const uint64_t db = operand_desc<B_MN>(base + s * STAGE_BYTES + TILE_BYTES);
          umma_pair_warp_at<0, 0>(d, da, db, IDESC, k > part.k0);
          umma_pair_warp_at<AS, BS>(d, da, db, IDESC, 1);
          umma_pair_warp_at<2 * AS, 2 * BS>(d, da, db, IDESC, 1);
          umma_pair_warp_at<3 * AS, 3 * BS>(d, da, db, IDESC, 1);
          umma_commit_pair_warp(mapa_shared(&bar[B_EMPTY + s], 0));
          umma_commit_pair_warp(mapa_shared(&bar[B_EMPTY + s], 1));
        }
        if (!ok) break;
        umma_commit_pair_warp(mapa_shared(&bar[B_ACCF + ab], 0));
        umma_commit_pair_warp(mapa_shared(&bar[B_ACCF + ab], 1));
      }
      if (!ok && lane == 0) *abort_flag = 1;
      // every MMA issued has completed before TMEM is released
      umma_commit_pair_warp(mapa_shared(&bar[B_FINAL], 0));
      mbar_wait(&bar[B_FINAL], 0, nullptr);
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- epilogue
    // A warp takes its 32 accumulator rows 32 columns at a time, one row per lane: bias, activation,
    // gate and residual (16-byte loads of the lane's own row, one chunk ahead) in registers, the
    // rounded row to shared memory (16-byte pieces, TMA's swizzle: no bank conflicts), and a TMA
    // store writes the 32 x 32 box while the next chunk is computed (two buffers a warp; the float32
    // pre-activations take both).  Where pitches or bases do not suit that (`vec` is 0) the float32
    // chunk goes through shared memory instead and a lane takes a column.
    const int w = warp - 4, q = w & 3, half = w >> 2;  // TMEM lane quadrant, column half
    constexpr int COLS = (GATED ? BN / 2 : BN) / 2;   // result columns of this warp
    const uint32_t acce = mapa_shared(&bar[B_ACCE], 0);
    const uint32_t stage = smem_addr(smem + OFF_STAGING + w * (32 * 32 * 4));
    const bool vec = p.vec != 0, pre_f32 = p.pre_f32 != 0;
    const T* res = EPI == EPI_LINEAR ? static_cast<const T*>(p.res) : nullptr;
    const T* bias = EPI == EPI_LINEAR ? static_cast<const T*>(p.bias) : nullptr;
    void* const pre = EPI == EPI_STORE ? nullptr : p.pre;
    const int act = EPI == EPI_STORE ? KVS_ACT_NONE : p.act;
    // this lane's row of a 64-byte-row box (16-byte piece c at c ^ ((row >> 1) & 3)) and of a
    // 128-byte-row box (at c ^ (row & 7))
    const uint32_t row64 = lane * 64 + (((lane >> 1) & 3) << 4), row128 = stage + lane * 128 + ((lane & 7) << 4);
    uint32_t flip = 0;  // which of the two 2 KB buffers is next
    // 32 rounded values of this lane's row to the next buffer, and the box to x, y
    auto put_half = [&](const CUtensorMap* map, const uint32_t (&o)[16], int x, int y) {
      if (lane == 0) bulk_wait_read<1>();
      __syncwarp();
      const uint32_t at = stage + flip + row64;
#pragma unroll
      for (int c = 0; c < 4; ++c) st_shared_u4(at ^ (c << 4), o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(map, stage + flip, x, y);
        bulk_commit();
      }
      flip ^= 2048;
    };
    auto put_f32 = [&](const CUtensorMap* map, const uint32_t (&v)[32], int x, int y) {  // both buffers
      if (lane == 0) bulk_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 8; ++c) st_shared_u4(row128 ^ (c << 4), v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(map, stage, x, y);
        bulk_commit();
        bulk_wait_read<0>();
      }
      __syncwarp();
    };
    auto keep_pre = [&](const CUtensorMap* map, const uint32_t (&v)[32], int x, int y) {
      if (pre_f32) {
        put_f32(map, v, x, y);
      } else {
        uint32_t o[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = pack2<T>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
        put_half(map, o, x, y);
      }
    };
    // the scalar path's exchange: row r, column `lane` of a float32 chunk
    auto exchange = [&](const uint32_t (&v)[32]) {
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 8; ++c) st_shared_u4(row128 ^ (c << 4), v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      __syncwarp();
    };
    auto single = [&](int r) {
      float f;
      asm volatile("ld.shared.f32 %0, [%1];\n"
                   : "=f"(f)
                   : "r"(stage + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4));
      return f;
    };
    bool dead = false;
    Part seg;
    for (int ui = 0; part_of(p, kb_all, pair, n_pairs, ui, seg); ++ui) {
      const int ab = ui & 1;
      int part, mb, nb;
      unit_of(p, seg.u, part, mb, nb);
      const int row0 = mb * 2 * BM + (int)rank * BM + q * 32;
      const int n0 = nb * (GATED ? BN / 2 : BN) + half * COLS;
      const int rows = min(32, p.M - row0);  // existing rows of this warp (may be none)
      // the residual of the chunk at hand, as it lies: 32 columns of this lane's row, or without `vec`
      // 32 rows of its column, one to a register
      uint32_t rv[32];
      auto load_res = [&](int c) {
        const int col = n0 + c * 32;
        if (vec) {
          const T* from = res + (int64_t)(row0 + lane) * p.ld_res + col;
          if (lane < rows)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (col + k * 8 < p.N) {
                const uint4 q = *reinterpret_cast<const uint4*>(from + k * 8);
                rv[4 * k] = q.x, rv[4 * k + 1] = q.y, rv[4 * k + 2] = q.z, rv[4 * k + 3] = q.w;
              }
        } else if (col + lane < p.N) {
          const unsigned short* from = reinterpret_cast<const unsigned short*>(res) + (int64_t)row0 * p.ld_res + col + lane;
#pragma unroll
          for (int r = 0; r < 32; ++r, from += p.ld_res)
            if (r < rows) rv[r] = *from;
        }
      };
      const bool owner = seg.k0 == 0;
      if (res && owner) load_res(0);
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(&bar[B_ACCF + ab], (ui >> 1) & 1, abort_flag,
                                                                      run_polls(seg.k1 - seg.k0)));
      if (dead && lane == 0) *abort_flag = 1;
      tc_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + ab * BN + half * COLS;
      if constexpr (BN == 256) {
        if (!owner) {  // the unit's beginning is another pair's: leave the sums to it
          const int slot = (pair * 2 + (int)rank) * EPI_WARPS + w;
          float4* to = reinterpret_cast<float4*>(p.sums + (int64_t)slot * SUMS_PER_WARP) + lane;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32];
            if (!dead) {
              tmem_ld32(GATED ? taddr + (c & 1) * 32 + (c >> 1) * (BN / 2) : taddr + c * 32, v);
              tmem_wait_ld();
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = 0x7fc00000u;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              __stcg(to + (c * 8 + j) * 32, make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]),
                                                        __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])));
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_cluster(acce + ab * 8);
            __threadfence();
            flag_give(p.ready + slot, p.token);
          }
          continue;
        }
      }
      // the pairs that hold the rest of the unit: pair + 1 .. pair + others
      int others = 0;
      if (BN == 256 && seg.k1 < kb_all) {
        const int64_t unit_end = (int64_t)(seg.u - p.whole + 1) * kb_all;
        while (pair + others + 1 < p.cut_pairs && cut_begin(p, kb_all, pair + others + 1) < unit_end) ++others;
        bool there = true;
        if (lane == 0) {
          // over a second for the first; after one that ran out the others are only looked at, so that each
          // flag is left as flag_take leaves it
          for (int r = 1; r <= others; ++r)
            there &= flag_take(p.ready + ((pair + r) * 2 + (int)rank) * EPI_WARPS + w, p.token, there ? 1 << 21 : 1);
        }
        if (!__all_sync(0xffffffffu, there)) dead = true;
        __syncwarp();  // lane 0 acquired the flags; a vote orders no memory, this does, before any lane reads the sums
      }
      const float4* sums = reinterpret_cast<const float4*>(p.sums) +
                           (int64_t)(((pair + 1) * 2 + (int)rank) * EPI_WARPS + w) * (SUMS_PER_WARP / 4) + lane;
      auto add_others = [&](uint32_t (&v)[32], int c) {
        for (int r = 0; r < others; ++r) {
          const float4* from = sums + (int64_t)r * 2 * EPI_WARPS * (SUMS_PER_WARP / 4) + c * 8 * 32;
          float4 f[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = __ldcg(from + j * 32);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[4 * j] = __float_as_uint(__uint_as_float(v[4 * j]) + f[j].x);
            v[4 * j + 1] = __float_as_uint(__uint_as_float(v[4 * j + 1]) + f[j].y);
            v[4 * j + 2] = __float_as_uint(__uint_as_float(v[4 * j + 2]) + f[j].z);
            v[4 * j + 3] = __float_as_uint(__uint_as_float(v[4 * j + 3]) + f[j].w);
          }
        }
      };
#pragma unroll 1
      for (int c = 0; c < COLS / 32; ++c) {
        const int col = n0 + c * 32;
        if (col >= p.N || rows <= 0) break;
        uint32_t v[32], u32[GATED ? 32 : 1];
        if (!dead) {
          tmem_ld32(taddr + c * 32, v);
          if constexpr (GATED) tmem_ld32(taddr + BN / 2 + c * 32, u32);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0x7fc00000u;
          if constexpr (GATED)
#pragma unroll
            for (int j = 0; j < 32; ++j) u32[j] = 0x7fc00000u;
        }
        if (others && !dead) {
          add_others(v, c);
          if constexpr (GATED) add_others(u32, c + 2);
        }
        if (!vec) {
          // ------------------------------------------------ a lane per column
          const bool in = col + lane < p.N;
          T* out = static_cast<T*>(part ? p.out1 : p.out0) + (int64_t)row0 * p.ld_out + col + lane;
          int64_t pi = (int64_t)row0 * p.ld_pre + col + lane;
          // the exchanged chunk's column, plus `add`: shared-memory reads of eight rows in flight together
          auto column = [&](auto* to, int64_t ld, float add) {
#pragma unroll 1
            for (int r0 = 0; r0 < rows; r0 += 8) {
              float f[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = single(r0 + i) + add;
#pragma unroll
              for (int i = 0; i < 8; ++i, to += ld)
                if (r0 + i < rows && in) *to = from_acc<std::remove_reference_t<decltype(*to)>>(f[i]);
            }
          };
          auto keep_column = [&](int64_t at, float add) {
            if (pre_f32) column(static_cast<float*>(pre) + at, p.ld_pre, add);
            else column(static_cast<T*>(pre) + at, p.ld_pre, add);
          };
          if constexpr (GATED) {
            if (pre)
              for (int g = 0; g < 2; ++g) {
                if (g) exchange(u32);
                else exchange(v);
                keep_column(pi + g * p.N, 0.f);
              }
            with_act_code(act, [&](auto code) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                v[j] = __float_as_uint(act_f(__uint_as_float(v[j]), decltype(code)::value) * __uint_as_float(u32[j]));
            });
            exchange(v);
            column(out, p.ld_out, 0.f);
          } else {
            exchange(v);
            const float b = bias && in ? to_acc<T>(bias[col + lane]) : 0.f;
            if (pre) keep_column(pi, b);
            if (act == KVS_ACT_NONE && !res) {
              column(out, p.ld_out, b);
            } else {
              with_act_code(act, [&](auto code) {
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += 8) {
                  if (r0 >= rows) break;
                  float f[8];
#pragma unroll
                  for (int i = 0; i < 8; ++i) f[i] = act_f(single(r0 + i) + b, decltype(code)::value);
#pragma unroll
                  for (int i = 0; i < 8; ++i, out += p.ld_out)
                    if (r0 + i < rows && in) {
                      const unsigned short h = (unsigned short)rv[r0 + i];
                      *out = from_acc<T>(res ? f[i] + to_acc<T>(*reinterpret_cast<const T*>(&h)) : f[i]);
                    }
                }
              });
              if (res && (c + 1) * 32 < COLS) load_res(c + 1);
            }
          }
          continue;
        }
        // -------------------------------------------------- a lane per row
        if constexpr (GATED) {
          if (pre) {
            keep_pre(&tm_pre, v, col, row0);
            keep_pre(&tm_o1, u32, col, row0);
          }
        } else if (bias) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (col + k * 8 < p.N) {
              const Vec8<T> b = *reinterpret_cast<const Vec8<T>*>(bias + col + k * 8);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[k * 8 + j] = __float_as_uint(__uint_as_float(v[k * 8 + j]) + to_acc<T>(b.v[j]));
            }
        }
        if constexpr (EPI == EPI_LINEAR)
          if (pre) keep_pre(&tm_pre, v, col, row0);
        auto apply = [&](auto code) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float y = act_f(__uint_as_float(v[j]), decltype(code)::value);
            if constexpr (GATED) y *= __uint_as_float(u32[j]);
            v[j] = __float_as_uint(y);
          }
        };
        if constexpr (EPI == EPI_STORE) apply(std::integral_constant<int, KVS_ACT_NONE>());
        else with_act_code(act, apply);
        if (res) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            Vec8<T> r8;
            *reinterpret_cast<uint4*>(&r8) = make_uint4(rv[4 * k], rv[4 * k + 1], rv[4 * k + 2], rv[4 * k + 3]);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k * 8 + j] = __float_as_uint(__uint_as_float(v[k * 8 + j]) + to_acc<T>(r8.v[j]));
          }
          if ((c + 1) * 32 < COLS) load_res(c + 1);
        }
        uint32_t o[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = pack2<T>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
        put_half(part ? &tm_o1 : &tm_o0, o, col, row0);
      }
      // this thread's TMEM reads are done: release the accumulator to the MMA warp
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acce + ab * 8);
    }
    if (lane == 0) bulk_wait_read<0>();  // the boxes have left shared memory before the CTA does
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs done with TMEM and with each other's barriers
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------------ stream GEMM (few rows)
// With few rows of x the product is bound by reading the weights once.  The operands change
// places: 128 weight rows (or, in dx, 128 columns of W) are the M = 128 rows of the MMA and a tile
// of 16..128 rows of x its N columns, so the tensor cores' work follows the rows that exist and
// TMEM lane = result column.  A cluster of S CTAs takes one tile and splits the reduced index
// between them, so that (result tiles x S) CTAs stream the weights at once, one per SM (147 KB of copies in
// flight at 16 rows, eight stages, to 229 KB at 128) or two (98 to 111 KB each); stream_plan has the rule and both
// sides' times.  The S
// partial sums meet in distributed shared memory: CTA r adds up, in rank order, the 128 / S result
// columns that it then finishes (bias, activation, gate product, residual) and stores.  Nothing
// passes through global memory, no counters, no second launch, and the order of the sum is fixed.
// The gated form's 128 weight rows are 64 of Wg and the 64 of Wu that belong to them: g and u of an
// output are 64 columns apart in the partial sums.
//
// 256 threads: warp 0 lane 0 = TMA producer, warp 1 = TMEM allocation and MMA issuer, warps 4..7
// take the accumulators to shared memory; all of them finish and store.
//
// Bound by HBM where the weights are large: 1 x 14336 gated x 4096 takes 40.8 us (235 MB, 5.8 TB/s, 89 %
// of a copy's rate), 48 rows 43.3, 64 x 4096 x 14336 22.9 in a graph (117 MB, 5.1 TB/s); else by what
// lies beside the stream, 5 us of launch, first loads and join: 1 x 4096 x 4096 10 us for 34 MB.
constexpr int SNT = 256;
constexpr int SMAX_STAGES = 8;
constexpr int SMAX_SPLIT = 8;
constexpr int HALF_SM_SMEM = 113 * 1024;  // two CTAs per SM: 228 KB less 1 KB each that the system keeps
constexpr int S_BARS = 2 * SMAX_STAGES + 3;
constexpr int S_BAR_BYTES = S_BARS * 8 + 8;

struct StreamParams {
  int M, N;      // rows of x (or dz), result columns
  int n_kb;      // K blocks of one operand pair
  int k_parts;   // 2: the sum runs over (weights 0, x 0), then (weights 1, x 1)
  int tn;        // rows of x per tile, a multiple of 16
  int nt;        // tiles of 128 result columns (64 when gated)
  int stages;    // ring depth
  int split;     // CTAs per tile (cluster size, a power of two)
  int lsplit;    // its logarithm
  int act, vec, pre_f32;
  void* out;
  const void* bias;
  const void* res;
  void* pre;
  int64_t ld_out, ld_res, ld_pre;
};

// A walk round a ring of stages: the stage at hand and the parity of its barriers' phase.  (Counted
// on, not divided out of a running index: the one thread that issues copies, or MMAs, does nothing else,
// and at 16 rows of x its instructions, not the copies, bounded a K block.)
struct Ring {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ void next(uint32_t stages) {
    if (++slot == stages) {
      slot = 0;
      phase ^= 1;
      wrapped = true;
    }
  }
  // whether stage j was filled, and the parity of its last fill's phase
  __device__ __forceinline__ bool used(uint32_t j) const { return wrapped || j < slot; }
  __device__ __forceinline__ uint32_t last_phase(uint32_t j) const { return j < slot ? phase : phase ^ 1; }

 private:
  bool wrapped = false;
};

template <typename T, bool W_MN, bool GATED>
__global__ void __launch_bounds__(SNT)
stream_gemm_kernel(const __grid_constant__ CUtensorMap tm_w0, const __grid_constant__ CUtensorMap tm_w1,
                   const __grid_constant__ CUtensorMap tm_x0, const __grid_constant__ CUtensorMap tm_x1,
                   const StreamParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int COLS = GATED ? 64 : 128;  // result columns of a tile
  const int stage_bytes = TILE_BYTES + p.tn * BK * 2;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + p.stages * stage_bytes);
  uint64_t *full = bar, *empty = bar + SMAX_STAGES, *done = bar + 2 * SMAX_STAGES, *last = done + 1,
           *drained = done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tmem_cols = p.tn <= 32 ? 32 : p.tn <= 64 ? 64 : 128;
  const int rank = (int)(blockIdx.x % p.split);  // cluster rank (the clusters are along x)
  const int tile = (int)(blockIdx.x / p.split);
  const int n0 = (tile % p.nt) * COLS, m0 = (tile / p.nt) * p.tn;

  if (tid == 0) {
    for (int i = 0; i < S_BARS; ++i) mbar_init(&bar[i], 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_let_next_start();
  pdl_wait_for_previous();
  // this CTA's share of the K blocks
  const int kb_all = p.n_kb * p.k_parts;
  const int kb_beg = (int)((int64_t)kb_all * rank / p.split), kb_end = (int)((int64_t)kb_all * (rank + 1) / p.split);

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      Ring at;
      for (int k = kb_beg; k < kb_end; ++k, at.next(p.stages)) {
        const int s = at.slot;
        if (!mbar_wait_fast(&empty[s], at.phase ^ 1, abort_flag)) {  // (true the first time round)
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        uint8_t* st = smem + s * stage_bytes;
        const bool second = k >= p.n_kb;
        const int kb = second ? k - p.n_kb : k;
        const CUtensorMap* w = second ? &tm_w1 : &tm_w0;
        if (GATED) {  // (boxes of 64 rows)
          tma_load_2d(st, &tm_w0, kb * BK, n0, &full[s]);
          tma_load_2d(st + HALF_TILE, &tm_w1, kb * BK, n0, &full[s]);
        } else if (W_MN) {
          tma_load_2d(st, w, n0, kb * BK, &full[s]);
          tma_load_2d(st + HALF_TILE, w, n0 + 64, kb * BK, &full[s]);
        } else {
          tma_load_2d(st, w, kb * BK, n0, &full[s]);
        }
        tma_load_2d(st + TILE_BYTES, second ? &tm_x1 : &tm_x0, kb * BK, m0, &full[s]);
      }
      if (!ok) *abort_flag = 1;
      // every copy has landed before the CTA may go on to leave; immediate unless aborting
      for (int j = 0; j < p.stages; ++j)
        if (at.used(j)) mbar_wait(&full[j], at.last_phase(j), nullptr, ok ? 400000 : 20000);
      mbar_arrive(drained);
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_of<T>(128, p.tn, W_MN, 0);
    constexpr uint32_t AS = W_MN ? 128 : 2;
    const uint64_t dw0 = operand_desc<W_MN>(smem_addr(smem)), dx0 = desc_kmajor_sw128(smem_addr(smem) + TILE_BYTES);
    bool ok = true;
    Ring at;
    for (int k = kb_beg; k < kb_end; ++k, at.next(p.stages)) {
      const int s = at.slot;
      ok = __all_sync(0xffffffffu, mbar_wait_fast(&full[s], at.phase, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const uint64_t dw = dw0 + s * (stage_bytes >> 4), dx = dx0 + s * (stage_bytes >> 4);
      umma_bf16_warp_at<0, 0>(tmem, dw, dx, idesc, k > kb_beg);
      umma_bf16_warp_at<AS, 2>(tmem, dw, dx, idesc, 1);
      umma_bf16_warp_at<2 * AS, 4>(tmem, dw, dx, idesc, 1);
      umma_bf16_warp_at<3 * AS, 6>(tmem, dw, dx, idesc, 1);
      umma_commit_warp(&empty[s]);
    }
    if (ok) umma_commit_warp(done);
    else if (lane == 0) *abort_flag = 1;
    // every MMA issued has completed before TMEM is released
    umma_commit_warp(last);
    mbar_wait(last, 0, nullptr);
    __syncwarp();
  } else if (warp >= 4) {
    // partial sums to shared memory, [row of x][128 weight rows]: over the ring,
    // which nothing uses any more once the last MMA has completed
    const int q = warp & 3;  // TMEM lane quadrant
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag, run_polls(kb_end - kb_beg)));
    if (!ok) {  // the NaNs go where copies may still be landing: after those
      if (lane == 0) *abort_flag = 1;
      mbar_wait(drained, 0, nullptr);
      __syncwarp();
    }
    tc_fence_after();
    const uint32_t part = smem_addr(smem) + (q * 32 + lane) * 4;
    const int live = min(p.tn, p.M - m0);
#pragma unroll 1
    for (int c = 0; c < live; c += 32) {  // two loads in flight (the second may be past the tile)
      uint32_t v[16], w[16];
      const bool two = c + 16 < live;
      if (ok) {
        tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
        if (two) tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c + 16, w);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = w[j] = 0x7fc00000u;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) st_shared_f1(part + (c + j) * 512, __uint_as_float(v[j]));
      if (two)
#pragma unroll
        for (int j = 0; j < 16; ++j) st_shared_f1(part + (c + 16 + j) * 512, __uint_as_float(w[j]));
    }
    tc_fence_before();
  }
  if (p.split > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
  {
    // this CTA's share of the tile: 128 / S (64 / S) result columns in groups of four, one group per
    // thread, and rows of x in steps of (threads / groups)
    const int lq = (GATED ? 4 : 5) - p.lsplit;  // log2 of the groups
    const int c = (((rank << lq) + (tid & ((1 << lq) - 1)))) * 4, n = n0 + c;
    const int step = SNT >> lq;
    const int live = n < p.N ? min(p.tn, p.M - m0) : 0;
    int m = tid >> lq;
    const T* bias = static_cast<const T*>(p.bias);
    const bool pre_f32 = p.pre_f32 != 0, vec = p.vec != 0;  // (vec: N is a multiple of 4)
    const int have = min(4, p.N - n);
    float4 b4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (bias && live > 0) b4 = load_n(bias + n, have, vec);
    uint32_t at = smem_addr(smem) + (m * 128 + c) * 4;
    T* out = static_cast<T*>(p.out) + (int64_t)(m0 + m) * p.ld_out + n;
    const T* res = static_cast<const T*>(p.res) + (int64_t)(m0 + m) * p.ld_res + n;
    int64_t pi = (int64_t)(m0 + m) * p.ld_pre + n;
    // four partial columns of a row of x: every CTA's are asked for before any is added, in rank order
    auto ask = [&](auto s, uint32_t from, float4 (&v)[decltype(s)::value]) {
      constexpr int S = decltype(s)::value;
      if constexpr (S == 1) {
        v[0] = ld_shared_f4(from);
      } else {
#pragma unroll
        for (int r = 0; r < S; ++r) v[r] = ld_cluster_f4(mapa_addr(from, r));
      }
    };
    auto add_up = [&](const auto& v) {
      float4 t = v[0];
#pragma unroll
      for (int r = 1; r < (int)(sizeof(v) / sizeof(float4)); ++r)
        t = make_float4(t.x + v[r].x, t.y + v[r].y, t.z + v[r].z, t.w + v[r].w);
      return t;
    };
    auto finish = [&](auto code, float4 z, float4 u) {
      constexpr int ACT = decltype(code)::value;
      z = make_float4(z.x + b4.x, z.y + b4.y, z.z + b4.z, z.w + b4.w);
      if (p.pre) {
        if (pre_f32) {
          store_n(static_cast<float*>(p.pre) + pi, z, have, vec);
          if constexpr (GATED) store_n(static_cast<float*>(p.pre) + pi + p.N, u, have, vec);
        } else {
          store_n(static_cast<T*>(p.pre) + pi, z, have, vec);
          if constexpr (GATED) store_n(static_cast<T*>(p.pre) + pi + p.N, u, have, vec);
        }
        pi += step * p.ld_pre;
      }
      float4 y = make_float4(act_f(z.x, ACT), act_f(z.y, ACT), act_f(z.z, ACT), act_f(z.w, ACT));
      if constexpr (GATED) y = make_float4(y.x * u.x, y.y * u.y, y.z * u.z, y.w * u.w);
      if (p.res) {
        const float4 r = load_n(res, have, vec);
        y = make_float4(y.x + r.x, y.y + r.y, y.z + r.z, y.w + r.w);
        res += step * p.ld_res;
      }
      store_n(out, y, have, vec);
      out += step * p.ld_out;
    };
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    // One loop per activation and split: with both chosen at run time inside it, a row of four
    // columns cost 540 issue cycles instead of about 60, more than the product itself at 64 rows.
    auto rows = [&](auto code, auto s) {
      constexpr int S = decltype(s)::value;
      float4 v[S], w[S];
      if constexpr (GATED) {
        for (; m < live; m += step, at += step * 512) {
          ask(s, at, v);
          ask(s, at + 256, w);
          const float4 g = add_up(v);
          finish(code, g, add_up(w));
        }
      } else {  // two rows at a time
        for (; m < live; m += 2 * step, at += 2 * step * 512) {
          const bool two = m + step < live;
          ask(s, at, v);
          if (two) ask(s, at + step * 512, w);
          finish(code, add_up(v), none);
          if (two) finish(code, add_up(w), none);
        }
      }
    };
    auto with_act = [&](auto s) {
      if constexpr (W_MN) rows(std::integral_constant<int, KVS_ACT_NONE>(), s);  // (dx has none)
      else with_act_code(p.act, [&](auto code) { rows(code, s); });
    };
    if (p.split == 1) with_act(std::integral_constant<int, 1>());
    else if (p.split == 2) with_act(std::integral_constant<int, 2>());
    else if (p.split == 4) with_act(std::integral_constant<int, 4>());
    else with_act(std::integral_constant<int, 8>());
  }
  if (p.split > 1) cluster_sync();  // no CTA leaves while another reads its partials
}

// ------------------------------------------------------------------ gradients of the epilogue
// (No __restrict__ on what these kernels read: a kernel that starts before the one before it has ended may not load
// that one's results as read-only data, nor may the compiler move the loads up past the wait as such.)
// Eight consecutive elements as they lie in memory: as separate half-precision values they would
// be unpacked, and waited for, where they are loaded.
template <typename T> struct alignas(16) Raw8 {
  uint32_t v[2 * sizeof(T)];
};
// zeros from the n-th on
template <typename T> __device__ __forceinline__ Raw8<T> load8(const T* p, int n, bool vec) {
  if (vec) return *reinterpret_cast<const Raw8<T>*>(p);
  Vec8<T> r;
#pragma unroll
  for (int k = 0; k < 8; ++k) r.v[k] = k < n ? p[k] : from_acc<T>(0.f);
  return *reinterpret_cast<const Raw8<T>*>(&r);
}
template <typename T> __device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = to_acc<T>(e[k]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// dz = gy act'(pre) (or gy itself) into a row pitch the tensor maps take, and its column sums
// over a chunk of rows (the bias gradient's partials, added up in chunk order: the bits do not
// depend on scheduling).  64 x 4 threads: eight columns each, rows in steps of four, the loads
// of two to four steps in flight.  Bound by HBM: bias sums of 8192 x 4096 15.6 us (4.3 TB/s), with silu's
// gradient 47 us (268 MB, 5.7 TB/s).
template <typename T, typename Z>
__global__ void __launch_bounds__(256, 4)
dz_kernel(const T* gy, int64_t ld_gy, const Z* pre, int64_t ld_pre, int act, T* dz, int64_t ld_dz, float* part, int M,
          int N, int rows_per, int vec) {
  __shared__ float red[4][512];
  pdl_let_next_start();
  pdl_wait_for_previous();
  const int c0 = (blockIdx.x * 64 + threadIdx.x) * 8;
  const int r_beg = (int)min((int64_t)M, (int64_t)blockIdx.y * rows_per);
  const int r_end = (int)min((int64_t)M, ((int64_t)blockIdx.y + 1) * rows_per);
  const int nv = N - c0;
  float sum[8] = {};
  if (nv > 0)
    with_act_code(act, [&](auto code) {
      constexpr int ACT = decltype(code)::value;
      constexpr int U = ACT == KVS_ACT_NONE ? 4 : 2;
      for (int r0 = r_beg + threadIdx.y; r0 < r_end; r0 += 4 * U) {
        Raw8<T> gv[U];
        Raw8<Z> zv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t r = r0 + 4 * u;
          if (r < r_end) {
            gv[u] = load8(gy + r * ld_gy + c0, nv, vec);
            if (ACT != KVS_ACT_NONE) zv[u] = load8(pre + r * ld_pre + c0, nv, vec);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t r = r0 + 4 * u;
          if (r < r_end) {
            float d[8], z[8];
            unpack8(gv[u], d);
            if (ACT != KVS_ACT_NONE) {
              unpack8(zv[u], z);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                float a, da;
                act_grad_f(z[k], ACT, a, da);
                d[k] *= da;
              }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[k] += d[k];
            if (dz) store8(dz + r * ld_dz + c0, d);  // (its pitch is a multiple of 8)
          }
        }
      }
    });
  if (!part) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[threadIdx.y][threadIdx.x * 8 + k] = sum[k];
  __syncthreads();
  for (int i = threadIdx.y * 64 + threadIdx.x; i < 512; i += 256) {
    const int c = blockIdx.x * 512 + i;
    if (c < N) part[(int64_t)blockIdx.y * N + c] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
  }
}

// db[j] = sum of the chunks' partials: thread row y takes chunks y, y + 8, ..., then the eight are
// added in order
template <typename T>
__global__ void __launch_bounds__(256)
bias_grad_kernel(const float* part, T* db, int n_parts, int N) {
  __shared__ float red[8][32];
  pdl_let_next_start();
  pdl_wait_for_previous();
  const int j = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (j < N) {
#pragma unroll 8
    for (int c = threadIdx.y; c < n_parts; c += 8) s += part[(int64_t)c * N + j];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && j < N) {
    float t = red[0][threadIdx.x];
#pragma unroll
    for (int y = 1; y < 8; ++y) t += red[y][threadIdx.x];
    db[j] = from_acc<T>(t);
  }
}

// dg = gh u act'(g) and du = gh act(g), eight columns per thread; dgu rows hold dg at 0 and du
// at `half` (N rounded up to 8), zeros between.  Bound by HBM.
template <typename T, typename Z>
__global__ void __launch_bounds__(256)
gated_dz_kernel(const T* gh, int64_t ld_gh, const Z* pre, int64_t ld_pre, int act, T* dgu, int64_t ld_dgu, int half,
                int64_t M, int N, int vec) {
  pdl_let_next_start();
  pdl_wait_for_previous();
  const int nvec = half / 8;
  with_act_code(act, [&](auto code) {
    constexpr int ACT = decltype(code)::value;
    for (int64_t idx = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; idx < M * nvec;
         idx += (int64_t)gridDim.x * blockDim.x) {
      const int64_t r = idx / nvec;
      const int c0 = (int)(idx - r * nvec) * 8, nv = N - c0;
      const Z* g = pre + r * ld_pre + c0;
      const Raw8<Z> gr = load8(g, nv, vec), ur = load8(g + N, nv, vec);
      const Raw8<T> hr = load8(gh + r * ld_gh + c0, nv, vec);
      float gv[8], uv[8], hv[8], og[8], ou[8];
      unpack8(gr, gv);
      unpack8(ur, uv);
      unpack8(hr, hv);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float a, da;
        act_grad_f(gv[k], ACT, a, da);
        og[k] = hv[k] * uv[k] * da;
        ou[k] = hv[k] * a;
      }
      store8(dgu + r * ld_dgu + c0, og);
      store8(dgu + r * ld_dgu + half + c0, ou);
    }
  });
}

// ------------------------------------------------------------------ host
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// a [rows][cols] matrix of half-precision elements, rows `ld` elements apart, read in boxes of 64
// columns (one 128-byte swizzled row) x `box_rows` rows; elements outside read as zeros
bool make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, int32_t dtype) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  if (rows == 1) ld = (cols + 7) / 8 * 8;  // a single row has no pitch
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {BK, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, dtype == KVS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// a [rows][cols] result written in boxes of 32 x 32 (half precision: 64-byte rows, float32: 128)
bool make_out_map(CUtensorMap* m, void* base, int64_t rows, int64_t cols, int64_t ld, int32_t dtype) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const int size = dtype == KVS_F32 ? 4 : 2;
  if (rows == 1) ld = (cols + 7) / 8 * 8;  // a single row has no pitch
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * size};
  const cuuint32_t box[2] = {32, 32};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m,
            dtype == KVS_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
            : dtype == KVS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            size == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// An operand of a product: [rows][cols] as it lies in memory.  K-major operands have the reduced
// index along a row (box of 128 rows), MN-major ones down the rows (two boxes of 64 rows).
struct Operand {
  const void* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
};

bool al(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }

std::mutex g_mu;
struct KernelState {
  bool set[64] = {};
  int pairs[64] = {};
};

// pairs of CTAs of `kernel` that can run at once on the current device (0: it cannot be set up)
template <typename K> int max_pairs(K kernel, KernelState& s) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(g_mu);
  if (!s.set[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PAIR_SMEM) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    cudaLaunchConfig_t cfg = {};  // the cluster size (2) is the kernel's compile-time attribute
    cfg.gridDim = dim3(2, 1, 1);
    cfg.blockDim = dim3(NT, 1, 1);
    cfg.dynamicSmemBytes = PAIR_SMEM;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    s.pairs[dev] = n;
    s.set[dev] = true;
  }
  return s.pairs[dev];
}

// How a product is dealt out to the CTA pairs: unit width, units done whole, pairs that share the
// K blocks of the others, and the estimate in microseconds by which the cut was chosen: of a single
// launch at full clock whose operands come from L2.  About 6 outside the loop, 1.5 a unit, and per K block
// 0.29 for 256 columns, near the tensor cores' nominal rate, but 0.235 for 128, which the 64 bytes per clock
// that an SM takes from L2 bound (24 KB a block against 32).  Cut units cost about 7 (19 MB of sums
// written at once; less with fewer pairs) and 2 for each pair whose sums the last one to finish has to add.
//
// The estimates compare ways of one product; they are not its time.  Fitted on 512..2048 x 4096 x 4096, they come
// out low as products grow, since the clock falls under the power cap and long reduced indexes wait for HBM:
// 8192 x 4096 x 4096 146 (measured 168-199), 4096 x 14336 gated x 4096 507 (590), 1999 x 6144 x 4096 66 (69-90),
// a 4096 x 4096 weight gradient from 16384 rows whole 309 (532), from 32768 606 (790-970).  What they chose, whole
// tiles against cut: 1024 x 6144 x 4096 46 -> 43 us, 2048 x 2560 x 4096 46 -> 37, 640 x 4096 x 14336 99 -> 81,
// 2304 x 2304 x 16384 168 -> 159, 900 x 1500 x 14344 76 -> 50, 300 x 2048 x 32768 139 -> 63; of 12 sizes cut one
// lost, 3000 x 2560 x 8192 91 -> 96.
//
// Pairs with cut units are at different K blocks and share operands only through L2, of which about
// 90 MB holds them (110 where both operands lie MN-major: a K block of all tiles is then contiguous):
// what does not fit comes from HBM again for every pair, 64 KB a K block of a full tile.  Units are cut where
// the larger of the two times gains four percent.  Weight gradients, whole tiles against cut: 4096 x 4096
// from 8192 rows 239 -> 220 us, from 16384 532 -> 439, 6144 x 4096 from 16384 782 -> 674; forward
// 4000 x 2560 x 8192 172 -> 138.  Not cut: a 4096 x 4096 weight gradient from 32768 rows (971 us,
// cut 1065), 2048 x 4096 x 14336 (165, cut 231), 8192 x 4096 over 28672 (1885, cut 2050): past 250 MB only in
// equal cuts, at most half as many units as pairs, whose pairs stay as near in K as those of whole units do and
// which would leave the others idle (weight gradients of a narrow layer, whole tiles against cut: 64 x 64 from
// 262144 rows 1097 -> 99 us, 1 x 4096 from 65536 291 -> 120, 1001 x 520 from 131072 567 -> 190).
constexpr int PAIRS = 74;  // of a B200's 148 SMs
struct PairPlan {
  int bn, whole, cut_pairs;
  double us;
  size_t scratch() const { return (size_t)cut_pairs * 2 * EPI_WARPS * (SUMS_PER_WARP * 4 + 8); }
};
// A group of row blocks passes over all of B once: where B is too large to stay in L2 (126 MB, shared
// with A and the results), fewer passes of it are worth more rows of A in flight.  8192 x 14336
// gated x 4096: 1345 us in groups of 16, 1390 of 8; with B of 34 MB 215 us of 8, 218 of 16; and where
// 16 row blocks do not stay in L2 themselves, 16384 x 4096 x 14336 takes 1513 in groups of 8, 1548 of 16.
int group_of(int64_t N, int kb, bool gated) {
  const int64_t row = 2 * (int64_t)kb * BK;  // bytes
  return N * (gated ? 2 : 1) * row > (48 << 20) && 16 * 256 * row <= (48 << 20) ? 16 : 8;
}
PairPlan pair_plan_of(int64_t M_part, int m_parts, int64_t N, int kb, bool gated, bool both_mn, bool cut_allowed) {
  const int64_t M = M_part * m_parts, row_blocks = (M_part + 2 * BM - 1) / (2 * BM) * m_parts;
  auto units_of = [&](int bn) { return row_blocks * ((N + (gated ? bn / 2 : bn) - 1) / (gated ? bn / 2 : bn)); };
  auto rounds = [](int64_t units) { return (double)((units + PAIRS - 1) / PAIRS); };
  const int64_t units = units_of(256);
  PairPlan best = {256, (int)std::min<int64_t>(units, 1 << 30), 0, 6.0 + rounds(units) * (1.5 + kb * 0.29)};
  const double narrow = 6.0 + rounds(units_of(128)) * (1.5 + kb * 0.235);
  if (narrow < best.us) best = {128, (int)std::min<int64_t>(units_of(128), 1 << 30), 0, narrow};
  if (!cut_allowed || units % PAIRS == 0 || units >= (1 << 30)) return best;
  const int64_t whole = std::max<int64_t>(0, units / PAIRS - 1) * PAIRS, rest = units - whole;
  // bytes that the cut units' tiles read, in rows and columns that exist, and a K block of one of them
  const int64_t cols = units / row_blocks, n_cols = gated ? 2 * N : N;
  const int64_t r = std::max(std::min<int64_t>(row_blocks, group_of(N, kb, gated)), (rest + cols - 1) / cols);
  const int64_t c = std::min(cols, (rest + r - 1) / r);
  const double shared_mb = (double)(std::min(r * 256, M) + std::min(c * 256, n_cols)) * kb * BK * 2 / 1e6;
  const double block_mb = (double)(std::min<int64_t>(256, M) + std::min<int64_t>(256, n_cols)) * BK * 2 / 1e6;
  const double fits_mb = both_mn ? 110.0 : 90.0;
  const double hbm_us = shared_mb > fits_mb ? (double)rest * kb * block_mb * (1.0 - fits_mb / shared_mb) / 6.4 : 0.0;
  const double uncut = best.us;
  auto consider = [&](int64_t pairs, int others, bool in_step) {
    const double run = (double)rest * kb / pairs;  // K blocks a pair
    if (run < 4) return;
    const double us = 6.0 + (double)(whole / PAIRS) * (1.5 + kb * 0.29) + std::max(run * 0.29, in_step ? 0.0 : hbm_us) +
                      1.5 * (1 + (run > kb)) + 7.0 * (double)pairs / PAIRS + 2.0 * others;
    if (us < best.us && us < 0.96 * uncut) best = {256, (int)whole, (int)pairs, us};
  };
  // equal cuts of every unit (pairs with the same part of theirs keep in step, whatever the length), or all pairs
  // whatever the cuts come to
  for (int s = 2; rest < PAIRS && rest * s <= PAIRS; ++s) consider(rest * s, s - 1, true);
  if (shared_mb <= 250.0) consider(PAIRS, rest >= PAIRS ? 1 : (int)((PAIRS + rest - 1) / rest), false);
  return best;
}

struct Product {
  Operand a[2], b[2];
  PairParams p = {};
  void* scratch = nullptr;  // for cut units' sums
  size_t scratch_bytes = 0;
};

// a value that no other launch of this process has, and that memory does not hold by chance
unsigned long long launch_token() {
  static std::atomic<unsigned long long> count{(unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
  unsigned long long z = count.fetch_add(0x9E3779B97F4A7C15ull) + 0x9E3779B97F4A7C15ull;  // SplitMix64 (Steele, Lea, Flood 2014)
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  z ^= z >> 31;
  return z && ~z ? z : 1;  // (a clean word, 0, is neither a token nor the complement that a given-up flag holds)
}

template <typename T, bool A_MN, bool B_MN, int EPI, int BN>
int launch_pair_n(const Product& g, const PairPlan& plan, int32_t dtype, cudaStream_t st) {
  constexpr bool GATED = EPI == EPI_GATED;
  static KernelState state;
  const auto kernel = pair_gemm_kernel<T, A_MN, B_MN, EPI, BN>;
  const int most = max_pairs(kernel, state);
  if (most <= 0) return KVS_E_UNSUPPORTED;
  CUtensorMap m[4];
  for (int i = 0; i < 2; ++i) {
    const Operand &a = g.a[i], &b = g.b[i];
    if (!a.p) m[i] = m[0];  // (no second operand)
    else if (!make_map(&m[i], a.p, a.rows, a.cols, a.ld, A_MN ? 64 : 128, dtype)) return KVS_E_UNSUPPORTED;
    if (!b.p) m[2 + i] = m[2];
    else if (!make_map(&m[2 + i], b.p, b.rows, b.cols, b.ld, B_MN ? 64 : BN / 2, dtype)) return KVS_E_UNSUPPORTED;
  }
  PairParams p = g.p;
  CUtensorMap o[3] = {m[0], m[0], m[0]};  // (those not written are not used)
  if (p.vec) {
    if (!make_out_map(&o[0], p.out0, p.M, p.N, p.ld_out, dtype)) return KVS_E_UNSUPPORTED;
    if (p.m_parts > 1 && !make_out_map(&o[1], p.out1, p.M, p.N, p.ld_out, dtype)) return KVS_E_UNSUPPORTED;
    if (p.pre) {  // gate and up have a map each, so that a box at the end of one leaves the other alone
      const int32_t type = p.pre_f32 ? KVS_F32 : dtype;
      if (!make_out_map(&o[2], p.pre, p.M, p.N, p.ld_pre, type)) return KVS_E_UNSUPPORTED;
      uint8_t* up = static_cast<uint8_t*>(p.pre) + (size_t)p.N * (p.pre_f32 ? 4 : 2);
      if (GATED && !make_out_map(&o[1], up, p.M, p.N, p.ld_pre, type)) return KVS_E_UNSUPPORTED;
    }
  }
  p.mb = (p.M + 2 * BM - 1) / (2 * BM);
  p.nb = GATED ? (p.N + BN / 2 - 1) / (BN / 2) : (p.N + BN - 1) / BN;
  const int64_t units = (int64_t)p.mb * p.m_parts * p.nb;
  if (units > (1 << 30)) return KVS_E_UNSUPPORTED;
  p.n_units = p.whole = (int)units;
  p.cut_pairs = 0;
  p.group = group_of(p.N, p.n_kb * p.k_parts, GATED);
  int pairs = std::min(most, p.n_units);
  if (BN == 256 && plan.cut_pairs > 0 && most >= PAIRS) {
    p.whole = plan.whole;
    p.cut_pairs = plan.cut_pairs;
    pairs = plan.whole > 0 ? PAIRS : plan.cut_pairs;
    p.ready = static_cast<unsigned long long*>(g.scratch);
    p.sums = reinterpret_cast<float*>(p.ready + (size_t)plan.cut_pairs * 2 * EPI_WARPS);
    p.token = launch_token();
  }
  return launch_overlapped(kernel, 2 * pairs, NT, PAIR_SMEM, st, 0, m[0], m[1], m[2], m[3], o[0], o[1],
                           o[2], p);
}

// clusters of `size` (2, 4, 8) of the stream kernel's CTAs that run at once, one CTA an SM
int clusters_at_once(int size) {
  static int most[64][3];  // by device; 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return size == 2 ? 74 : size == 4 ? 33 : 15;  // planning without a device: a B200's
  }
  std::lock_guard<std::mutex> lock(g_mu);
  int& n = most[dev][size / 4];
  if (n == 0) {
    const auto kernel = stream_gemm_kernel<__nv_bfloat16, false, false>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size, 1, 1);
    cfg.blockDim = dim3(SNT, 1, 1);
    cfg.dynamicSmemBytes = 200 * 1024;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
  }
  return n;
}

// ---- few rows: how a product is cut for the stream kernel
struct StreamPlan {
  int tn, stages, split, per_sm;
  size_t smem;
};
StreamPlan stream_plan(int64_t M, int64_t N, int kb_all, bool gated) {
  StreamPlan s;
  const int most = 128;  // rows per tile
  const int64_t mt = (M + most - 1) / most;
  s.tn = (int)(((M + mt - 1) / mt + 15) / 16 * 16);
  const int stage = TILE_BYTES + s.tn * BK * 2;
  const int fixed = S_BAR_BYTES + 1024;
  const int64_t tiles = ((N + (gated ? 63 : 127)) / (gated ? 64 : 128)) * mt;
  // As many CTAs a tile as run at once with the whole shared memory as their ring, but with two K blocks
  // each, four where the partial sums are large (128 x 1024 x 1024: 6.6 us in fours, 7.4 in eights).  What
  // does not run at once waits for a whole round: 64 x 4608 x 4096 takes 12.4 us in clusters of two, 18.0
  // of four, and 2048 columns of K 4096 8.6 in fours, 14.5 in eights.  (Powers of two: clusters of other
  // sizes pack badly into the GPCs; 1 x 6144 x 4096 took 18.6 us with six CTAs a tile, 13.4 with four.)
  auto cut = [&](int per_sm, int least) {
    int split = 1;
    while (split < SMAX_SPLIT && tiles <= (int64_t)per_sm * clusters_at_once(split * 2) && kb_all / (split * 2) >= least)
      split *= 2;
    return split;
  };
  // One CTA an SM has the deeper ring and exchanges half the partial sums: 64 x 1024 x 4096 7.2 us against
  // 7.9 with two an SM, 128 x 2048 x 14336 18.7 against 21.8.  Two an SM are better
  //   for one to 16 rows, where their number lets a tile be cut once more: 1 x 4608 x 4096 9.9 against 11.1,
  //   1 x 4608 x 14336 25.5 against 30.3;
  //   for up to 64 rows of K >= 2048, where whole tiles leave SMs idle: 32 x 10240 x 4096 18.2 against 19.4;
  //   and where there are more tiles than SMs: 64 x 28672 x 4096 45.4 against 47.8.
  const int least = s.tn > 32 ? 4 : 2;
  const int one = cut(1, least), two = cut(2, least);
  const bool spread = two > one && (s.tn <= 16 || (one == 1 && s.tn <= 64 && kb_all >= 32));
  s.per_sm = spread || tiles > 148 ? 2 : 1;
  const int room = (s.per_sm == 1 ? 232448 : HALF_SM_SMEM) - fixed;
  s.stages = std::min(room / stage, SMAX_STAGES);  // three at least, which hold the 512 tn bytes of partial sums
  s.split = s.per_sm == 2 ? two : one;
  s.smem = (size_t)s.stages * stage + fixed;
  return s;
}

template <typename T, bool W_MN, bool GATED>
int launch_stream(const Operand (&w)[2], const Operand (&x)[2], StreamParams p, int32_t dtype, cudaStream_t st) {
  static bool set[64] = {};
  const auto kernel = stream_gemm_kernel<T, W_MN, GATED>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return KVS_E_UNSUPPORTED;
  {
    std::lock_guard<std::mutex> lock(g_mu);
    if (!set[dev]) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess) {
        cudaGetLastError();
        return KVS_E_UNSUPPORTED;
      }
      set[dev] = true;
    }
  }
  const StreamPlan s = stream_plan(p.M, p.N, p.n_kb * p.k_parts, GATED);
  CUtensorMap m[4];
  for (int i = 0; i < 2; ++i) {
    if (!w[i].p) m[i] = m[0];  // (no second operand)
    else if (!make_map(&m[i], w[i].p, w[i].rows, w[i].cols, w[i].ld, W_MN || GATED ? 64 : 128, dtype))
      return KVS_E_UNSUPPORTED;
    if (!x[i].p) m[2 + i] = m[2];
    else if (!make_map(&m[2 + i], x[i].p, x[i].rows, x[i].cols, x[i].ld, s.tn, dtype)) return KVS_E_UNSUPPORTED;
  }
  p.tn = s.tn;
  p.stages = s.stages;
  p.split = s.split;
  p.lsplit = s.split == 8 ? 3 : s.split / 2;  // 1, 2, 4, 8
  p.nt = (p.N + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
  const int64_t ctas = (int64_t)p.nt * ((p.M + s.tn - 1) / s.tn) * s.split;
  if (ctas > (1 << 30)) return KVS_E_UNSUPPORTED;
  return launch_overlapped(kernel, (unsigned)ctas, SNT, s.smem, st, s.split, m[0], m[1], m[2], m[3], p);
}

template <typename T, bool A_MN, bool B_MN, int EPI>
int launch_pair(const Product& g, int32_t dtype, cudaStream_t st) {
  PairPlan plan = pair_plan_of(g.p.M, g.p.m_parts, g.p.N, g.p.n_kb * g.p.k_parts, EPI == EPI_GATED, A_MN && B_MN, true);
  if (plan.scratch() > g.scratch_bytes)
    plan = pair_plan_of(g.p.M, g.p.m_parts, g.p.N, g.p.n_kb * g.p.k_parts, EPI == EPI_GATED, A_MN && B_MN, false);
  return plan.bn == 128 ? launch_pair_n<T, A_MN, B_MN, EPI, 128>(g, plan, dtype, st)
                        : launch_pair_n<T, A_MN, B_MN, EPI, 256>(g, plan, dtype, st);
}

// Whether a product of M rows goes to the stream kernel.  Up to 128 rows the weights' bytes bound
// it (128 x 14336 gated x 4096: 48.1 us against 57 in pair units; 64 x 4096 x 14336: 22.9 against
// 62).  Beyond, two estimates decide, fitted to both kernels' times over 144..1536 rows, 1024..14336
// columns and K 520..14336, back to back.  Here a K block takes a CTA 0.27 us, an SM takes 147 KB
// and all of them 18 MB a microsecond from L2; a row of a tile costs 0.021 us to finish, a doubling of
// the cluster 0.27.  What pair_plan says of the pairs is its time alone: of its 6 us about 3 are
// hidden in a row of calls.  300 x 6144 x 4096 takes 19.7 us here, 26.2 in pairs; 256 x 1024 x 1024
// 7.2 against 7.4; 640 x 4096 x 2048 18.7 against 15.4.  The choice is within 24 % of the better
// one everywhere in that range, within 1 % on average.
bool use_stream(int64_t M, int64_t N, int kb_all, bool gated) {
  if (M <= 128) return true;
  const StreamPlan s = stream_plan(M, N, kb_all, gated);
  const int64_t ctas = ((N + (gated ? 63 : 127)) / (gated ? 64 : 128)) * ((M + s.tn - 1) / s.tn) * s.split;
  const double rounds = (double)((ctas + 148 * s.per_sm - 1) / (148 * s.per_sm)), on_an_sm = (double)((ctas + 147) / 148);
  const double blocks = (kb_all + s.split - 1) / s.split, bytes = blocks * (TILE_BYTES + s.tn * BK * 2);
  const double us = 3.0 + std::max({rounds * blocks * 0.27, on_an_sm * bytes / 147e3, (double)ctas * bytes / 18.1e6}) +
                    rounds * s.tn * 0.021 + std::log2((double)s.split) * 0.27 + (rounds - 1) * 3.3;
  return us < 3.1 + 1.065 * (pair_plan_of(M, 1, N, kb_all, gated, false, true).us - 6.0);
}

// scratch of one product for its cut units (0: none)
// (a weight gradient's operands both lie MN-major, and it has no few-rows form)
size_t product_scratch(int64_t M, int m_parts, int64_t N, int kb_all, bool gated, bool weight_grad) {
  if (!weight_grad && use_stream(M, N, kb_all, gated)) return 0;
  return pair_plan_of(M, m_parts, N, kb_all, gated, weight_grad, true).scratch();
}

bool act_ok(int32_t a) { return a >= KVS_ACT_NONE && a <= KVS_ACT_GELU; }

// sizes whose block counts and columns stay inside 32 bits
bool sizes_ok(const kvs_linear_args* a) {
  return a->n > 0 && a->k > 0 && a->rows <= (1 << 30) && a->n <= (1 << 29) && a->k <= (1 << 30);
}

// what both directions ask of x and the weights
int check_common(const kvs_linear_args* a) {
  if (!a || a->rows < 0 || a->n <= 0 || a->k <= 0 || !act_ok(a->activation)) return KVS_E_ARG;
  if (a->dtype != KVS_BF16 && a->dtype != KVS_F16) return KVS_E_UNSUPPORTED;
  if (a->k % 8 || !sizes_ok(a)) return KVS_E_UNSUPPORTED;
  if (!a->weight || (a->rows > 0 && !a->x)) return KVS_E_ARG;
  if ((a->rows > 1 && a->ld_x < a->k) || (a->n > 1 && a->ld_w < a->k) ||
      (a->weight_up && a->n > 1 && a->ld_w_up < a->k))
    return KVS_E_ARG;
  if ((a->rows > 1 && a->ld_x % 8) || (a->n > 1 && a->ld_w % 8) || (a->weight_up && a->n > 1 && a->ld_w_up % 8) ||
      !al(a->x, 16) || !al(a->weight, 16) || !al(a->weight_up, 16))
    return KVS_E_UNSUPPORTED;
  if (a->weight_up && (a->bias || a->residual)) return KVS_E_ARG;
  if (a->pre && a->pre_dtype != KVS_F32 && a->pre_dtype != a->dtype) return KVS_E_UNSUPPORTED;
  return KVS_OK;
}

template <typename T> int forward(const kvs_linear_args* a, cudaStream_t st) {
  Product g;
  g.a[0] = {a->x, a->rows, a->k, a->ld_x};
  g.b[0] = {a->weight, a->n, a->k, a->ld_w};
  if (a->weight_up) g.b[1] = {a->weight_up, a->n, a->k, a->ld_w_up};
  PairParams& p = g.p;
  p.M = a->rows;
  p.N = a->n;
  p.n_kb = (a->k + BK - 1) / BK;
  p.k_parts = p.m_parts = 1;
  p.act = a->activation;
  p.out0 = a->out;
  p.bias = a->bias;
  p.res = a->residual;
  p.pre = a->pre;
  p.pre_f32 = a->pre_dtype == KVS_F32;
  p.ld_out = a->ld_out;
  p.ld_res = a->ld_res;
  p.ld_pre = a->ld_pre;
  auto fits = [&](int e) {  // e elements at a time, everywhere
    const int bytes = 2 * e;
    return a->n % e == 0 && a->ld_out % e == 0 && al(a->out, bytes) && al(a->bias, bytes) &&
           (!a->residual || (a->ld_res % e == 0 && al(a->residual, bytes))) &&
           (!a->pre || (a->ld_pre % e == 0 && al(a->pre, 16)));
  };
  const bool gated = a->weight_up != nullptr;
  if (use_stream(a->rows, a->n, p.n_kb, gated)) {
    StreamParams s = {};
    s.M = p.M, s.N = p.N, s.n_kb = p.n_kb, s.k_parts = 1;
    s.act = p.act, s.vec = fits(4), s.pre_f32 = p.pre_f32;
    s.out = p.out0, s.bias = p.bias, s.res = p.res, s.pre = p.pre;
    s.ld_out = p.ld_out, s.ld_res = p.ld_res, s.ld_pre = p.ld_pre;
    return gated ? launch_stream<T, false, true>(g.b, g.a, s, a->dtype, st)
                 : launch_stream<T, false, false>(g.b, g.a, s, a->dtype, st);
  }
  p.vec = fits(8);
  g.scratch = a->scratch;
  g.scratch_bytes = a->scratch && al(a->scratch, 16) ? a->scratch_bytes : 0;
  return gated ? launch_pair<T, false, false, EPI_GATED>(g, a->dtype, st)
                      : launch_pair<T, false, false, EPI_LINEAR>(g, a->dtype, st);
}

// rows per chunk of the bias-gradient partials: at most 256 chunks, enough of them that the
// column blocks (512 wide) fill the machine about four times over
int bias_rows_per(int64_t rows, int32_t n) {
  const int64_t cols = (n + 511) / 512;
  const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({(rows + 15) / 16, 592 / cols + 1, 256}));
  return (int)((rows + chunks - 1) / chunks);
}

// whether the plain form needs dz as a tensor of its own: an activation, or a gradient whose
// rows the tensor maps cannot take as they lie
bool needs_dz(const kvs_linear_args* a, const kvs_linear_grads* g) {
  return a->activation != KVS_ACT_NONE || !al(g->gy, 16) || (a->rows > 1 && g->ld_gy % 8);
}

// the backward's products: K blocks of dx (over n, twice when gated) and of dw (over the rows)
int dx_blocks(const kvs_linear_args* a) { return (a->n + BK - 1) / BK * (a->weight_up ? 2 : 1); }
int dw_blocks(const kvs_linear_args* a) { return (a->rows + BK - 1) / BK; }
// scratch of the larger of the two (they run one after the other)
size_t backward_product_scratch(const kvs_linear_args* a, const kvs_linear_grads* g) {
  const size_t x = g->dx ? product_scratch(a->rows, 1, a->k, dx_blocks(a), false, false) : 0;
  const size_t w = g->dw ? product_scratch(a->n, a->weight_up ? 2 : 1, a->k, dw_blocks(a), false, true) : 0;
  return std::max(x, w);
}
// what lies before it: dz and the bias partials
size_t backward_front_scratch(const kvs_linear_args* a, const kvs_linear_grads* g) {
  const size_t pitch = (size_t)up8(a->n);
  if (a->weight_up) return align_up((size_t)a->rows * 2 * pitch * 2, 256);
  size_t bytes = needs_dz(a, g) ? align_up((size_t)a->rows * pitch * 2, 256) : 0;
  if (g->db) {
    const int per = bias_rows_per(a->rows, a->n);
    bytes += align_up((size_t)((a->rows + per - 1) / per) * a->n * sizeof(float), 256);
  }
  return bytes;
}

template <typename T, typename Z> int backward(const kvs_linear_args* a, const kvs_linear_grads* g, cudaStream_t st) {
  const bool gated = a->weight_up != nullptr;
  const int M = a->rows, N = a->n, K = a->k;
  const int64_t pitch = up8(N);
  uint8_t* sp = static_cast<uint8_t*>(g->scratch);
  const T* gy = static_cast<const T*>(g->gy);
  const Z* pre = static_cast<const Z*>(a->pre);
  Operand dz[2];
  int rc;
  const size_t front = backward_front_scratch(a, g);
  void* const cut = sp + front;
  const size_t cut_bytes = g->scratch_bytes > front ? g->scratch_bytes - front : 0;
  if (gated) {
    const bool vec = N % 8 == 0 && al(gy, 16) && al(pre, 16) && g->ld_gy % 8 == 0 && a->ld_pre % 8 == 0;
    T* dgu = reinterpret_cast<T*>(sp);
    const int64_t work = (int64_t)M * (pitch / 8);
    rc = launch_overlapped(gated_dz_kernel<T, Z>, (unsigned)std::min<int64_t>((work + 255) / 256, 148 * 16), 256, 0, st, 0,
                           gy, g->ld_gy, pre, a->ld_pre, a->activation, dgu, 2 * pitch, (int)pitch, (int64_t)M, N,
                           (int)vec);
    if (rc) return rc;
    dz[0] = {dgu, M, N, 2 * pitch};
    dz[1] = {dgu + pitch, M, N, 2 * pitch};
  } else {
    dz[0] = {gy, M, N, g->ld_gy};
    T* own_dz = nullptr;
    if (needs_dz(a, g)) {
      own_dz = reinterpret_cast<T*>(sp);
      sp += align_up((size_t)M * pitch * sizeof(T), 256);
      dz[0] = {own_dz, M, N, pitch};
    }
    if (own_dz || g->db) {
      const int per = bias_rows_per(M, N), chunks = (M + per - 1) / per;
      float* part = g->db ? reinterpret_cast<float*>(sp) : nullptr;
      const bool act = a->activation != KVS_ACT_NONE;
      const bool vec = N % 8 == 0 && al(gy, 16) && g->ld_gy % 8 == 0 && (!act || (al(pre, 16) && a->ld_pre % 8 == 0));
      rc = launch_overlapped(dz_kernel<T, Z>, dim3((N + 511) / 512, chunks), dim3(64, 4), 0, st, 0, gy, g->ld_gy,
                             act ? pre : nullptr, a->ld_pre, a->activation, own_dz, pitch, part, M, N, per, (int)vec);
      if (rc) return rc;
      if (part) {
        rc = launch_overlapped(bias_grad_kernel<T>, (N + 31) / 32, dim3(32, 8), 0, st, 0, part, static_cast<T*>(g->db),
                               chunks, N);
        if (rc) return rc;
      }
    }
  }
  if (g->dx) {  // [M][K] = dz [M][N] W [N][K], summed over N (twice when gated)
    Product x;
    x.scratch = cut;
    x.scratch_bytes = cut_bytes;
    x.a[0] = dz[0];
    x.a[1] = dz[1];
    x.b[0] = {a->weight, N, K, a->ld_w};
    if (gated) x.b[1] = {a->weight_up, N, K, a->ld_w_up};
    x.p.M = M;
    x.p.N = K;
    x.p.k_parts = gated ? 2 : 1;
    x.p.n_kb = dx_blocks(a) / x.p.k_parts;
    x.p.m_parts = 1;
    x.p.out0 = g->dx;
    x.p.ld_out = g->ld_dx;
    x.p.vec = g->ld_dx % 8 == 0 && al(g->dx, 16);  // (K is a multiple of 8)
    if (use_stream(M, K, x.p.n_kb * x.p.k_parts, false)) {
      StreamParams s = {};
      s.M = M, s.N = K, s.n_kb = x.p.n_kb, s.k_parts = x.p.k_parts;
      s.vec = g->ld_dx % 4 == 0 && al(g->dx, 8), s.out = g->dx, s.ld_out = g->ld_dx;
      rc = launch_stream<T, true, false>(x.b, x.a, s, a->dtype, st);
    } else {
      rc = launch_pair<T, false, true, EPI_STORE>(x, a->dtype, st);
    }
    if (rc) return rc;
  }
  if (g->dw) {  // [N][K] = dz^T [N][M] x [M][K], summed over the rows (two results when gated)
    Product w;
    w.scratch = cut;
    w.scratch_bytes = cut_bytes;
    w.a[0] = dz[0];
    w.a[1] = dz[1];
    w.b[0] = {a->x, M, K, a->ld_x};
    w.p.M = N;
    w.p.N = K;
    w.p.n_kb = dw_blocks(a);
    w.p.k_parts = 1;
    w.p.m_parts = gated ? 2 : 1;
    w.p.out0 = g->dw;
    w.p.out1 = g->dw_up;
    w.p.ld_out = g->ld_dw;
    w.p.vec = g->ld_dw % 8 == 0 && al(g->dw, 16) && al(g->dw_up, 16);
    if ((rc = launch_pair<T, true, true, EPI_STORE>(w, a->dtype, st))) return rc;
  }
  return KVS_OK;
}

}  // namespace

KVS_API size_t kvs_linear_scratch_bytes(const kvs_linear_args* a) {
  if (!a || a->rows <= 0 || !sizes_ok(a)) return 0;
  return product_scratch(a->rows, 1, a->n, (a->k + BK - 1) / BK, a->weight_up != nullptr, false);
}

KVS_API int kvs_linear(const kvs_linear_args* a, kvs_stream_t stream) {
  if (int rc = check_common(a)) return rc;
  const bool gated = a->weight_up != nullptr;
  if (a->rows == 0) return KVS_OK;
  if (!a->out || a->ld_out < a->n || (a->residual && a->ld_res < a->n) ||
      (a->pre && a->ld_pre < (int64_t)a->n * (gated ? 2 : 1)))
    return KVS_E_ARG;
  return a->dtype == KVS_F16 ? forward<__half>(a, to_cuda(stream)) : forward<__nv_bfloat16>(a, to_cuda(stream));
}

KVS_API size_t kvs_linear_backward_scratch_bytes(const kvs_linear_args* a, const kvs_linear_grads* g) {
  if (!a || !g || a->rows <= 0 || !sizes_ok(a)) return 0;
  return backward_front_scratch(a, g) + backward_product_scratch(a, g);
}

KVS_API int kvs_linear_backward(const kvs_linear_args* a, const kvs_linear_grads* g, kvs_stream_t stream) {
  if (int rc = check_common(a)) return rc;
  const bool gated = a->weight_up != nullptr;
  if (!g || (gated && ((g->dw != nullptr) != (g->dw_up != nullptr) || g->db)) || (!gated && g->dw_up)) return KVS_E_ARG;
  if ((g->dx && g->ld_dx < a->k) || (g->dw && g->ld_dw < a->k)) return KVS_E_ARG;
  const cudaStream_t st = to_cuda(stream);
  if (a->rows == 0) {  // sums over no rows
    cudaError_t e = cudaSuccess;
    for (void* w : {g->dw, g->dw_up})
      if (w && e == cudaSuccess) e = cudaMemset2DAsync(w, (size_t)g->ld_dw * 2, 0, (size_t)a->k * 2, a->n, st);
    if (g->db && e == cudaSuccess) e = cudaMemsetAsync(g->db, 0, (size_t)a->n * 2, st);
    return e == cudaSuccess ? KVS_OK : KVS_E_LAUNCH;
  }
  const bool needs_pre = gated || a->activation != KVS_ACT_NONE;
  if (!g->gy || g->ld_gy < a->n || (needs_pre && (!a->pre || a->ld_pre < (int64_t)a->n * (gated ? 2 : 1))))
    return KVS_E_ARG;
  if ((g->dx && !al(g->dx, 2)) || (g->dw && !al(g->dw, 2))) return KVS_E_ARG;
  const size_t need = kvs_linear_backward_scratch_bytes(a, g);
  if (need && (!g->scratch || g->scratch_bytes < need || !al(g->scratch, 256))) return KVS_E_SCRATCH;
  const bool f32 = a->pre_dtype == KVS_F32;
  if (a->dtype == KVS_F16) return f32 ? backward<__half, float>(a, g, st) : backward<__half, __half>(a, g, st);
  return f32 ? backward<__nv_bfloat16, float>(a, g, st) : backward<__nv_bfloat16, __nv_bfloat16>(a, g, st);
}

namespace {
// One thread plays both sides of a flag between CTAs.  late 0: gives, then takes.  late 1: takes before anything
// was given, and gives after that, as a part does whose owner's wait ran out.  out[0]: whether the take saw the
// flag; out[1]: whether the word is 0 when both are done; out[2]: whether a take of the same token, by a replay
// whose giver has not come yet, sees a flag.
__global__ void flag_selftest_kernel(int late, int polls, unsigned long long token, unsigned long long* flag, int32_t* out) {
  if (!late) flag_give(flag, token);
  out[0] = flag_take(flag, token, polls);
  if (late) flag_give(flag, token);
  out[1] = *flag == 0;
  out[2] = flag_take(flag, token, polls);
}
}  // namespace

KVS_API int kvs_selftest_flag(int32_t late, int32_t polls, uint64_t token, uint64_t* flag, int32_t* out,
                              kvs_stream_t stream) {
  if (!flag || !out || late < 0 || late > 1 || polls < 1 || token == 0 || token == ~(uint64_t)0) return KVS_E_ARG;
  flag_selftest_kernel<<<1, 1, 0, to_cuda(stream)>>>(late, polls, token, reinterpret_cast<unsigned long long*>(flag), out);
  return launch_rc();
}
