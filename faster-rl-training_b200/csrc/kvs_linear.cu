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
#include "kvs_common.cuh"
#include "kvs_sm100.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>

using namespace kvs;
using namespace kvs::sm100;

namespace {

// ------------------------------------------------------------------ element-wise helpers
__device__ __forceinline__ float sigmoid_f(float z) { return 1.f / (1.f + __expf(-z)); }

__device__ __forceinline__ float act_f(float z, int act) {
  if (act == KVS_ACT_RELU) return z <= 0.f ? 0.f : z;  // a NaN stays one
  if (act == KVS_ACT_SILU) return z * sigmoid_f(z);
  if (act == KVS_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
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
    const float c = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    a = z * c;
    da = c + z * 0.39894228040143268f * __expf(-0.5f * z * z);
  } else {
    a = z;
    da = 1.f;
  }
}

template <typename T> struct alignas(sizeof(T) * 4) Vec4 { T v[4]; };
template <typename T> struct alignas(16) Vec8 { T v[8]; };

// four consecutive elements in one access
template <typename T> __device__ __forceinline__ float4 load4(const T* p) {
  const Vec4<T> q = *reinterpret_cast<const Vec4<T>*>(p);
  return make_float4(to_acc<T>(q.v[0]), to_acc<T>(q.v[1]), to_acc<T>(q.v[2]), to_acc<T>(q.v[3]));
}
template <typename T> __device__ __forceinline__ void store4(T* p, float4 f) {
  Vec4<T> q;
  q.v[0] = from_acc<T>(f.x);
  q.v[1] = from_acc<T>(f.y);
  q.v[2] = from_acc<T>(f.z);
  q.v[3] = from_acc<T>(f.w);
  *reinterpret_cast<Vec4<T>*>(p) = q;
}
template <typename T> __device__ __forceinline__ void store_pre(void* pre, int64_t i, float4 f, bool f32) {
  if (f32) store4(static_cast<float*>(pre) + i, f);
  else store4(static_cast<T*>(pre) + i, f);
}
// a running pointer the compiler may not turn into one precomputed address per unrolled step
// (they would cost the epilogue its registers)
template <typename P> __device__ __forceinline__ void advance(P*& p, int64_t step) {
  p += step;
  asm volatile("" : "+l"(p));
}
template <typename T> __device__ __forceinline__ void store_pre1(void* pre, int64_t i, float f, bool f32) {
  if (f32) static_cast<float*>(pre)[i] = f;
  else static_cast<T*>(pre)[i] = from_acc<T>(f);
}

// ------------------------------------------------------------------ pair GEMM
constexpr int BM = 128;  // result rows per CTA (256 per pair)
constexpr int BN = 256;  // accumulator columns per unit (128 per CTA's share of B)
constexpr int BK = 64;   // reduced elements per stage
constexpr int STAGES = 6;
constexpr int TILE_BYTES = 128 * BK * 2;     // 16 KB, either major
constexpr int HALF_TILE = TILE_BYTES / 2;    // MN-major: 64 MN elements x 64 K rows
constexpr int STAGE_BYTES = 2 * TILE_BYTES;  // A + B of one CTA
constexpr int EPI_WARPS = 8;  // two per TMEM lane quadrant, each half of the columns
constexpr int NT = 128 + 32 * EPI_WARPS;
constexpr int OFF_STAGING = STAGES * STAGE_BYTES;  // per epilogue warp 32 rows x 32 float32
constexpr int STAGING_BYTES = EPI_WARPS * 32 * 32 * 4;
constexpr int OFF_BAR = OFF_STAGING + STAGING_BYTES;
enum { B_FULL = 0, B_EMPTY = STAGES, B_ACCF = 2 * STAGES, B_ACCE = 2 * STAGES + 2, B_FINAL = 2 * STAGES + 4,
       NBAR = 2 * STAGES + 5 };
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
  int act;
  int vec;         // N is a multiple of 4 and every row of out / res / pre may be accessed four at a time
  int pre_f32;     // pre is float32 (else of the activations' type)
  void* out0;
  void* out1;
  const void* bias;
  const void* res;
  void* pre;
  int64_t ld_out, ld_res, ld_pre;
};

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

// 128 rows (MN index `row`) x 64 reduced elements (block kb) of an operand into `dst`
template <bool MN>
__device__ __forceinline__ void load_tile_pair(uint8_t* dst, const CUtensorMap* map, int kb, int row, uint32_t bar) {
  if (MN) {  // map: inner index MN, outer K
    tma_load_2d_pair(dst, map, row, kb * BK, bar);
    tma_load_2d_pair(dst + HALF_TILE, map, row + 64, kb * BK, bar);
  } else {
    tma_load_2d_pair(dst, map, kb * BK, row, bar);
  }
}

// what the epilogue does with an accumulator: store it, the plain product's whole epilogue, or the
// gate's product
enum { EPI_STORE = 0, EPI_LINEAR = 1, EPI_GATED = 2 };

template <typename T, bool A_MN, bool B_MN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NT, 1)
pair_gemm_kernel(const __grid_constant__ CUtensorMap tm_a0, const __grid_constant__ CUtensorMap tm_a1,
                 const __grid_constant__ CUtensorMap tm_b0, const __grid_constant__ CUtensorMap tm_b1,
                 const PairParams p) {
  constexpr bool GATED = EPI == EPI_GATED;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_MISC + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();  // 0: the even CTA, which issues the MMAs
  const int pair = (int)(blockIdx.x >> 1), n_pairs = (int)(gridDim.x >> 1);

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

  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------------- producer
      bool ok = true;
      int it = 0;
      for (int u = pair; ok && u < p.n_units; u += n_pairs) {
        int part, mb, nb;
        unit_of(p, u, part, mb, nb);
        const int row = mb * 2 * BM + (int)rank * BM;
        const int col = GATED ? nb * (BN / 2) : nb * BN + (int)rank * (BN / 2);
        for (int k = 0; k < kb_all; ++k, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES && !mbar_wait(&bar[B_EMPTY + s], ((it / STAGES) - 1) & 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t full = mapa_shared(&bar[B_FULL + s], 0);
          if (rank == 0) mbar_arrive_expect_tx(&bar[B_FULL + s], 2 * STAGE_BYTES);
          uint8_t* st = smem + s * STAGE_BYTES;
          const bool second = k >= p.n_kb;  // of two K parts
          const int kb = second ? k - p.n_kb : k;
          load_tile_pair<A_MN>(st, part || second ? &tm_a1 : &tm_a0, kb, row, full);
          load_tile_pair<B_MN>(st + TILE_BYTES, second || (GATED && rank) ? &tm_b1 : &tm_b0, kb, col, full);
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
      int it = 0, ui = 0;
      for (int u = pair; ok && u < p.n_units; u += n_pairs, ++ui) {
        const int ab = ui & 1;
        if (ui >= 2) {
          ok = __all_sync(0xffffffffu, mbar_wait_fast(&bar[B_ACCE + ab], ((ui >> 1) - 1) & 1, abort_flag));
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t d = tmem + ab * BN;
        for (int k = 0; k < kb_all; ++k, ++it) {
          const int s = it % STAGES;
          ok = __all_sync(0xffffffffu, mbar_wait_fast(&bar[B_FULL + s], (it / STAGES) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = operand_desc<A_MN>(base + s * STAGE_BYTES);
          const uint64_t db = operand_desc<B_MN>(base + s * STAGE_BYTES + TILE_BYTES);
          umma_pair_warp_at<0, 0>(d, da, db, IDESC, k > 0);
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
    // A warp takes its 32 accumulator rows 32 columns at a time: one row per lane out of TMEM,
    // through shared memory (16-byte chunks swizzled by the row, no bank conflicts), so that
    // eight lanes then hold one row's 32 columns and global accesses are 64-byte runs; rows whose
    // pitch or base does not allow that go one element per lane.  The residual of a chunk is read
    // before its accumulators are waited for.
    const int w = warp - 4, q = w & 3, half = w >> 2;  // TMEM lane quadrant, column half
    constexpr int COLS = (GATED ? BN / 2 : BN) / 2;   // result columns of this warp
    const uint32_t acce = mapa_shared(&bar[B_ACCE], 0);
    uint8_t* stage = smem + OFF_STAGING + w * (32 * 32 * 4);
    const int rr = lane >> 3, cc = lane & 7;
    const bool vec = p.vec != 0, pre_f32 = p.pre_f32 != 0;
    const T* res = EPI == EPI_LINEAR ? static_cast<const T*>(p.res) : nullptr;
    const T* bias = EPI == EPI_LINEAR ? static_cast<const T*>(p.bias) : nullptr;
    void* const pre = EPI == EPI_STORE ? nullptr : p.pre;
    const int act = EPI == EPI_STORE ? KVS_ACT_NONE : p.act;
    // addresses as 32-bit offsets formed at their use: row r, 16-byte chunk c lies at
    // 128 r + 16 (c ^ (r & 7))
    const uint32_t stage_at = smem_addr(stage);
    const uint32_t put_at = stage_at + lane * 128 + ((lane & 7) << 4);
    const uint32_t four_at = stage_at + rr * 128 + ((cc ^ rr) << 4);
    auto to_smem = [&](const uint32_t (&v)[32]) {
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 8; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(put_at ^ (c << 4)), "r"(v[4 * c]),
                     "r"(v[4 * c + 1]), "r"(v[4 * c + 2]), "r"(v[4 * c + 3])
                     : "memory");
      __syncwarp();
    };
    // row 4 i + rr, columns 4 cc .. 4 cc + 3 (r & 7 = rr + 4 (i & 1): the chunk's bit 2 flips)
    auto four = [&](int i) {
      float4 f;
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                   : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                   : "r"((four_at ^ ((i & 1) << 6)) + i * 512));
      return f;
    };
    auto single = [&](int r) {  // row r, column `lane`
      float f;
      asm volatile("ld.shared.f32 %0, [%1];\n"
                   : "=f"(f)
                   : "r"(stage_at + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4));
      return f;
    };
    bool dead = false;
    int ui = 0;
    for (int u = pair; u < p.n_units; u += n_pairs, ++ui) {
      const int ab = ui & 1;
      int part, mb, nb;
      unit_of(p, u, part, mb, nb);
      const int64_t row0 = (int64_t)mb * 2 * BM + (int)rank * BM + q * 32;
      const int n0 = nb * (GATED ? BN / 2 : BN) + half * COLS;
      const int rows = (int)min((int64_t)32, p.M - row0);  // existing rows of this warp
      T* out = static_cast<T*>(part ? p.out1 : p.out0);
      uint2 rv[8];  // the residual of the chunk at hand, four elements each
      if (res && vec) {
        const T* first = res + (row0 + rr) * p.ld_res + n0 + cc * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i * 4 + rr < rows && n0 + cc * 4 < p.N) rv[i] = *reinterpret_cast<const uint2*>(first);
          advance(first, 4 * p.ld_res);
        }
      }
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait(&bar[B_ACCF + ab], (ui >> 1) & 1, abort_flag));
      if (dead && lane == 0) *abort_flag = 1;
      tc_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + ab * BN + half * COLS;
#pragma unroll 1
      for (int c = 0; c < COLS / 32; ++c) {
        if (n0 + c * 32 >= p.N) break;
        const int col = n0 + c * 32 + (vec ? cc * 4 : lane);
        const bool in = col < p.N;  // (vec: N is a multiple of 4)
        uint32_t v[32];
        if (!dead) {
          tmem_ld32(taddr + c * 32, v);
          if constexpr (!GATED) tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0x7fc00000u;
        }
        if constexpr (GATED) {
          // g and u of one output lie in the same lane: the product is formed before the exchange
          uint32_t u32[32];
          if (!dead) {
            tmem_ld32(taddr + BN / 2 + c * 32, u32);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) u32[j] = 0x7fc00000u;
          }
          // the chunk in shared memory to 32 rows of `to`
          auto rows_to = [&](auto* to, int64_t ld) {
            if (vec) {
              to += (row0 + rr) * ld + col;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if (i * 4 + rr < rows && in) store4(to, four(i));
                advance(to, 4 * ld);
              }
            } else {
              to += row0 * ld + col;
#pragma unroll 4
              for (int r = 0; r < rows; ++r) {
                if (in) *to = from_acc<std::remove_reference_t<decltype(*to)>>(single(r));
                advance(to, ld);
              }
            }
          };
          auto keep = [&](const uint32_t(&s)[32], int64_t off) {
            to_smem(s);
            if (pre_f32) rows_to(static_cast<float*>(pre) + off, p.ld_pre);
            else rows_to(static_cast<T*>(pre) + off, p.ld_pre);
          };
          if (pre) {
            keep(v, 0);
            keep(u32, p.N);
          }
          auto gate = [&](auto code) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              v[j] = __float_as_uint(act_f(__uint_as_float(v[j]), decltype(code)::value) * __uint_as_float(u32[j]));
          };
          if (act == KVS_ACT_SILU) gate(std::integral_constant<int, KVS_ACT_SILU>());
          else if (act == KVS_ACT_GELU) gate(std::integral_constant<int, KVS_ACT_GELU>());
          else if (act == KVS_ACT_RELU) gate(std::integral_constant<int, KVS_ACT_RELU>());
          else gate(std::integral_constant<int, KVS_ACT_NONE>());
          to_smem(v);
          rows_to(out, p.ld_out);
          continue;
        }
        to_smem(v);
        auto finish = [&](auto code) {
          constexpr int ACT = decltype(code)::value;
          if (vec) {
            float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
            if (bias && in) b = load4(bias + col);
            T* o = out + (row0 + rr) * p.ld_out + col;
            const T* next = res + (row0 + rr) * p.ld_res + col + 32;
            const bool more = (c + 1) * 32 < COLS && col + 32 < p.N;
            int64_t pi = (row0 + rr) * p.ld_pre + col;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool on = i * 4 + rr < rows && in;
              const float4 f = four(i);
              const float4 z = make_float4(f.x + b.x, f.y + b.y, f.z + b.z, f.w + b.w);
              if (pre) {
                if (on) store_pre<T>(pre, pi, z, pre_f32);
                pi += 4 * p.ld_pre;
                asm volatile("" : "+l"(pi));
              }
              float4 y = make_float4(act_f(z.x, ACT), act_f(z.y, ACT), act_f(z.z, ACT), act_f(z.w, ACT));
              if (res) {  // the next chunk's load goes out as soon as this one's value is taken
                Vec4<T> r4;
                *reinterpret_cast<uint2*>(&r4) = rv[i];
                y.x += to_acc<T>(r4.v[0]);
                y.y += to_acc<T>(r4.v[1]);
                y.z += to_acc<T>(r4.v[2]);
                y.w += to_acc<T>(r4.v[3]);
                if (more && i * 4 + rr < rows) rv[i] = *reinterpret_cast<const uint2*>(next);
                advance(next, 4 * p.ld_res);
              }
              if (on) store4(o, y);
              advance(o, 4 * p.ld_out);
            }
          } else {
            const float b = bias && in ? to_acc<T>(bias[col]) : 0.f;
            T* o = out + row0 * p.ld_out + col;
            const T* rp = res + row0 * p.ld_res + col;
            int64_t pi = row0 * p.ld_pre + col;
#pragma unroll 1
            for (int r0 = 0; r0 < rows; r0 += 8) {
              float y[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                y[i] = res && r0 + i < rows && in ? to_acc<T>(*rp) : 0.f;
                if (res) advance(rp, p.ld_res);
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = r0 + i;
                if (r < rows && in) {
                  const float z = single(r) + b;
                  if (pre) store_pre1<T>(pre, pi + i * p.ld_pre, z, pre_f32);
                  *o = from_acc<T>(act_f(z, ACT) + y[i]);
                }
                advance(o, p.ld_out);
              }
              pi += 8 * p.ld_pre;
            }
          }
        };
        if (EPI == EPI_STORE || act == KVS_ACT_NONE) finish(std::integral_constant<int, KVS_ACT_NONE>());
        else if (act == KVS_ACT_SILU) finish(std::integral_constant<int, KVS_ACT_SILU>());
        else if (act == KVS_ACT_GELU) finish(std::integral_constant<int, KVS_ACT_GELU>());
        else finish(std::integral_constant<int, KVS_ACT_RELU>());
      }
      // this thread's TMEM reads are done: release the accumulator to the MMA warp
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acce + ab * 8);
    }
  }
  tc_fence_before();
  cluster_sync();  // both CTAs done with TMEM and with each other's barriers
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------------ gradients of the epilogue
// eight consecutive elements, zeros from the n-th on
template <typename T> __device__ __forceinline__ Vec8<T> load8(const T* p, int n, bool vec) {
  if (vec) return *reinterpret_cast<const Vec8<T>*>(p);
  Vec8<T> r;
#pragma unroll
  for (int k = 0; k < 8; ++k) r.v[k] = k < n ? p[k] : from_acc<T>(0.f);
  return r;
}

// dz = gy act'(pre) (or gy itself) into a row pitch the tensor maps take, and its column sums
// over a chunk of rows (the bias gradient's partials, added up in chunk order: the bits do not
// depend on scheduling).  64 x 4 threads: eight columns each, rows in steps of four.
template <typename T, typename Z>
__global__ void __launch_bounds__(256)
dz_kernel(const T* __restrict__ gy, int64_t ld_gy, const Z* __restrict__ pre, int64_t ld_pre, int act,
          T* __restrict__ dz, int64_t ld_dz, float* __restrict__ part, int M, int N, int rows_per, int vec) {
  __shared__ float red[4][512];
  const int c0 = (blockIdx.x * 64 + threadIdx.x) * 8;
  const int r_end = min(M, (int)(blockIdx.y + 1) * rows_per);
  const int nv = N - c0;
  float sum[8] = {};
  if (nv > 0) {
    for (int r = blockIdx.y * rows_per + threadIdx.y; r < r_end; r += 4) {
      const T* g = gy + (int64_t)r * ld_gy + c0;
      const Z* z = pre ? pre + (int64_t)r * ld_pre + c0 : nullptr;
      Vec8<T> o;
      const Vec8<T> gv = load8(g, nv, vec);
      Vec8<Z> zv;
      if (z) zv = load8(z, nv, vec);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float d = to_acc<T>(gv.v[k]);
        if (z) {
          float a, da;
          act_grad_f(to_acc<Z>(zv.v[k]), act, a, da);
          d *= da;
        }
        sum[k] += d;
        o.v[k] = from_acc<T>(d);
      }
      if (dz) *reinterpret_cast<Vec8<T>*>(dz + (int64_t)r * ld_dz + c0) = o;  // pitch a multiple of 8
    }
  }
  if (!part) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[threadIdx.y][threadIdx.x * 8 + k] = sum[k];
  __syncthreads();
  for (int i = threadIdx.y * 64 + threadIdx.x; i < 512; i += 256) {
    const int c = blockIdx.x * 512 + i;
    if (c < N) part[(int64_t)blockIdx.y * N + c] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
  }
}

template <typename T>
__global__ void bias_grad_kernel(const float* __restrict__ part, T* __restrict__ db, int n_parts, int N) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= N) return;
  float s = 0.f;
  for (int c = 0; c < n_parts; ++c) s += part[(int64_t)c * N + j];
  db[j] = from_acc<T>(s);
}

// dg = gh u act'(g) and du = gh act(g), eight columns per thread; dgu rows hold dg at 0 and du
// at `half` (N rounded up to 8), zeros between
template <typename T, typename Z>
__global__ void __launch_bounds__(256)
gated_dz_kernel(const T* __restrict__ gh, int64_t ld_gh, const Z* __restrict__ pre, int64_t ld_pre, int act,
                T* __restrict__ dgu, int64_t ld_dgu, int half, int64_t M, int N, int vec) {
  const int nvec = half / 8;
  for (int64_t idx = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; idx < M * nvec;
       idx += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = idx / nvec;
    const int c0 = (int)(idx - r * nvec) * 8, nv = N - c0;
    const Z* g = pre + r * ld_pre + c0;
    const Vec8<Z> gv = load8(g, nv, vec), uv = load8(g + N, nv, vec);
    const Vec8<T> hv = load8(gh + r * ld_gh + c0, nv, vec);
    Vec8<T> og, ou;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float a, da;
      act_grad_f(to_acc<Z>(gv.v[k]), act, a, da);
      const float hf = to_acc<T>(hv.v[k]);
      og.v[k] = from_acc<T>(hf * to_acc<Z>(uv.v[k]) * da);
      ou.v[k] = from_acc<T>(hf * a);
    }
    *reinterpret_cast<Vec8<T>*>(dgu + r * ld_dgu + c0) = og;
    *reinterpret_cast<Vec8<T>*>(dgu + r * ld_dgu + half + c0) = ou;
  }
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

struct Product {
  Operand a[2], b[2];
  PairParams p = {};
};

template <typename T, bool A_MN, bool B_MN, int EPI>
int launch_pair(const Product& g, int32_t dtype, cudaStream_t st) {
  constexpr bool GATED = EPI == EPI_GATED;
  static KernelState state;
  const auto kernel = pair_gemm_kernel<T, A_MN, B_MN, EPI>;
  const int most = max_pairs(kernel, state);
  if (most <= 0) return KVS_E_UNSUPPORTED;
  CUtensorMap m[4];
  for (int i = 0; i < 2; ++i) {
    const Operand& a = g.a[i].p ? g.a[i] : g.a[0];
    const Operand& b = g.b[i].p ? g.b[i] : g.b[0];
    if (!make_map(&m[i], a.p, a.rows, a.cols, a.ld, A_MN ? 64 : 128, dtype) ||
        !make_map(&m[2 + i], b.p, b.rows, b.cols, b.ld, B_MN ? 64 : 128, dtype))
      return KVS_E_UNSUPPORTED;
  }
  PairParams p = g.p;
  p.mb = (p.M + 2 * BM - 1) / (2 * BM);
  p.nb = GATED ? (p.N + BN / 2 - 1) / (BN / 2) : (p.N + BN - 1) / BN;
  const int64_t units = (int64_t)p.mb * p.m_parts * p.nb;
  if (units > (1 << 30)) return KVS_E_UNSUPPORTED;
  p.n_units = (int)units;
  p.group = 8;
  kernel<<<2 * std::min(most, p.n_units), NT, PAIR_SMEM, st>>>(m[0], m[1], m[2], m[3], p);
  return launch_rc();
}

bool act_ok(int32_t a) { return a >= KVS_ACT_NONE && a <= KVS_ACT_GELU; }

// what both directions ask of x and the weights
int check_common(const kvs_linear_args* a) {
  if (!a || a->rows < 0 || a->n <= 0 || a->k <= 0 || !act_ok(a->activation)) return KVS_E_ARG;
  if (a->dtype != KVS_BF16 && a->dtype != KVS_F16) return KVS_E_UNSUPPORTED;
  if (a->k % 8) return KVS_E_UNSUPPORTED;
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
  p.vec = a->n % 4 == 0 && a->ld_out % 4 == 0 && al(a->out, 8) && al(a->bias, 8) && (!a->residual || (a->ld_res % 4 == 0 && al(a->residual, 8))) &&
          (!a->pre || (a->ld_pre % 4 == 0 && al(a->pre, a->pre_dtype == KVS_F32 ? 16 : 8)));
  return a->weight_up ? launch_pair<T, false, false, EPI_GATED>(g, a->dtype, st)
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

template <typename T, typename Z> int backward(const kvs_linear_args* a, const kvs_linear_grads* g, cudaStream_t st) {
  const bool gated = a->weight_up != nullptr;
  const int M = a->rows, N = a->n, K = a->k;
  const int64_t pitch = up8(N);
  uint8_t* sp = static_cast<uint8_t*>(g->scratch);
  const T* gy = static_cast<const T*>(g->gy);
  const Z* pre = static_cast<const Z*>(a->pre);
  Operand dz[2];
  int rc;
  if (gated) {
    const bool vec = N % 8 == 0 && al(gy, 16) && al(pre, 16) && g->ld_gy % 8 == 0 && a->ld_pre % 8 == 0;
    T* dgu = reinterpret_cast<T*>(sp);
    const int64_t work = (int64_t)M * (pitch / 8);
    gated_dz_kernel<T, Z><<<(unsigned)std::min<int64_t>((work + 255) / 256, 148 * 16), 256, 0, st>>>(
        gy, g->ld_gy, pre, a->ld_pre, a->activation, dgu, 2 * pitch, (int)pitch, M, N, vec);
    if ((rc = launch_rc())) return rc;
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
      dz_kernel<T, Z><<<dim3((N + 511) / 512, chunks), dim3(64, 4), 0, st>>>(
          gy, g->ld_gy, act ? pre : nullptr, a->ld_pre, a->activation, own_dz, pitch, part, M, N, per, vec);
      if ((rc = launch_rc())) return rc;
      if (part) {
        bias_grad_kernel<T><<<(N + 255) / 256, 256, 0, st>>>(part, static_cast<T*>(g->db), chunks, N);
        if ((rc = launch_rc())) return rc;
      }
    }
  }
  if (g->dx) {  // [M][K] = dz [M][N] W [N][K], summed over N (twice when gated)
    Product x;
    x.a[0] = dz[0];
    x.a[1] = dz[1];
    x.b[0] = {a->weight, N, K, a->ld_w};
    if (gated) x.b[1] = {a->weight_up, N, K, a->ld_w_up};
    x.p.M = M;
    x.p.N = K;
    x.p.n_kb = (N + BK - 1) / BK;
    x.p.k_parts = gated ? 2 : 1;
    x.p.m_parts = 1;
    x.p.out0 = g->dx;
    x.p.ld_out = g->ld_dx;
    x.p.vec = g->ld_dx % 4 == 0 && al(g->dx, 8);
    if ((rc = launch_pair<T, false, true, EPI_STORE>(x, a->dtype, st))) return rc;
  }
  if (g->dw) {  // [N][K] = dz^T [N][M] x [M][K], summed over the rows (two results when gated)
    Product w;
    w.a[0] = dz[0];
    w.a[1] = dz[1];
    w.b[0] = {a->x, M, K, a->ld_x};
    w.p.M = N;
    w.p.N = K;
    w.p.n_kb = (M + BK - 1) / BK;
    w.p.k_parts = 1;
    w.p.m_parts = gated ? 2 : 1;
    w.p.out0 = g->dw;
    w.p.out1 = g->dw_up;
    w.p.ld_out = g->ld_dw;
    w.p.vec = g->ld_dw % 4 == 0 && al(g->dw, 8) && al(g->dw_up, 8);
    if ((rc = launch_pair<T, true, true, EPI_STORE>(w, a->dtype, st))) return rc;
  }
  return KVS_OK;
}

}  // namespace

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
  if (!a || !g || a->rows <= 0 || a->n <= 0) return 0;
  const size_t pitch = (size_t)up8(a->n);
  if (a->weight_up) return (size_t)a->rows * 2 * pitch * 2;
  size_t bytes = needs_dz(a, g) ? align_up((size_t)a->rows * pitch * 2, 256) : 0;
  if (g->db) {
    const int per = bias_rows_per(a->rows, a->n);
    bytes += (size_t)((a->rows + per - 1) / per) * a->n * sizeof(float);
  }
  return bytes;
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
