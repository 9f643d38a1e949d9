// gemm_tc.cu: the matrix products of the transformer-block operators in
// bf16 / f16 on the 5th-generation tensor cores (tcgen05 + TMEM).
//
//   acc[m, n] = sum over segments s, k of a[s](m, k) b[s](n, k)
//
// Persistent, warp-specialised. A tile is 128 rows per CTA by BN columns;
// with CG = 2 two CTAs of a cluster share one 256 x BN tile: each stages its
// own 128 rows of A and half the rows of B, and one MMA instruction of the
// pair (tcgen05.mma.cta_group::2) reads both halves, so every byte of B
// crosses into shared memory once per 256 rows. (One CTA alone at 128 x 256
// writes 12 KB and reads 12 KB of shared memory per 128-cycle MMA step,
// more than its 128 B/clk; the pair writes and reads 8 KB.)
//  * warp 0: TMA producer. Steps of 64 along the reduction into a ring of
//    stages, 128-byte swizzled. An operand whose reduced dimension is
//    contiguous is staged K-major (one box of 64 x rows); one whose rows
//    are contiguous, MN-major (boxes of 64 rows x 64): weight and input
//    gradients read their operands as they lie in memory, with no
//    transpose.
//  * warp 1: issues the MMAs (of the pair: its first CTA only). Two
//    accumulators in TMEM, so the next tile's product runs during this
//    one's epilogue.
//  * warp 2 allocates TMEM; warps 4-11 are the epilogue: two warps per TMEM
//    lane quarter, each half the columns. A lane holds one row; results are
//    packed and turned through shared memory so that global loads (the
//    residual) and stores run along rows in whole 128-byte lines.
// A gated layer's B tile is BN / 2 gate rows and the same BN / 2 up rows:
// one MMA makes both projections, and the epilogue finds both factors of an
// output in its row.
//
// A reduction too long for its few tiles is cut into parts that write
// float32 sums to the workspace; launch_split_finish adds them in order.
// Every wait is bounded (error word and early exit).
#include <atomic>

#include "block_common.cuh"
#include "gemm_tc.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

using namespace tc;

constexpr int kBM = 128;        // rows per CTA
constexpr int kBK = 64;         // reduction per stage: one 128-byte row
constexpr int kCtrlWarps = 4;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kCtrlWarps + kEpiWarps) * 32;
constexpr int kStagePitch = 144;  // epilogue turning buffer: 128 B + 16

template <int BN, int CG>
struct Cfg {
  static constexpr int B_ROWS = BN / CG;  // rows of B staged per CTA
  static constexpr int A_BYTES = kBM * kBK * 2;
  static constexpr int B_BYTES = B_ROWS * kBK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int EPI_BYTES = kEpiWarps * (32 * kStagePitch + 512);
  static constexpr int MAX_BYTES = 227 * 1024 - 2048 - EPI_BYTES;
  static constexpr int STAGES = MAX_BYTES / STAGE < 8 ? MAX_BYTES / STAGE : 8;
  static constexpr int OFF_EPI = STAGES * STAGE;
  static constexpr int OFF_BAR = OFF_EPI + EPI_BYTES;
  static constexpr int NBAR = 2 * STAGES + 4;
  static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16;
  static constexpr int SMEM_ALLOC = SMEM + 1024;  // 1024-byte alignment
  static constexpr int TMEM_COLS = 2 * BN;        // two accumulators
  static_assert(SMEM_ALLOC <= 227 * 1024, "shared memory");
  static_assert(TMEM_COLS == 512 || TMEM_COLS == 256 || TMEM_COLS == 128,
                "TMEM columns");
};

struct TcArgs {
  GemmProblem p;
  float* partial;     // split > 1: [split][planes][M][N]
  int tiles_m, tiles_n;
  int steps_seg;      // stages of one segment
  int steps;          // of all segments
  int split;
  int steps_part;     // steps of one part
  int64_t units;      // tiles * split
  uint8_t a_mn, b_mn;  // operand staged MN-major
  uint8_t vec_out, vec_pre, vec_res, vec_f32;
};

// The tile of a unit: groups of eight row tiles sweep the columns, so the
// tiles in flight share their operands in L2.
struct Unit {
  int m, n, part;
};
__device__ __forceinline__ Unit unit_of(const TcArgs& a, int64_t u) {
  constexpr int kGroup = 8;
  Unit r;
  int64_t tile = u;
  r.part = 0;
  if (a.split > 1) {
    tile = u / a.split;
    r.part = int(u - tile * a.split);
  }
  const int64_t per_group = int64_t(kGroup) * a.tiles_n;
  const int64_t g = tile / per_group;
  const int in = int(tile - g * per_group);
  const int first = int(g) * kGroup;
  const int rows = a.tiles_m - first < kGroup ? a.tiles_m - first : kGroup;
  r.m = first + in % rows;
  r.n = in / rows;
  return r;
}

// ---------------------------------------------------------------------------
// cta_group::2 forms and cluster helpers.
// ---------------------------------------------------------------------------
template <int CG>
__device__ __forceinline__ uint32_t cta_rank() {
  if constexpr (CG == 1) return 0;
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r)
               : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];"
               ::"r"(bar)
               : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void* map,
                                            uint32_t bar, int c0, int c1) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::"
        "complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global."
        "mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b,
                                        uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1) {
    tc_mma(d, a, b, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// Arrives on `bar` (of both CTAs of a pair) when the MMAs issued so far are
// done.
template <int CG>
__device__ __forceinline__ void commit_all(uint32_t bar) {
  if constexpr (CG == 1) {
    tc_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster."
        "multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(uint16_t(3))
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void alloc_cols(uint32_t slot, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile(
        "tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
        ::"r"(slot),
        "r"(cols)
        : "memory");
    asm volatile(
        "tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" :::
            "memory");
  }
}
template <int CG>
__device__ __forceinline__ void dealloc_cols(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_dealloc(addr, cols);
  } else {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(
                     addr),
                 "r"(cols)
                 : "memory");
  }
}

// ---------------------------------------------------------------------------
// Epilogue pieces. `stage` is the warp's 32 x kStagePitch turning buffer.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void activate32(float* v, int act) {
  switch (act) {
    case VECTRA_ACT_RELU:
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_fwd<false, VECTRA_ACT_RELU>(v[i]);
      break;
    case VECTRA_ACT_GELU:
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_fwd<false, VECTRA_ACT_GELU>(v[i]);
      break;
    case VECTRA_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < 32; ++i)
        v[i] = act_fwd<false, VECTRA_ACT_GELU_TANH>(v[i]);
      break;
    case VECTRA_ACT_SILU:
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = act_fwd<false, VECTRA_ACT_SILU>(v[i]);
      break;
    default:
      break;
  }
}

// Writes the warp's 32 x COLS block (row = lane, packed 16-bit pairs) to
// global rows row0.., columns col0.., through the turning buffer.
template <typename T, int COLS>
__device__ __forceinline__ void store_block(uint8_t* stage, const uint32_t* pk,
                                            T* out, int64_t ld, int64_t row0,
                                            int64_t rows, int64_t col0,
                                            int64_t cols, bool vec,
                                            int lane) {
#pragma unroll
  for (int c = 0; c < COLS / 8; ++c)
    *reinterpret_cast<uint4*>(stage + lane * kStagePitch + c * 16) =
        make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
  __syncwarp();
  if (vec) {
    constexpr int kLanes = COLS / 8;  // lanes per row
    const int c = lane % kLanes;
    const int64_t col = col0 + c * 8;
    if (col < cols) {
#pragma unroll
      for (int i = 0; i < kLanes; ++i) {
        const int r = i * (32 / kLanes) + lane / kLanes;
        if (row0 + r < rows)
          *reinterpret_cast<uint4*>(out + (row0 + r) * ld + col) =
              *reinterpret_cast<const uint4*>(stage + r * kStagePitch +
                                              c * 16);
      }
    }
  } else {
    for (int r = 0; r < 32 && row0 + r < rows; ++r) {
      const T* s = reinterpret_cast<const T*>(stage + r * kStagePitch);
#pragma unroll
      for (int c = 0; c < COLS; c += 32)
        if (col0 + c + lane < cols)
          out[(row0 + r) * ld + col0 + c + lane] = s[c + lane];
    }
  }
  __syncwarp();
}

// The same for 32 float32 columns.
__device__ __forceinline__ void store_block_f32(uint8_t* stage, const float* v,
                                                float* out, int64_t ld,
                                                int64_t row0, int64_t rows,
                                                int64_t col0, int64_t cols,
                                                bool vec, int lane) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4*>(stage + lane * kStagePitch + c * 16) =
        make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  __syncwarp();
  if (vec) {
    const int c = lane % 8;
    const int64_t col = col0 + c * 4;
    if (col < cols) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + lane / 8;
        if (row0 + r < rows)
          *reinterpret_cast<float4*>(out + (row0 + r) * ld + col) =
              *reinterpret_cast<const float4*>(stage + r * kStagePitch +
                                               c * 16);
      }
    }
  } else {
    for (int r = 0; r < 32 && row0 + r < rows; ++r)
      if (col0 + lane < cols)
        out[(row0 + r) * ld + col0 + lane] = reinterpret_cast<const float*>(
            stage + r * kStagePitch)[lane];
  }
  __syncwarp();
}

// Reads the warp's 32 x COLS block of the residual into pk (row = lane).
template <typename T, int COLS>
__device__ __forceinline__ void load_block(uint8_t* stage, uint32_t* pk,
                                           const GemmProblem& p, int64_t row0,
                                           int64_t col0, bool vec, int lane) {
  const T* res = static_cast<const T*>(p.res);
  if (vec) {
    constexpr int kLanes = COLS / 8;
    const int c = lane % kLanes;
    const int64_t col = col0 + c * 8;
    uint4 raw[kLanes];
#pragma unroll
    for (int i = 0; i < kLanes; ++i) {
      const int64_t row = row0 + i * (32 / kLanes) + lane / kLanes;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (row < p.M && col < p.N)
        raw[i] = *reinterpret_cast<const uint4*>(res + row * p.res_sm + col);
    }
#pragma unroll
    for (int i = 0; i < kLanes; ++i)
      *reinterpret_cast<uint4*>(
          stage + (i * (32 / kLanes) + lane / kLanes) * kStagePitch + c * 16) =
          raw[i];
  } else {
    for (int r = 0; r < 32; ++r) {
      T* s = reinterpret_cast<T*>(stage + r * kStagePitch);
#pragma unroll
      for (int c = 0; c < COLS; c += 32) {
        const int64_t row = row0 + r, col = col0 + c + lane;
        s[c + lane] = row < p.M && col < p.N
                          ? res[row * p.res_sm + col * p.res_sn]
                          : from_f32<T>(0.f);
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < COLS / 8; ++c) {
    const uint4 q = *reinterpret_cast<const uint4*>(
        stage + lane * kStagePitch + c * 16);
    pk[4 * c] = q.x;
    pk[4 * c + 1] = q.y;
    pk[4 * c + 2] = q.z;
    pk[4 * c + 3] = q.w;
  }
  __syncwarp();
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(w << 16),
                       __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Column terms of a group (bias), as floats in the warp's buffer.
template <typename T>
__device__ __forceinline__ void load_bias_cols(float* dst, const void* bias,
                                               int64_t stride, int64_t col0,
                                               int64_t cols, int n,
                                               int lane) {
  for (int c = lane; c < n; c += 32)
    dst[c] = bias && col0 + c < cols
                 ? to_f32(static_cast<const T*>(bias)[(col0 + c) * stride])
                 : 0.f;
}

template <int EPI, typename T, int BN, int CG>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap ta0,
                   const __grid_constant__ CUtensorMap ta1,
                   const __grid_constant__ CUtensorMap tb0,
                   const __grid_constant__ CUtensorMap tb1,
                   const __grid_constant__ TcArgs g) {
  using C = Cfg<BN, CG>;
  constexpr bool kGated = EPI == kEpiGated;
  constexpr int kTileN = kGated ? BN / 2 : BN;  // output columns of a tile
  constexpr int FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_addr(smem);
  const uint32_t bars = sbase + C::OFF_BAR;
  auto bar_full = [&](int s) { return bars + uint32_t(s) * 8; };
  auto bar_empty = [&](int s) { return bars + uint32_t(C::STAGES + s) * 8; };
  auto bar_acc_full = [&](int b) {
    return bars + uint32_t(2 * C::STAGES + b) * 8;
  };
  auto bar_acc_empty = [&](int b) {
    return bars + uint32_t(2 * C::STAGES + 2 + b) * 8;
  };
  uint32_t* tmem_slot =
      reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + C::NBAR * 8);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank<CG>();
  const GemmProblem& p = g.p;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), kEpiWarps * CG);
    }
    fence_barrier_init();
  }
  if (warp == 2) alloc_cols<CG>(smem_addr(tmem_slot), C::TMEM_COLS);
  allow_dependents();
  tc_fence_before();
  __syncthreads();
  // The peer's barriers exist before anything signals them.
  if constexpr (CG == 2) cluster_sync_all();
  tc_fence_after();
  grid_dependency_wait();
  const uint32_t tmem = *tmem_slot;
  const int64_t first = blockIdx.x / CG, stride = gridDim.x / CG;
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int s = 0;
      uint32_t phase = 0;
      int64_t issued = 0;
      for (int64_t u = first; u < g.units && ok; u += stride) {
        const Unit t = unit_of(g, u);
        const int m0 = (t.m * CG + int(rank)) * kBM;
        const int n0 = t.n * kTileN;
        const int k_first = t.part * g.steps_part;
        const int k_last = k_first + g.steps_part < g.steps
                               ? k_first + g.steps_part
                               : g.steps;
        for (int k = k_first; k < k_last; ++k) {
          ok = mbar_wait(bar_empty(s), phase ^ 1, p.err);
          if (!ok) break;
          uint32_t full = bar_full(s);
          if (CG == 1 || rank == 0)
            mbar_arrive_expect_tx(full, C::STAGE * CG);
          if constexpr (CG == 2) full = map_cta(full, 0);
          const int seg = k >= g.steps_seg ? 1 : 0;
          const int k0 = (k - seg * g.steps_seg) * kBK;
          const uint32_t sa = sbase + uint32_t(s) * C::STAGE;
          const uint32_t sb = sa + C::A_BYTES;
          const CUtensorMap* ma = seg ? &ta1 : &ta0;
          if (g.a_mn) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i)
              tma_load_2d<CG>(sa + i * 8192, ma, full, m0 + i * 64, k0);
          } else {
            tma_load_2d<CG>(sa, ma, full, k0, m0);
          }
          // Rows of B: in a pair, half each. A gated tile's first half is
          // the gate weight's rows, its second half the up weight's.
          constexpr int kBoxRows = kGated && CG == 1 ? BN / 2 : C::B_ROWS;
#pragma unroll
          for (int h = 0; h < C::B_ROWS / kBoxRows; ++h) {
            const CUtensorMap* mb =
                kGated ? ((CG == 2 ? int(rank) : h) ? &tb1 : &tb0)
                       : (seg ? &tb1 : &tb0);
            const int row =
                kGated ? n0 : n0 + int(rank) * C::B_ROWS;
            const uint32_t dst = sb + h * kBoxRows * 128;
            if (g.b_mn) {
#pragma unroll
              for (int i = 0; i < kBoxRows / 64; ++i)
                tma_load_2d<CG>(dst + i * 8192, mb, full, row + i * 64, k0);
            } else {
              tma_load_2d<CG>(dst, mb, full, k0, row);
            }
          }
          ++issued;
          if (++s == C::STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      // After a wait ran out, copies may still be in flight: let them land
      // (the barriers of the stages issued last) before shared memory goes.
      if (!ok && (CG == 1 || rank == 0)) {
        for (int i = 0; i < C::STAGES && i < issued; ++i) {
          s = s == 0 ? C::STAGES - 1 : s - 1;
          if (s == C::STAGES - 1) phase ^= 1;
          mbar_wait(bar_full(s), phase, p.err);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = f16_idesc(FMT, kBM * CG, BN, g.b_mn) |
                             (uint32_t(g.a_mn) << 15);
      // K-major: rows of 128 bytes, 8-row groups 1,024 bytes apart, a step
      // of 16 is 32 bytes. MN-major: blocks of 64 rows x 64 steps 8,192
      // bytes apart, a step of 16 is 16 lines of 128 bytes.
      const uint64_t da0 = sw128_desc(sbase, g.a_mn ? 8192 : 16, 1024);
      const uint64_t db0 =
          sw128_desc(sbase + C::A_BYTES, g.b_mn ? 8192 : 16, 1024);
      const uint32_t ka = (g.a_mn ? 2048 : 32) >> 4;
      const uint32_t kb = (g.b_mn ? 2048 : 32) >> 4;
      int s = 0;
      uint32_t phase = 0;
      int buf = 0;
      uint32_t buf_phase = 0;
      for (int64_t u = first; u < g.units && ok; u += stride) {
        int part = 0;
        if (g.split > 1) part = int(u % g.split);
        const int k_first = part * g.steps_part;
        const int k_last = k_first + g.steps_part < g.steps
                               ? k_first + g.steps_part
                               : g.steps;
        ok = mbar_wait(bar_acc_empty(buf), buf_phase ^ 1, p.err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(buf * BN);
        for (int k = k_first; k < k_last; ++k) {
          ok = mbar_wait(bar_full(s), phase, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = da0 + uint64_t((uint32_t(s) * C::STAGE) >> 4);
          const uint64_t db = db0 + uint64_t((uint32_t(s) * C::STAGE) >> 4);
#pragma unroll
          for (int i = 0; i < kBK / 16; ++i)
            mma_f16<CG>(d, da + i * ka, db + i * kb, idesc,
                        k > k_first || i > 0);
          commit_all<CG>(bar_empty(s));
          if (++s == C::STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        commit_all<CG>(bar_acc_full(buf));
        buf ^= 1;
        if (buf == 0) buf_phase ^= 1;
      }
    }
  } else if (warp >= kCtrlWarps) {
    // ------------------------------------------------------------ epilogue
    constexpr int kWarpCols = kTileN / 2;
    constexpr int kGroupCols = kWarpCols < 64 ? kWarpCols : 64;
    const int w = warp - kCtrlWarps;
    const int quarter = w & 3, half = w >> 2;
    uint8_t* stage = smem + C::OFF_EPI + w * (32 * kStagePitch + 512);
    float* cols = reinterpret_cast<float*>(stage + 32 * kStagePitch);
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int64_t u = first; u < g.units; u += stride) {
      const Unit t = unit_of(g, u);
      const int64_t row0 =
          int64_t(t.m * CG + int(rank)) * kBM + quarter * 32;
      const int64_t tile_col = int64_t(t.n) * kTileN + half * kWarpCols;
      ok = mbar_wait(bar_acc_full(buf), buf_phase, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = lanes + uint32_t(buf * BN + half * kWarpCols);
#pragma unroll 1
      for (int c0 = 0; c0 < kWarpCols; c0 += kGroupCols) {
        const int64_t col0 = tile_col + c0;
        const bool live = row0 < p.M && col0 < p.N;
        const bool final_part = g.split == 1;
        uint32_t pk[kGroupCols / 2];
        if (EPI != kEpiStore && final_part && live) {
          load_bias_cols<T>(cols, p.bias[0], p.bias_stride[0], col0, p.N,
                            kGroupCols, lane);
          if constexpr (kGated)
            load_bias_cols<T>(cols + 64, p.bias[1], p.bias_stride[1], col0,
                              p.N, kGroupCols, lane);
          __syncwarp();
          if (EPI == kEpiLinear && p.res)
            load_block<T, kGroupCols>(stage, pk, p, row0, col0, g.vec_res,
                                      lane);
        }
#pragma unroll
        for (int i = 0; i < kGroupCols / 32; ++i) {
          uint32_t r0[32];
          uint32_t r1[kGated ? 32 : 1];
          tmem_ld32u(acc + c0 + i * 32, r0);
          if constexpr (kGated)
            tmem_ld32u(acc + BN / 2 + c0 + i * 32, r1);
          tmem_wait_ld_tied(r0);
          if constexpr (kGated) regs_tie32(r1);
          if (c0 + (i + 1) * 32 == kWarpCols) {
            // This warp's last read of the accumulator.
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 1)
                mbar_arrive(bar_acc_empty(buf));
              else
                mbar_arrive_cluster(map_cta(bar_acc_empty(buf), 0));
            }
          }
          if (!live) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r0[j]);
          const int64_t col = col0 + i * 32;
          if (!final_part) {
            const int64_t plane = p.M * p.N;
            float* q = g.partial + int64_t(t.part) * (kGated ? 2 : 1) * plane;
            store_block_f32(stage, v, q, p.N, row0, p.M, col, p.N, g.vec_f32,
                            lane);
            if constexpr (kGated) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r1[j]);
              store_block_f32(stage, v, q + plane, p.N, row0, p.M, col, p.N,
                              g.vec_f32, lane);
            }
            continue;
          }
          if constexpr (EPI != kEpiStore) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 b =
                  *reinterpret_cast<const float4*>(cols + i * 32 + j);
              v[j] += b.x;
              v[j + 1] += b.y;
              v[j + 2] += b.z;
              v[j + 3] += b.w;
            }
          }
          if constexpr (EPI == kEpiLinear) {
            if (p.pre) {
              uint32_t zk[16];
#pragma unroll
              for (int j = 0; j < 16; ++j)
                zk[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
              store_block<T, 32>(stage, zk, static_cast<T*>(p.pre), p.pre_ld,
                                 row0, p.M, col, p.N, g.vec_pre, lane);
            }
            activate32(v, p.act);
            if (p.res) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 q = unpack2<T>(pk[i * 16 + j]);
                v[2 * j] += q.x;
                v[2 * j + 1] += q.y;
              }
            }
          }
          if constexpr (kGated) {
            float up[32];
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 b =
                  *reinterpret_cast<const float4*>(cols + 64 + i * 32 + j);
              up[j] = __uint_as_float(r1[j]) + b.x;
              up[j + 1] = __uint_as_float(r1[j + 1]) + b.y;
              up[j + 2] = __uint_as_float(r1[j + 2]) + b.z;
              up[j + 3] = __uint_as_float(r1[j + 3]) + b.w;
            }
            if (p.gate) {
              store_block_f32(stage, v, p.gate, p.gate_ld, row0, p.M, col,
                              p.N, g.vec_f32, lane);
              store_block_f32(stage, up, p.up, p.up_ld, row0, p.M, col, p.N,
                              g.vec_f32, lane);
            }
            activate32(v, p.act);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= up[j];
          }
#pragma unroll
          for (int j = 0; j < 16; ++j)
            pk[i * 16 + j] = pack2<T>(v[2 * j], v[2 * j + 1]);
        }
        if (live && final_part)
          store_block<T, kGroupCols>(stage, pk, static_cast<T*>(p.out),
                                     p.out_ld, row0, p.M, col0, p.N,
                                     g.vec_out, lane);
      }
      buf ^= 1;
      if (buf == 0) buf_phase ^= 1;
    }
  }

  // Teardown: every TMEM access is done before the allocating warp frees it,
  // and neither CTA of a pair leaves while the other may signal it.
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    dealloc_cols<CG>(tmem, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// Packing: operands the tensor maps cannot describe (odd strides, unaligned
// rows) are first copied to rows of a multiple of 16 bytes.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    pack_kernel(const uint16_t* src, int64_t s_outer, int64_t s_inner,
                uint16_t* dst, int64_t ld, int64_t outer, int64_t inner) {
  allow_dependents();
  grid_dependency_wait();
  const int64_t total = outer * inner;
  const int64_t step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += step) {
    const int64_t o = e / inner, i = e - o * inner;
    dst[o * ld + i] = src[o * s_outer + i * s_inner];
  }
}

bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// An operand as the tensor maps see it.
struct TmaOperand {
  const void* p;
  bool mn;        // rows contiguous
  int64_t ld;     // elements between lines of the other direction
};

bool describable(const MatView& m, int64_t rows, int64_t k, bool mn) {
  const int64_t inner = mn ? m.sr : m.sk, outer = mn ? m.sk : m.sr;
  const int64_t lines = mn ? k : rows;
  if (!aligned16(m.p) || (inner != 1 && (mn ? rows : k) > 1)) return false;
  return lines <= 1 || (outer > 0 && outer % 8 == 0 &&
                        outer < (int64_t(1) << 36));
}

// Which form an operand is staged in, or -1: it has to be packed.
int form_of(const MatView& m, int64_t rows, int64_t k) {
  if (describable(m, rows, k, false)) return 0;
  if (describable(m, rows, k, true)) return 1;
  return -1;
}

cudaError_t pack(const MatView& m, int64_t rows, int64_t k, bool mn,
                 Workspace& ws, TmaOperand* out, cudaStream_t stream) {
  const int64_t outer = mn ? k : rows, inner = mn ? rows : k;
  const int64_t ld = (inner + 7) / 8 * 8;
  uint16_t* dst = static_cast<uint16_t*>(ws.take(size_t(outer) * ld * 2));
  *out = {dst, mn, ld};
  if (ws.dry || ws.overflow) return cudaSuccess;
  const int64_t blocks = (outer * inner + 255) / 256;
  const int64_t most = int64_t(device_sm_count()) * 16;
  const cudaError_t e = launch_pdl(
      pack_kernel, dim3(unsigned(blocks < most ? blocks : most)), dim3(256),
      0, stream, static_cast<const uint16_t*>(m.p), mn ? m.sk : m.sr,
      mn ? m.sr : m.sk, dst, ld, outer, inner);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

template <int EPI, typename T, int BN, int CG>
cudaError_t launch_cfg(const CUtensorMap* maps, const TcArgs& g,
                       cudaStream_t stream) {
  using C = Cfg<BN, CG>;
  auto kern = gemm_tc_kernel<EPI, T, BN, CG>;
  static std::atomic<int> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return cudaErrorInvalidDevice;
  if (dev < 0 || dev >= 64 || !configured[dev].load()) {
    const cudaError_t e = cudaFuncSetAttribute(
        kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_ALLOC);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(1);
  }
  const int64_t slots = device_sm_count() / CG;
  const int64_t ctas = (g.units < slots ? g.units : slots) * CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM_ALLOC;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 1 ? 1 : 2;
  return cudaLaunchKernelEx(&cfg, kern, maps[0], maps[1], maps[2], maps[3],
                            g);
}

template <int EPI, typename T>
cudaError_t launch_shape(int bn, int cg, const CUtensorMap* maps,
                         const TcArgs& g, cudaStream_t stream) {
  if (cg == 2) return launch_cfg<EPI, T, 256, 2>(maps, g, stream);
  if (bn == 256) return launch_cfg<EPI, T, 256, 1>(maps, g, stream);
  if constexpr (EPI != kEpiGated)
    if (bn == 64) return launch_cfg<EPI, T, 64, 1>(maps, g, stream);
  return launch_cfg<EPI, T, 128, 1>(maps, g, stream);
}

template <typename T>
cudaError_t launch_epi(int epi, int bn, int cg, const CUtensorMap* maps,
                       const TcArgs& g, cudaStream_t stream) {
  if (epi == kEpiGated)
    return launch_shape<kEpiGated, T>(bn, cg, maps, g, stream);
  if (epi == kEpiLinear)
    return launch_shape<kEpiLinear, T>(bn, cg, maps, g, stream);
  return launch_shape<kEpiStore, T>(bn, cg, maps, g, stream);
}

}  // namespace

bool gemm_tc_supports(const GemmProblem& p) {
  return (p.dtype == VECTRA_BF16 || p.dtype == VECTRA_F16) && p.K > 0 &&
         p.K < (int64_t(1) << 30);
}

cudaError_t run_gemm_tc(const GemmProblem& p, const TcShape& shape,
                        Workspace& ws, cudaStream_t stream) {
  const bool gated = p.epilogue == kEpiGated;
  const int tile_n = gated ? shape.bn / 2 : shape.bn;
  if (tile_n < 64) return cudaErrorInvalidValue;
  TcArgs g{};
  g.p = p;
  g.tiles_m = int((p.M + kBM * shape.cg - 1) / (kBM * shape.cg));
  g.tiles_n = int((p.N + tile_n - 1) / tile_n);
  g.steps_seg = int((p.K + kBK - 1) / kBK);
  g.steps = g.steps_seg * p.segments;
  g.split = shape.split;
  g.steps_part = (g.steps + g.split - 1) / g.split;
  g.split = (g.steps + g.steps_part - 1) / g.steps_part;  // no empty parts
  g.units = int64_t(g.tiles_m) * g.tiles_n * g.split;

  // Both A's (and both B's) of a call are staged in one form.
  const int n_a = p.segments, n_b = gated ? 2 : p.segments;
  TmaOperand op[4];
  for (int side = 0; side < 2; ++side) {
    const MatView* v = side ? p.b : p.a;
    const int n = side ? n_b : n_a;
    const int64_t rows = side ? p.N : p.M;
    int form = form_of(v[0], rows, p.K);
    if (form < 0) form = v[0].sr == 1 && v[0].sk != 1;
    for (int i = 0; i < n; ++i) {
      if (describable(v[i], rows, p.K, form == 1)) {
        op[2 * side + i] = {v[i].p, form == 1, form ? v[i].sk : v[i].sr};
      } else {
        const cudaError_t e =
            pack(v[i], rows, p.K, form == 1, ws, &op[2 * side + i], stream);
        if (e != cudaSuccess) return e;
      }
    }
    if (n == 1) op[2 * side + 1] = op[2 * side];
    (side ? g.b_mn : g.a_mn) = uint8_t(form == 1);
  }
  if (g.split > 1)
    g.partial = static_cast<float*>(ws.take(
        size_t(g.split) * (gated ? 2 : 1) * p.M * p.N * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;

  const auto vec = [](const void* q, int64_t ld, int64_t es) {
    return uint8_t(aligned16(q) && (ld * es) % 16 == 0);
  };
  const bool n8 = p.N % 8 == 0;
  g.vec_out = n8 && vec(p.out, p.out_ld, 2);
  g.vec_pre = n8 && vec(p.pre, p.pre_ld, 2);
  g.vec_res = n8 && p.res_sn == 1 && vec(p.res, p.res_sm, 2);
  g.vec_f32 = g.split > 1 ? p.N % 4 == 0
                          : p.N % 4 == 0 && vec(p.gate, p.gate_ld, 4) &&
                                vec(p.up, p.up_ld, 4);

  CUtensorMap maps[4];
  const int b_rows = gated && shape.cg == 1 ? shape.bn / 2
                                            : shape.bn / shape.cg;
  for (int i = 0; i < 4; ++i) {
    const int64_t rows = i < 2 ? p.M : p.N;
    const TmaOperand& o = op[i];
    const int64_t inner = o.mn ? rows : p.K, outer = o.mn ? p.K : rows;
    const int box = o.mn ? kBK : (i < 2 ? kBM : b_rows);
    if (!make_line_map(&maps[i], o.p, p.dtype, inner, outer, o.ld, box))
      return cudaErrorInvalidValue;
  }
  const cudaError_t e =
      p.dtype == VECTRA_BF16
          ? launch_epi<__nv_bfloat16>(p.epilogue, shape.bn, shape.cg, maps, g,
                                      stream)
          : launch_epi<__half>(p.epilogue, shape.bn, shape.cg, maps, g,
                               stream);
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (g.split > 1) {
    const cudaError_t f = launch_split_finish(p, g.split, g.partial, stream);
    if (f == cudaSuccess) count_launches(1);
    return f;
  }
  return cudaSuccess;
}

}  // namespace vectra
