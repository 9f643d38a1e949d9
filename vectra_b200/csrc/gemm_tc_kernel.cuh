// gemm_tc_kernel.cuh: the matrix products of the transformer-block operators in
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
//  * warp 1: allocates TMEM and issues the MMAs (of the pair: its first CTA
//    only). Two accumulators in TMEM, so the next tile's product runs during
//    this one's epilogue.
//  * the other warps are the epilogue: two or four per TMEM lane quarter,
//    which share its columns. A lane holds one row;
//    results are packed and turned through shared memory so that global
//    loads (the residual) and stores run along rows.
// A gated layer's B tile is BN / 2 gate rows and the same BN / 2 up rows:
// one MMA makes both projections, and the epilogue finds both factors of an
// output in its row.
//
// float32 tensors: each operand is first split into three bf16 planes, hi +
// mid + lo, 24 bits in all, and the product is the sum of the six plane
// products that matter (lo hi, hi lo, mid mid, mid hi, hi mid, hi hi, small
// ones first), as further segments of the same reduction: 6 bf16 products
// run at 3.5 times the FP32 pipe's rate.
//
// A reduction too long for its few tiles is cut into parts that write
// float32 sums to the workspace; launch_split_finish adds them in order.
// Every wait is bounded (error word and early exit).
#pragma once

#include <atomic>

#include "block_common.cuh"
#include "gemm_tc.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

using namespace tc;

constexpr int kCtrlWarps = 2;
constexpr int kStagePitch = 80;  // epilogue turning buffer: rows of 64 B + 16
constexpr int kEpiWarpBytes = 32 * kStagePitch + 512;  // and the biases

template <int BN, int CG>
struct Cfg {
  // Epilogue warps: each TMEM lane quarter (a warp reads the quarter of its
  // index modulo 4) is shared by EPI_WARPS / 4 of them, with at least 32
  // accumulator columns each. Four per scheduler at
  // BN = 256: an epilogue with an activation is bound by instruction
  // latency (two per scheduler issued on 39 % of cycles and took 109 us for
  // 66,560 x 256 x 1,024 with GELU).
  static constexpr int EPI_WARPS = BN == 256 ? 16 : 8;
  static constexpr int THREADS = (kCtrlWarps + EPI_WARPS) * 32;
  static constexpr int B_ROWS = BN / CG;  // rows of B staged per CTA
  static constexpr int A_BYTES = kTcRows * kTcStep * 2;
  static constexpr int B_BYTES = B_ROWS * kTcStep * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int EPI_BYTES = EPI_WARPS * kEpiWarpBytes;
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

// float32: where the accumulation that starts at step `from` ends. The tensor
// cores add into the accumulator rounding toward zero, so a long sum drifts
// (by -2e-8 of itself for every 16 products: 1.4e-5 after 4,096 positive
// ones). The five small plane products are too small for that to matter, but
// of the last, hi hi, every 512 of the reduction is accumulated apart and
// added by the epilogue, which rounds to nearest.
constexpr int kChunkSteps = 8;
__device__ __forceinline__ int chunk_end(const TcArgs& g, int from,
                                         int last) {
  const int small = g.steps / 6 * 5;  // steps before hi hi
  const int at = from < small ? 0 : (from - small) / kChunkSteps;
  const int end = small + (at + 1) * kChunkSteps;
  return end < last ? end : last;
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
// Relaxed: what it announces are tensor-memory reads that tcgen05.wait::ld
// has completed. A release at cluster scope would also wait for the warp's
// global stores of the tile before.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];"
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
// Activations of a lane's values, in pairs.
//
// The smooth ones are z * sigmoid(g(z)): silu g = z, gelu_tanh g = 2 c (z +
// 0.044715 z^3), and gelu g = logit(Phi(z)) = z Q(z^2) with a polynomial Q
// fitted on |z| <= 5 for the least error of the result (7e-8; beyond, its
// leading term keeps driving the sigmoid to 0 or 1). With x = -g log2(e),
// sigmoid = 1 / (1 + 2^x); two of them share one reciprocal, 1/a = b / (ab),
// so a value costs 1.5 MUFU operations instead of 2. z is capped from below
// (NaN kept) where x reaches 63, so that ab stays finite; the result there
// is within 3e-10 of the activation, and -infinity gives that, not NaN.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// -log2(e) logit(Phi(z)) / z as a polynomial in t = z^2.
__device__ __forceinline__ float gelu_q(float t) {
  float q = fmaf(-5.2620424e-09f, t, 3.8715868e-07f);
  q = fmaf(q, t, -1.1483583e-05f);
  q = fmaf(q, t, 1.5959822e-04f);
  q = fmaf(q, t, 9.4943171e-05f);
  q = fmaf(q, t, -1.0483774e-01f);
  return fmaf(q, t, -2.3022075f);
}

template <int ACT>
__device__ __forceinline__ void activate2(float& z0, float& z1) {
  if constexpr (ACT == VECTRA_ACT_RELU) {
    z0 = max_nan(z0, 0.f);
    z1 = max_nan(z1, 0.f);
  } else if constexpr (ACT != VECTRA_ACT_NONE) {
    // Below kLow, x would pass 63.
    constexpr float kLow = ACT == VECTRA_ACT_SILU        ? -43.6f
                           : ACT == VECTRA_ACT_GELU_TANH ? -7.6f
                                                         : -6.5f;
    z0 = max_nan(z0, kLow);
    z1 = max_nan(z1, kLow);
    float x0, x1;
    if constexpr (ACT == VECTRA_ACT_SILU) {
      x0 = -kLog2e * z0;
      x1 = -kLog2e * z1;
    } else {
      const float t0 = z0 * z0, t1 = z1 * z1;
      if constexpr (ACT == VECTRA_ACT_GELU_TANH) {
        constexpr float k0 = -2.f * kGeluTanhC * kLog2e;
        x0 = fmaf(k0 * kGeluTanhA, t0, k0) * z0;
        x1 = fmaf(k0 * kGeluTanhA, t1, k0) * z1;
      } else {
        x0 = gelu_q(t0) * z0;
        x1 = gelu_q(t1) * z1;
      }
    }
    const float a = 1.f + fast_exp2(x0), b = 1.f + fast_exp2(x1);
    const float r = fast_rcp(a * b);
    z0 *= b * r;
    z1 *= a * r;
  }
}

// Keeps the compiler from interleaving more than eight values at a time: 32
// at once want more registers than four warps per scheduler leave (96), and
// spilled.
__device__ __forceinline__ void tie8(float* v) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]),
                 "+f"(v[5]), "+f"(v[6]), "+f"(v[7]));
}

template <int ACT, int N>
__device__ __forceinline__ void activate(float* v) {
  if constexpr (ACT != VECTRA_ACT_NONE) {
#pragma unroll
    for (int j = 0; j < N; j += 8) {
      tie8(v + j);
#pragma unroll
      for (int i = 0; i < 8; i += 2) activate2<ACT>(v[j + i], v[j + i + 1]);
      tie8(v + j);
    }
  }
}

// ---------------------------------------------------------------------------
// Epilogue pieces. `stage` is the warp's 32 x kStagePitch turning buffer.
// ---------------------------------------------------------------------------
// Where a warp's 32-row block lies: rows left in the matrix (0 .. 32) and
// the pointer walk of the coalesced passes.
struct RowBlock {
  int64_t row0;
  int rows;
};

// Writes the warp's 32 x 32 block (row = lane, packed 16-bit pairs) to rows
// row0.., columns col.. through the turning buffer: four lanes per row of
// 64 bytes.
template <typename T>
__device__ __forceinline__ void store_block(uint8_t* stage, const uint32_t* pk,
                                            T* out, int64_t ld,
                                            const RowBlock& rb, int64_t col,
                                            int64_t cols, bool vec,
                                            int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(stage + lane * kStagePitch + c * 16) =
        make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
  __syncwarp();
  if (vec) {
    const int r = lane / 4, c = (lane % 4) * 8;
    if (col + c < cols) {
      T* q = out + (rb.row0 + r) * ld + col + c;
      const uint8_t* s = stage + r * kStagePitch + c * 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r + 8 * i < rb.rows)
          *reinterpret_cast<uint4*>(q) =
              *reinterpret_cast<const uint4*>(s + i * 8 * kStagePitch);
        q += 8 * ld;
      }
    }
  } else if (col + lane < cols) {
    T* q = out + rb.row0 * ld + col + lane;
    for (int r = 0; r < rb.rows; ++r, q += ld)
      *q = reinterpret_cast<const T*>(stage + r * kStagePitch)[lane];
  }
  __syncwarp();
}

// The same for 16 columns of float32.
__device__ __forceinline__ void store_half_f32(uint8_t* stage, const float* v,
                                               float* out, int64_t ld,
                                               const RowBlock& rb,
                                               int64_t col, int64_t cols,
                                               bool vec, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<float4*>(stage + lane * kStagePitch + c * 16) =
        make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  __syncwarp();
  if (vec) {
    const int r = lane / 4, c = (lane % 4) * 4;
    if (col + c < cols) {
      float* q = out + (rb.row0 + r) * ld + col + c;
      const uint8_t* s = stage + r * kStagePitch + c * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r + 8 * i < rb.rows)
          *reinterpret_cast<float4*>(q) =
              *reinterpret_cast<const float4*>(s + i * 8 * kStagePitch);
        q += 8 * ld;
      }
    }
  } else if (col + lane % 16 < cols) {
    float* q = out + (rb.row0 + lane / 16) * ld + col + lane % 16;
    for (int r = lane / 16; r < rb.rows; r += 2, q += 2 * ld)
      *q =
          reinterpret_cast<const float*>(stage + r * kStagePitch)[lane % 16];
  }
  __syncwarp();
}
__device__ __forceinline__ void store_block_f32(uint8_t* stage, const float* v,
                                                float* out, int64_t ld,
                                                const RowBlock& rb,
                                                int64_t col, int64_t cols,
                                                bool vec, int lane) {
  store_half_f32(stage, v, out, ld, rb, col, cols, vec, lane);
  store_half_f32(stage, v + 16, out, ld, rb, col + 16, cols, vec, lane);
}

// The residual's 32 x 32 block: asynchronous copies into the turning buffer
// (coalesced, in flight while the accumulator is waited for and read), from
// which a lane then takes its row.
template <typename T>
__device__ __forceinline__ void fetch_residual(uint8_t* stage,
                                               const GemmProblem& p,
                                               const RowBlock& rb,
                                               int64_t col, int lane) {
  const int r = lane / 4, c = (lane % 4) * 8;
  const T* q = static_cast<const T*>(p.res) + (rb.row0 + r) * p.res_sm + col +
               c;
  const uint32_t dst = smem_addr(stage) + r * kStagePitch + c * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r + 8 * i < rb.rows && col + c < p.N)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(
                       dst + i * 8 * kStagePitch),
                   "l"(q)
                   : "memory");
    q += 8 * p.res_sm;
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(w << 16),
                       __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <typename T>
__device__ __forceinline__ void add_residual(uint8_t* stage, float* v,
                                             bool vec, const GemmProblem& p,
                                             const RowBlock& rb, int64_t col,
                                             int lane) {
  if (vec) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    const T* q = static_cast<const T*>(p.res) + rb.row0 * p.res_sm +
                 (col + lane) * p.res_sn;
    for (int r = 0; r < rb.rows; ++r, q += p.res_sm)
      if (col + lane < p.N)
        reinterpret_cast<T*>(stage + r * kStagePitch)[lane] = *q;
  }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 q = *reinterpret_cast<const uint4*>(
        stage + lane * kStagePitch + c * 16);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[c * 8 + 2 * i] += f.x;
      v[c * 8 + 2 * i + 1] += f.y;
    }
  }
  __syncwarp();
}

// Adds a float32 residual, 16 columns at a time.
__device__ __forceinline__ void add_residual_f32(uint8_t* stage, float* v,
                                                 bool vec,
                                                 const GemmProblem& p,
                                                 const RowBlock& rb,
                                                 int64_t col0, int lane) {
  const float* res = static_cast<const float*>(p.res);
#pragma unroll
  for (int h = 0; h < 32; h += 16) {
    const int64_t col = col0 + h;
    if (vec) {
      const int r = lane / 4, c = (lane % 4) * 4;
      const float* q = res + (rb.row0 + r) * p.res_sm + col + c;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r + 8 * i < rb.rows && col + c < p.N)
          *reinterpret_cast<float4*>(stage + (r + 8 * i) * kStagePitch +
                                     c * 4) =
              __ldg(reinterpret_cast<const float4*>(q));
        q += 8 * p.res_sm;
      }
    } else if (col + lane % 16 < p.N) {
      for (int r = lane / 16; r < rb.rows; r += 2)
        reinterpret_cast<float*>(stage + r * kStagePitch)[lane % 16] =
            res[(rb.row0 + r) * p.res_sm + (col + lane % 16) * p.res_sn];
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 q = *reinterpret_cast<const float4*>(
          stage + lane * kStagePitch + c * 16);
      v[h + 4 * c] += q.x;
      v[h + 4 * c + 1] += q.y;
      v[h + 4 * c + 2] += q.z;
      v[h + 4 * c + 3] += q.w;
    }
    __syncwarp();
  }
}

// A block of 32 x 32 results (or saved values) in T.
template <typename T>
__device__ __forceinline__ void store_values(uint8_t* stage, const float* v,
                                             T* out, int64_t ld,
                                             const RowBlock& rb, int64_t col,
                                             int64_t cols, bool vec,
                                             int lane) {
  if constexpr (std::is_same<T, float>::value) {
    store_block_f32(stage, v, out, ld, rb, col, cols, vec, lane);
  } else {
    uint32_t pk[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) pk[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
    store_block<T>(stage, pk, out, ld, rb, col, cols, vec, lane);
  }
}

// Biases of a warp's columns, as floats in its shared memory; zeros without
// a bias, so that the columns' loop needs no branch.
template <typename T>
__device__ __forceinline__ void load_bias(float* dst, const void* bias,
                                          int64_t stride, int64_t col,
                                          int64_t cols, int n, int lane) {
  for (int c = lane; c < n; c += 32)
    dst[c] = bias && col + c < cols
                 ? to_f32(static_cast<const T*>(bias)[(col + c) * stride])
                 : 0.f;
}
template <int N>
__device__ __forceinline__ void add_bias(float* v, const float* cols) {
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 b = *reinterpret_cast<const float4*>(cols + j);
    v[j] += b.x;
    v[j + 1] += b.y;
    v[j + 2] += b.z;
    v[j + 3] += b.w;
  }
}

// One tile of one epilogue warp: `cols` its bias values in shared memory (a
// gated layer's up biases 64 behind). `wait` waits for the next accumulator
// and gives the TMEM address of the warp's rows and first column, `release`
// gives it back after the last read. What a call does not need is compiled out: with
// the residual, the saved values and the partial sums behind run-time
// branches the values were copied between registers at every join, 10
// instructions for each result where the bare store takes 6.
template <int EPI, int ACT, bool RES, bool PRE, typename T, int TILE_N,
          int WARP_COLS, typename Wait, typename Release>
__device__ __forceinline__ void epilogue_tile(const TcArgs& g, uint8_t* stage,
                                              float* cols, int chunks,
                                              const RowBlock& rb,
                                              int64_t tile_col, int part,
                                              int lane, Wait&& wait,
                                              Release&& release) {
  constexpr bool kGated = EPI == kEpiGated || EPI == kEpiGatedPartial;
  constexpr bool kPartial = EPI == kEpiPartial || EPI == kEpiGatedPartial;
  static_assert(WARP_COLS % 32 == 0 && WARP_COLS <= 64, "columns");
  const GemmProblem& p = g.p;
  if constexpr (EPI == kEpiLinear || EPI == kEpiGated) {
    load_bias<T>(cols, p.bias[0], p.bias_stride[0], tile_col, p.N, WARP_COLS,
                 lane);
    if constexpr (kGated)
      load_bias<T>(cols + 64, p.bias[1], p.bias_stride[1], tile_col, p.N,
                   WARP_COLS, lane);
    __syncwarp();
  }
  // With saved values in the same buffer the residual comes after them.
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr bool kEarly = RES && !PRE && !kF32;
  if constexpr (kEarly)
    if (g.vec_res) fetch_residual<T>(stage, p, rb, tile_col, lane);
  // 32 columns: `v` their sums, `up` a gated layer's second ones.
  auto finish = [&](float* v, float* up, int c0) {
    const int64_t col = tile_col + c0;
    if constexpr (kPartial) {
      const int64_t plane = p.M * p.N;
      float* q = g.partial + int64_t(part) * (kGated ? 2 : 1) * plane;
      store_block_f32(stage, v, q, p.N, rb, col, p.N, g.vec_f32, lane);
      if constexpr (kGated)
        store_block_f32(stage, up, q + plane, p.N, rb, col, p.N, g.vec_f32,
                        lane);
    } else {
      if constexpr (EPI == kEpiLinear) {
        add_bias<32>(v, cols + c0);
        if constexpr (PRE) {
          store_values<T>(stage, v, static_cast<T*>(p.pre), p.pre_ld, rb,
                          col, p.N, g.vec_pre, lane);
          if constexpr (RES && !kF32)
            if (g.vec_res) fetch_residual<T>(stage, p, rb, col, lane);
        }
        activate<ACT, 32>(v);
        if constexpr (RES && kF32)
          add_residual_f32(stage, v, g.vec_res, p, rb, col, lane);
        else if constexpr (RES)
          add_residual<T>(stage, v, g.vec_res, p, rb, col, lane);
      }
      if constexpr (EPI == kEpiGated) {
        add_bias<32>(v, cols + c0);
        add_bias<32>(up, cols + 64 + c0);
        if constexpr (PRE) {
          store_block_f32(stage, v, p.gate, p.gate_ld, rb, col, p.N,
                          g.vec_f32, lane);
          store_block_f32(stage, up, p.up, p.up_ld, rb, col, p.N, g.vec_f32,
                          lane);
        }
        activate<ACT, 32>(v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= up[j];
      }
      store_values<T>(stage, v, static_cast<T*>(p.out), p.out_ld, rb, col,
                      p.N, g.vec_out, lane);
    }
  };
  if constexpr (kF32) {
    // The chunks of the reduction are added here, rounding to nearest (see
    // chunk_end).
    constexpr int kSums = kGated ? 2 * WARP_COLS : WARP_COLS;
    float sum[kSums];
    for (int chunk = 0; chunk < chunks; ++chunk) {
      uint32_t acc = 0;
      if (!wait(&acc)) return;
#pragma unroll
      for (int c = 0; c < kSums; c += 16) {
        uint32_t r[16];
        tmem_ld16u(acc + (c < WARP_COLS ? c : TILE_N + c - WARP_COLS), r);
        tmem_wait_ld();
        regs_tie16(r);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sum[c + j] = chunk == 0 ? __uint_as_float(r[j])
                                  : sum[c + j] + __uint_as_float(r[j]);
      }
      release();
    }
#pragma unroll
    for (int c0 = 0; c0 < WARP_COLS; c0 += 32)
      if (rb.rows > 0 && tile_col + c0 < p.N)
        finish(sum + c0, sum + (kGated ? WARP_COLS + c0 : 0), c0);
  } else if constexpr (EPI == kEpiGated) {
    // Both factors of 16 columns at a time: 32 of each would not fit the 96
    // registers beside the packed results.
    uint32_t acc = 0;
    if (!wait(&acc)) return;
#pragma unroll 1
    for (int c0 = 0; c0 < WARP_COLS; c0 += 32) {
      const int64_t col = tile_col + c0;
      const bool live = rb.rows > 0 && col < p.N;
      uint32_t pk[16];
#pragma unroll
      for (int h = 0; h < 32; h += 16) {
        uint32_t r0[16], r1[16];
        tmem_ld16u(acc + c0 + h, r0);
        tmem_ld16u(acc + TILE_N + c0 + h, r1);
        tmem_wait_ld();
        regs_tie16(r0);
        regs_tie16(r1);
        if (c0 + h + 16 == WARP_COLS) release();
        float v[16], up[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[j] = __uint_as_float(r0[j]);
          up[j] = __uint_as_float(r1[j]);
        }
        add_bias<16>(v, cols + c0 + h);
        add_bias<16>(up, cols + 64 + c0 + h);
        if constexpr (PRE) {
          if (live) {
            store_half_f32(stage, v, p.gate, p.gate_ld, rb, col + h, p.N,
                           g.vec_f32, lane);
            store_half_f32(stage, up, p.up, p.up_ld, rb, col + h, p.N,
                           g.vec_f32, lane);
          }
        }
        activate<ACT, 16>(v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          pk[h / 2 + j] = pack2<T>(v[2 * j] * up[2 * j],
                                   v[2 * j + 1] * up[2 * j + 1]);
      }
      if (live)
        store_block<T>(stage, pk, static_cast<T*>(p.out), p.out_ld, rb, col,
                       p.N, g.vec_out, lane);
    }
  } else {
    uint32_t acc = 0;
    if (!wait(&acc)) return;
#pragma unroll 1
    for (int c0 = 0; c0 < WARP_COLS; c0 += 32) {
      if constexpr (kEarly)
        if (g.vec_res && c0 > 0)
          fetch_residual<T>(stage, p, rb, tile_col + c0, lane);
      uint32_t r0[32];
      uint32_t r1[kGated ? 32 : 1];
      tmem_ld32u(acc + c0, r0);
      if constexpr (kGated) tmem_ld32u(acc + TILE_N + c0, r1);
      tmem_wait_ld_tied(r0);
      if constexpr (kGated) regs_tie32(r1);
      if (c0 + 32 == WARP_COLS) release();
      if (rb.rows <= 0 || tile_col + c0 >= p.N) continue;
      float v[32], up[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r0[j]);
      if constexpr (kGated) {
#pragma unroll
        for (int j = 0; j < 32; ++j) up[j] = __uint_as_float(r1[j]);
      }
      finish(v, up, c0);
    }
  }
}

template <int EPI, bool RES, bool PRE, typename T, int BN, int CG>
__global__ void __launch_bounds__(Cfg<BN, CG>::THREADS, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap ta0,
                   const __grid_constant__ CUtensorMap ta1,
                   const __grid_constant__ CUtensorMap tb0,
                   const __grid_constant__ CUtensorMap tb1,
                   const __grid_constant__ TcArgs g) {
  using C = Cfg<BN, CG>;
  constexpr bool kGated = EPI == kEpiGated || EPI == kEpiGatedPartial;
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int kTileN = kGated ? BN / 2 : BN;  // output columns of a tile
  // Operand format: bf16 (also float32's planes) or f16.
  constexpr int FMT = std::is_same<T, __half>::value ? 0 : 1;
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
      mbar_init(bar_acc_empty(b), C::EPI_WARPS * CG);
    }
    fence_barrier_init();
  }
  if (warp == 1) alloc_cols<CG>(smem_addr(tmem_slot), C::TMEM_COLS);
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
        const int m0 = (t.m * CG + int(rank)) * kTcRows;
        const int n0 = t.n * kTileN;
        const int k_first = t.part * g.steps_part;
        const int k_last = k_first + g.steps_part < g.steps
                               ? k_first + g.steps_part
                               : g.steps;
        int seg_at = k_first / g.steps_seg;
        int in_seg = k_first - seg_at * g.steps_seg;
        TcSegment seg = g.seg[seg_at];
        for (int k = k_first; k < k_last; ++k) {
          ok = mbar_wait(bar_empty(s), phase ^ 1, p.err);
          if (!ok) break;
          uint32_t full = bar_full(s);
          if (CG == 1 || rank == 0)
            mbar_arrive_expect_tx(full, C::STAGE * CG);
          if constexpr (CG == 2) full = map_cta(full, 0);
          if (in_seg == g.steps_seg) {
            in_seg = 0;
            seg = g.seg[++seg_at];
          }
          const int k0 = in_seg++ * kTcStep;
          const uint32_t sa = sbase + uint32_t(s) * C::STAGE;
          const uint32_t sb = sa + C::A_BYTES;
          const CUtensorMap* ma = seg.map ? &ta1 : &ta0;
          if (g.a_mn) {
#pragma unroll
            for (int i = 0; i < kTcRows / 64; ++i)
              tma_load_2d<CG>(sa + i * 8192, ma, full, m0 + i * 64,
                              k0 + seg.a_line);
          } else {
            tma_load_2d<CG>(sa, ma, full, k0, m0 + seg.a_line);
          }
          // Rows of B: in a pair, half each. A gated tile's first half is
          // the gate weight's rows, its second half the up weight's.
          constexpr int kBoxRows = kGated && CG == 1 ? BN / 2 : C::B_ROWS;
#pragma unroll
          for (int h = 0; h < C::B_ROWS / kBoxRows; ++h) {
            const CUtensorMap* mb =
                (kGated ? (CG == 2 ? int(rank) : h) : seg.map) ? &tb1 : &tb0;
            const int row =
                kGated ? n0 : n0 + int(rank) * C::B_ROWS;
            const uint32_t dst = sb + h * kBoxRows * 128;
            if (g.b_mn) {
#pragma unroll
              for (int i = 0; i < kBoxRows / 64; ++i)
                tma_load_2d<CG>(dst + i * 8192, mb, full, row + i * 64,
                                k0 + seg.b_line);
            } else {
              tma_load_2d<CG>(dst, mb, full, k0, row + seg.b_line);
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
      const uint32_t idesc = f16_idesc(FMT, kTcRows * CG, BN, g.b_mn) |
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
        for (int from = k_first; from < k_last && ok;) {
        const int to = kF32 ? chunk_end(g, from, k_last) : k_last;
        ok = mbar_wait(bar_acc_empty(buf), buf_phase ^ 1, p.err);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(buf * BN);
        for (int k = from; k < to; ++k) {
          ok = mbar_wait(bar_full(s), phase, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = da0 + uint64_t((uint32_t(s) * C::STAGE) >> 4);
          const uint64_t db = db0 + uint64_t((uint32_t(s) * C::STAGE) >> 4);
#pragma unroll
          for (int i = 0; i < kTcStep / 16; ++i)
            mma_f16<CG>(d, da + i * ka, db + i * kb, idesc,
                        k > from || i > 0);
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
        from = to;
        }
      }
    }
  } else if (warp >= kCtrlWarps) {
    // ------------------------------------------------------------ epilogue
    const int w = warp - kCtrlWarps;
    constexpr int kWarpCols = kTileN / (C::EPI_WARPS / 4);
    const int quarter = warp & 3, share = w >> 2;
    uint8_t* stage = smem + C::OFF_EPI + w * kEpiWarpBytes;
    float* cols = reinterpret_cast<float*>(stage + 32 * kStagePitch);
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    // One copy of the whole loop per activation: with the choice inside it,
    // the copies' registers met again after every tile and spilled.
    auto role = [&](auto act) {
      int buf = 0;
      uint32_t buf_phase = 0;
      for (int64_t u = first; u < g.units && ok; u += stride) {
        const Unit t = unit_of(g, u);
        RowBlock rb;
        rb.row0 = int64_t(t.m * CG + int(rank)) * kTcRows + quarter * 32;
        const int64_t left = p.M - rb.row0;
        rb.rows = int(left < 0 ? 0 : (left < 32 ? left : 32));
        const int64_t tile_col = int64_t(t.n) * kTileN + share * kWarpCols;
        int chunks = 1;
        if constexpr (kF32) {
          const int k_first = t.part * g.steps_part;
          const int k_last = k_first + g.steps_part < g.steps
                                 ? k_first + g.steps_part
                                 : g.steps;
          chunks = 0;
          for (int k = k_first; k < k_last; k = chunk_end(g, k, k_last))
            ++chunks;
        }
        auto wait = [&](uint32_t* acc) {
          ok = mbar_wait(bar_acc_full(buf), buf_phase, p.err);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) tc_fence_after();
          *acc = lanes + uint32_t(buf * BN + share * kWarpCols);
          return ok;
        };
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 1)
              mbar_arrive(bar_acc_empty(buf));
            else
              mbar_arrive_cluster(map_cta(bar_acc_empty(buf), 0));
          }
          buf ^= 1;
          if (buf == 0) buf_phase ^= 1;
        };
        epilogue_tile<EPI, decltype(act)::value, RES, PRE, T, kTileN,
                      kWarpCols>(g, stage, cols, chunks, rb, tile_col,
                                 t.part, lane, wait, release);
      }
    };
    if constexpr (EPI != kEpiLinear && EPI != kEpiGated) {
      role(std::integral_constant<int, VECTRA_ACT_NONE>{});
    } else {
      switch (p.act) {
        case VECTRA_ACT_RELU:
          role(std::integral_constant<int, VECTRA_ACT_RELU>{});
          break;
        case VECTRA_ACT_GELU:
          role(std::integral_constant<int, VECTRA_ACT_GELU>{});
          break;
        case VECTRA_ACT_GELU_TANH:
          role(std::integral_constant<int, VECTRA_ACT_GELU_TANH>{});
          break;
        case VECTRA_ACT_SILU:
          role(std::integral_constant<int, VECTRA_ACT_SILU>{});
          break;
        default:
          role(std::integral_constant<int, VECTRA_ACT_NONE>{});
          break;
      }
    }
  }

  // Teardown: every TMEM access is done before the allocating warp frees it,
  // and neither CTA of a pair leaves while the other may signal it.
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    dealloc_cols<CG>(tmem, C::TMEM_COLS);
  }
}

template <int EPI, bool RES, bool PRE, typename T, int BN, int CG>
cudaError_t launch_cfg(const CUtensorMap* maps, const TcArgs& g,
                       cudaStream_t stream) {
  using C = Cfg<BN, CG>;
  auto kern = gemm_tc_kernel<EPI, RES, PRE, T, BN, CG>;
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
  cfg.blockDim = dim3(C::THREADS);
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

template <int EPI, bool RES, bool PRE, typename T>
cudaError_t launch_shape(int bn, int cg, const CUtensorMap* maps,
                         const TcArgs& g, cudaStream_t stream) {
  // float32 keeps its sums in registers across chunks: the pair's tile, with
  // 96 registers a thread, has no room for them.
  if constexpr (!std::is_same<T, float>::value)
    if (cg == 2)
      return launch_cfg<EPI, RES, PRE, T, 256, 2>(maps, g, stream);
  if constexpr (EPI != kEpiGated && EPI != kEpiGatedPartial)
    if (bn == 64) return launch_cfg<EPI, RES, PRE, T, 64, 1>(maps, g, stream);
  return launch_cfg<EPI, RES, PRE, T, 128, 1>(maps, g, stream);
}

}  // namespace

// Products with an activation, bias or residual.
template <typename T>
cudaError_t launch_tc_linear(int bn, int cg, const CUtensorMap* maps,
                             const TcArgs& g, cudaStream_t stream) {
  if (g.p.res)
    return g.p.pre ? launch_shape<kEpiLinear, true, true, T>(bn, cg, maps, g,
                                                             stream)
                   : launch_shape<kEpiLinear, true, false, T>(bn, cg, maps, g,
                                                              stream);
  return g.p.pre ? launch_shape<kEpiLinear, false, true, T>(bn, cg, maps, g,
                                                            stream)
                 : launch_shape<kEpiLinear, false, false, T>(bn, cg, maps, g,
                                                             stream);
}

// The others: gated layers, bare products, partial sums.
template <typename T>
cudaError_t launch_tc_other(int epilogue, int bn, int cg,
                            const CUtensorMap* maps, const TcArgs& g,
                            cudaStream_t stream) {
  switch (epilogue) {
    case kEpiGated:
      return g.p.gate ? launch_shape<kEpiGated, false, true, T>(bn, cg, maps,
                                                                g, stream)
                      : launch_shape<kEpiGated, false, false, T>(bn, cg, maps,
                                                                 g, stream);
    case kEpiPartial:
      return launch_shape<kEpiPartial, false, false, T>(bn, cg, maps, g,
                                                        stream);
    case kEpiGatedPartial:
      return launch_shape<kEpiGatedPartial, false, false, T>(bn, cg, maps, g,
                                                             stream);
    default:
      return launch_shape<kEpiStore, false, false, T>(bn, cg, maps, g,
                                                      stream);
  }
}

}  // namespace vectra
