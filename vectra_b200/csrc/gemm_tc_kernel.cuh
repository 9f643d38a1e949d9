// gemm_tc_kernel.cuh: the matrix products of the transformer-block operators
// on the 5th-generation tensor cores (tcgen05 + TMEM).
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
//    which share its columns. A lane holds one row; results are packed and
//    turned through shared memory, from where the copy engine stores them.
// A gated layer's B tile is BN / 2 gate rows and the same BN / 2 up rows:
// one MMA makes both projections, and the epilogue finds both factors of an
// output in its row.
//
// float32 tensors: each operand is first split into three bf16 planes, hi +
// mid + lo, 24 bits in all; a stage brings in all planes of both, and the
// product is the sum of the six plane products that matter (lo hi, hi lo,
// mid mid, mid hi, hi mid, hi hi): 6 bf16 products run at 3.5 times the FP32
// pipe's rate. (What that costs beside the product: splitting x and a small
// weight is 12 of the 52 us of 65,536 x 128 -> 256.)
//
// A reduction too long for its few tiles is cut into parts that write
// float32 sums to the workspace; launch_split_finish adds them in order.
// Every wait is bounded (error word and early exit).
//
// Measured (B200): 8,191 x 4096 -> 4096 f16 with a whole epilogue 187-212 us
// for a few calls at a time, the tensor pipe 91 % busy, and 232-245 us call
// after call, where the power limit lowers the clock: 1.12-1.47 PFLOP/s, 0.68
// to 0.89 of the library's burst rate. Gated 8,192 x 4096 -> 10240 840 us,
// 1.64 PFLOP/s. With a reduction of 256 the results bound it: 66,560 x 256 ->
// 1024 bare 39 us (3.5 TB/s of writes, a fill's rate), with bias and GELU 62.
#pragma once

#include <atomic>

#include "block_common.cuh"
#include "gemm_tc.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

using namespace tc;

constexpr int kCtrlWarps = 2;
// A warp's turning buffer, 32 rows of 64 bytes in the 64-byte-swizzled order
// of the tensor maps' stores, and its biases.
constexpr int kTurnBytes = 2048;
constexpr int kBiasBytes = 512;

template <int BN, int CG, bool F32>
struct Cfg {
  // Epilogue warps: each TMEM lane quarter (a warp reads the quarter of its
  // index modulo 4) is shared by EPI_WARPS / 4 of them, with at least 32
  // accumulator columns each. Four per scheduler at BN = 256: an epilogue
  // with an activation is bound by instruction latency (66,560 x 256 -> 1024
  // with GELU took 109 us with two, which issued on 39 % of cycles, and 95
  // with four).
  static constexpr int EPI_WARPS = BN == 256 ? 16 : 8;
  static constexpr int THREADS = (kCtrlWarps + EPI_WARPS) * 32;
  static constexpr int B_ROWS = BN / CG;  // rows of B staged per CTA
  static constexpr int A_BYTES = kTcRows * kTcStep * 2;
  static constexpr int B_BYTES = B_ROWS * kTcStep * 2;
  static constexpr int PLANES = F32 ? 3 : 1;
  static constexpr int PLANE = A_BYTES + B_BYTES;  // one plane's A, then B
  static constexpr int STAGE = PLANES * PLANE;
  static constexpr int ACC_COLS = F32 ? 2 * BN : BN;  // see multiply_planes
  static constexpr int EPI_BYTES = EPI_WARPS * (kTurnBytes + kBiasBytes);
  static constexpr int MAX_BYTES = 227 * 1024 - 2048 - EPI_BYTES;
  static constexpr int STAGES = MAX_BYTES / STAGE < 8 ? MAX_BYTES / STAGE : 8;
  static constexpr int OFF_EPI = STAGES * STAGE;
  static constexpr int OFF_BAR = OFF_EPI + EPI_BYTES;
  static constexpr int NBAR = 2 * STAGES + 4;
  static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16;
  static constexpr int SMEM_ALLOC = SMEM + 1024;  // 1024-byte alignment
  static constexpr int TMEM_COLS = 2 * ACC_COLS;  // two accumulators
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
// ones). Every 512 of the reduction is accumulated apart and added by the
// epilogue, which rounds to nearest.
constexpr int kChunkSteps = 8;
__device__ __forceinline__ int chunk_end(int from, int last) {
  return from + kChunkSteps < last ? from + kChunkSteps : last;
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
// sigmoid = 1 / (1 + 2^x). Each value has a reciprocal of its own: one for
// two, 1/a = b / (ab), would carry a NaN into the neighbouring column. Far
// out, 2^x is 0 or infinity and the sigmoid 1 or 0; an infinite z gives what
// the definition gives in floating point, infinity or (-infinity times 0)
// NaN, here as in every other kernel of the operators.
// Packed multiplications and additions halve the instructions.
// float32 results take the same forms of silu and gelu_tanh, whose error is
// relative and below that of the product before them. gelu's is absolute and
// would lose a float32 result's tail (4 % of gelu(-5)): normal_cdf2. In 16
// bits, results below 2e-5 carry that error beyond their own rounding.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float c) { return f2pk(c, c); }

// -log2(e) logit(Phi(z)) / z as a polynomial in t = z^2, of two values.
__device__ __forceinline__ uint64_t gelu_q(uint64_t t) {
  uint64_t q = ffma2(both(-5.2620424e-09f), t, both(3.8715868e-07f));
  q = ffma2(q, t, both(-1.1483583e-05f));
  q = ffma2(q, t, both(1.5959822e-04f));
  q = ffma2(q, t, both(9.4943171e-05f));
  q = ffma2(q, t, both(-1.0483774e-01f));
  return ffma2(q, t, both(-2.3022075f));
}

// Phi of two values, to 5e-7 of itself for z < 0 and to 3e-7 for z > 0, beside
// the exponential's argument (z^2 2^-24): with a = |z|, Phi(-a) =
// exp(-a^2 / 2) F(a), where (a + k) F(a) is smooth up to its limit at infinity
// and a polynomial of degree 9 in (a - k) / (a + k), fitted for the
// least relative error on 0 <= a <= 14.5 (2e-8). Measured: 65,536 x 128 -> 256
// takes 52 us with it, 47 with the fit of the 16-bit results, 82 with erfcf.
__device__ __forceinline__ void normal_cdf2(float z0, float z1, float& p0,
                                            float& p1) {
  constexpr float k = 2.75f;
  const uint64_t z = f2pk(z0, z1);
  const uint64_t w = f2pk(fast_rcp(fabsf(z0) + k), fast_rcp(fabsf(z1) + k));
  const uint64_t x = ffma2(w, both(-2.f * k), both(1.f));
  uint64_t q = ffma2(both(-7.0936112e-05f), x, both(-4.0973665e-04f));
  q = ffma2(q, x, both(-2.4665534e-04f));
  q = ffma2(q, x, both(2.4838729e-03f));
  q = ffma2(q, x, both(3.1877409e-03f));
  q = ffma2(q, x, both(-1.6440826e-02f));
  q = ffma2(q, x, both(-1.6562568e-02f));
  q = ffma2(q, x, both(1.8233395e-01f));
  q = ffma2(q, x, both(-4.7435427e-01f));
  q = ffma2(q, x, both(7.1898603e-01f));
  const float2 t = f2upk(fmul2(fmul2(z, z), both(-0.5f * kLog2e)));
  const float2 half = f2upk(
      fmul2(fmul2(q, w), f2pk(fast_exp2(t.x), fast_exp2(t.y))));
  p0 = z0 < 0.f ? half.x : 1.f - half.x;
  p1 = z1 < 0.f ? half.y : 1.f - half.y;
}

// The sigmoids s of two smooth activations and r = 1 - s, formed as 2^x s:
// far out, where s is 1 but for its last bit, a difference would leave that
// bit for the slope to multiply by z^3. Where 2^x passes 2^126, s is 0.
template <int ACT>
__device__ __forceinline__ void sigmoid2(float z0, float z1, float& s0,
                                         float& s1, float& r0, float& r1) {
  const uint64_t z = f2pk(z0, z1);
  uint64_t x;
  if constexpr (ACT == VECTRA_ACT_SILU) {
    x = fmul2(z, both(-kLog2e));
  } else {
    const uint64_t t = fmul2(z, z);
    if constexpr (ACT == VECTRA_ACT_GELU_TANH) {
      constexpr float k0 = -2.f * kGeluTanhC * kLog2e;
      x = fmul2(z, ffma2(t, both(k0 * kGeluTanhA), both(k0)));
    } else {
      x = fmul2(z, gelu_q(t));
    }
  }
  const float2 xs = f2upk(x);
  const float e0 = fast_exp2(xs.x), e1 = fast_exp2(xs.y);
  s0 = fast_rcp(1.f + e0);
  s1 = fast_rcp(1.f + e1);
  r0 = fminf(e0, 0x1p126f) * s0;
  r1 = fminf(e1, 0x1p126f) * s1;
}

template <int ACT, bool F32>
__device__ __forceinline__ void activate2(float& z0, float& z1) {
  if constexpr (ACT == VECTRA_ACT_RELU) {
    z0 = max_nan(z0, 0.f);
    z1 = max_nan(z1, 0.f);
  } else if constexpr (F32 && ACT == VECTRA_ACT_GELU) {
    float p0, p1;
    normal_cdf2(z0, z1, p0, p1);
    z0 *= p0;
    z1 *= p1;
  } else if constexpr (ACT != VECTRA_ACT_NONE) {
    float s0, s1, r0, r1;
    sigmoid2<ACT>(z0, z1, s0, s1, r0, r1);
    z0 *= s0;
    z1 *= s1;
  }
}

// act'(z) from z, its sigmoid s and r = 1 - s: s + z ds/dz.
template <int ACT>
__device__ __forceinline__ float slope_of(float z, float s, float r) {
  if constexpr (ACT == VECTRA_ACT_SILU) {
    return fmaf(z * s, r, s);
  } else if constexpr (ACT == VECTRA_ACT_GELU_TANH) {
    // 0 * z^2 far out has to stay 0.
    const float t = fminf(z * z, 1e4f);
    const float du = 2.f * kGeluTanhC * fmaf(3.f * kGeluTanhA, t, 1.f);
    return fmaf(z * s * r, du, s);
  } else {  // gelu: s is Phi, and Phi' the normal density
    const float t = fminf(z * z, 1e4f);
    return fmaf(z * 0.3989422804f, fast_exp2(-0.5f * kLog2e * t), s);
  }
}
// z0, z1 become act(z), s0, s1 act'(z).
template <int ACT>
__device__ __forceinline__ void activate_grad2(float& z0, float& z1,
                                               float& s0, float& s1) {
  if constexpr (ACT == VECTRA_ACT_NONE) {
    s0 = s1 = 1.f;
  } else if constexpr (ACT == VECTRA_ACT_RELU) {
    s0 = z0 > 0.f ? 1.f : 0.f;
    s1 = z1 > 0.f ? 1.f : 0.f;
    z0 = max_nan(z0, 0.f);
    z1 = max_nan(z1, 0.f);
  } else {
    float p0, p1, r0, r1;
    sigmoid2<ACT>(z0, z1, p0, p1, r0, r1);
    s0 = slope_of<ACT>(z0, p0, r0);
    s1 = slope_of<ACT>(z1, p1, r1);
    z0 *= p0;
    z1 *= p1;
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

template <int ACT, bool F32, int N>
__device__ __forceinline__ void activate(float* v) {
  if constexpr (ACT != VECTRA_ACT_NONE) {
#pragma unroll
    for (int j = 0; j < N; j += 8) {
      tie8(v + j);
#pragma unroll
      for (int i = 0; i < 8; i += 2) activate2<ACT, F32>(v[j + i], v[j + i + 1]);
      tie8(v + j);
    }
  }
}

// ---------------------------------------------------------------------------
// Epilogue pieces. `stage` is the warp's turning buffer: a lane writes (or
// reads) its row, and rows are moved whole by the copy engine where the
// result's layout allows a tensor map, else by the warp. The copy engine
// spares the shared-memory reads and the stores of the warp: with K = 256
// the SM's one 128 B/clk path through L1 and shared memory, which the
// operands also take, is what bounds a tile.
// ---------------------------------------------------------------------------
struct RowBlock {
  int64_t row0;
  int rows;  // of the 32 that lie in the matrix
};

// Byte offset of 16-byte chunk c of row r.
__device__ __forceinline__ int turn_at(int r, int c) {
  return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// The buffer is free: the last store has read it. (Lane 0 issues them all.)
__device__ __forceinline__ void turn_acquire(int lane) {
  if (lane == 0)
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}

// The buffer's rows to rows `row`.. and columns `col`.. of the matrix; what
// lies outside it is not written.
__device__ __forceinline__ void turn_store_2d(const CUtensorMap* map,
                                              uint8_t* stage, int col,
                                              int row, int lane) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    asm volatile(
        "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group "
        "[%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
        "r"(smem_addr(stage)), "r"(col), "r"(row)
        : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
__device__ __forceinline__ void turn_store_3d(const CUtensorMap* map,
                                              uint8_t* stage, int col,
                                              int row, int plane, int lane) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    asm volatile(
        "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group "
        "[%0, {%2, %3, %4}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
        "r"(smem_addr(stage)), "r"(col), "r"(row), "r"(plane)
        : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}

// Where a block of results goes: by the copy engine through `map`, else to
// rows of `ld` elements at `out`.
template <typename T>
struct Target {
  const CUtensorMap* map;
  bool tma;
  T* out;
  int64_t ld, cols;
};

// Writes 32 rows of 64 bytes (a lane's row in `words`) to columns col..:
// 32 16-bit or 16 float32 columns.
template <typename T>
__device__ __forceinline__ void store_rows(uint8_t* stage,
                                           const uint32_t* words,
                                           const Target<T>& to,
                                           const RowBlock& rb, int64_t col,
                                           int lane) {
  constexpr int kCols = 64 / int(sizeof(T));
  turn_acquire(lane);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(stage + turn_at(lane, c)) =
        make_uint4(words[4 * c], words[4 * c + 1], words[4 * c + 2],
                   words[4 * c + 3]);
  if (to.tma) {
    turn_store_2d(to.map, stage, int(col), int(rb.row0), lane);
  } else {
    __syncwarp();
    for (int e = lane; e < 32 * kCols; e += 32) {
      const int r = e / kCols, c = e % kCols;
      if (r < rb.rows && col + c < to.cols)
        to.out[(rb.row0 + r) * to.ld + col + c] =
            *reinterpret_cast<const T*>(
                stage + turn_at(r, c * int(sizeof(T)) / 16) +
                c * int(sizeof(T)) % 16);
    }
    __syncwarp();
  }
}
__device__ __forceinline__ void store_half_f32(uint8_t* stage, const float* v,
                                               const Target<float>& to,
                                               const RowBlock& rb,
                                               int64_t col, int lane) {
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[j]);
  if (col < to.cols) store_rows<float>(stage, w, to, rb, col, lane);
}

// A block of 32 x 32 results (or saved values) in T.
template <typename T>
__device__ __forceinline__ void store_values(uint8_t* stage, const float* v,
                                             const Target<T>& to,
                                             const RowBlock& rb, int64_t col,
                                             int lane) {
  if constexpr (std::is_same<T, float>::value) {
    store_half_f32(stage, v, to, rb, col, lane);
    store_half_f32(stage, v + 16, to, rb, col + 16, lane);
  } else {
    uint32_t pk[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) pk[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
    store_rows<T>(stage, pk, to, rb, col, lane);
  }
}

// 32 columns of one part's float32 sums.
__device__ __forceinline__ void store_partial(uint8_t* stage, const float* v,
                                              const TcArgs& g,
                                              const CUtensorMap* map,
                                              const RowBlock& rb, int plane,
                                              int64_t col0, int lane) {
#pragma unroll
  for (int h = 0; h < 32; h += 16) {
    const int64_t col = col0 + h;
    if (col >= g.p.N) continue;
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[h + j]);
    if (g.tma_out) {
      turn_acquire(lane);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(stage + turn_at(lane, c)) = make_uint4(
            w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
      turn_store_3d(map, stage, int(col), int(rb.row0), plane, lane);
    } else {
      const Target<float> to{
          nullptr, false, g.partial + int64_t(plane) * g.p.M * g.p.N, g.p.N,
          g.p.N};
      store_rows<float>(stage, w, to, rb, col, lane);
    }
  }
}

// The residual's 32 x 32 block: asynchronous copies into the turning buffer
// (coalesced, in flight while the accumulator is waited for and read), from
// which a lane then takes its row.
template <typename T>
__device__ __forceinline__ void fetch_residual(uint8_t* stage,
                                               const GemmProblem& p,
                                               const RowBlock& rb,
                                               int64_t col, int lane) {
  turn_acquire(lane);
  const int r = lane / 4, c = lane % 4;
  const T* q = static_cast<const T*>(p.res) + (rb.row0 + r) * p.res_sm + col +
               c * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r + 8 * i < rb.rows && col + c * 8 < p.N)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(
                       smem_addr(stage + turn_at(r + 8 * i, c))),
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

// The residual block's rows are in the turning buffer: waits for the copies,
// or, without whole 16-byte pieces, reads it here.
template <typename T>
__device__ __forceinline__ void residual_ready(uint8_t* stage, bool vec,
                                               const GemmProblem& p,
                                               const RowBlock& rb,
                                               int64_t col, int lane) {
  if (vec) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    turn_acquire(lane);
    const T* q = static_cast<const T*>(p.res) + rb.row0 * p.res_sm +
                 (col + lane) * p.res_sn;
    if (col + lane < p.N)
      for (int r = 0; r < rb.rows; ++r, q += p.res_sm)
        *reinterpret_cast<T*>(stage + turn_at(r, lane / 8) + lane % 8 * 2) =
            *q;
  }
  __syncwarp();
}

template <typename T>
__device__ __forceinline__ void add_residual(uint8_t* stage, float* v,
                                             bool vec, const GemmProblem& p,
                                             const RowBlock& rb, int64_t col,
                                             int lane) {
  residual_ready<T>(stage, vec, p, rb, col, lane);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 q =
        *reinterpret_cast<const uint4*>(stage + turn_at(lane, c));
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

// Adds 16 columns over the warp's 32 rows (lanes), destroying x: every step
// halves the columns a lane keeps and hands the other half to its partner,
// so that lanes 2 c and 2 c + 1 end with column c.
__device__ __forceinline__ float column_sums16(float* x, int lane) {
#pragma unroll
  for (int n = 8; n >= 1; n >>= 1) {
    const bool upper = (lane & (2 * n)) != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= n) break;
      const float keep = upper ? x[i + n] : x[i];
      const float give = upper ? x[i] : x[i + n];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * n);
    }
  }
  return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 1);
}

// A float32 residual, 16 columns at a time.
__device__ __forceinline__ void add_residual_f32(uint8_t* stage, float* v,
                                                 bool vec,
                                                 const GemmProblem& p,
                                                 const RowBlock& rb,
                                                 int64_t col0, int lane) {
  const float* res = static_cast<const float*>(p.res);
#pragma unroll
  for (int h = 0; h < 32; h += 16) {
    const int64_t col = col0 + h;
    turn_acquire(lane);
    if (vec) {
      const int r = lane / 4, c = lane % 4;
      const float* q = res + (rb.row0 + r) * p.res_sm + col + c * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r + 8 * i < rb.rows && col + c * 4 < p.N)
          *reinterpret_cast<float4*>(stage + turn_at(r + 8 * i, c)) =
              __ldg(reinterpret_cast<const float4*>(q));
        q += 8 * p.res_sm;
      }
    } else if (col + lane % 16 < p.N) {
      for (int r = lane / 16; r < rb.rows; r += 2)
        *reinterpret_cast<float*>(stage + turn_at(r, lane % 16 / 4) +
                                  lane % 4 * 4) =
            res[(rb.row0 + r) * p.res_sm + (col + lane % 16) * p.res_sn];
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 q =
          *reinterpret_cast<const float4*>(stage + turn_at(lane, c));
      v[h + 4 * c] += q.x;
      v[h + 4 * c + 1] += q.y;
      v[h + 4 * c + 2] += q.z;
      v[h + 4 * c + 3] += q.w;
    }
    __syncwarp();
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
// branches the values were copied between registers at every join: 10
// instructions for each result where the bare store took 6.
template <int EPI, int ACT, bool RES, bool PRE, typename T, int TILE_N,
          int WARP_COLS, typename Wait, typename Release>
__device__ __forceinline__ void epilogue_tile(const TcArgs& g,
                                              const CUtensorMap* const* maps,
                                              uint8_t* stage, float* cols,
                                              int chunks,
                                              const RowBlock& rb,
                                              int64_t tile_col, int part,
                                              int lane, Wait&& wait,
                                              Release&& release) {
  constexpr bool kGated = EPI == kEpiGated || EPI == kEpiGatedPartial ||
                          EPI == kEpiGatedGrad;
  constexpr bool kPartial = EPI == kEpiPartial || EPI == kEpiGatedPartial;
  static_assert(WARP_COLS % 32 == 0 && WARP_COLS <= 64, "columns");
  const GemmProblem& p = g.p;
  if constexpr (EPI == kEpiLinear || EPI == kEpiGated ||
                EPI == kEpiGatedGrad) {
    load_bias<T>(cols, p.bias[0], p.bias_stride[0], tile_col, p.N, WARP_COLS,
                 lane);
    if constexpr (kGated)
      load_bias<T>(cols + 64, p.bias[1], p.bias_stride[1], tile_col, p.N,
                   WARP_COLS, lane);
    __syncwarp();
  }
  const Target<T> out{maps[0], g.tma_out != 0, static_cast<T*>(p.out),
                      p.out_ld, p.N};
  const Target<T> pre{maps[1], g.tma_pre != 0, static_cast<T*>(p.pre),
                      p.pre_ld, p.N};
  const Target<float> gate_to{maps[1], g.tma_pre != 0, p.gate, p.gate_ld,
                              p.N};
  const Target<float> up_to{maps[2], g.tma_pre != 0, p.up, p.up_ld, p.N};
  // With saved values in the same buffer the residual comes after them.
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr bool kEarly = RES && !PRE && !kF32;
  if constexpr (kEarly)
    if (g.vec_res) fetch_residual<T>(stage, p, rb, tile_col, lane);
  // 32 columns: `v` their sums, `up` a gated layer's second ones.
  auto finish = [&](float* v, float* up, int c0) {
    const int64_t col = tile_col + c0;
    if constexpr (kPartial) {
      const int plane = part * (kGated ? 2 : 1);
      store_partial(stage, v, g, maps[0], rb, plane, col, lane);
      if constexpr (kGated)
        store_partial(stage, up, g, maps[0], rb, plane + 1, col, lane);
    } else {
      if constexpr (EPI == kEpiLinear) {
        add_bias<32>(v, cols + c0);
        if constexpr (PRE) {
          store_values<T>(stage, v, pre, rb, col, lane);
          if constexpr (RES && !kF32)
            if (g.vec_res) fetch_residual<T>(stage, p, rb, col, lane);
        }
        activate<ACT, kF32, 32>(v);
        if constexpr (RES && kF32)
          add_residual_f32(stage, v, g.vec_res, p, rb, col, lane);
        else if constexpr (RES)
          add_residual<T>(stage, v, g.vec_res, p, rb, col, lane);
      }
      if constexpr (EPI == kEpiGated) {
        add_bias<32>(v, cols + c0);
        add_bias<32>(up, cols + 64 + c0);
        if constexpr (PRE) {
          store_values<float>(stage, v, gate_to, rb, col, lane);
          store_values<float>(stage, up, up_to, rb, col, lane);
        }
        activate<ACT, kF32, 32>(v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= up[j];
      }
      store_values<T>(stage, v, out, rb, col, lane);
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
        // hi hi, and the five small products.
        constexpr int kSmall = kGated ? 2 * TILE_N : TILE_N;
        const uint32_t at =
            acc + (c < WARP_COLS ? c : TILE_N + c - WARP_COLS);
        uint32_t r[16], q[16];
        tmem_load16x2(at, r, at + kSmall, q);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float part_sum = __uint_as_float(r[j]) + __uint_as_float(q[j]);
          sum[c + j] = chunk == 0 ? part_sum : sum[c + j] + part_sum;
        }
      }
      release();
    }
#pragma unroll
    for (int c0 = 0; c0 < WARP_COLS; c0 += 32)
      if (rb.rows > 0 && tile_col + c0 < p.N)
        finish(sum + c0, sum + (kGated ? WARP_COLS + c0 : 0), c0);
  } else if constexpr (EPI == kEpiGatedGrad) {
    // g and u again, and with dh (read like a residual) dg = dh u act'(g)
    // and du = dh act(g). RES: their sums over the warp's rows as well, from
    // the unrounded values.
    uint32_t acc = 0;
    if (g.vec_res) fetch_residual<T>(stage, p, rb, tile_col, lane);
    if (!wait(&acc)) return;
#pragma unroll 1
    for (int c0 = 0; c0 < WARP_COLS; c0 += 32) {
      const int64_t col = tile_col + c0;
      const bool live = rb.rows > 0 && col < p.N;
      if (g.vec_res && c0 > 0) fetch_residual<T>(stage, p, rb, col, lane);
      residual_ready<T>(stage, g.vec_res, p, rb, col, lane);
      uint32_t dg[16], du[16];
#pragma unroll
      for (int h = 0; h < 32; h += 16) {
        uint32_t dh[8];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint4 q = *reinterpret_cast<const uint4*>(
              stage + turn_at(lane, h / 8 + c));
          const bool in = lane < rb.rows;  // rows past the end count nothing
          dh[4 * c] = in ? q.x : 0;
          dh[4 * c + 1] = in ? q.y : 0;
          dh[4 * c + 2] = in ? q.z : 0;
          dh[4 * c + 3] = in ? q.w : 0;
        }
        uint32_t r0[16], r1[16];
        tmem_load16x2(acc + c0 + h, r0, acc + TILE_N + c0 + h, r1);
        if (c0 + h + 16 == WARP_COLS) release();
        float v[16], up[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[j] = __uint_as_float(r0[j]);
          up[j] = __uint_as_float(r1[j]);
        }
        add_bias<16>(v, cols + c0 + h);
        add_bias<16>(up, cols + 64 + c0 + h);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          if (j % 8 == 0) tie8(v + j);
          float s0, s1;
          activate_grad2<ACT>(v[j], v[j + 1], s0, s1);
          const float2 d = unpack2<T>(dh[j / 2]);
          up[j] *= d.x * s0;
          up[j + 1] *= d.y * s1;
          v[j] *= d.x;
          v[j + 1] *= d.y;
          if (j % 8 == 6) tie8(v + j - 6);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dg[h / 2 + j] = pack2<T>(up[2 * j], up[2 * j + 1]);
          du[h / 2 + j] = pack2<T>(v[2 * j], v[2 * j + 1]);
        }
        if constexpr (RES) {
          const float sg = column_sums16(up, lane);
          const float su = column_sums16(v, lane);
          const int64_t c = col + h + (lane >> 1);
          if (live && (lane & 1) == 0 && c < p.N) {
            const int64_t at = rb.row0 / 32 * p.N + c;
            p.gate[at] = sg;
            p.up[at] = su;
          }
        }
      }
      __syncwarp();  // dh's rows are read
      if (live) {
        store_rows<T>(stage, dg, out, rb, col, lane);
        store_rows<T>(stage, du, pre, rb, col, lane);
      }
    }
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
        tmem_load16x2(acc + c0 + h, r0, acc + TILE_N + c0 + h, r1);
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
            store_half_f32(stage, v, gate_to, rb, col + h, lane);
            store_half_f32(stage, up, up_to, rb, col + h, lane);
          }
        }
        activate<ACT, kF32, 16>(v);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          pk[h / 2 + j] = pack2<T>(v[2 * j] * up[2 * j],
                                   v[2 * j + 1] * up[2 * j + 1]);
      }
      if (live)
        store_rows<T>(stage, pk, out, rb, col, lane);
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
      tmem_load32(acc + c0, r0);
      if constexpr (kGated) tmem_load32(acc + TILE_N + c0, r1);
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
__global__ void __launch_bounds__(Cfg<BN, CG, std::is_same<T, float>::value>::THREADS, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap ta0,
                   const __grid_constant__ CUtensorMap ta1,
                   const __grid_constant__ CUtensorMap tb0,
                   const __grid_constant__ CUtensorMap tb1,
                   const __grid_constant__ CUtensorMap tout,
                   const __grid_constant__ CUtensorMap tpre,
                   const __grid_constant__ CUtensorMap tpre2,
                   const __grid_constant__ TcArgs g) {
  using C = Cfg<BN, CG, std::is_same<T, float>::value>;
  constexpr bool kGated = EPI == kEpiGated || EPI == kEpiGatedPartial ||
                          EPI == kEpiGatedGrad;
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
        int seg = k_first / g.steps_seg;
        int in_seg = k_first - seg * g.steps_seg;
        for (int k = k_first; k < k_last; ++k) {
          ok = mbar_wait(bar_empty(s), phase ^ 1, p.err);
          if (!ok) break;
          uint32_t full = bar_full(s);
          if (CG == 1 || rank == 0)
            mbar_arrive_expect_tx(full, C::STAGE * CG);
          if constexpr (CG == 2) full = map_cta(full, 0);
          if (in_seg == g.steps_seg) {
            in_seg = 0;
            ++seg;
          }
          const int k0 = in_seg++ * kTcStep;
          const CUtensorMap* ma = seg ? &ta1 : &ta0;
#pragma unroll
          for (int plane = 0; plane < C::PLANES; ++plane) {
            const int a_line = plane * g.a_lines, b_line = plane * g.b_lines;
            const uint32_t sa =
                sbase + uint32_t(s) * C::STAGE + plane * C::PLANE;
            const uint32_t sb = sa + C::A_BYTES;
            if (g.a_mn) {
#pragma unroll
              for (int i = 0; i < kTcRows / 64; ++i)
                tma_load_2d<CG>(sa + i * 8192, ma, full, m0 + i * 64,
                                k0 + a_line);
            } else {
              tma_load_2d<CG>(sa, ma, full, k0, m0 + a_line);
            }
            // Rows of B: in a pair, half each. A gated tile's first half is
            // the gate weight's rows, its second half the up weight's.
            constexpr int kBoxRows = kGated && CG == 1 ? BN / 2 : C::B_ROWS;
#pragma unroll
            for (int h = 0; h < C::B_ROWS / kBoxRows; ++h) {
              const CUtensorMap* mb =
                  (kGated ? (CG == 2 ? int(rank) : h) : seg) ? &tb1 : &tb0;
              const int row = kGated ? n0 : n0 + int(rank) * C::B_ROWS;
              const uint32_t dst = sb + h * kBoxRows * 128;
              if (g.b_mn) {
#pragma unroll
                for (int i = 0; i < kBoxRows / 64; ++i)
                  tma_load_2d<CG>(dst + i * 8192, mb, full, row + i * 64,
                                  k0 + b_line);
              } else {
                tma_load_2d<CG>(dst, mb, full, k0, row + b_line);
              }
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
          const int to = kF32 ? chunk_end(from, k_last) : k_last;
          ok = mbar_wait(bar_acc_empty(buf), buf_phase ^ 1, p.err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + uint32_t(buf * C::ACC_COLS);
          for (int k = from; k < to; ++k) {
            ok = mbar_wait(bar_full(s), phase, p.err);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = da0 + uint64_t((uint32_t(s) * C::STAGE) >> 4);
            const uint64_t db = db0 + uint64_t((uint32_t(s) * C::STAGE) >> 4);
            if constexpr (kF32) {
              // Planes 0, 1, 2 are hi, mid, lo. hi hi has an accumulator of
              // its own: the others are too small beside it for their
              // truncation to matter, but would add five more truncations of
              // its sum.
              constexpr int kPairs[6][2] = {{2, 0}, {0, 2}, {1, 1},
                                            {1, 0}, {0, 1}, {0, 0}};
#pragma unroll
              for (int i = 0; i < kTcStep / 16; ++i)
#pragma unroll
                for (int q = 0; q < 6; ++q)
                  mma_f16<CG>(q == 5 ? d : d + BN,
                              da + i * ka + ((kPairs[q][0] * C::PLANE) >> 4),
                              db + i * kb + ((kPairs[q][1] * C::PLANE) >> 4),
                              idesc, k > from || i > 0 || (q > 0 && q < 5));
            } else {
#pragma unroll
              for (int i = 0; i < kTcStep / 16; ++i)
                mma_f16<CG>(d, da + i * ka, db + i * kb, idesc,
                            k > from || i > 0);
            }
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
    uint8_t* stage = smem + C::OFF_EPI + w * kTurnBytes;
    float* cols = reinterpret_cast<float*>(
        smem + C::OFF_EPI + C::EPI_WARPS * kTurnBytes + w * kBiasBytes);
    const CUtensorMap* const maps[3] = {&tout, &tpre, &tpre2};
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
          for (int k = k_first; k < k_last; k = chunk_end(k, k_last))
            ++chunks;
        }
        auto wait = [&](uint32_t* acc) {
          ok = mbar_wait(bar_acc_full(buf), buf_phase, p.err);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) tc_fence_after();
          *acc = lanes + uint32_t(buf * C::ACC_COLS + share * kWarpCols);
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
                      kWarpCols>(g, maps, stage, cols, chunks, rb, tile_col,
                                 t.part, lane, wait, release);
      }
    };
    if constexpr (EPI != kEpiLinear && EPI != kEpiGated &&
                  EPI != kEpiGatedGrad) {
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
    // The last stores have left shared memory and reached global memory.
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
  using C = Cfg<BN, CG, std::is_same<T, float>::value>;
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
                            maps[4], maps[5], maps[6], g);
}

template <int EPI, bool RES, bool PRE, typename T>
cudaError_t launch_shape(int bn, int cg, const CUtensorMap* maps,
                         const TcArgs& g, cudaStream_t stream) {
  // float32 keeps its sums in registers across chunks: the pair's tile, with
  // 96 registers a thread, has no room for them.
  if constexpr (!std::is_same<T, float>::value)
    if (cg == 2)
      return launch_cfg<EPI, RES, PRE, T, 256, 2>(maps, g, stream);
  if constexpr (EPI != kEpiGated && EPI != kEpiGatedPartial &&
                EPI != kEpiGatedGrad)
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
    case kEpiGatedGrad:
      if constexpr (std::is_same<T, float>::value)
        return cudaErrorInvalidValue;
      else
        return g.p.gate
                   ? launch_shape<kEpiGatedGrad, true, false, T>(bn, cg, maps,
                                                                 g, stream)
                   : launch_shape<kEpiGatedGrad, false, false, T>(
                         bn, cg, maps, g, stream);
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
