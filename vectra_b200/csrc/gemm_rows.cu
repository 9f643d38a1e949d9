// gemm_rows.cu: the products of a serving step, act(x W^T + b) + r or the
// gated layer for a few rows of x, eight at a time.
//
// Bound by reading the weights: 2 N K bytes against 16 N K operations. There is no reuse to stage for, so the weights go straight
// from global memory into mma.sync operands: in m16n8k16 the weight rows are
// the 16 rows, the tokens the 8 columns, and since a sum may run over the
// reduction in any order, a lane's 16-byte load (eight neighbours of one
// weight row) supplies its share of two MMAs when the token operand is read
// with the same assignment.
//
// A block of 8 warps owns 16 weight rows; a gated layer's block 8 rows of
// each weight, gate rows as MMA rows 0-7 and up rows as 8-15, so that both
// factors of an output meet in it. The warps cut the reduction into eight
// contiguous ranges, keep kDepth steps of 32 elements in flight each, and
// are added in order through shared memory. Two blocks per SM keep 128 KB in
// flight, which covers DRAM latency at full rate. Measured (B200): the gated
// layer of one token, 4096 -> 10240, 27.8 us (6.0 TB/s, 0.92 of the copy
// rate), 8 x 4096 -> 4096 8.0 us (33 MB: 4.2 TB/s, start and join included);
// the tensor-core kernel takes 48 and 13. (Two token tiles per pass, for 16
// rows, took 12.7 us where that kernel takes 10.1.)
#include "block_common.cuh"
#include "gemm_rows.cuh"
#include "mma_sync.cuh"

namespace vectra {
namespace {

constexpr int kWarps = 8;
constexpr int kTokens = 8;
constexpr int kStep = 32;   // reduction per load of a lane quad
constexpr int kDepth = 8;

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <bool kExact>
__device__ __forceinline__ float act_any(float z, int act) {
  switch (act) {
    case VECTRA_ACT_RELU:
      return act_fwd<kExact, VECTRA_ACT_RELU>(z);
    case VECTRA_ACT_GELU:
      return act_fwd<kExact, VECTRA_ACT_GELU>(z);
    case VECTRA_ACT_GELU_TANH:
      return act_fwd<kExact, VECTRA_ACT_GELU_TANH>(z);
    case VECTRA_ACT_SILU:
      return act_fwd<kExact, VECTRA_ACT_SILU>(z);
    default:
      return z;
  }
}

// The warps' sums, added in order, and the epilogue: one output per thread.
template <typename T, bool GATED>
__device__ __forceinline__ void finish_rows(
    const GemmProblem& p, const float (*sums)[kTokens][16 + 1], int64_t n0,
    int64_t m0) {
  constexpr int kCols = GATED ? 8 : 16;
  constexpr bool kExact = std::is_same<T, float>::value;
  const int t = threadIdx.x / kCols, r = threadIdx.x % kCols;
  const int64_t n = n0 + r, m = m0 + t;
  if (m >= p.M || t >= kTokens || n >= p.N) return;
  float z = 0.f, u = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    z += sums[w][t][r];
    if constexpr (GATED) u += sums[w][t][8 + r];
  }
  if (p.bias[0])
    z += to_f32(static_cast<const T*>(p.bias[0])[n * p.bias_stride[0]]);
  T* out = static_cast<T*>(p.out) + m * p.out_ld + n;
  if constexpr (GATED) {
    if (p.bias[1])
      u += to_f32(static_cast<const T*>(p.bias[1])[n * p.bias_stride[1]]);
    if (p.gate) {
      p.gate[m * p.gate_ld + n] = z;
      p.up[m * p.up_ld + n] = u;
    }
    *out = from_f32<T>(act_any<kExact>(z, p.act) * u);
  } else {
    if (p.pre) static_cast<T*>(p.pre)[m * p.pre_ld + n] = from_f32<T>(z);
    float y = act_any<kExact>(z, p.act);
    if (p.res)
      y += to_f32(static_cast<const T*>(p.res)[m * p.res_sm + n * p.res_sn]);
    *out = from_f32<T>(y);
  }
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kWarps * 32, 2)
    gemm_rows_kernel(const __grid_constant__ GemmProblem p) {
  constexpr int kCols = GATED ? 8 : 16;  // outputs per token of a block
  __shared__ float sums[kWarps][kTokens][16 + 1];
  allow_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  const int64_t n0 = int64_t(blockIdx.x) * kCols;
  // Contiguous ranges of whole 128-byte lines.
  const int64_t steps = (p.K + kStep - 1) / kStep;
  const int64_t per = ((steps + kWarps - 1) / kWarps + 1) / 2 * 2;
  const int64_t s0 = warp * per;
  const int64_t s1 = s0 + per < steps ? s0 + per : steps;

  // MMA rows g and g + 8 of this lane.
  const T* wp[2];
  bool wok[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t n = n0 + g + (GATED ? 0 : 8 * h);
    const MatView& w = p.b[GATED ? h : 0];
    wok[h] = n < p.N;
    wp[h] = static_cast<const T*>(w.p) + (wok[h] ? n : 0) * w.sr + t * 8;
  }
  const int64_t m0 = int64_t(blockIdx.y) * kTokens;
  const bool xok = m0 + g < p.M;
  const T* xp = static_cast<const T*>(p.a[0].p) +
                (xok ? m0 + g : 0) * p.a[0].sr + t * 8;

  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t step = s0; step < s1; step += kDepth) {
    uint4 w[kDepth][2], x[kDepth];
#pragma unroll
    for (int q = 0; q < kDepth; ++q) {
      const int64_t k = (step + q) * kStep;
      const bool in = step + q < s1 && k + t * 8 < p.K;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[q][h] = in && wok[h] ? load_stream(wp[h] + k)
                               : make_uint4(0, 0, 0, 0);
      x[q] = in && xok ? __ldg(reinterpret_cast<const uint4*>(xp + k))
                       : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int q = 0; q < kDepth; ++q) {
      const uint4 &a = w[q][0], &b = w[q][1];
      const uint32_t lo[4] = {a.x, b.x, a.y, b.y};
      const uint32_t hi[4] = {a.z, b.z, a.w, b.w};
      mma16816<T>(acc, lo, x[q].x, x[q].y);
      mma16816<T>(acc, hi, x[q].z, x[q].w);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    sums[warp][2 * t + (c & 1)][g + 8 * (c >> 1)] = acc[c];
  __syncthreads();
  finish_rows<T, GATED>(p, sums, n0, m0);
}

// The same for float32, on the FP32 pipe: a lane's 16 bytes are four
// neighbours of a weight row, multiplied by the same four of every token and
// added over the quad at the end.
// Measured (B200): 1 x 4096 -> 4096 13.3 us (67 MB: 5.0 TB/s), gated 1 x 4096 ->
// 10240 52.7 (336 MB: 6.4), 8 x 4096 -> 4096 22.6, gated 8 x 4096 -> 10240
// 94.9. With eight tokens it is bound by latency, not by the pipe (issue 0.35
// per scheduler, DRAM 31 %, two blocks an SM at 128 registers): the tokens'
// pieces, eight 16-byte loads for every two of the weights, leave registers
// for four steps in flight.
template <bool GATED, int TOKENS>
__global__ void __launch_bounds__(kWarps * 32, 2)
    gemm_rows_f32_kernel(const __grid_constant__ GemmProblem p) {
  constexpr int kCols = GATED ? 8 : 16;
  constexpr int kStep32 = 16, kDepth32 = 4;
  __shared__ float sums[kWarps][kTokens][16 + 1];
  allow_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  const int64_t n0 = int64_t(blockIdx.x) * kCols;
  const int64_t steps = (p.K + kStep32 - 1) / kStep32;
  const int64_t per = ((steps + kWarps - 1) / kWarps + 1) / 2 * 2;
  const int64_t s0 = warp * per;
  const int64_t s1 = s0 + per < steps ? s0 + per : steps;
  const float* wp[2];
  bool wok[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t n = n0 + g + (GATED ? 0 : 8 * h);
    const MatView& w = p.b[GATED ? h : 0];
    wok[h] = n < p.N;
    wp[h] = static_cast<const float*>(w.p) + (wok[h] ? n : 0) * w.sr + t * 4;
  }
  // Tokens past M repeat the last one; nothing of theirs is written.
  const int64_t m0 = int64_t(blockIdx.y) * kTokens;
  const float* xp[TOKENS];
#pragma unroll
  for (int m = 0; m < TOKENS; ++m)
    xp[m] = static_cast<const float*>(p.a[0].p) +
            (m0 + m < p.M ? m0 + m : p.M - 1) * p.a[0].sr + t * 4;
  float acc[2][TOKENS];
#pragma unroll
  for (int m = 0; m < TOKENS; ++m) acc[0][m] = acc[1][m] = 0.f;
  for (int64_t step = s0; step < s1; step += kDepth32) {
    union {
      uint4 u;
      float f[4];
    } w[kDepth32][2];
#pragma unroll
    for (int q = 0; q < kDepth32; ++q) {
      const int64_t k = (step + q) * kStep32;
      const bool in = step + q < s1 && k + t * 4 < p.K;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[q][h].u = in && wok[h] ? load_stream(wp[h] + k)
                                 : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int q = 0; q < kDepth32; ++q) {
      const int64_t k = (step + q) * kStep32;
      const bool in = step + q < s1 && k + t * 4 < p.K;
      float4 x[TOKENS];
#pragma unroll
      for (int m = 0; m < TOKENS; ++m)
        x[m] = in ? __ldg(reinterpret_cast<const float4*>(xp[m] + k))
                  : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int m = 0; m < TOKENS; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v = acc[h][m];
          v = fmaf(w[q][h].f[0], x[m].x, v);
          v = fmaf(w[q][h].f[1], x[m].y, v);
          v = fmaf(w[q][h].f[2], x[m].z, v);
          acc[h][m] = fmaf(w[q][h].f[3], x[m].w, v);
        }
    }
  }
#pragma unroll
  for (int m = 0; m < TOKENS; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = acc[h][m];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (t == 0) sums[warp][m][g + 8 * h] = v;
    }
  __syncthreads();
  finish_rows<float, GATED>(p, sums, n0, m0);
}

bool line_view(const MatView& m, int64_t rows, int64_t es) {
  return m.sk == 1 && (reinterpret_cast<uintptr_t>(m.p) & 15) == 0 &&
         (rows <= 1 || m.sr * es % 16 == 0);
}

}  // namespace

// Up to eight rows read the weights once and always run here. More rows take
// passes over them, which still beats the tensor-core kernel's start and
// second launch while the blocks' work is small. B200, us, here against
// there: bf16 32 x 1024 -> 1024 3.1 and 5.9, 64 x 1024 -> 1024 5.3 and 6.0,
// 32 x 1472 -> 1984 6.0 and 7.4, 64 x 1472 -> 1984 9.7 and 7.4, 16 x 4096 ->
// 4096 13.5 and 10.1; f32, whose other kernel also splits its operands first,
// 16 x 4096 -> 4096 41 and 56, 32 x 1024 -> 1024 6.2 and 11.5, 32 x 1472 ->
// 1984 16.1 and 15.2.
bool gemm_rows_supports(const GemmProblem& p) {
  const bool f32 = p.dtype == VECTRA_F32;
  const int64_t es = f32 ? 4 : 2;
  if (p.segments != 1 || p.K * es % 16 != 0 || p.a[0].plane_lines)
    return false;
  if (p.M > (f32 ? 2 * kTokens : kTokens)) {
    const int64_t cols = p.epilogue == kEpiGated ? 8 : 16;
    const int64_t blocks =
        ((p.N + cols - 1) / cols) * ((p.M + kTokens - 1) / kTokens);
    if (p.M > kRowsMost || blocks * p.K > (f32 ? 400000 : 800000))
      return false;
  }
  return line_view(p.a[0], p.M, es) && line_view(p.b[0], p.N, es) &&
         (p.epilogue != kEpiGated || line_view(p.b[1], p.N, es));
}

cudaError_t launch_gemm_rows(const GemmProblem& p, cudaStream_t stream) {
  const bool gated = p.epilogue == kEpiGated;
  const int64_t cols = gated ? 8 : 16;
  const dim3 grid(unsigned((p.N + cols - 1) / cols),
                  unsigned((p.M + kTokens - 1) / kTokens));
  const dim3 block(kWarps * 32);
  auto run = [&](auto kernel) {
    return launch_pdl(kernel, grid, block, 0, stream, p);
  };
  if (p.dtype == VECTRA_F32) {
    if (p.M == 1)
      return gated ? run(gemm_rows_f32_kernel<true, 1>)
                   : run(gemm_rows_f32_kernel<false, 1>);
    if (p.M <= 4)
      return gated ? run(gemm_rows_f32_kernel<true, 4>)
                   : run(gemm_rows_f32_kernel<false, 4>);
    return gated ? run(gemm_rows_f32_kernel<true, 8>)
                 : run(gemm_rows_f32_kernel<false, 8>);
  }
  if (p.dtype == VECTRA_F16)
    return gated ? run(gemm_rows_kernel<__half, true>)
                 : run(gemm_rows_kernel<__half, false>);
  return gated ? run(gemm_rows_kernel<__nv_bfloat16, true>)
               : run(gemm_rows_kernel<__nv_bfloat16, false>);
}

}  // namespace vectra
