// block_common.cuh: activations, problem descriptions and the workspace of
// the transformer-block operators (include/vectra_block.h).
//
// Every matrix product of these operators is one GemmProblem,
//   acc[m, n] = sum over segments s, k of a[s](m, k) b[s](n, k),
// followed by an epilogue on acc in float32. Operands are [rows][reduction]
// views with two strides, so a forward product (x W^T), an input gradient
// (dz W) and a weight gradient (dz^T x) differ only in strides.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "rbf_common.cuh"
#include "vectra_block.h"

namespace vectra {

// ---------------------------------------------------------------------------
// Activations. kExact: CUDA's expf and erfcf, for float32 tensors, in forms
// that keep their relative accuracy in the negative tail (0.5 z (1 + erf),
// and the same with tanh, lose it from z = -3 on).
// Otherwise forms on ex2.approx and rcp.approx whose error (below 1e-6
// absolute) is far under the rounding of the 16-bit results.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool kExact>
__device__ __forceinline__ float sigmoid_f(float z) {
  if constexpr (kExact) return 1.f / (1.f + expf(-z));
  return fast_rcp(1.f + fast_exp2(-kLog2e * z));
}
// The same, and in `rest` 1 - sigmoid without the difference's cancellation,
// which the slopes would multiply by z or z^3.
template <bool kExact>
__device__ __forceinline__ float sigmoid_f(float z, float* rest) {
  const float e = kExact ? expf(-z) : fast_exp2(-kLog2e * z);
  const float s = kExact ? 1.f / (1.f + e) : fast_rcp(1.f + e);
  *rest = fminf(e, 0x1p126f) * s;  // s is 0 where e is infinite
  return s;
}

constexpr float kGeluTanhC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluTanhA = 0.044715f;

// Phi(z) = erfc(-z / sqrt 2) / 2, and exp(-z^2 / 2) on the way: Abramowitz
// and Stegun 7.1.26, erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2) with
// t = 1 / (1 + p x) for x >= 0 (absolute error 1.5e-7).
__device__ __forceinline__ float phi_fast(float z, float* e_out) {
  const float x = fabsf(z) * 0.70710678f;
  const float t = fast_rcp(fmaf(0.3275911f, x, 1.f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float e = fast_exp2(-kLog2e * x * x);
  *e_out = e;
  const float half = 0.5f * p * t * e;  // erfc(|z| / sqrt 2) / 2
  return z < 0.f ? half : 1.f - half;
}

template <bool kExact, int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == VECTRA_ACT_RELU) {
    return z > 0.f || z != z ? z : 0.f;  // NaN stays NaN
  } else if constexpr (ACT == VECTRA_ACT_SILU) {
    if constexpr (kExact) return z / (1.f + expf(-z));
    return z * sigmoid_f<false>(z);
  } else if constexpr (ACT == VECTRA_ACT_GELU) {
    if constexpr (kExact) return 0.5f * z * erfcf(z * -0.70710678118f);
    float e;
    return z * phi_fast(z, &e);
  } else if constexpr (ACT == VECTRA_ACT_GELU_TANH) {
    const float u = kGeluTanhC * fmaf(kGeluTanhA * z * z, z, z);
    // (1 + tanh u) / 2 = sigmoid(2 u)
    if constexpr (kExact) return z / (1.f + expf(-2.f * u));
    return z * sigmoid_f<false>(2.f * u);
  } else {
    return z;
  }
}

// act(z) and act'(z) together (the backward of a gated layer needs both).
template <bool kExact, int ACT>
__device__ __forceinline__ float act_grad(float z, float* value) {
  if constexpr (ACT == VECTRA_ACT_RELU) {
    *value = z > 0.f || z != z ? z : 0.f;
    return z > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == VECTRA_ACT_SILU) {
    float rest;
    const float s = sigmoid_f<kExact>(z, &rest);
    *value = z * s;
    return s * (1.f + z * rest);
  } else if constexpr (ACT == VECTRA_ACT_GELU) {
    float phi, e;
    if constexpr (kExact) {
      phi = 0.5f * erfcf(z * -0.70710678118f);
      e = expf(-0.5f * z * z);
    } else {
      phi = phi_fast(z, &e);
    }
    *value = z * phi;
    return phi + z * 0.3989422804f * e;
  } else if constexpr (ACT == VECTRA_ACT_GELU_TANH) {
    const float u = kGeluTanhC * fmaf(kGeluTanhA * z * z, z, z);
    float rest;
    const float s = sigmoid_f<kExact>(2.f * u, &rest);
    *value = z * s;
    // Past |z| = 100, s or rest is exactly 0; its product with z^2 has to
    // stay 0.
    const float t = fminf(z * z, 1e4f);
    const float du = kGeluTanhC * fmaf(3.f * kGeluTanhA, t, 1.f);
    return s + 2.f * z * s * rest * du;
  } else {
    *value = z;
    return 1.f;
  }
}

// Calls f with the activation as a compile-time constant.
template <typename F>
cudaError_t with_activation(int act, F&& f) {
  switch (act) {
    case VECTRA_ACT_RELU:
      return f(std::integral_constant<int, VECTRA_ACT_RELU>{});
    case VECTRA_ACT_GELU:
      return f(std::integral_constant<int, VECTRA_ACT_GELU>{});
    case VECTRA_ACT_GELU_TANH:
      return f(std::integral_constant<int, VECTRA_ACT_GELU_TANH>{});
    case VECTRA_ACT_SILU:
      return f(std::integral_constant<int, VECTRA_ACT_SILU>{});
    default:
      return f(std::integral_constant<int, VECTRA_ACT_NONE>{});
  }
}

// Calls f with a null pointer of the element type.
template <typename F>
cudaError_t with_dtype(int dtype, F&& f) {
  if (dtype == VECTRA_F32) return f(static_cast<float*>(nullptr));
  if (dtype == VECTRA_F16) return f(static_cast<__half*>(nullptr));
  return f(static_cast<__nv_bfloat16*>(nullptr));
}

// ---------------------------------------------------------------------------
// Matrix products.
// ---------------------------------------------------------------------------
// A view of [rows][K], K the reduced dimension; strides in elements.
struct MatView {
  const void* p = nullptr;
  int64_t sr = 0, sk = 0;
  // float32 split beforehand (split_for_products): p holds three bf16 planes
  // of this many lines, in the order of the view's own rows in memory.
  int64_t plane_lines = 0;
};

// What happens to acc[m, n].
enum GemmEpilogue {
  kEpiStore = 0,   // out = acc
  kEpiLinear = 1,  // z = acc + bias; pre = z; out = act(z) + residual
  kEpiGated = 2,   // g = acc + bias, u = acc2 + bias2; out = act(g) * u
  // The backward of that without saved values (bf16 / f16): with g and u
  // formed again and dh in `res`, out = dh u act'(g), pre = dh act(g), and
  // their sums over blocks of 32 rows in gate and up ([blocks][N]).
  kEpiGatedGrad = 3
};

struct GemmProblem {
  int32_t dtype = VECTRA_F32;
  int32_t epilogue = kEpiStore;
  int32_t act = VECTRA_ACT_NONE;
  int32_t segments = 1;  // products summed: 1 or 2 (kEpiGated: 1)
  int64_t M = 0, N = 0, K = 0;  // every segment reduces over K
  MatView a[2], b[2];    // gated: b[0] gate, b[1] up, both with a[0]
  const void* bias[2] = {nullptr, nullptr};
  int64_t bias_stride[2] = {0, 0};
  const void* res = nullptr;
  int64_t res_sm = 0, res_sn = 0;
  void* out = nullptr;
  int64_t out_ld = 0;
  void* pre = nullptr;   // kEpiLinear: z in dtype
  int64_t pre_ld = 0;
  float* gate = nullptr;  // kEpiGated: g and u
  float* up = nullptr;
  int64_t gate_ld = 0, up_ld = 0;
  unsigned int* err = nullptr;  // device error word (set at launch)
};

// Bump allocator over the caller's workspace. With no base it only counts,
// so one function both sizes a call and runs it.
struct Workspace {
  char* base = nullptr;
  size_t size = 0;
  size_t used = 0;
  bool dry = true;
  bool overflow = false;
  void* take(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) / 256 * 256;
    if (dry) return nullptr;
    if (used > size) {
      overflow = true;
      return nullptr;
    }
    return base + at;
  }
};

// Runs (or, when ws.dry, sizes) one product; picks the kernel.
cudaError_t run_gemm(const GemmProblem& p, Workspace& ws, cudaStream_t stream);

// A float32 matrix [lines][inner] (rows `ld` apart, unit inner stride) split
// into planes once for several products; returns it as the operand that
// reduces over the lines (`cols`) and the one that reduces over the inner
// dimension (`rows`).
cudaError_t split_for_products(const void* p, int64_t lines, int64_t inner,
                               int64_t s_line, int64_t s_inner, Workspace& ws,
                               MatView* rows, MatView* cols,
                               cudaStream_t stream);

// gemm_finish.cu: `partial` holds [split][M][N] float32 sums (for kEpiGated
// [split][2][M][N]).
// Adds the parts in order and applies the epilogue.
cudaError_t launch_split_finish(const GemmProblem& p, int split,
                                const float* partial, cudaStream_t stream);

// block_grad.cu: elementwise parts of the backward passes.
// dz (and du) are written in the operands' type: 16-bit tensors' products run
// on 16-bit operands, and two planes of them would double both products of a
// backward pass. It costs a gated layer's bf16 gradients 2.3e-3 of their size
// against 1.7e-3 for the result's rounding alone; db is of the unrounded sums.
struct GradProblem {
  int32_t dtype = VECTRA_F32;
  int32_t act = VECTRA_ACT_NONE;
  bool gated = false;
  int64_t M = 0, N = 0;
  const void* dy = nullptr;
  int64_t dy_sm = 0, dy_sn = 0;
  const void* pre = nullptr;  // linear: z [M, pre_ld]
  int64_t pre_ld = 0;
  const float* gate = nullptr;  // gated: g and u
  const float* up = nullptr;
  int64_t gate_ld = 0, up_ld = 0;
  void* dz = nullptr;   // linear: dz; gated: dg; null: only the sums
  void* dz2 = nullptr;  // gated: du
  int64_t dz_ld = 0;
  void* db = nullptr;   // column sums in dtype; null: not wanted
  void* db2 = nullptr;
};
cudaError_t run_grad(const GradProblem& p, Workspace& ws, cudaStream_t stream);
// db = column sums of `partial` [chunks][N], in order; db2 likewise.
cudaError_t launch_column_finish(int32_t dtype, const float* partial,
                                 const float* partial2, int chunks, int64_t N,
                                 void* db, void* db2, cudaStream_t stream);

// qk_norm_rope.cu
struct QkSide {
  const void* x = nullptr;
  int64_t sx[4] = {0, 0, 0, 0};
  void* out = nullptr;       // forward: the result; backward: dx
  int64_t so[4] = {0, 0, 0, 0};
  const void* dy = nullptr;  // backward
  int64_t sy[4] = {0, 0, 0, 0};
  const void* w = nullptr;
  int64_t sw = 0;
  void* dw = nullptr;        // backward, [D] in the weight's type
  int64_t sdw = 0;
  int32_t w_dtype = VECTRA_F32;
  int32_t H = 0;
};
struct QkProblem {
  QkSide side[2];  // queries, keys
  int32_t dtype = VECTRA_F32;
  int32_t interleaved = 0;
  int64_t B = 0, N = 0;
  int32_t D = 0, R2 = 0;
  int64_t P = 0;
  const float* cos = nullptr;
  const float* sin = nullptr;
  int64_t cos_ld = 0, sin_ld = 0;
  const void* pos = nullptr;
  int32_t pos_bytes = 8;
  int64_t pos_sb = 0, pos_sn = 0;
  float eps = 0.f;
};
cudaError_t launch_qk_forward(const QkProblem& p, cudaStream_t stream);
cudaError_t run_qk_backward(const QkProblem& p, Workspace& ws,
                            cudaStream_t stream);

// Largest size of one dimension: tensor-map coordinates are 32-bit, and
// float32 operands keep three planes of lines in one map.
constexpr int64_t kMaxSize = (int64_t(1) << 29) - 256;

// Adds to the library's launch counter (capi.cu).
void count_launches(int n);

}  // namespace vectra
