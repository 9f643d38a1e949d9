// gemm_finish.cu: the end of a product whose reduction was cut into parts:
// adds the parts' float32 sums in order (so the result does not depend on
// scheduling) and applies the epilogue. With no parts it is the product over
// an empty reduction.
//
// Memory-bound, mostly from L2, where the parts were just written: a thread
// takes VEC neighbouring columns of a row and issues the parts' loads four
// at a time.
#include "block_common.cuh"

namespace vectra {
namespace {

template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* p, bool vec, int64_t stride,
                                         int n, float* v) {
  if (VEC == 4 && vec) {
    union {
      uint2 u2;
      uint4 u4;
      T e[4];
    } raw;
    if constexpr (sizeof(T) == 4)
      raw.u4 = __ldg(reinterpret_cast<const uint4*>(p));
    else
      raw.u2 = __ldg(reinterpret_cast<const uint2*>(p));
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(raw.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i < n ? to_f32(p[i * stride]) : 0.f;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, bool vec, int n,
                                          const float* v) {
  if (VEC == 4 && vec) {
    union {
      uint2 u2;
      uint4 u4;
      T e[4];
    } raw;
#pragma unroll
    for (int i = 0; i < VEC; ++i) raw.e[i] = from_f32<T>(v[i]);
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<uint4*>(p) = raw.u4;
    else
      *reinterpret_cast<uint2*>(p) = raw.u2;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}

struct FinishArgs {
  GemmProblem p;
  const float* partial;
  int split;
  // Four elements at once: of the results, of the saved values, of the
  // residual.
  uint8_t vec_out, vec_pre, vec_res, vec_f32;
};

template <typename T, int ACT, int VEC>
__global__ void __launch_bounds__(256)
    split_finish_kernel(const __grid_constant__ FinishArgs f) {
  constexpr bool kExact = std::is_same<T, float>::value;
  const GemmProblem& p = f.p;
  allow_dependents();
  grid_dependency_wait();
  const bool gated = p.epilogue == kEpiGated;
  const int64_t plane = p.M * p.N;
  const int64_t n = (int64_t(blockIdx.x) * 32 + threadIdx.x % 32) * VEC;
  if (n >= p.N) return;
  const int cols = int(p.N - n < VEC ? p.N - n : VEC);
  float b[2][VEC];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      b[s][i] = p.epilogue != kEpiStore && p.bias[s] && i < cols
                    ? to_f32(static_cast<const T*>(
                          p.bias[s])[(n + i) * p.bias_stride[s]])
                    : 0.f;
  for (int64_t m = int64_t(blockIdx.y) * 8 + threadIdx.x / 32; m < p.M;
       m += int64_t(gridDim.y) * 8) {
    float z[VEC], u[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) z[i] = u[i] = 0.f;
    const float* q = f.partial + m * p.N + n;
    const int64_t step = gated ? 2 * plane : plane;
    for (int s0 = 0; s0 < f.split; s0 += 4) {
      float x[4][VEC], y[4][VEC];
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s0 + s < f.split) {
          load_row<float, VEC>(q + (s0 + s) * step, true, 1, cols, x[s]);
          if (gated)
            load_row<float, VEC>(q + (s0 + s) * step + plane, true, 1, cols,
                                 y[s]);
        }
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s0 + s < f.split) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            z[i] += x[s][i];
            if (gated) u[i] += y[s][i];
          }
        }
    }
    float out[VEC];
    if (p.epilogue == kEpiStore) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = z[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        z[i] += b[0][i];
        u[i] += b[1][i];
      }
      if (p.pre)
        store_row<T, VEC>(static_cast<T*>(p.pre) + m * p.pre_ld + n,
                          f.vec_pre, cols, z);
      if (p.gate) {
        store_row<float, VEC>(p.gate + m * p.gate_ld + n, f.vec_f32, cols, z);
        store_row<float, VEC>(p.up + m * p.up_ld + n, f.vec_f32, cols, u);
      }
      float r[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) r[i] = 0.f;
      if (p.res)
        load_row<T, VEC>(static_cast<const T*>(p.res) + m * p.res_sm +
                             n * p.res_sn,
                         f.vec_res, p.res_sn, cols, r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        out[i] = act_fwd<kExact, ACT>(z[i]);
        out[i] = gated ? out[i] * u[i] : out[i] + r[i];
      }
    }
    store_row<T, VEC>(static_cast<T*>(p.out) + m * p.out_ld + n, f.vec_out,
                      cols, out);
  }
}

}  // namespace

cudaError_t launch_split_finish(const GemmProblem& p, int split,
                                const float* partial, cudaStream_t stream) {
  const int es = p.dtype == VECTRA_F32 ? 4 : 2;
  const auto vec = [&](const void* q, int64_t ld, int size) {
    return uint8_t(reinterpret_cast<uintptr_t>(q) % (4 * size) == 0 &&
                   ld % 4 == 0);
  };
  FinishArgs f{p, partial, split, 0, 0, 0, 0};
  f.vec_out = vec(p.out, p.out_ld, es);
  f.vec_pre = vec(p.pre, p.pre_ld, es);
  f.vec_res = p.res_sn == 1 && vec(p.res, p.res_sm, es);
  f.vec_f32 = vec(p.gate, p.gate_ld, 4) && vec(p.up, p.up_ld, 4);
  const bool four = p.N % 4 == 0;  // rows of the sums stay 16-byte aligned
  const int64_t bx = (p.N + (four ? 127 : 31)) / (four ? 128 : 32);
  int64_t by = (p.M + 7) / 8;
  const int64_t most = int64_t(device_sm_count()) * 32 / bx + 1;
  if (by > most) by = most;
  if (by > 65535) by = 65535;
  const dim3 grid{unsigned(bx), unsigned(by)};
  return with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_activation(p.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      return four ? launch_pdl(split_finish_kernel<T, ACT, 4>, grid,
                               dim3(256), 0, stream, f)
                  : launch_pdl(split_finish_kernel<T, ACT, 1>, grid,
                               dim3(256), 0, stream, f);
    });
  });
}

}  // namespace vectra
