// gemm_finish.cu: the end of a product whose reduction was cut into parts:
// adds the parts' float32 sums in order (so the result does not depend on
// scheduling) and applies the epilogue. With no parts it is the product over
// an empty reduction.
#include "block_common.cuh"

namespace vectra {
namespace {

template <typename T>
__device__ __forceinline__ float ld_any(const void* p, int64_t i) {
  return to_f32(static_cast<const T*>(p)[i]);
}

// z -> outputs for one element.
template <typename T, int ACT>
__device__ __forceinline__ void finish_element(const GemmProblem& p,
                                               int64_t m, int64_t n,
                                               float acc, float acc2) {
  constexpr bool kExact = std::is_same<T, float>::value;
  T* out = static_cast<T*>(p.out) + m * p.out_ld + n;
  if (p.epilogue == kEpiStore) {
    *out = from_f32<T>(acc);
    return;
  }
  float z = acc;
  if (p.bias[0]) z += ld_any<T>(p.bias[0], n * p.bias_stride[0]);
  if (p.epilogue == kEpiLinear) {
    if (p.pre)
      static_cast<T*>(p.pre)[m * p.pre_ld + n] = from_f32<T>(z);
    float y = act_fwd<kExact, ACT>(z);
    if (p.res) y += ld_any<T>(p.res, m * p.res_sm + n * p.res_sn);
    *out = from_f32<T>(y);
    return;
  }
  float u = acc2;
  if (p.bias[1]) u += ld_any<T>(p.bias[1], n * p.bias_stride[1]);
  if (p.gate) {
    p.gate[m * p.gate_ld + n] = z;
    p.up[m * p.up_ld + n] = u;
  }
  *out = from_f32<T>(act_fwd<kExact, ACT>(z) * u);
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256)
    split_finish_kernel(const GemmProblem p, int split, const float* partial) {
  allow_dependents();
  grid_dependency_wait();
  const int64_t plane = p.M * p.N;
  const int64_t step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < plane;
       e += step) {
    const int64_t m = e / p.N, n = e - m * p.N;
    float acc = 0.f, acc2 = 0.f;
    if (p.epilogue == kEpiGated) {
      for (int s = 0; s < split; ++s) {
        acc += partial[2 * s * plane + e];
        acc2 += partial[(2 * s + 1) * plane + e];
      }
    } else {
      for (int s = 0; s < split; ++s) acc += partial[s * plane + e];
    }
    finish_element<T, ACT>(p, m, n, acc, acc2);
  }
}

}  // namespace

cudaError_t launch_split_finish(const GemmProblem& p, int split,
                                const float* partial, cudaStream_t stream) {
  const int64_t blocks = (p.M * p.N + 255) / 256;
  const int64_t most = int64_t(device_sm_count()) * 8;
  return with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_activation(p.act, [&](auto act) {
      return launch_pdl(split_finish_kernel<T, decltype(act)::value>,
                        dim3(unsigned(blocks < most ? blocks : most)),
                        dim3(256), 0, stream, p, split, partial);
    });
  });
}

}  // namespace vectra
