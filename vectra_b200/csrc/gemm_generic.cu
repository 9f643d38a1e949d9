// gemm_generic.cu: the matrix products of the transformer-block operators
// for any strides and element type, on the FP32 pipe.
//
// A block of 256 threads computes a 128 x 128 tile of acc in steps of 16
// along the reduction: both operands are staged in shared memory as float32,
// transposed to [k][row], and each thread accumulates 8 x 8 values (two
// groups of four rows and four columns, so the shared-memory reads are
// 16-byte and conflict-free). The next step's elements are loaded into
// registers while the current one is multiplied. A gated layer's tile is 64
// gate columns and the same 64 up columns, so one thread holds both factors
// of its outputs.
//
// The bound is the FP32 pipe: 128 x 128 x 16 x 2 operations against 16 KB
// staged per step.
#include "block_common.cuh"

namespace vectra {
namespace {

constexpr int kBM = 128, kBN = 128, kBK = 16, kThreads = 256;

struct GenericArgs {
  GemmProblem p;
  int64_t k_per_split;  // reduction of one part, over all segments
  int split;
  float* partial;
};

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

// Eight staged elements of one operand, held in registers between the global
// load and the shared store. Consecutive threads walk the direction whose
// stride is 1 (`k_fast`).
struct Stage {
  float v[8];
};

template <typename T>
__device__ __forceinline__ void load_stage(Stage& st, const MatView& m,
                                           bool k_fast, int64_t row0,
                                           int64_t rows, int64_t k0,
                                           int64_t k_end) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = i * kThreads + threadIdx.x;
    const int r = k_fast ? e / kBK : e % kBM;
    const int k = k_fast ? e % kBK : e / kBM;
    const int64_t row = row0 + r, kk = k0 + k;
    st.v[i] = (row < rows && kk < k_end)
                  ? ld_any<T>(m.p, row * m.sr + kk * m.sk)
                  : 0.f;
  }
}

// The gated layer's B tile: rows 0..63 from the gate weight, 64..127 from
// the up weight.
template <typename T>
__device__ __forceinline__ void load_stage_gated(Stage& st, const MatView& g,
                                                 const MatView& u,
                                                 bool k_fast, int64_t row0,
                                                 int64_t rows, int64_t k0,
                                                 int64_t k_end) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = i * kThreads + threadIdx.x;
    const int r = k_fast ? e / kBK : e % kBN;
    const int k = k_fast ? e % kBK : e / kBN;
    const MatView& m = r < kBN / 2 ? g : u;
    const int64_t row = row0 + (r & (kBN / 2 - 1)), kk = k0 + k;
    st.v[i] = (row < rows && kk < k_end)
                  ? ld_any<T>(m.p, row * m.sr + kk * m.sk)
                  : 0.f;
  }
}

constexpr int kPitch = kBM + 4;  // 16-byte rows, transposed stores spread

__device__ __forceinline__ void store_stage(float* s, const Stage& st,
                                            bool k_fast) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = i * kThreads + threadIdx.x;
    const int r = k_fast ? e / kBK : e % kBM;
    const int k = k_fast ? e % kBK : e / kBM;
    s[k * kPitch + r] = st.v[i];
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads)
    gemm_generic_kernel(const GenericArgs g) {
  __shared__ __align__(16) float sa[2][kBK * kPitch];
  __shared__ __align__(16) float sb[2][kBK * kPitch];
  const GemmProblem& p = g.p;
  allow_dependents();
  grid_dependency_wait();
  const bool gated = p.epilogue == kEpiGated;
  const int n_tile = gated ? kBN / 2 : kBN;
  const int64_t tiles_n = (p.N + n_tile - 1) / n_tile;
  const int64_t tile_m = blockIdx.x / tiles_n, tile_n = blockIdx.x % tiles_n;
  const int64_t m0 = tile_m * kBM, n0 = tile_n * n_tile;
  const int part = blockIdx.y;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const bool a_k_fast = p.a[0].sk == 1, b_k_fast = p.b[0].sk == 1;

  // This part's steps run over [first, last) of the reduction as it would
  // be with the segments laid end to end, each padded to whole steps.
  const int64_t steps_seg = (p.K + kBK - 1) / kBK;
  const int64_t steps = steps_seg * p.segments;
  const int64_t per = (steps + g.split - 1) / g.split;
  const int64_t first = part * per;
  const int64_t last = first + per < steps ? first + per : steps;

  float acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;

  Stage ra, rb;
  auto load = [&](int64_t step) {
    const int s = step >= steps_seg ? 1 : 0;
    const int64_t k0 = (step - s * steps_seg) * kBK;
    load_stage<T>(ra, p.a[s], a_k_fast, m0, p.M, k0, p.K);
    if (gated)
      load_stage_gated<T>(rb, p.b[0], p.b[1], b_k_fast, n0, p.N, k0, p.K);
    else
      load_stage<T>(rb, p.b[s], b_k_fast, n0, p.N, k0, p.K);
  };
  if (first < last) {
    load(first);
    store_stage(sa[0], ra, a_k_fast);
    store_stage(sb[0], rb, b_k_fast);
  }
  __syncthreads();
  for (int64_t step = first; step < last; ++step) {
    const int cur = int(step - first) & 1;
    const bool more = step + 1 < last;
    if (more) load(step + 1);
    const float* pa = sa[cur];
    const float* pb = sb[cur];
#pragma unroll
    for (int k = 0; k < kBK; ++k) {
      float av[8], bv[8];
      *reinterpret_cast<float4*>(av) =
          *reinterpret_cast<const float4*>(pa + k * kPitch + ty * 4);
      *reinterpret_cast<float4*>(av + 4) =
          *reinterpret_cast<const float4*>(pa + k * kPitch + 64 + ty * 4);
      *reinterpret_cast<float4*>(bv) =
          *reinterpret_cast<const float4*>(pb + k * kPitch + tx * 4);
      *reinterpret_cast<float4*>(bv + 4) =
          *reinterpret_cast<const float4*>(pb + k * kPitch + 64 + tx * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
    }
    if (more) {
      store_stage(sa[cur ^ 1], ra, a_k_fast);
      store_stage(sb[cur ^ 1], rb, b_k_fast);
    }
    __syncthreads();
  }

  const int64_t plane = p.M * p.N;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t m = m0 + (i < 4 ? ty * 4 + i : 64 + ty * 4 + i - 4);
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (gated) {
        if (j >= 4) continue;
        const int64_t n = n0 + tx * 4 + j;
        if (n >= p.N) continue;
        if (g.split > 1) {
          float* q = g.partial + part * 2 * plane + m * p.N + n;
          q[0] = acc[i][j & 3];
          q[plane] = acc[i][(j & 3) + 4];
        } else {
          finish_element<T, ACT>(p, m, n, acc[i][j & 3],
                                 acc[i][(j & 3) + 4]);
        }
      } else {
        const int64_t n = n0 + (j < 4 ? tx * 4 + j : 64 + tx * 4 + j - 4);
        if (n >= p.N) continue;
        if (g.split > 1)
          g.partial[part * plane + m * p.N + n] = acc[i][j];
        else
          finish_element<T, ACT>(p, m, n, acc[i][j], 0.f);
      }
    }
  }
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

cudaError_t launch_gemm_generic(const GemmProblem& p, int split,
                                float* partial, cudaStream_t stream) {
  const int n_tile = p.epilogue == kEpiGated ? kBN / 2 : kBN;
  const int64_t tiles =
      ((p.M + kBM - 1) / kBM) * ((p.N + n_tile - 1) / n_tile);
  if (tiles > 0x7fffffff || split > 65535) return cudaErrorInvalidValue;
  GenericArgs g{p, 0, split, partial};
  return with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_activation(split > 1 ? VECTRA_ACT_NONE : p.act, [&](auto act) {
      return launch_pdl(gemm_generic_kernel<T, decltype(act)::value>,
                        dim3(unsigned(tiles), unsigned(split)),
                        dim3(kThreads), 0, stream, g);
    });
  });
}

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
