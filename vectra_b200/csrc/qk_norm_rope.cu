// qk_norm_rope.cu: the RMS norm of every query and key head vector and the
// rotation of its position, in one pass, with its backward pass.
//
//   n = v * r, r = 1 / sqrt(mean(v^2) + eps);  y = n * w
//   (a, b) -> (a cos - b sin, b cos + a sin) for the first R2 pairs of y
// and for an upstream gradient g, with g' its rotation by the opposite
// angle:
//   dw = sum over vectors of g' * n,  dv = r (w g' - n mean(w g' n)).
// Rotation and norm run in float32 on the values as loaded; each result is
// rounded once.
//
// Memory-bound: each vector is read once and written once.
#include "block_common.cuh"

namespace vectra {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxPairs = 8;  // per lane: D <= 512 has 256 pairs

struct QkArgs {
  QkProblem p;
  float* partial;  // backward: [2][blocks][D] weight-gradient sums
};

__device__ __forceinline__ int64_t load_pos(const QkProblem& p, int64_t b,
                                            int64_t n) {
  if (p.pos == nullptr) return n;
  const int64_t i = b * p.pos_sb + n * p.pos_sn;
  return p.pos_bytes == 8 ? static_cast<const int64_t*>(p.pos)[i]
                          : int64_t(static_cast<const int32_t*>(p.pos)[i]);
}

// The general kernel: one warp per head vector, any strides. A lane holds
// the element pairs lane, lane + 32, ... of the vector; pairs past R2 are
// two unrotated elements (2 j, 2 j + 1 counted from 2 R2), so each lane's
// elements, and its share of the weight gradient, are the same for every
// vector.
__device__ __forceinline__ void pair_elements(int j, int r2, int d,
                                              int interleaved, int* e0,
                                              int* e1) {
  if (j < r2) {
    *e0 = interleaved ? 2 * j : j;
    *e1 = interleaved ? 2 * j + 1 : j + r2;
  } else {
    *e0 = 2 * j;
    *e1 = 2 * j + 1;
  }
  if (*e0 >= d) *e0 = -1;
  if (*e1 >= d) *e1 = -1;
}

template <typename T, bool BACKWARD>
__global__ void __launch_bounds__(kWarps * 32)
    qk_general_kernel(const QkArgs a) {
  __shared__ float sums[kWarps][512];
  const QkProblem& p = a.p;
  const QkSide& s = p.side[blockIdx.y];
  allow_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int D = p.D;
  int e0[kMaxPairs], e1[kMaxPairs];
  float w0[kMaxPairs], w1[kMaxPairs], dw0[kMaxPairs], dw1[kMaxPairs];
#pragma unroll
  for (int i = 0; i < kMaxPairs; ++i) {
    pair_elements(lane + 32 * i, p.R2, D, p.interleaved, &e0[i], &e1[i]);
    w0[i] = w1[i] = 1.f;
    dw0[i] = dw1[i] = 0.f;
    if (s.w) {
      if (e0[i] >= 0) w0[i] = load_any(s.w, s.w_dtype, e0[i] * s.sw);
      if (e1[i] >= 0) w1[i] = load_any(s.w, s.w_dtype, e1[i] * s.sw);
    }
  }
  const int64_t vectors = p.B * p.N * s.H;
  const float inv_d = 1.f / float(D);
  for (int64_t v = int64_t(blockIdx.x) * kWarps + warp; v < vectors;
       v += int64_t(gridDim.x) * kWarps) {
    const int64_t token = v / s.H;
    const int64_t h = v - token * s.H, b = token / p.N, n = token - b * p.N;
    const T* x = static_cast<const T*>(s.x) + b * s.sx[0] + h * s.sx[1] +
                 n * s.sx[2];
    const int64_t pos = load_pos(p, b, n);
    const bool known = pos >= 0 && pos < p.P;
    float x0[kMaxPairs], x1[kMaxPairs];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
      x0[i] = e0[i] >= 0 ? to_f32(x[e0[i] * s.sx[3]]) : 0.f;
      x1[i] = e1[i] >= 0 ? to_f32(x[e1[i] * s.sx[3]]) : 0.f;
      ss += x0[i] * x0[i] + x1[i] * x1[i];
    }
    const float r = rsqrtf(warp_sum(ss) * inv_d + p.eps);
    T* out = static_cast<T*>(s.out) + b * s.so[0] + h * s.so[1] + n * s.so[2];
    if constexpr (!BACKWARD) {
#pragma unroll
      for (int i = 0; i < kMaxPairs; ++i) {
        const int j = lane + 32 * i;
        const float y0 = x0[i] * r * w0[i], y1 = x1[i] * r * w1[i];
        float o0 = y0, o1 = y1;
        if (j < p.R2) {
          const float c = known ? __ldg(p.cos + pos * p.cos_ld + j) : NAN;
          const float sn = known ? __ldg(p.sin + pos * p.sin_ld + j) : NAN;
          o0 = y0 * c - y1 * sn;
          o1 = y1 * c + y0 * sn;
        } else if (!known) {
          o0 = o1 = NAN;
        }
        if (e0[i] >= 0) out[e0[i]] = from_f32<T>(o0);
        if (e1[i] >= 0) out[e1[i]] = from_f32<T>(o1);
      }
    } else {
      const T* dy = static_cast<const T*>(s.dy) + b * s.sy[0] + h * s.sy[1] +
                    n * s.sy[2];
      float g0[kMaxPairs], g1[kMaxPairs];
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < kMaxPairs; ++i) {
        const int j = lane + 32 * i;
        const float y0 = e0[i] >= 0 ? to_f32(dy[e0[i] * s.sy[3]]) : 0.f;
        const float y1 = e1[i] >= 0 ? to_f32(dy[e1[i] * s.sy[3]]) : 0.f;
        g0[i] = y0;
        g1[i] = y1;
        if (j < p.R2) {
          const float c = known ? __ldg(p.cos + pos * p.cos_ld + j) : NAN;
          const float sn = known ? __ldg(p.sin + pos * p.sin_ld + j) : NAN;
          g0[i] = y0 * c + y1 * sn;
          g1[i] = y1 * c - y0 * sn;
        } else if (!known && e0[i] >= 0) {
          g0[i] = g1[i] = NAN;
        }
        dw0[i] += g0[i] * x0[i] * r;
        dw1[i] += g1[i] * x1[i] * r;
        g0[i] *= w0[i];
        g1[i] *= w1[i];
        dot += g0[i] * x0[i] + g1[i] * x1[i];
      }
      const float c = warp_sum(dot) * r * r * inv_d;
#pragma unroll
      for (int i = 0; i < kMaxPairs; ++i) {
        if (e0[i] >= 0) out[e0[i]] = from_f32<T>(r * (g0[i] - x0[i] * c));
        if (e1[i] >= 0) out[e1[i]] = from_f32<T>(r * (g1[i] - x1[i] * c));
      }
    }
  }
  if constexpr (BACKWARD) {
    if (s.dw == nullptr) return;
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
      if (e0[i] >= 0) sums[warp][e0[i]] = dw0[i];
      if (e1[i] >= 0) sums[warp][e1[i]] = dw1[i];
    }
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kWarps * 32) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += sums[w][d];
      a.partial[(int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * D + d] = t;
    }
  }
}

// Adds the blocks' weight-gradient sums in order.
__global__ void __launch_bounds__(256)
    qk_weight_finish_kernel(const QkProblem p, const float* partial,
                            int blocks) {
  __shared__ float sums[8][32];
  allow_dependents();
  grid_dependency_wait();
  const QkSide& s = p.side[blockIdx.y];
  if (s.dw == nullptr) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int d = blockIdx.x * 32 + lane;
  const float* src = partial + int64_t(blockIdx.y) * blocks * p.D;
  float t = 0.f;
  if (d < p.D)
    for (int c = warp; c < blocks; c += 8) t += src[int64_t(c) * p.D + d];
  sums[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && d < p.D) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += sums[w][lane];
    const int64_t i = d * s.sdw;
    if (s.w_dtype == VECTRA_F32)
      static_cast<float*>(s.dw)[i] = total;
    else if (s.w_dtype == VECTRA_F16)
      static_cast<__half*>(s.dw)[i] = from_f32<__half>(total);
    else
      static_cast<__nv_bfloat16*>(s.dw)[i] = from_f32<__nv_bfloat16>(total);
  }
}

int general_blocks(const QkProblem& p) {
  const int64_t h = p.side[0].H > p.side[1].H ? p.side[0].H : p.side[1].H;
  const int64_t blocks = (p.B * p.N * h + kWarps - 1) / kWarps;
  const int64_t most = int64_t(device_sm_count()) * 4;
  return int(blocks < 1 ? 1 : (blocks < most ? blocks : most));
}

}  // namespace

cudaError_t launch_qk_forward(const QkProblem& p, cudaStream_t stream) {
  if (p.B * p.N == 0 || p.D == 0 || p.side[0].H + p.side[1].H == 0)
    return cudaSuccess;
  const QkArgs a{p, nullptr};
  const cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(qk_general_kernel<T, false>,
                      dim3(unsigned(general_blocks(p)), 2), dim3(kWarps * 32),
                      0, stream, a);
  });
  if (e == cudaSuccess) count_launches(1);
  return e;
}

cudaError_t run_qk_backward(const QkProblem& p, Workspace& ws,
                            cudaStream_t stream) {
  if (p.D == 0) return cudaSuccess;
  const int blocks = general_blocks(p);
  const bool weights = p.side[0].dw || p.side[1].dw;
  QkArgs a{p, nullptr};
  if (weights)
    a.partial = static_cast<float*>(
        ws.take(size_t(2) * blocks * p.D * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;
  cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(qk_general_kernel<T, true>, dim3(unsigned(blocks), 2),
                      dim3(kWarps * 32), 0, stream, a);
  });
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (!weights) return cudaSuccess;
  e = launch_pdl(qk_weight_finish_kernel,
                 dim3(unsigned((p.D + 31) / 32), 2), dim3(256), 0, stream, p,
                 static_cast<const float*>(a.partial), blocks);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace vectra
