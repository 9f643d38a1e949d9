// cross_finish.cu: what attention to an encoder's states needs beside its
// tile kernels (cross.cuh): c_i = e_i . out_i before the backward pass, and
// the joins of an axis that was split over blocks, in the parts' order.
#include "cross.cuh"

namespace vectra {
namespace {

// Sixteen lanes a row, 16-byte pieces where rows allow them (VEC); memory-bound.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    delta_kernel(const __grid_constant__ CrossProblem p, float* delta) {
  allow_dependents();
  grid_dependency_wait();
  const int64_t rows = p.B * p.H * p.Nq;
  const int lane = threadIdx.x % 16;
  // The loop runs to the warp's last row: the sums need every lane.
  for (int64_t r0 = (int64_t(blockIdx.x) * 8 + threadIdx.x / 32) * 2; r0 < rows;
       r0 += int64_t(gridDim.x) * 16) {
    const int64_t r = r0 + threadIdx.x % 32 / 16;
    float t = 0.f;
    if (r < rows) {
      const int64_t bh = r / p.Nq, i = r - bh * p.Nq;
      const int64_t b = bh / p.H, h = bh - b * p.H;
      const T* o = static_cast<const T*>(p.out) + b * p.so[0] + h * p.so[1] +
                   i * p.so[2];
      const T* e = static_cast<const T*>(p.dout) + b * p.se[0] +
                   h * p.se[1] + i * p.se[2];
      const T* rest =
          p.rest ? static_cast<const T*>(p.rest) + r * p.Dv : nullptr;
      constexpr int N = VEC ? 16 / int(sizeof(T)) : 1;
      for (int d = lane * N; d < p.Dv; d += 16 * N) {
        union Piece {
          uint4 u;
          T e[N];
        } x, y, z;
        if constexpr (VEC) {
          x.u = __ldg(reinterpret_cast<const uint4*>(o + d));
          y.u = __ldg(reinterpret_cast<const uint4*>(e + d));
          if (rest) z.u = __ldg(reinterpret_cast<const uint4*>(rest + d));
        } else {
          x.e[0] = o[d];
          y.e[0] = e[d * p.se[3]];
          if (rest) z.e[0] = rest[d];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
          float v = to_f32(x.e[j]);
          if (rest) v = fmaf(to_f32(z.e[j]), 1.f / kRestLift<T>, v);
          t = fmaf(v, to_f32(y.e[j]), t);
        }
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0 && r < rows) delta[r] = t;
  }
}

// The sum of squares of a vector, by sixteen neighbouring lanes of a warp, all
// of which call it; `live`: there is one. 16-byte pieces.
template <typename T>
__device__ __forceinline__ float vector_square(const T* x, bool live,
                                               int width) {
  float t = 0.f;
  if (live) {
    for (int d = threadIdx.x % 16 * 8; d < width; d += 128) {
      union {
        uint4 u;
        T e[8];
      } y;
      if (d + 8 <= width) {
        y.u = __ldg(reinterpret_cast<const uint4*>(x + d));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          y.e[j] = d + j < width ? x[d + j] : from_f32<T>(0.f);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = to_f32(y.e[j]);
        t = fmaf(v, v, t);
      }
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// Sixteen lanes a key (bf16 and f16).
template <typename T>
__global__ void __launch_bounds__(256)
    squares_kernel(const __grid_constant__ CrossProblem p, float* squares) {
  allow_dependents();
  grid_dependency_wait();
  const int64_t rows = p.B * p.Hk * p.Nk;
  const int lane = threadIdx.x % 16;
  for (int64_t r0 = (int64_t(blockIdx.x) * 8 + threadIdx.x / 32) * 2; r0 < rows;
       r0 += int64_t(gridDim.x) * 16) {
    const int64_t r = r0 + threadIdx.x % 32 / 16;
    const bool live = r < rows;
    const int64_t bh = live ? r / p.Nk : 0, i = live ? r - bh * p.Nk : 0;
    const int64_t b = bh / p.Hk, h = bh - b * p.Hk;
    const float t = vector_square<T>(static_cast<const T*>(p.k) + b * p.sk[0] +
                                         h * p.sk[1] + i * p.sk[2],
                                     live, p.D);
    if (lane == 0 && live) squares[r] = t;
  }
}

// `parts` blocks a key head of a sequence, which take its seen values and then
// its packed queries' gradients in turn. Maxima do not depend on the order.
__global__ void __launch_bounds__(256)
    bounds_kernel(const __grid_constant__ CrossProblem p, float* bounds,
                  int parts) {
  using T = __half;
  __shared__ float tops[8][2];
  allow_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t plane = blockIdx.x / parts;
  const int part = int(blockIdx.x - plane * parts);
  const int64_t b = plane / p.Hk, hk = plane - b * p.Hk;
  const int64_t len = cross_length(p, b), rows = len > 0 ? p.Nq * p.G : 0;
  const int64_t first = (int64_t(part) * 8 + warp) * 2 + lane / 16;
  const int64_t step = int64_t(parts) * 16;
  float top[2] = {0.f, 0.f};
  // The loops run to the warp's last row: the sums need every lane.
  for (int64_t r = first; r - lane / 16 < len; r += step) {
    const bool live = r < len;
    const T* v = static_cast<const T*>(p.v) + b * p.sv[0] + hk * p.sv[1] +
                 (live ? r : 0) * p.sv[2];
    top[1] = fmaxf(top[1], sqrtf(vector_square<T>(v, live, p.Dv)));
  }
  for (int64_t r = first; r - lane / 16 < rows; r += step) {
    const bool live = r < rows;
    const int64_t i = live ? r / p.G : 0;
    const int64_t h = hk * p.G + (live ? r - i * p.G : 0);
    const T* e = static_cast<const T*>(p.dout) + b * p.se[0] + h * p.se[1] +
                 i * p.se[2];
    const float size = sqrtf(vector_square<T>(e, live, p.Dv));
    top[0] = fmaxf(top[0], 2.f * fabsf(cross_scale(p, b, h)) * size);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top[i] = warp_max(top[i]);
    if (lane == 0) tops[warp][i] = top[i];
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    float t = 0.f;
    for (int w = 0; w < 8; ++w) t = fmaxf(t, tops[w][threadIdx.x]);
    // Floats that are not negative are ordered as their bits are.
    atomicMax(reinterpret_cast<unsigned int*>(bounds + plane * 2) +
                  threadIdx.x,
              __float_as_uint(t));
  }
}

// One warp a row: the largest maximum over the parts, then every part's sum
// and result brought to it.
template <typename T>
__global__ void __launch_bounds__(256)
    join_kernel(const __grid_constant__ CrossProblem p) {
  allow_dependents();
  grid_dependency_wait();
  const int64_t rows = p.B * p.H * p.Nq;
  const int lane = threadIdx.x % 32;
  for (int64_t r = int64_t(blockIdx.x) * 8 + threadIdx.x / 32; r < rows;
       r += int64_t(gridDim.x) * 8) {
    const int64_t bh = r / p.Nq, i = r - bh * p.Nq;
    const int64_t b = bh / p.H, h = bh - b * p.H;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + r;
    // Two parts a lane (64 at most): their factors, then the sums over parts
    // with four parts' loads under way.
    float2 own[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = lane + 32 * i;
      own[i] = s < p.splits ? ml[s * rows] : make_float2(kNegInf, 0.f);
    }
    // A maximum leaves NaN out, a sum does not: either makes the row NaN.
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      odd = odd || own[i].x != own[i].x || own[i].y != own[i].y;
    const float m = __any_sync(0xffffffffu, odd)
                        ? NAN
                        : warp_max(fmaxf(own[0].x, own[1].x));
    float f[2], l = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // A part whose keys all weigh nothing (or that has none) adds nothing.
      f[i] = own[i].x == kNegInf ? 0.f : fast_exp2(own[i].x - m);
      l += own[i].y * f[i];
    }
    l = warp_sum(l);
    float acc[kMaxCrossWidth / 32];
#pragma unroll
    for (int c = 0; c < kMaxCrossWidth / 32; ++c) acc[c] = 0.f;
    for (int s0 = 0; s0 < p.splits; s0 += 4) {
      float v[4][kMaxCrossWidth / 32];
      float by[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = s0 + i;
        by[i] = __shfl_sync(0xffffffffu, s < 32 ? f[0] : f[1], s & 31);
        const float* o = p.part + (s * rows + r) * p.Dv;
#pragma unroll
        for (int c = 0; c < kMaxCrossWidth / 32; ++c)
          v[i][c] = s < p.splits && c * 32 + lane < p.Dv ? o[c * 32 + lane]
                                                         : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < kMaxCrossWidth / 32; ++c)
          acc[c] = fmaf(v[i][c], by[i], acc[c]);  // 0 * NaN of a far part too
    }
    const bool any = cross_length(p, b) > 0;
    T* out = static_cast<T*>(p.out) + b * p.so[0] + h * p.so[1] + i * p.so[2];
    T* rest = p.rest ? static_cast<T*>(p.rest) + r * p.Dv : nullptr;
#pragma unroll
    for (int c = 0; c < kMaxCrossWidth / 32; ++c) {
      const int d = c * 32 + lane;
      if (d < p.Dv)
        store_with_rest<T>(out + d, rest ? rest + d : nullptr,
                           any ? acc[c] / l : 0.f);
    }
    if (p.lse && lane == 0) p.lse[r] = any ? m + log2f(l) : INFINITY;
  }
}

struct SumArgs {
  const float* part;
  void* out;
  int64_t H, N, rows;
  int64_t so[3];
  int splits, width;
};
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const SumArgs a) {
  allow_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x % 32;
  for (int64_t r = int64_t(blockIdx.x) * 8 + threadIdx.x / 32; r < a.rows;
       r += int64_t(gridDim.x) * 8) {
    const int64_t bh = r / a.N, i = r - bh * a.N;
    const int64_t b = bh / a.H, h = bh - b * a.H;
    T* out = static_cast<T*>(a.out) + b * a.so[0] + h * a.so[1] + i * a.so[2];
    for (int d = lane; d < a.width; d += 32) {
      float t = 0.f;
#pragma unroll 4
      for (int s = 0; s < a.splits; ++s)
        t += __ldg(a.part + (s * a.rows + r) * a.width + d);
      out[d] = from_f32<T>(t);
    }
  }
}

// `warps` warps (of a block of eight) a head of a sequence. A row's three sums
// over its parts are X = sum z d, Y = sum P d and Z = sum z, of distances d; its
// share is -(X - Y Z), where Z is what rounding left of zero.
__global__ void __launch_bounds__(256)
    dscale_kernel(const __grid_constant__ CrossProblem p, int splits,
                  int warps) {
  __shared__ double sums[8];
  allow_dependents();
  grid_dependency_wait();
  const int64_t rows = p.B * p.H * p.Nq;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t head = int64_t(blockIdx.x) * (8 / warps) + warp / warps;
  double t = 0.0;
  if (head < p.B * p.H) {
    const int64_t first = head * p.Nq;
    for (int64_t i = warp % warps * 32 + lane; i < p.Nq; i += warps * 32) {
      float x = 0.f, y = 0.f, z = 0.f;
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const float* w = p.dscale_rows + (s * rows + first + i) * 3;
        x += __ldg(w);
        y += __ldg(w + 1);
        z += __ldg(w + 2);
      }
      // Rounded products: over a single key the difference is exactly zero.
      t -= double(__fsub_rn(x, __fmul_rn(y, z)));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (lane == 0) sums[warp] = t;
  __syncthreads();
  if (lane == 0 && warp % warps == 0 && head < p.B * p.H) {
    for (int w = 1; w < warps; ++w) t += sums[warp + w];
    p.dscale[head] = float(t);
  }
}

unsigned row_blocks(int64_t rows) {
  const int64_t blocks = (rows + 7) / 8;
  const int64_t most = int64_t(device_sm_count()) * 16;
  return unsigned(blocks < most ? blocks : most);
}

}  // namespace

cudaError_t launch_cross_delta(const CrossProblem& p, float* delta,
                               cudaStream_t stream) {
  const int64_t rows = p.B * p.H * p.Nq;
  if (rows == 0) return cudaSuccess;
  count_launches(1);
  return with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int64_t sizes[3] = {p.B, p.H, p.Nq};
    const auto whole = [&](const void* base, const int64_t* s) {
      bool ok = (reinterpret_cast<uintptr_t>(base) & 15) == 0;
      for (int i = 0; i < 3; ++i)
        ok = ok && (sizes[i] <= 1 || s[i] * int64_t(sizeof(T)) % 16 == 0);
      return ok;
    };
    const bool vec = p.Dv * sizeof(T) % 16 == 0 && whole(p.out, p.so) &&
                     whole(p.dout, p.se) && (p.se[3] == 1 || p.Dv == 1) &&
                     (reinterpret_cast<uintptr_t>(p.rest) & 15) == 0;
    return launch_pdl(vec ? delta_kernel<T, true> : delta_kernel<T, false>,
                      dim3(row_blocks((rows + 1) / 2)), dim3(256), 0, stream,
                      p, delta);
  });
}

cudaError_t launch_cross_squares(const CrossProblem& p, float* squares,
                                 cudaStream_t stream) {
  const int64_t rows = p.B * p.Hk * p.Nk;
  if (rows == 0) return cudaSuccess;
  count_launches(1);
  const dim3 grid(row_blocks((rows + 1) / 2));
  if (p.dtype == VECTRA_BF16)
    return launch_pdl(squares_kernel<__nv_bfloat16>, grid, dim3(256), 0,
                      stream, p, squares);
  return launch_pdl(squares_kernel<__half>, grid, dim3(256), 0, stream, p,
                    squares);
}

cudaError_t launch_cross_bounds(const CrossProblem& p, float* bounds,
                                cudaStream_t stream) {
  const int64_t planes = p.B * p.Hk;
  const cudaError_t e =
      cudaMemsetAsync(bounds, 0, size_t(planes) * 2 * sizeof(float), stream);
  if (e != cudaSuccess) return e;
  // A block takes 64 rows or more of each kind.
  const int64_t most = p.Nk > p.Nq * p.G ? p.Nk : p.Nq * p.G;
  int64_t parts = int64_t(device_sm_count()) * 8 / planes;
  if (parts > most / 64) parts = most / 64;
  if (parts < 1) parts = 1;
  if (planes * parts > 0x7fffffff) return cudaErrorInvalidValue;
  count_launches(1);
  return launch_pdl(bounds_kernel, dim3(unsigned(planes * parts)), dim3(256),
                    0, stream, p, bounds, int(parts));
}

cudaError_t launch_cross_join(const CrossProblem& p, cudaStream_t stream) {
  const int64_t rows = p.B * p.H * p.Nq;
  if (rows == 0) return cudaSuccess;
  count_launches(1);
  return with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(join_kernel<T>, dim3(row_blocks(rows)), dim3(256), 0,
                      stream, p);
  });
}

cudaError_t launch_cross_sum(int32_t dtype, const float* part, int splits,
                             int64_t B, int64_t H, int64_t N, int width,
                             void* out, const int64_t* so,
                             cudaStream_t stream) {
  const SumArgs a{part, out, H, N, B * H * N, {so[0], so[1], so[2]}, splits,
                  width};
  if (a.rows == 0 || width == 0) return cudaSuccess;
  count_launches(1);
  return with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(sum_kernel<T>, dim3(row_blocks(a.rows)), dim3(256), 0,
                      stream, a);
  });
}

cudaError_t launch_cross_dscale(const CrossProblem& p, int splits,
                                cudaStream_t stream) {
  if (p.B * p.H == 0) return cudaSuccess;
  count_launches(1);
  const int warps = p.Nq > 64 ? 8 : 1;
  const int64_t per = 8 / warps;
  return launch_pdl(dscale_kernel, dim3(unsigned((p.B * p.H + per - 1) / per)),
                    dim3(256), 0, stream, p, splits, warps);
}

}  // namespace vectra
