// block_grad.cu: the elementwise half of the backward passes, with the bias
// gradients in the same read.
//
//   linear: dz = dy * act'(z), db = sum of dz over rows
//   gated:  dg = dh * u * act'(g), du = dh * act(g), and their column sums
//
// Memory-bound: each input element is read once and each result written
// once. A block of 8 warps takes 32 * VEC columns and a chunk of rows; a
// thread keeps the sums of its columns in float32 (from the unrounded dz),
// the warps' sums are joined in shared memory and written per chunk, and a
// second kernel adds the chunks in order, so the result does not depend on
// scheduling. Measured (B200): gated, 66,560 x 704 bf16, 106 us for 656 MB (6.2
// TB/s, 0.95 of the copy rate) with the sums; rows' loads one at a time took
// 203.
#include "block_common.cuh"

namespace vectra {
namespace {

constexpr int kWarps = 8;
constexpr int kBlocksPerSm = 8;

struct GradArgs {
  GradProblem p;
  int64_t rows_per_chunk;
  float* partial;   // [chunks][N] sums (null: not wanted)
  float* partial2;
};

// VEC elements as loaded, converted when used.
template <typename T, int VEC>
struct Raw {
  union {
    uint4 u[VEC * sizeof(T) / 16 > 0 ? VEC * sizeof(T) / 16 : 1];
    T e[VEC];
  };
  __device__ __forceinline__ Raw() {}
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) {
      e[0] = *p;
    } else {
#pragma unroll
      for (int w = 0; w < int(VEC * sizeof(T) / 16); ++w)
        u[w] = __ldg(reinterpret_cast<const uint4*>(p) + w);
    }
  }
  __device__ __forceinline__ float at(int i) const { return to_f32(e[i]); }
};

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(v[0]);
  } else {
    constexpr int kWords = VEC * int(sizeof(T)) / 16;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      union {
        uint4 u;
        T e[16 / sizeof(T)];
      } raw;
#pragma unroll
      for (int i = 0; i < int(16 / sizeof(T)); ++i)
        raw.e[i] = from_f32<T>(v[w * int(16 / sizeof(T)) + i]);
      *(reinterpret_cast<uint4*>(p) + w) = raw.u;
    }
  }
}

template <typename T, int VEC, int ACT, bool GATED>
__global__ void __launch_bounds__(kWarps * 32)
    grad_kernel(const GradArgs a) {
  constexpr bool kExact = std::is_same<T, float>::value;
  constexpr int kSides = GATED ? 2 : 1;
  constexpr int kBatch = GATED ? 2 : 4;
  __shared__ float sums[kSides][kWarps][32 * VEC];
  const GradProblem& p = a.p;
  allow_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t n = int64_t(blockIdx.x) * 32 * VEC + lane * VEC;
  const int64_t r0 = int64_t(blockIdx.y) * a.rows_per_chunk;
  const int64_t r1 =
      r0 + a.rows_per_chunk < p.M ? r0 + a.rows_per_chunk : p.M;
  float sg[VEC], su[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sg[i] = su[i] = 0.f;
  if (n < p.N) {
    // kBatch rows' loads are issued before any of them is used.
    for (int64_t m0 = r0 + warp; m0 < r1; m0 += kWarps * kBatch) {
      Raw<T, VEC> dy[kBatch], z[GATED ? 1 : kBatch];
      Raw<float, VEC> g[GATED ? kBatch : 1], u[GATED ? kBatch : 1];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int64_t m = m0 + i * kWarps;
        if (m >= r1) break;
        dy[i].load(static_cast<const T*>(p.dy) + m * p.dy_sm + n * p.dy_sn);
        if constexpr (GATED) {
          g[i].load(p.gate + m * p.gate_ld + n);
          u[i].load(p.up + m * p.up_ld + n);
        } else if constexpr (ACT != VECTRA_ACT_NONE) {
          z[i].load(static_cast<const T*>(p.pre) + m * p.pre_ld + n);
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int64_t m = m0 + i * kWarps;
        if (m >= r1) break;
        float d1[VEC], d2[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = dy[i].at(j);
          float value;
          if constexpr (GATED) {
            const float slope = act_grad<kExact, ACT>(g[i].at(j), &value);
            d1[j] = d * u[i].at(j) * slope;
            d2[j] = d * value;
            su[j] += d2[j];
          } else if constexpr (ACT != VECTRA_ACT_NONE) {
            d1[j] = d * act_grad<kExact, ACT>(z[i].at(j), &value);
          } else {
            d1[j] = d;
          }
          sg[j] += d1[j];
        }
        if (GATED || p.dz)
          store_vec<T, VEC>(static_cast<T*>(p.dz) + m * p.dz_ld + n, d1);
        if constexpr (GATED)
          store_vec<T, VEC>(static_cast<T*>(p.dz2) + m * p.dz_ld + n, d2);
      }
    }
  }
  if (a.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    sums[0][warp][lane * VEC + i] = sg[i];
    if constexpr (GATED) sums[1][warp][lane * VEC + i] = su[i];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * VEC; c += kWarps * 32) {
    const int64_t col = int64_t(blockIdx.x) * 32 * VEC + c;
    if (col >= p.N) continue;
#pragma unroll
    for (int s = 0; s < kSides; ++s) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += sums[s][w][c];
      (s == 0 ? a.partial : a.partial2)[blockIdx.y * p.N + col] = t;
    }
  }
}

// Adds the chunks' sums: 32 warps share the chunks of 32 columns and are
// joined in shared memory.
template <typename T>
__global__ void __launch_bounds__(1024)
    colsum_finish_kernel(const float* partial, const float* partial2,
                         int chunks, int64_t N, T* out, T* out2) {
  __shared__ float sums[32][32];
  allow_dependents();
  grid_dependency_wait();
  const float* src = blockIdx.y ? partial2 : partial;
  T* dst = blockIdx.y ? out2 : out;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t n = int64_t(blockIdx.x) * 32 + lane;
  float t = 0.f;
  if (n < N) {
#pragma unroll 4
    for (int c = warp; c < chunks; c += 32) t += __ldg(src + c * N + n);
  }
  sums[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && n < N) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) total += sums[w][lane];
    dst[n] = from_f32<T>(total);
  }
}

template <typename T, int VEC>
cudaError_t launch_grad(const GradArgs& a, int chunks, cudaStream_t stream) {
  const GradProblem& p = a.p;
  const dim3 grid(unsigned((p.N + 32 * VEC - 1) / (32 * VEC)),
                  unsigned(chunks));
  return with_activation(p.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    return p.gated ? launch_pdl(grad_kernel<T, VEC, ACT, true>, grid,
                                dim3(kWarps * 32), 0, stream, a)
                   : launch_pdl(grad_kernel<T, VEC, ACT, false>, grid,
                                dim3(kWarps * 32), 0, stream, a);
  });
}

bool aligned(const void* p, int64_t ld, size_t es) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * es) % 16 == 0;
}

}  // namespace

cudaError_t run_grad(const GradProblem& p, Workspace& ws,
                     cudaStream_t stream) {
  if (p.N == 0 || (p.M == 0 && p.db == nullptr)) return cudaSuccess;
  const size_t es = p.dtype == VECTRA_F32 ? 4 : 2;
  // dz lies in the workspace, whose rows are aligned.
  const bool vec = p.N % 8 == 0 && p.dy_sn == 1 &&
                   aligned(p.dy, p.dy_sm, es) &&
                   (!p.pre || aligned(p.pre, p.pre_ld, es)) &&
                   (!p.gate || (aligned(p.gate, p.gate_ld, 4) &&
                                aligned(p.up, p.up_ld, 4)));
  // Chunks: enough blocks for kBlocksPerSm, at least 16 rows each, and
  // few enough that the chunk sums stay small beside the data.
  const int64_t cols = (p.N + (vec ? 255 : 31)) / (vec ? 256 : 32);
  int64_t chunks = (int64_t(device_sm_count()) * kBlocksPerSm + cols - 1) / cols;
  const int64_t most = (p.M + 15) / 16;
  if (chunks > most) chunks = most;
  if (chunks > 4096) chunks = 4096;
  if (chunks < 1) chunks = 1;
  GradArgs a{p, (p.M + chunks - 1) / chunks, nullptr, nullptr};
  if (a.rows_per_chunk < 1) a.rows_per_chunk = 1;
  if (p.db) {
    a.partial = static_cast<float*>(ws.take(chunks * p.N * sizeof(float)));
    if (p.gated)
      a.partial2 = static_cast<float*>(ws.take(chunks * p.N * sizeof(float)));
  }
  if (ws.dry || ws.overflow) return cudaSuccess;
  cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return vec ? launch_grad<T, 8>(a, int(chunks), stream)
               : launch_grad<T, 1>(a, int(chunks), stream);
  });
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (!p.db) return cudaSuccess;
  return launch_column_finish(p.dtype, a.partial, a.partial2, int(chunks),
                              p.N, p.db, p.db2, stream);
}

cudaError_t launch_column_finish(int32_t dtype, const float* partial,
                                 const float* partial2, int chunks, int64_t N,
                                 void* db, void* db2, cudaStream_t stream) {
  const cudaError_t e = with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(colsum_finish_kernel<T>,
                      dim3(unsigned((N + 31) / 32), db2 ? 2 : 1), dim3(1024),
                      0, stream, partial, partial2, chunks, N,
                      static_cast<T*>(db), static_cast<T*>(db2));
  });
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace vectra
