// residual_norm.cu: dropout, and what stands between two sublayers of a
// transformer block: the norm of a sublayer's result, dropout, its gate, the
// scaled residual and the next sublayer's norm, in one pass, with its
// backward pass.
//
//   u = n0 bw, n0 = norm(branch)          (bw given; else u = branch)
//   x_out = a x + gate d, d = dropout(u)
//   y = n1 w + b, n1 = norm(x_out)
// and for upstream gradients e of x_out and f of y, with c(.) the mean of a
// row and r the factors of the norms:
//   dw = sum f n1, db = sum f
//   g = e + r1 (f w - n1 c(f w n1) [- c(f w)])     (brackets: layer norm)
//   dx = a g, dgate = sum g d, h = dropout'(g gate)
//   dbw = sum h n0, dbranch = r0 (h bw - n0 c(h bw n0) [- c(h bw)])
// Rows are held in float32 registers between their reading and writing; sums
// over rows are joined in a fixed order, without atomics.
//
// Memory-bound. A team of threads (a warp up to 512 columns, else a block)
// owns a row: each thread holds one or two chunks of 8 neighbouring columns,
// the same for every row, so that it can keep its columns' sums over rows in
// registers.
#include <type_traits>

#include "block_common.cuh"
#include "philox.cuh"
#include "residual_norm.cuh"

namespace vectra {
namespace {

constexpr int kChunk = 8;  // columns a thread reads at once

template <typename T>
struct Raw {
  static constexpr int N = int(sizeof(T)) / 2;  // 16-byte pieces
  uint4 u[N];
};

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float* v) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(r.u[i].x);
      v[4 * i + 1] = __uint_as_float(r.u[i].y);
      v[4 * i + 2] = __uint_as_float(r.u[i].z);
      v[4 * i + 3] = __uint_as_float(r.u[i].w);
    }
  } else {
    const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f =
            __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw<T> pack(const float* v) {
  Raw<T> r;
  union {
    T e[kChunk];
    uint4 u[Raw<T>::N];
  } c;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) c.e[i] = from_f32<T>(v[i]);
#pragma unroll
  for (int i = 0; i < Raw<T>::N; ++i) r.u[i] = c.u[i];
  return r;
}

// Eight columns from `col` of a row of `cols`; columns outside are 0. VEC:
// whole 16-byte pieces, cols a multiple of 8.
template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> load_raw(const void* row, int64_t inner,
                                           int col, int cols) {
  Raw<T> r;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < Raw<T>::N; ++i) {
      r.u[i] = make_uint4(0, 0, 0, 0);
      if (col < cols)
        r.u[i] = __ldg(reinterpret_cast<const uint4*>(
                           static_cast<const T*>(row) + col) +
                       i);
    }
  } else {
    union {
      T e[kChunk];
      uint4 u[Raw<T>::N];
    } c;
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      c.e[i] = col + i < cols
                   ? static_cast<const T*>(row)[(col + i) * inner]
                   : from_f32<T>(0.f);
#pragma unroll
    for (int i = 0; i < Raw<T>::N; ++i) r.u[i] = c.u[i];
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const void* row, int64_t inner, int col,
                                      int cols, float* v) {
  unpack<T>(load_raw<T, VEC>(row, inner, col, cols), v);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(void* row, int col, int cols,
                                       const float* v) {
  T* p = static_cast<T*>(row) + col;
  if constexpr (VEC) {
    if (col >= cols) return;
    const Raw<T> r = pack<T>(v);
#pragma unroll
    for (int i = 0; i < Raw<T>::N; ++i)
      reinterpret_cast<uint4*>(p)[i] = r.u[i];
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (col + i < cols) p[i] = from_f32<T>(v[i]);
  }
}

// Whether elements first .. first + 7 are kept. ALIGNED: first is a multiple
// of 8, else two groups' numbers meet in a chunk.
template <bool ALIGNED>
__device__ __forceinline__ uint32_t keep8(const PhiloxKey& key, int64_t first,
                                          uint32_t cut) {
  const uint64_t g = uint64_t(first) >> 3;
  uint32_t bits = keep_bits(key, g, cut);
  if constexpr (!ALIGNED) {
    const int off = int(first & 7);
    bits = (bits | keep_bits(key, g + 1, cut) << 8) >> off;
  }
  return bits;
}

// ---------------------------------------------------------------------------
// Dropout.
// ---------------------------------------------------------------------------
struct DropArgs {
  const void* x;
  void* y;
  int64_t rows, cols, ld, inner;  // x; y is contiguous
  Drop drop;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const DropArgs a) {
  allow_dependents();
  grid_dependency_wait();
  const PhiloxKey key = load_key(a.drop);
  const int64_t n = a.rows * a.cols;
  const int64_t groups = (n + kChunk - 1) / kChunk;
  for (int64_t g = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; g < groups;
       g += int64_t(gridDim.x) * blockDim.x) {
    const int64_t e = g * kChunk;
    float v[kChunk];
    if constexpr (VEC) {
      const int64_t r = a.rows == 1 ? 0 : e / a.cols;
      const T* p = static_cast<const T*>(a.x) + r * a.ld + (e - r * a.cols);
      load8<T, true>(p, 1, 0, kChunk, v);
    } else {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        v[i] = 0.f;
        if (e + i >= n) continue;
        const int64_t r = (e + i) / a.cols, c = e + i - r * a.cols;
        v[i] = to_f32(static_cast<const T*>(a.x)[r * a.ld + c * a.inner]);
      }
    }
    const uint32_t keep = keep_bits(key, uint64_t(g), a.drop.cut);
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      v[i] = keep >> i & 1 ? v[i] * a.drop.scale : 0.f;
    T* out = static_cast<T*>(a.y) + e;
    if constexpr (VEC) {
      store8<T, true>(out, 0, kChunk, v);
    } else {
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
        if (e + i < n) out[i] = from_f32<T>(v[i]);
    }
  }
}

// ---------------------------------------------------------------------------
// Norms.
// ---------------------------------------------------------------------------
// Sums of two values over the team. A block's team writes its warps' sums to
// one of two places in turn, so one barrier a sum is enough.
struct TeamSum {
  float2 (*part)[32];
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float a, float b) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (blockDim.x == 32) return make_float2(a, b);
    const int lane = threadIdx.x % 32;
    if (lane == 0) part[turn][threadIdx.x / 32] = make_float2(a, b);
    __syncthreads();
    float2 v = make_float2(0.f, 0.f);
    if (lane < int(blockDim.x) / 32) v = part[turn][lane];
    turn ^= 1;
    return make_float2(warp_sum(v.x), warp_sum(v.y));
  }
};

// mean (0 unless LAYER) and factor of the row in v, `count` of whose NC * 8
// values a thread holds are in the row.
template <int NC>
__device__ __forceinline__ float2 row_norm(TeamSum& sum, bool layer,
                                           const float (*v)[kChunk],
                                           const int* live, float inv_c,
                                           float eps) {
  float s = 0.f, mean = 0.f;
  if (layer) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < kChunk; ++i) s += v[c][i];  // 0 outside the row
    mean = sum(s, 0.f).x * inv_c;
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const float t = v[c][i] - mean;
      ss += i < live[c] ? t * t : 0.f;
    }
  return make_float2(mean, rsqrtf(sum(ss, 0.f).x * inv_c + eps));
}

template <typename T, int NC, bool VEC>
__global__ void __launch_bounds__(1024)
    norm_forward_kernel(const __grid_constant__ NormProblem p) {
  __shared__ float2 part[2][32];
  TeamSum sum{part};
  allow_dependents();
  grid_dependency_wait();
  const int C = p.C;
  const float inv_c = 1.f / float(C);
  const PhiloxKey key = load_key(p.drop);
  int col[NC], live[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = (c * int(blockDim.x) + int(threadIdx.x)) * kChunk;
    live[c] = min(max(C - col[c], 0), kChunk);
  }
  for (int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
       row < p.M; row += int64_t(gridDim.x) * blockDim.y) {
    float v[NC][kChunk];
    float4 stats = make_float4(0.f, 0.f, 0.f, 0.f);
    const char* x = p.x.row<T>(row);
    if (p.branch.p == nullptr) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        load8<T, VEC>(x, p.x.inner, col[c], C, v[c]);
    } else {
      Raw<T> rx[NC];
      const char* br = p.branch.row<T>(row);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        rx[c] = load_raw<T, VEC>(x, p.x.inner, col[c], C);
        load8<T, VEC>(br, p.branch.inner, col[c], C, v[c]);
      }
      if (p.branch_weight.p) {
        const float2 n = row_norm<NC>(sum, p.layer, v, live, inv_c, p.eps);
        stats.z = n.x;
        stats.w = n.y;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float w[kChunk];
          load8<T, VEC>(p.branch_weight.p, p.branch_weight.inner, col[c], C,
                        w);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) v[c][i] = (v[c][i] - n.x) * n.y * w[i];
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (p.drop.cut && live[c] > 0) {
          const uint32_t keep =
              keep8<VEC>(key, row * C + col[c], p.drop.cut);
#pragma unroll
          for (int i = 0; i < kChunk; ++i)
            v[c][i] = keep >> i & 1 ? v[c][i] * p.drop.scale : 0.f;
        }
        if (p.gate.p) {
          float g[kChunk];
          load8<T, VEC>(p.gate.row<T>(row / p.gate_rows), p.gate.inner, col[c],
                        C, g);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) v[c][i] *= g[i];
        }
        float xv[kChunk];
        unpack<T>(rx[c], xv);
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
          v[c][i] = fmaf(p.residual_scale, xv[i], v[c][i]);
        store8<T, VEC>(static_cast<T*>(p.x_out) + row * C, col[c], C, v[c]);
      }
    }
    if (p.y) {
      const float2 n = row_norm<NC>(sum, p.layer, v, live, inv_c, p.eps);
      stats.x = n.x;
      stats.y = n.y;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float w[kChunk], b[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          w[i] = 1.f;
          b[i] = 0.f;
        }
        if (p.weight.p)
          load8<T, VEC>(p.weight.p, p.weight.inner, col[c], C, w);
        if (p.bias.p) load8<T, VEC>(p.bias.p, p.bias.inner, col[c], C, b);
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
          v[c][i] = fmaf((v[c][i] - n.x) * n.y, w[i], b[i]);
        store8<T, VEC>(static_cast<T*>(p.y) + row * C, col[c], C, v[c]);
      }
    }
    if (p.stats && threadIdx.x == 0)
      reinterpret_cast<float4*>(p.stats)[row] = stats;
  }
}

// Backward. A unit is `unit_rows` rows of one gate row's group; the teams take
// units in turn. A team's sums for the weights stay in registers to its end;
// those for a gate that rows share are written at the end of each unit.
template <typename T, int NC, bool VEC, bool NORM0, bool GATE>
__global__ void __launch_bounds__(NC == 1 ? 256 : 512)
    norm_backward_kernel(const __grid_constant__ NormProblem p) {
  __shared__ float2 part[2][32];
  TeamSum sum{part};
  allow_dependents();
  grid_dependency_wait();
  const int C = p.C;
  const float inv_c = 1.f / float(C);
  const PhiloxKey key = load_key(p.drop);
  int col[NC];
  float dw[NC][kChunk], db[NC][kChunk];
  float dbw[NORM0 ? NC : 1][kChunk];
  float dgate[GATE ? NC : 1][kChunk];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = (c * int(blockDim.x) + int(threadIdx.x)) * kChunk;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      dw[c][i] = db[c][i] = 0.f;
      if constexpr (NORM0) dbw[c][i] = 0.f;
      if constexpr (GATE) dgate[c][i] = 0.f;
    }
  }
  const int64_t team = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t teams = int64_t(gridDim.x) * blockDim.y;
  for (int64_t unit = team; unit < p.units; unit += teams) {
    const int64_t group = unit / p.units_per_group;
    const int64_t first = (unit - group * p.units_per_group) * p.unit_rows;
    const int64_t group_rows = GATE ? p.gate_rows : p.M;
    const int64_t row0 = group * group_rows + first;
    const int64_t row1 = group * group_rows +
                         min(first + int64_t(p.unit_rows), group_rows);
    for (int64_t row = row0; row < row1; ++row) {
      // g, the gradient of x_out.
      float g[NC][kChunk];
      Raw<T> rb[NC];
      float4 stats = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.stats) stats = __ldg(reinterpret_cast<const float4*>(p.stats) + row);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        if (p.branch.p)
          rb[c] = load_raw<T, VEC>(p.branch.row<T>(row), p.branch.inner,
                                   col[c], C);
        else
          rb[c] = Raw<T>{};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (p.e.p) {
          load8<T, VEC>(p.e.row<T>(row), p.e.inner, col[c], C, g[c]);
        } else {
#pragma unroll
          for (int i = 0; i < kChunk; ++i) g[c][i] = 0.f;
        }
      }
      if (p.f.p) {
        Raw<T> rn[NC], rf[NC];
        float fn = 0.f, fs = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          rn[c] = load_raw<T, VEC>(p.x.row<T>(row), p.x.inner, col[c], C);
          rf[c] = load_raw<T, VEC>(p.f.row<T>(row), p.f.inner, col[c], C);
        }
        float w[NC][kChunk];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
          for (int i = 0; i < kChunk; ++i) w[c][i] = 1.f;
          if (p.weight.p)
            load8<T, VEC>(p.weight.p, p.weight.inner, col[c], C, w[c]);
          float n[kChunk], f[kChunk];
          unpack<T>(rn[c], n);
          unpack<T>(rf[c], f);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            n[i] = (n[i] - stats.x) * stats.y;
            // Outside the row f is 0.
            dw[c][i] = fmaf(f[i], n[i], dw[c][i]);
            db[c][i] += f[i];
            const float fw = f[i] * w[c][i];
            fn = fmaf(fw, n[i], fn);
            fs += fw;
          }
        }
        const float2 s = sum(fn, p.layer ? fs : 0.f);
        const float cn = s.x * inv_c, cs = s.y * inv_c;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float n[kChunk], f[kChunk];
          unpack<T>(rn[c], n);
          unpack<T>(rf[c], f);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            n[i] = (n[i] - stats.x) * stats.y;
            g[c][i] = fmaf(stats.y, f[i] * w[c][i] - n[i] * cn - cs, g[c][i]);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (!p.dx) break;
        float t[kChunk];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) t[i] = g[c][i] * p.residual_scale;
        store8<T, VEC>(static_cast<T*>(p.dx) + row * C, col[c], C, t);
      }
      if (!NORM0 && !p.dbranch && !p.dgate) continue;
      // h, the gradient of u.
      float hn = 0.f, hs = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float u[kChunk];
        unpack<T>(rb[c], u);
        uint32_t keep = 0xff;
        if (p.drop.cut) keep = keep8<VEC>(key, row * C + col[c], p.drop.cut);
        float bw[kChunk];
        if constexpr (NORM0) {
          load8<T, VEC>(p.branch_weight.p, p.branch_weight.inner, col[c], C,
                        bw);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) u[i] = (u[i] - stats.z) * stats.w;
        }
        if constexpr (GATE) {
          float gate[kChunk], own[kChunk];
          load8<T, VEC>(p.gate.row<T>(group), p.gate.inner, col[c], C, gate);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            float d = NORM0 ? u[i] * bw[i] : u[i];
            d = keep >> i & 1 ? d * p.drop.scale : 0.f;
            own[i] = g[c][i] * d;
            dgate[c][i] += own[i];
            g[c][i] *= gate[i];
          }
        }
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          const float h = keep >> i & 1 ? g[c][i] * p.drop.scale : 0.f;
          g[c][i] = h;
          if constexpr (NORM0) {
            if (col[c] + i < C) dbw[c][i] = fmaf(h, u[i], dbw[c][i]);
            g[c][i] = h * bw[i];  // 0 outside the row
            hn = fmaf(g[c][i], u[i], hn);
            hs += g[c][i];
          }
        }
      }
      if constexpr (NORM0) {
        const float2 s = sum(hn, p.layer ? hs : 0.f);
        const float cn = s.x * inv_c, cs = s.y * inv_c;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float u[kChunk];
          unpack<T>(rb[c], u);
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            u[i] = (u[i] - stats.z) * stats.w;
            g[c][i] = stats.w * (g[c][i] - u[i] * cn - cs);
          }
        }
      }
      if (p.dbranch) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          store8<T, VEC>(static_cast<T*>(p.dbranch) + row * C, col[c], C,
                         g[c]);
      }
    }
    if constexpr (GATE) {
      // One unit a gate row: its sum is the gradient.
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (p.dgate && p.units_per_group == 1)
          store8<T, VEC>(static_cast<T*>(p.dgate) + group * C, col[c], C,
                         dgate[c]);
        else if (p.dgate)
          store8<float, VEC>(p.gate_part + unit * C, col[c], C, dgate[c]);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) dgate[c][i] = 0.f;
      }
    }
  }
  // The blocks' sums: a block's teams join theirs through shared memory.
  __shared__ float joined[8][512 + 8];
  const auto flush = [&](int k, const float (*own)[kChunk]) {
    if (p.part[k] == nullptr) return;
    float* out = p.part[k] + int64_t(blockIdx.x) * C;
    if (blockDim.y == 1) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        store8<float, VEC>(out, col[c], C, own[c]);
      return;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
        if (col[c] + i < C) joined[threadIdx.y][col[c] + i] = own[c][i];
    __syncthreads();
    for (int q = threadIdx.y * 32 + threadIdx.x; q < C;
         q += blockDim.y * blockDim.x) {
      float t = 0.f;
      for (int j = 0; j < int(blockDim.y); ++j) t += joined[j][q];
      out[q] = t;
    }
  };
  flush(0, dw);
  flush(1, db);
  if constexpr (NORM0) flush(2, dbw);
}

// out[g, col] = sum over `count` consecutive rows of `part` in order.
struct FinishArgs {
  const float* part[3];
  void* out[3];
  int64_t count;   // rows a sum
  int64_t groups;  // sums
  int C;
};
template <typename T>
__global__ void __launch_bounds__(256) norm_finish_kernel(const FinishArgs a) {
  __shared__ float sums[8][33];
  allow_dependents();
  grid_dependency_wait();
  const int k = blockIdx.z;
  if (a.out[k] == nullptr) return;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int col = blockIdx.x * 32 + lane;
  for (int64_t g = blockIdx.y; g < a.groups; g += gridDim.y) {
    const float* p = a.part[k] + g * a.count * a.C;
    float t = 0.f;
    if (col < a.C) {
#pragma unroll 4
      for (int64_t r = warp; r < a.count; r += 8) t += __ldg(p + r * a.C + col);
    }
    sums[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && col < a.C) {
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) total += sums[w][lane];
      static_cast<T*>(a.out[k])[g * a.C + col] = from_f32<T>(total);
    }
    __syncthreads();
  }
}

bool rows_vec(const RowView& v, int64_t rows, int es) {
  return v.p == nullptr ||
         ((reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.inner == 1 &&
          (rows <= 1 || v.ld * es % 16 == 0));
}
bool ptr_vec(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

bool all_vec(const NormProblem& p) {
  const int es = p.dtype == VECTRA_F32 ? 4 : 2;
  return p.C % kChunk == 0 && rows_vec(p.x, p.M, es) &&
         rows_vec(p.branch, p.M, es) && rows_vec(p.weight, 1, es) &&
         rows_vec(p.bias, 1, es) && rows_vec(p.branch_weight, 1, es) &&
         rows_vec(p.gate, p.gate_count, es) && rows_vec(p.e, p.M, es) &&
         rows_vec(p.f, p.M, es) && ptr_vec(p.x_out) && ptr_vec(p.y) &&
         ptr_vec(p.dx) && ptr_vec(p.dbranch) && ptr_vec(p.dgate);
}

// A row's team: chunks a thread, threads, teams a block. A warp up to 512
// columns; above, a block, whose threads hold two chunks.
struct Team {
  int nc;
  dim3 block;
};
Team team_of(int C) {
  if (C <= 512) return {C <= 256 ? 1 : 2, dim3(32, 8)};
  const int per = 2 * 32 * kChunk;
  return {2, dim3(unsigned((C + per - 1) / per * 32), 1)};
}

template <typename F>
cudaError_t with_bool(bool v, F&& f) {
  return v ? f(std::true_type{}) : f(std::false_type{});
}

template <typename F>
cudaError_t with_chunks(int nc, F&& f) {
  return nc == 1 ? f(std::integral_constant<int, 1>{})
                 : f(std::integral_constant<int, 2>{});
}
// The backward kernel's block has 512 threads at most, for their registers;
// four chunks cover the rows that two do not (and spill: rows that wide are
// rare).
template <typename F>
cudaError_t with_more_chunks(int nc, F&& f) {
  return nc == 4 ? f(std::integral_constant<int, 4>{})
                 : with_chunks(nc, std::forward<F>(f));
}

}  // namespace

cudaError_t launch_dropout(int32_t dtype, const RowView& x, int64_t rows,
                           int64_t cols, void* y, const Drop& drop,
                           cudaStream_t stream) {
  if (rows * cols == 0) return cudaSuccess;
  DropArgs a{x.p, y, rows, cols, x.ld, x.inner, drop};
  const bool flat = x.inner == 1 && (rows == 1 || x.ld == cols);
  if (flat) {
    a.cols = rows * cols;
    a.rows = 1;
  }
  const int es = dtype == VECTRA_F32 ? 4 : 2;
  const bool vec =
      a.cols % kChunk == 0 && rows_vec(x, a.rows, es) && ptr_vec(y);
  const int64_t groups = (a.rows * a.cols + kChunk - 1) / kChunk;
  int64_t blocks = (groups + 255) / 256;
  const int64_t most = int64_t(device_sm_count()) * 8;
  if (blocks > most) blocks = most;
  const cudaError_t e = with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_pdl(vec ? dropout_kernel<T, true> : dropout_kernel<T, false>,
                      dim3(unsigned(blocks)), dim3(256), 0, stream, a);
  });
  if (e == cudaSuccess) count_launches(1);
  return e;
}

cudaError_t launch_norm_forward(const NormProblem& p, cudaStream_t stream) {
  if (p.M == 0 || p.C == 0) return cudaSuccess;
  const Team team = team_of(p.C);
  int64_t blocks = (p.M + team.block.y - 1) / team.block.y;
  const int64_t most = int64_t(device_sm_count()) *
                       (2048 / int(team.block.x * team.block.y));
  if (blocks > most) blocks = most;
  const bool vec = all_vec(p);
  const cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_chunks(team.nc, [&](auto nc) {
      constexpr int NC = decltype(nc)::value;
      return launch_pdl(vec ? norm_forward_kernel<T, NC, true>
                            : norm_forward_kernel<T, NC, false>,
                        dim3(unsigned(blocks)), team.block, 0, stream, p);
    });
  });
  if (e == cudaSuccess) count_launches(1);
  return e;
}

cudaError_t run_norm_backward(const NormProblem& problem, Workspace& ws,
                              cudaStream_t stream) {
  NormProblem p = problem;
  if (p.C == 0) return cudaSuccess;
  Team team = team_of(p.C);
  if (team.block.x > 512) team = {4, dim3((team.block.x / 32 + 1) / 2 * 32, 1)};
  const bool gate = p.gate.p != nullptr;
  const bool norm0 = p.branch_weight.p != nullptr;
  // Two resident blocks an SM, teams that each get a unit at least.
  int64_t blocks = int64_t(device_sm_count()) * 2;
  const int64_t groups = gate ? p.gate_count : 1;
  const int64_t group_rows = gate ? p.gate_rows : p.M;
  const int64_t teams = blocks * team.block.y;
  int64_t per_group = groups > 0 ? (teams + groups - 1) / groups : 1;
  // Units of eight rows or more, where a gate's sums are written for each.
  const int64_t most = (group_rows + 7) / 8;
  if (gate && per_group > most) per_group = most;
  if (per_group > group_rows) per_group = group_rows;
  if (per_group < 1) per_group = 1;
  p.unit_rows = int32_t((group_rows + per_group - 1) / per_group);
  if (p.unit_rows < 1) p.unit_rows = 1;
  p.units_per_group = (group_rows + p.unit_rows - 1) / p.unit_rows;
  if (p.units_per_group < 1) p.units_per_group = 1;
  p.units = p.M > 0 ? groups * p.units_per_group : 0;
  const int64_t need = (p.units + team.block.y - 1) / team.block.y;
  if (blocks > need) blocks = need;
  if (blocks < 1) blocks = 1;

  void* outs[3] = {p.dweight, p.dbias, norm0 ? p.dbranch_weight : nullptr};
  bool sums = false;
  for (int k = 0; k < 3; ++k) {
    p.part[k] = nullptr;
    if (!outs[k]) continue;
    sums = true;
    p.part[k] = static_cast<float*>(
        ws.take(size_t(blocks) * p.C * sizeof(float)));
  }
  p.gate_part = nullptr;
  const bool gate_sums = gate && p.dgate && p.units_per_group > 1;
  if (gate_sums)
    p.gate_part =
        static_cast<float*>(ws.take(size_t(p.units) * p.C * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;
  if (p.M == 0 && p.dgate) {
    const size_t es = p.dtype == VECTRA_F32 ? 4 : 2;
    const cudaError_t st =
        cudaMemsetAsync(p.dgate, 0, size_t(p.gate_count) * p.C * es, stream);
    if (st != cudaSuccess) return st;
  }
  const bool vec = all_vec(p);
  cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    cudaError_t st = with_more_chunks(team.nc, [&](auto nc) {
      return with_bool(norm0, [&](auto n0) {
        return with_bool(gate, [&](auto ga) {
          return with_bool(vec, [&](auto ve) {
            return launch_pdl(
                norm_backward_kernel<T, decltype(nc)::value,
                                     decltype(ve)::value, decltype(n0)::value,
                                     decltype(ga)::value>,
                dim3(unsigned(blocks)), team.block, 0, stream, p);
          });
        });
      });
    });
    if (st == cudaSuccess) count_launches(1);
    const unsigned across = unsigned((p.C + 31) / 32);
    if (st == cudaSuccess && sums) {
      const FinishArgs f{{p.part[0], p.part[1], p.part[2]},
                         {outs[0], outs[1], outs[2]}, blocks, 1, p.C};
      st = launch_pdl(norm_finish_kernel<T>, dim3(across, 1, 3), dim3(256), 0,
                      stream, f);
      if (st == cudaSuccess) count_launches(1);
    }
    if (st == cudaSuccess && gate_sums) {
      const FinishArgs f{{p.gate_part, nullptr, nullptr},
                         {p.dgate, nullptr, nullptr}, p.units_per_group,
                         groups, p.C};
      const unsigned down = unsigned(groups < 32768 ? groups : 32768);
      st = launch_pdl(norm_finish_kernel<T>, dim3(across, down, 1), dim3(256),
                      0, stream, f);
      if (st == cudaSuccess) count_launches(1);
    }
    return st;
  });
  return e;
}

}  // namespace vectra
