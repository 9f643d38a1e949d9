// residual_norm_kernel.cuh: dropout, and what stands between two sublayers of a
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
// over rows are joined in a fixed order, without atomics. 16-bit tensors keep
// what x_out's rounding left as well, for n1: without it dw of a bf16 row of
// mean 0 was 0.60 of a unit roundoff off instead of 0.41, and with the layer
// norm by the ratio of mean to deviation more.
//
// Memory-bound. A team of threads (a warp up to 512 columns, else a block)
// owns a row: each thread holds one or two chunks of 8 neighbouring columns,
// the same for every row, so that it can keep its columns' sums over rows in
// registers. The next rows are on their way into shared memory meanwhile, by
// asynchronous copies; a thread reads only what it copied itself, so they need
// no barrier.
//
// Measured, bf16: 66,560 rows of 256, layer norm, one gate row, dropout:
// forward for training 40 us (170 MB: 4.3 TB/s; 37 without the rest), bound by
// instructions (issue 68 %, DRAM 33 %); backward 69 us (239 MB: 3.5 TB/s, of
// which the joins of the column sums 9), the same (issue 63 % with two blocks
// an SM). 8,193 rows of 5,120, norms on both sides, a gate row for each
// 2,731: forward for training 85 us (420 MB, 4.9 TB/s; 77 without the rest);
// backward 230 us (587 MB, 2.6 TB/s; 207 without the rest), bound by
// instructions (issue 49 %) and by the column sums, 64 of which a thread keeps,
// in part in spilled registers. Of 207 us no loads would have left 188, no
// stores 195; one block of 640 threads an SM with half the sums each took 313.
// With loads to registers in turn instead of copies ahead it was 280. Dropout
// alone, 16,396 rows of 4,096: 55 us a pass (269 MB, 4.8 TB/s), bound by the
// numbers' integer products (issue 57 %, half of the stalls on that pipe) and by
// a thread's one load under way.
#pragma once

#include <type_traits>

#include "block_common.cuh"
#include "philox.cuh"
#include "residual_norm.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

using tc::f2pk;
using tc::f2upk;
using tc::fadd2;
using tc::ffma2;

constexpr int kPairs = kChunk / 2;  // as the packed float pipe takes them

template <typename T>
struct Raw {
  static constexpr int N = int(sizeof(T)) / 2;  // 16-byte pieces
  uint4 u[N];
};

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return f2pk(x, x); }
__device__ __forceinline__ float halves(uint64_t x) {
  const float2 f = f2upk(x);
  return f.x + f.y;
}

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, uint64_t* v) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[2 * i] = f2pk(__uint_as_float(r.u[i].x), __uint_as_float(r.u[i].y));
      v[2 * i + 1] =
          f2pk(__uint_as_float(r.u[i].z), __uint_as_float(r.u[i].w));
    }
  } else {
    const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[i] = f2pk(__uint_as_float(w[i] << 16),
                    __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 f =
            __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[i] = f2pk(f.x, f.y);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw<T> pack(const uint64_t* v) {
  Raw<T> r;
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 a = f2upk(v[2 * i]), b = f2upk(v[2 * i + 1]);
      r.u[i] = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y),
                          __float_as_uint(b.x), __float_as_uint(b.y));
    }
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = f2upk(v[i]);
      w[i] = tc::pack2<T>(a.x, a.y);
    }
    r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
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
                                      int cols, uint64_t* v) {
  unpack<T>(load_raw<T, VEC>(row, inner, col, cols), v);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(void* row, int col, int cols,
                                       const uint64_t* v) {
  T* p = static_cast<T*>(row) + col;
  if constexpr (VEC) {
    if (col >= cols) return;
    const Raw<T> r = pack<T>(v);
#pragma unroll
    for (int i = 0; i < Raw<T>::N; ++i)
      reinterpret_cast<uint4*>(p)[i] = r.u[i];
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float2 f = f2upk(v[i]);
      if (col + 2 * i < cols) p[2 * i] = from_f32<T>(f.x);
      if (col + 2 * i + 1 < cols) p[2 * i + 1] = from_f32<T>(f.y);
    }
  }
}

// What rounding v to T leaves, as it is kept.
template <typename T>
__device__ __forceinline__ void left_over(const uint64_t* v, uint64_t* rest) {
  uint64_t rounded[kPairs];
  unpack<T>(pack<T>(v), rounded);
  const uint64_t minus = both(-1.f);
#pragma unroll
  for (int i = 0; i < kPairs; ++i)
    rest[i] = mul2(ffma2(rounded[i], minus, v[i]), both(kRestLift<T>));
}

// Kept elements times `scale`, 0 for the others.
__device__ __forceinline__ void drop8(uint32_t keep, float scale,
                                      uint64_t* v) {
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const float2 f = f2upk(v[i]);
    v[i] = f2pk(keep >> (2 * i) & 1 ? f.x * scale : 0.f,
                keep >> (2 * i + 1) & 1 ? f.y * scale : 0.f);
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

// What a thread reads row by row, in shared memory: `stages` rows of the
// tensors (and of the saved statistics), and once the vectors over the columns.
//   [stage][statistics, then tensor, chunk, piece][thread]
//   [vector, chunk, piece][thread]
// A thread reads only what it put there itself, so nothing waits for another.
// Where rows have no 16-byte pieces (VEC false) everything is read from global
// memory when it is needed. Addresses are kept in 32 bits and per thread:
// formed anew for every piece in 64, they were half of all instructions; and
// vectors that were read again for every row from L1, of which the rows leave
// little, cost a row 4,500 of 11,000 cycles.
template <typename T, int NC, bool VEC>
struct Rows {
  static constexpr int N = Raw<T>::N;
  uint32_t mine;       // this thread's first piece
  uint32_t pitch;      // bytes between its pieces
  uint32_t stage;      // bytes of a stage
  uint32_t vectors;    // where they start
  uint32_t from[NC];   // where its chunks start in a row, in bytes
  uint32_t bytes[NC];  // 16 a piece; 0 outside the row, which then is zeros
  const int* col;
  int cols;

  __device__ __forceinline__ void init(const uint4* memory, const int* columns,
                                       const NormProblem& p) {
    const uint32_t tid = threadIdx.y * blockDim.x + threadIdx.x;
    mine = smem_addr(memory) + tid * 16;
    pitch = blockDim.x * blockDim.y * 16;
    stage = pitch * (1 + p.tensors * NC * N);
    vectors = mine + stage * p.stages;
    cols = p.C;
    col = columns;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bool in = columns[c] < cols;
      from[c] = in ? columns[c] * uint32_t(sizeof(T)) : 0;
      bytes[c] = in ? 16 : 0;
    }
  }
  __device__ __forceinline__ uint32_t place(uint32_t at, int tensor, int c,
                                            int i) const {
    return mine + at + (1 + (tensor * NC + c) * N + i) * pitch;
  }
  // `at`: the stage, in bytes.
  __device__ __forceinline__ void fetch(uint32_t at, int tensor,
                                        const RowView& view, int row) {
    if (!VEC || view.p == nullptr) return;
    const char* src = view.row<T>(row);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         place(at, tensor, c, i)),
                     "l"(src + from[c] + i * 16), "r"(bytes[c])
                     : "memory");
  }
  __device__ __forceinline__ void fetch_stats(uint32_t at, const float* stats,
                                              int row) {
    if (VEC && stats)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + at),
                   "l"(stats + 4 * int64_t(row))
                   : "memory");
  }
  static __device__ __forceinline__ void commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // All but the last `stages` - 1 rows have landed.
  static __device__ __forceinline__ void wait(int stages) {
    if (!VEC) return;
    if (stages == 3)
      asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (stages == 2)
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
      asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  static __device__ __forceinline__ uint4 load(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
  }
  __device__ __forceinline__ void get(uint32_t at, int tensor,
                                      const RowView& view, int row, int c,
                                      uint64_t* v) {
    Raw<T> r;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < N; ++i) r.u[i] = load(place(at, tensor, c, i));
    } else {
      r = load_raw<T, false>(view.row<T>(row), view.inner, col[c], cols);
    }
    unpack<T>(r, v);
  }
  __device__ __forceinline__ float4 get_stats(uint32_t at, const float* stats,
                                              int row) {
    if (!stats) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (!VEC) return __ldg(reinterpret_cast<const float4*>(stats) + row);
    const uint4 u = load(mine + at);
    return make_float4(__uint_as_float(u.x), __uint_as_float(u.y),
                       __uint_as_float(u.z), __uint_as_float(u.w));
  }
  // Vector `which`: row `row` of a view, or `missing` everywhere.
  __device__ __forceinline__ void keep(int which, const RowView& view, int row,
                                       float missing) {
    if constexpr (VEC) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        Raw<T> r;
        if (view.p) {
          r = load_raw<T, true>(view.row<T>(row), 1, col[c], cols);
        } else {
          uint64_t v[kPairs];
#pragma unroll
          for (int i = 0; i < kPairs; ++i) v[i] = both(missing);
          r = pack<T>(v);
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                           vectors + ((which * NC + c) * N + i) * pitch),
                       "r"(r.u[i].x), "r"(r.u[i].y), "r"(r.u[i].z),
                       "r"(r.u[i].w)
                       : "memory");
      }
    }
  }
  __device__ __forceinline__ void vector(int which, const RowView& view,
                                         int row, float missing, int c,
                                         uint64_t* v) {
    if constexpr (VEC) {
      Raw<T> r;
#pragma unroll
      for (int i = 0; i < N; ++i)
        r.u[i] = load(vectors + ((which * NC + c) * N + i) * pitch);
      unpack<T>(r, v);
    } else if (view.p) {
      unpack<T>(load_raw<T, false>(view.row<T>(row), view.inner, col[c], cols),
                v);
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) v[i] = both(missing);
    }
  }
};

// The vectors' places.
enum { kWeight = 0, kBranchWeight = 1, kGate = 2, kBias = 3 };
static_assert(kBias == kNormVectors - 1, "a backward pass keeps no bias");

// ---------------------------------------------------------------------------
// Dropout.
// ---------------------------------------------------------------------------
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
    uint64_t v[kPairs];
    if constexpr (VEC) {
      const int64_t r = a.rows == 1 ? 0 : e / a.cols;
      const T* p = static_cast<const T*>(a.x) + r * a.ld + (e - r * a.cols);
      load8<T, true>(p, 1, 0, kChunk, v);
    } else {
      float f[kChunk];
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        f[i] = 0.f;
        if (e + i >= n) continue;
        const int64_t r = (e + i) / a.cols, c = e + i - r * a.cols;
        f[i] = to_f32(static_cast<const T*>(a.x)[r * a.ld + c * a.inner]);
      }
#pragma unroll
      for (int i = 0; i < kPairs; ++i) v[i] = f2pk(f[2 * i], f[2 * i + 1]);
    }
    drop8(keep_bits(key, uint64_t(g), a.drop.cut), a.drop.scale, v);
    store8<T, VEC>(static_cast<T*>(a.y) + e, 0,
                   n - e < kChunk ? int(n - e) : kChunk, v);
  }
}

// ---------------------------------------------------------------------------
// Norms.
// ---------------------------------------------------------------------------
// Sums of one or two values over the team. A block's team writes its warps'
// sums to one of two places in turn, so one barrier a sum is enough.
struct TeamSum {
  float2 (*part)[32];
  int turn = 0;
  template <bool TWO>
  __device__ __forceinline__ float2 sum(float a, float b) {
    a = warp_sum(a);
    if constexpr (TWO) b = warp_sum(b);
    if (blockDim.x == 32) return make_float2(a, TWO ? b : 0.f);
    const int lane = threadIdx.x % 32, warps = int(blockDim.x) / 32;
    if (lane == 0) part[turn][threadIdx.x / 32] = make_float2(a, TWO ? b : 0.f);
    __syncthreads();
    float2 v = make_float2(0.f, 0.f);
    if (lane < warps) v = part[turn][lane];
    turn ^= 1;
    // A block of at most 16 warps: lanes past them hold zeros.
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (o >= 16 && warps <= 16) continue;
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      if constexpr (TWO) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (warps <= 16) {  // lanes 0 .. 15 have the sum
      v.x = __shfl_sync(0xffffffffu, v.x, lane & 15);
      if constexpr (TWO) v.y = __shfl_sync(0xffffffffu, v.y, lane & 15);
    }
    return v;
  }
  __device__ __forceinline__ float one(float a) { return sum<false>(a, 0.f).x; }
};

// mean (0 unless `layer`) and factor of the row in v, which is 0 outside it;
// `live` of a chunk's values are in the row.
template <int NC, bool VEC>
__device__ __forceinline__ float2 row_norm(TeamSum& team, bool layer,
                                           const uint64_t (*v)[kPairs],
                                           const int* live, float inv_c,
                                           float eps) {
  float mean = 0.f;
  if (layer) {
    uint64_t s = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < kPairs; ++i) s = fadd2(s, v[c][i]);
    mean = team.one(halves(s)) * inv_c;
  }
  const uint64_t minus = both(-mean);
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    uint64_t part = 0;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      uint64_t t = fadd2(v[c][i], minus);
      if constexpr (!VEC) {
        const float2 f = f2upk(t);
        t = f2pk(2 * i < live[c] ? f.x : 0.f, 2 * i + 1 < live[c] ? f.y : 0.f);
      }
      part = ffma2(t, t, part);
    }
    ss += live[c] > 0 ? halves(part) : 0.f;
  }
  return make_float2(mean, rsqrtf(team.one(ss) * inv_c + eps));
}

template <typename T, int NC, bool VEC>
__global__ void __launch_bounds__(1024)
    norm_forward_kernel(const __grid_constant__ NormProblem p) {
  __shared__ float2 part[2][32];
  TeamSum team{part};
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
  extern __shared__ uint4 ahead[];
  Rows<T, NC, VEC> rows;
  rows.init(ahead, col, p);
  rows.keep(kWeight, p.weight, 0, 1.f);
  rows.keep(kBranchWeight, p.branch_weight, 0, 1.f);
  rows.keep(kBias, p.bias, 0, 0.f);
  const int M = int(p.M), gate_rows = int(p.gate_rows);
  // A gate that differs from row to row comes as the rows do.
  const bool gate_moves = p.gate.p && gate_rows == 1;
  int gate_row = -1;
  const int first = int(blockIdx.x * blockDim.y + threadIdx.y);
  const int teams = int(gridDim.x * blockDim.y);
  const uint32_t end = rows.stage * p.stages;
  const auto fetch = [&](uint32_t stage, int64_t row) {
    if (row < M) {
      rows.fetch(stage, 0, p.x, int(row));
      rows.fetch(stage, 1, p.branch, int(row));
      if (gate_moves) rows.fetch(stage, 2, p.gate, int(row));
    }
    rows.commit();
  };
  if (VEC)
    for (int i = 0; i + 1 < p.stages; ++i)
      fetch(i * rows.stage, first + int64_t(i) * teams);
  uint32_t stage = 0;
  for (int row = first; row < M; row += teams) {
    if (VEC) {
      fetch(stage == 0 ? end - rows.stage : stage - rows.stage,
            row + int64_t(p.stages - 1) * teams);
      rows.wait(p.stages);
    }
    const int64_t at = int64_t(row) * C;
    uint64_t v[NC][kPairs];
    float4 stats = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.branch.p == nullptr) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        rows.get(stage, 0, p.x, row, c, v[c]);
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        rows.get(stage, 1, p.branch, row, c, v[c]);
      if (p.branch_weight.p) {
        const float2 n =
            row_norm<NC, VEC>(team, p.layer, v, live, inv_c, p.eps);
        stats.z = n.x;
        stats.w = n.y;
        const uint64_t r = both(n.y), minus = both(-n.x);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          uint64_t w[kPairs];
          rows.vector(kBranchWeight, p.branch_weight, 0, 1.f, c, w);
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            v[c][i] = mul2(mul2(fadd2(v[c][i], minus), r), w[i]);
        }
      }
      const int own_gate = p.gate_count == 1 ? 0 : row / gate_rows;
      if (p.gate.p && !gate_moves && own_gate != gate_row) {
        rows.keep(kGate, p.gate, own_gate, 1.f);
        gate_row = own_gate;
      }
      const uint64_t scale = both(p.residual_scale);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (p.drop.cut && live[c] > 0)
          drop8(keep8<VEC>(key, at + col[c], p.drop.cut), p.drop.scale,
                v[c]);
        if (p.gate.p) {
          uint64_t g[kPairs];
          if (gate_moves)
            rows.get(stage, 2, p.gate, row, c, g);
          else
            rows.vector(kGate, p.gate, own_gate, 1.f, c, g);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) v[c][i] = mul2(v[c][i], g[i]);
        }
        uint64_t x[kPairs];
        rows.get(stage, 0, p.x, row, c, x);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[c][i] = ffma2(scale, x[i], v[c][i]);
        store8<T, VEC>(static_cast<T*>(p.x_out) + at, col[c], C, v[c]);
        if constexpr (!std::is_same<T, float>::value) {
          if (p.rest) {
            left_over<T>(v[c], x);
            store8<T, VEC>(static_cast<T*>(p.rest) + at, col[c], C, x);
          }
        }
      }
    }
    if (p.y) {
      const float2 n =
          row_norm<NC, VEC>(team, p.layer, v, live, inv_c, p.eps);
      stats.x = n.x;
      stats.y = n.y;
      const uint64_t r = both(n.y), minus = both(-n.x);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint64_t w[kPairs], b[kPairs];
        rows.vector(kWeight, p.weight, 0, 1.f, c, w);
        rows.vector(kBias, p.bias, 0, 0.f, c, b);
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          v[c][i] = ffma2(mul2(fadd2(v[c][i], minus), r), w[i], b[i]);
        store8<T, VEC>(static_cast<T*>(p.y) + at, col[c], C, v[c]);
      }
    }
    if (p.stats && threadIdx.x == 0)
      reinterpret_cast<float4*>(p.stats)[row] = stats;
    stage += rows.stage;
    if (stage >= end) stage = 0;
    if (row > M - teams) break;  // row + teams may pass 32 bits
  }
}

// Backward. A unit is `unit_rows` rows of one gate row's group; the teams take
// units in turn. A team's sums for the weights stay in registers to its end;
// those for a gate that some rows share are written at the end of each unit.
// THREADS: the block's most; two blocks an SM up to 320.
template <typename T, int NC, bool VEC, bool NORM0, bool GATE, bool LAYER,
          int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS <= 320 ? 2 : 1)
    norm_backward_kernel(const __grid_constant__ NormProblem p) {
  __shared__ float2 part[2][32];
  TeamSum team_sum{part};
  allow_dependents();
  grid_dependency_wait();
  const int C = p.C;
  const float inv_c = 1.f / float(C);
  const PhiloxKey key = load_key(p.drop);
  int col[NC];
  uint64_t dw[NC][kPairs], db[NC][kPairs];
  uint64_t dbw[NORM0 ? NC : 1][kPairs];
  uint64_t dgate[GATE ? NC : 1][kPairs];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = (c * int(blockDim.x) + int(threadIdx.x)) * kChunk;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      dw[c][i] = db[c][i] = 0;
      if constexpr (NORM0) dbw[c][i] = 0;
      if constexpr (GATE) dgate[c][i] = 0;
    }
  }
  extern __shared__ uint4 ahead[];
  Rows<T, NC, VEC> rows;
  rows.init(ahead, col, p);
  rows.keep(kWeight, p.weight, 0, 1.f);
  if constexpr (NORM0) rows.keep(kBranchWeight, p.branch_weight, 0, 1.f);
  // A gate that differs from row to row comes as the rows do.
  const bool gate_moves = GATE && p.gate_rows == 1;
  // What x_out's rounding left, of 16-bit types.
  const bool has_rest = !std::is_same<T, float>::value && p.rest != nullptr;
  const RowView rest{p.rest, C, 1};
  const int rest_at = gate_moves ? 5 : 4;
  int gate_row = -1;
  const uint32_t end = rows.stage * p.stages;
  const int team = int(blockIdx.x * blockDim.y + threadIdx.y);
  const int teams = int(gridDim.x * blockDim.y);
  const int group_rows = int(GATE ? p.gate_rows : p.M);
  const int units = int(p.units), per_group = int(p.units_per_group);
  // The team's rows in order: row `row` of unit `unit`, which ends before
  // `end`; one walk ahead for the copies, one for the work.
  struct Walk {
    int unit, group, row, end;
  };
  const auto enter = [&](Walk* w, int64_t unit) {
    if (unit >= units) {
      w->unit = units;
      return;
    }
    w->unit = int(unit);
    w->group = w->unit / per_group;
    const int start = (w->unit - w->group * per_group) * p.unit_rows;
    w->row = w->group * group_rows + start;
    w->end = w->group * group_rows + min(start + p.unit_rows, group_rows);
  };
  const auto step = [&](Walk* w) {
    if (++w->row >= w->end) enter(w, int64_t(w->unit) + teams);
  };
  Walk now, later;
  enter(&now, team);
  later = now;
  const auto fetch = [&](uint32_t stage) {
    if (later.unit < units) {
      if (p.f.p) rows.fetch(stage, 0, p.x, later.row);
      rows.fetch(stage, 1, p.branch, later.row);
      rows.fetch(stage, 2, p.e, later.row);
      rows.fetch(stage, 3, p.f, later.row);
      if (gate_moves) rows.fetch(stage, 4, p.gate, later.row);
      if (has_rest) rows.fetch(stage, rest_at, rest, later.row);
      rows.fetch_stats(stage, p.stats, later.row);
      step(&later);
    }
    rows.commit();
  };
  if (VEC)
    for (int i = 0; i + 1 < p.stages; ++i) fetch(i * rows.stage);
  uint32_t stage = 0;
  while (now.unit < units) {
    const int row = now.row, group = now.group, unit = now.unit;
    if (VEC) {
      fetch(stage == 0 ? end - rows.stage : stage - rows.stage);
      rows.wait(p.stages);
    }
    const int64_t at = int64_t(row) * C;
    const float4 stats = rows.get_stats(stage, p.stats, row);
    // g, the gradient of x_out.
    uint64_t g[NC][kPairs];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (p.e.p) {
        rows.get(stage, 2, p.e, row, c, g[c]);
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) g[c][i] = 0;
      }
    }
    if (p.f.p) {
      const uint64_t minus = both(-stats.x), r = both(stats.y);
      // n1 and f w of a chunk, formed again behind the sums.
      const auto form = [&](int c, uint64_t* n, uint64_t* f, uint64_t* fw) {
        uint64_t w[kPairs];
        rows.vector(kWeight, p.weight, 0, 1.f, c, w);
        rows.get(stage, 0, p.x, row, c, n);
        if (has_rest) {
          rows.get(stage, rest_at, rest, row, c, f);
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            n[i] = ffma2(f[i], both(1.f / kRestLift<T>), n[i]);
        }
        rows.get(stage, 3, p.f, row, c, f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          n[i] = mul2(LAYER ? fadd2(n[i], minus) : n[i], r);
          fw[i] = mul2(f[i], w[i]);  // 0 outside the row, as f is
        }
      };
      uint64_t fn = 0, fs = 0;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint64_t n[kPairs], f[kPairs], fw[kPairs];
        form(c, n, f, fw);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          dw[c][i] = ffma2(f[i], n[i], dw[c][i]);
          db[c][i] = fadd2(db[c][i], f[i]);
          fn = ffma2(fw[i], n[i], fn);
          if constexpr (LAYER) fs = fadd2(fs, fw[i]);
        }
      }
      const float2 s = team_sum.sum<LAYER>(halves(fn), halves(fs));
      const uint64_t cn = both(-s.x * inv_c), cs = both(-s.y * inv_c);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint64_t n[kPairs], f[kPairs], fw[kPairs];
        form(c, n, f, fw);
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          g[c][i] = ffma2(r, LAYER ? fadd2(ffma2(n[i], cn, fw[i]), cs)
                                   : ffma2(n[i], cn, fw[i]),
                          g[c][i]);
      }
    }
    if (p.dx) {
      const uint64_t scale = both(p.residual_scale);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint64_t t[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) t[i] = mul2(g[c][i], scale);
        store8<T, VEC>(static_cast<T*>(p.dx) + at, col[c], C, t);
      }
    }
    if (NORM0 || p.dbranch || p.dgate) {
      // h, the gradient of u.
      if (GATE && !gate_moves && group != gate_row) {
        rows.keep(kGate, p.gate, group, 1.f);
        gate_row = group;
      }
      const uint64_t minus = both(-stats.z), r = both(stats.w);
      const auto form_u = [&](int c, uint64_t* u) {
        if (p.branch.p) {
          rows.get(stage, 1, p.branch, row, c, u);
        } else {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) u[i] = 0;
        }
        if constexpr (NORM0) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            u[i] = mul2(LAYER ? fadd2(u[i], minus) : u[i], r);
        }
      };
      uint64_t hn = 0, hs = 0;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint64_t u[kPairs], bw[kPairs];
        form_u(c, u);
        uint32_t keep = 0xff;
        if (p.drop.cut) keep = keep8<VEC>(key, at + col[c], p.drop.cut);
        if constexpr (NORM0)
          rows.vector(kBranchWeight, p.branch_weight, 0, 1.f, c, bw);
        if constexpr (GATE) {
          uint64_t gate[kPairs], d[kPairs];
          if (gate_moves)
            rows.get(stage, 4, p.gate, row, c, gate);
          else
            rows.vector(kGate, p.gate, group, 1.f, c, gate);
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            d[i] = NORM0 ? mul2(u[i], bw[i]) : u[i];
          if (p.drop.cut) drop8(keep, p.drop.scale, d);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            dgate[c][i] = ffma2(g[c][i], d[i], dgate[c][i]);
            g[c][i] = mul2(g[c][i], gate[i]);
          }
        }
        if (p.drop.cut) drop8(keep, p.drop.scale, g[c]);
        if constexpr (NORM0) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            dbw[c][i] = ffma2(g[c][i], u[i], dbw[c][i]);
            g[c][i] = mul2(g[c][i], bw[i]);  // 0 outside the row
            hn = ffma2(g[c][i], u[i], hn);
            if constexpr (LAYER) hs = fadd2(hs, g[c][i]);
          }
        }
      }
      if constexpr (NORM0) {
        const float2 s = team_sum.sum<LAYER>(halves(hn), halves(hs));
        const uint64_t cn = both(-s.x * inv_c), cs = both(-s.y * inv_c);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          uint64_t u[kPairs];
          form_u(c, u);
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            g[c][i] = mul2(r, LAYER ? fadd2(ffma2(u[i], cn, g[c][i]), cs)
                                    : ffma2(u[i], cn, g[c][i]));
        }
      }
      if (p.dbranch) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          store8<T, VEC>(static_cast<T*>(p.dbranch) + at, col[c], C,
                         g[c]);
      }
    }
    step(&now);
    stage += rows.stage;
    if (stage >= end) stage = 0;
    if constexpr (GATE) {
      // A gate row's sums: at the end of each unit, or with the weights' where
      // all rows share one.
      if (now.unit != unit && p.dgate && p.gate_count > 1) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (p.units_per_group == 1)
            store8<T, VEC>(static_cast<T*>(p.dgate) + int64_t(group) * C, col[c], C,
                           dgate[c]);
          else
            store8<float, VEC>(p.gate_part + int64_t(unit) * C, col[c], C, dgate[c]);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) dgate[c][i] = 0;
        }
      }
    }
  }
  // The blocks' sums: a block's teams join theirs through shared memory.
  // (The copies have landed and been read.)
  float(*joined)[512 + 8] = reinterpret_cast<float(*)[512 + 8]>(ahead);
  const auto flush = [&](int k, const uint64_t (*own)[kPairs]) {
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
      for (int i = 0; i < kPairs; ++i) {
        const float2 f = f2upk(own[c][i]);
        if (col[c] + 2 * i < C) joined[threadIdx.y][col[c] + 2 * i] = f.x;
        if (col[c] + 2 * i + 1 < C)
          joined[threadIdx.y][col[c] + 2 * i + 1] = f.y;
      }
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
  if constexpr (GATE) flush(3, dgate);
}

// out[g, col] = sum over `count` consecutive rows of `part` in order, by 32
// warps a block of 32 columns.
template <typename T>
__global__ void __launch_bounds__(1024) norm_finish_kernel(const FinishArgs a) {
  __shared__ float sums[32][33];
  allow_dependents();
  grid_dependency_wait();
  const int k = blockIdx.z;
  if (a.out[k] == nullptr) return;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int warps = blockDim.x / 32;
  const int col = blockIdx.x * 32 + lane;
  for (int64_t g = blockIdx.y; g < a.groups; g += gridDim.y) {
    const float* p = a.part[k] + g * a.count * a.C;
    float t = 0.f;
    if (col < a.C) {
#pragma unroll 8
      for (int64_t r = warp; r < a.count; r += warps)
        t += __ldg(p + r * a.C + col);
    }
    sums[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && col < a.C) {
      float total = 0.f;
      for (int w = 0; w < warps; ++w) total += sums[w][lane];
      static_cast<T*>(a.out[k])[g * a.C + col] = from_f32<T>(total);
    }
    __syncthreads();
  }
}

template <typename K>
cudaError_t allow_shared(K kern, size_t bytes) {
  return bytes > 32 * 1024
             ? cudaFuncSetAttribute(
                   kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                   int(bytes))
             : cudaSuccess;
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

template <typename T>
cudaError_t dropout_typed(const DropArgs& a, bool vec, unsigned blocks,
                          cudaStream_t stream) {
  return launch_pdl(vec ? dropout_kernel<T, true> : dropout_kernel<T, false>,
                    dim3(blocks), dim3(256), 0, stream, a);
}

template <typename T>
cudaError_t norm_forward_typed(const NormProblem& p, const NormLaunch& how,
                               cudaStream_t stream) {
  return with_chunks(how.chunks, [&](auto nc) {
    constexpr int NC = decltype(nc)::value;
    auto kern = how.vec ? norm_forward_kernel<T, NC, true>
                        : norm_forward_kernel<T, NC, false>;
    const cudaError_t st = allow_shared(kern, how.bytes);
    if (st != cudaSuccess) return st;
    return launch_pdl(kern, dim3(how.blocks), how.block, how.bytes, stream, p);
  });
}

template <typename T>
cudaError_t norm_backward_typed(const NormProblem& p, const NormLaunch& how,
                                cudaStream_t stream) {
  const auto run = [&](auto nc, auto n0, auto ga, auto ve, auto la) {
    constexpr int NC = decltype(nc)::value;
    constexpr bool N0 = decltype(n0)::value, GA = decltype(ga)::value;
    constexpr bool VE = decltype(ve)::value, LA = decltype(la)::value;
    auto kern = norm_backward_kernel<T, NC, VE, N0, GA, LA,
                                     NC == 1 ? 256 : 512>;
    if constexpr (NC == 2)
      if (how.two_blocks)
        kern = norm_backward_kernel<T, NC, VE, N0, GA, LA, 320>;
    const cudaError_t st = allow_shared(kern, how.bytes);
    if (st != cudaSuccess) return st;
    return launch_pdl(kern, dim3(how.blocks), how.block, how.bytes, stream, p);
  };
  return with_more_chunks(how.chunks, [&](auto nc) {
    return with_bool(p.branch_weight.p != nullptr, [&](auto n0) {
      return with_bool(p.gate.p != nullptr, [&](auto ga) {
        return with_bool(how.vec, [&](auto ve) {
          return with_bool(p.layer, [&](auto la) {
            return run(nc, n0, ga, ve, la);
          });
        });
      });
    });
  });
}

template <typename T>
cudaError_t norm_finish_typed(const FinishArgs& a, dim3 grid, int threads,
                              cudaStream_t stream) {
  return launch_pdl(norm_finish_kernel<T>, grid, dim3(unsigned(threads)), 0,
                    stream, a);
}

// One file a type, so that they compile side by side.
#define VECTRA_NORM_TYPE(T)                                                  \
  template cudaError_t dropout_typed<T>(const DropArgs&, bool, unsigned,     \
                                        cudaStream_t);                       \
  template cudaError_t norm_forward_typed<T>(                                \
      const NormProblem&, const NormLaunch&, cudaStream_t);                  \
  template cudaError_t norm_backward_typed<T>(                               \
      const NormProblem&, const NormLaunch&, cudaStream_t);                  \
  template cudaError_t norm_finish_typed<T>(const FinishArgs&, dim3, int,    \
                                            cudaStream_t);

}  // namespace vectra
