// cross_simple.cu: attention to an encoder's states (cross.cuh) on the float32
// pipes: every type, width up to 256 and stride, and all of float32, whose
// results no tensor core format holds.
//
// One kernel makes all three passes. A block owns R rows and walks tiles of CN
// columns: queries over keys (forward, dq) or keys over queries (dk and dv).
// With operands r, c (q and k) and r', c' (v and the upstream gradient, either
// way round) a tile is
//   s = |r - c|^2, t = r' . c'          (t in the backward passes)
//   P, z from s and t
//   acc += z c   (backward),  acc' += P c'  (forward, dk and dv).
// Distances are formed directly, sum (r - c)^2: twice the instructions of the
// product form in the first of up to four products, for float32's full
// accuracy where queries lie near their keys.
//
// All operands are staged in shared memory as [component][row], rows padded to
// 16-byte multiples, and P and z as [row][column]: every product then reads
// float4 pieces, for s and t along rows and columns, for acc along the summed
// columns. A thread owns R / 16 by CN / 16 of a tile and R / 16 by width / 16
// of a result. s and t take two columns an instruction (packed floats: 81 and
// 178 us of the figures below without).
//
// Bound by latency at the two blocks an SM that registers and shared memory
// hold (issue about 40 % of cycles, the FP32 pipe 30 %), and by a last wave of
// blocks. 257 queries on up to 700 keys, 8 heads of 64, batch 4, float32:
// forward 80 us, all gradients 172. Loading the next tile's operands by 4-byte
// asynchronous copies under the products changed 81 and 178 to 77 and 187.
#include <type_traits>

#include "cross.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

using tc::f2pk;
using tc::f2upk;
using tc::fadd2;
using tc::ffma2;

enum Pass { kForward = 0, kQueries = 1, kKeys = 2 };

constexpr int kThreads = 256;

template <int W, int R, int CN, int PASS>
struct Shape {
  static constexpr int LR = R + 4, LC = CN + 4;  // leading sizes
  static constexpr int RT = R / 16, CT = CN / 16, WT = W / 16;
  static constexpr bool kBack = PASS != kForward;
  // r, r' (backward), c, c', P (forward, keys), z (backward), column terms.
  static constexpr int OFF_R = 0;
  static constexpr int OFF_R2 = OFF_R + W * LR;
  static constexpr int OFF_C = OFF_R2 + (kBack ? W * LR : 0);
  static constexpr int OFF_C2 = OFF_C + W * LC;
  static constexpr int OFF_P = OFF_C2 + W * LC;
  static constexpr int OFF_Z = OFF_P + (PASS != kQueries ? R * LC : 0);
  static constexpr int OFF_COL = OFF_Z + (kBack ? R * LC : 0);
  static constexpr int FLOATS = OFF_COL + (PASS == kKeys ? 3 * CN : 0);
  static constexpr int BYTES = FLOATS * 4;
};

// Rows `first` .. of a matrix as [component][row]; rows at or past `rows`, and
// components at or past `width`, are zero. Packed rows are query, head of the
// group; `group` 1 for keys.
template <typename T, int W, int N, int L>
__device__ __forceinline__ void stage(float* dst, const void* base,
                                      const int64_t* s, int64_t b, int64_t h0,
                                      int64_t group, int64_t first,
                                      int64_t rows, int width) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if constexpr (std::is_same<T, float>::value) {
    // Whole 16-byte pieces: a warp takes one of 32 rows, whose components it
    // stores without conflicts.
    if (width % 4 == 0 && s[3] == 1 && s[0] % 4 == 0 && s[1] % 4 == 0 &&
        s[2] % 4 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) {
      constexpr int ROWS = N < 32 ? N : 32, SIDE = 32 / ROWS;
      const int r0 = lane % ROWS, d0 = lane / ROWS;
      for (int at = warp; at < N / ROWS * (W / 4) / SIDE; at += kThreads / 32) {
        const int r = at % (N / ROWS) * ROWS + r0;
        const int d = (at / (N / ROWS) * SIDE + d0) * 4;
        const int64_t row = first + r;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < rows && d < width) {
          const int64_t i = group == 1 ? row : row / group;
          const int64_t g = group == 1 ? 0 : row - i * group;
          v = __ldg(reinterpret_cast<const float4*>(
              static_cast<const float*>(base) + b * s[0] + (h0 + g) * s[1] +
              i * s[2] + d));
        }
        dst[d * L + r] = v.x;
        dst[(d + 1) * L + r] = v.y;
        dst[(d + 2) * L + r] = v.z;
        dst[(d + 3) * L + r] = v.w;
      }
      return;
    }
  }
  // A warp reads 8 components of 4 rows a step: whole 32-byte sectors of
  // 32-bit values, and stores that meet in at most 2 ways.
  const int dl = lane % 8, rl = lane / 8;
  for (int r = warp * 4 + rl; r < N; r += (kThreads / 32) * 4) {
    const int64_t row = first + r;
    const bool live = row < rows;
    const int64_t i = row / group, g = row - i * group;
    const T* src = static_cast<const T*>(base) + b * s[0] + (h0 + g) * s[1] +
                   i * s[2];
    for (int d = dl; d < W; d += 8)
      dst[d * L + r] = live && d < width ? to_f32(src[d * s[3]]) : 0.f;
  }
}

// lse leaves out the factor 2^(-g log2e |q_i|^2) of all of a row's weights in
// 16-bit types, as the tensor cores' kernels, which do not form it, do: the
// passes of one call may run on either (a copy of an argument may be aligned
// another way). float32 has these kernels alone, and keeps the whole logits.
template <typename T>
constexpr bool kLeaveOut = !std::is_same<T, float>::value;

// Rounded once, in all passes alike: a single key weighs exactly 1.
__device__ __forceinline__ float logit(float g, float distance) {
  return __fmul_rn(-g * kLog2e, distance);
}

// RT rows' components, each twice, and CT columns' in pairs.
template <int RT, int CT>
__device__ __forceinline__ void load_pairs(const float* rows,
                                           const float* columns, uint64_t* r,
                                           uint64_t* c) {
#pragma unroll
  for (int i = 0; i < RT; ++i) r[i] = f2pk(rows[i], rows[i]);
#pragma unroll
  for (int j = 0; j < CT; j += 2) {
    const float2 x = *reinterpret_cast<const float2*>(columns + j);
    c[j / 2] = f2pk(x.x, x.y);
  }
}

// One pass' work of one block: rows `block`, part `part` of the columns.
template <typename T, int W, int R, int CN, int PASS>
__device__ __forceinline__ void cross_pass(const CrossProblem& p,
                                           uint32_t block, int part,
                                           float* smem) {
  using S = Shape<W, R, CN, PASS>;
  constexpr int RT = S::RT, CT = S::CT, WT = S::WT;
  constexpr bool kRowsAreQueries = PASS != kKeys;
  float* sr = smem + S::OFF_R;
  float* sr2 = smem + S::OFF_R2;
  float* sc = smem + S::OFF_C;
  float* sc2 = smem + S::OFF_C2;
  float* sp = smem + S::OFF_P;
  float* sz = smem + S::OFF_Z;
  float* col_lse = smem + S::OFF_COL;
  float* col_delta = col_lse + CN;
  float* col_g = col_delta + CN;

  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t plane = block / p.row_blocks;
  const int64_t b = plane / p.Hk, hk = plane - b * p.Hk, h0 = hk * p.G;
  const int64_t first = (block - plane * p.row_blocks) * R;
  const int len = cross_length(p, b);
  const int64_t n_q = p.Nq * p.G;
  const int64_t rows = kRowsAreQueries ? n_q : int64_t(len);
  const int64_t cols = kRowsAreQueries ? int64_t(len) : n_q;
  const int tiles = first < rows ? int((cols + CN - 1) / CN) : 0;
  int t0, t1;
  split_range(tiles, part, p.splits, &t0, &t1);

  if (t0 < t1) {
    if constexpr (kRowsAreQueries) {
      stage<T, W, R, S::LR>(sr, p.q, p.sq, b, h0, p.G, first, rows, p.D);
      if constexpr (PASS == kQueries)
        stage<T, W, R, S::LR>(sr2, p.dout, p.se, b, h0, p.G, first, rows,
                              p.Dv);
    } else {
      stage<T, W, R, S::LR>(sr, p.k, p.sk, b, hk, 1, first, rows, p.D);
      stage<T, W, R, S::LR>(sr2, p.v, p.sv, b, hk, 1, first, rows, p.Dv);
    }
  }
  // Rows that are queries: scale, lse and c_i of each, and what lse leaves
  // out.
  float g2[RT], lse[RT], delta[RT], left_out[RT];
  int64_t qrow[RT];  // of [B, H, Nq]; -1: none
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    g2[i] = lse[i] = delta[i] = left_out[i] = 0.f;
    qrow[i] = -1;
    const int64_t r = first + ty * RT + i;
    if (kRowsAreQueries && r < rows) {
      const int64_t n = r / p.G, h = h0 + r - n * p.G;
      qrow[i] = (b * p.H + h) * p.Nq + n;
      g2[i] = cross_scale(p, b, h);
      if constexpr (PASS == kQueries) {
        lse[i] = p.lse[qrow[i]];
        delta[i] = p.delta[qrow[i]];
      }
    }
  }

  if constexpr (kLeaveOut<T> && kRowsAreQueries) {
    __syncthreads();
    if (t0 < t1) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float sq = 0.f;
        for (int d = tx; d < p.D; d += 16) {
          const float x = sr[d * S::LR + ty * RT + i];
          sq = fmaf(x, x, sq);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
          sq += __shfl_xor_sync(0xffffffffu, sq, o);
        left_out[i] = g2[i] * kLog2e * sq;
        lse[i] -= left_out[i];
      }
    }
  }

  float acc[S::kBack ? RT : 1][S::kBack ? WT : 1];   // z c
  float acc2[PASS != kQueries ? RT : 1][PASS != kQueries ? WT : 1];  // P c'
  float m[RT], l[RT], zs[RT], xs[RT], ys[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    m[i] = kNegInf;
    l[i] = zs[i] = xs[i] = ys[i] = 0.f;
#pragma unroll
    for (int j = 0; j < WT; ++j) {
      if constexpr (S::kBack) acc[i][j] = 0.f;
      if constexpr (PASS != kQueries) acc2[i][j] = 0.f;
    }
  }

  const bool works = first + threadIdx.x / 32 * 2 * RT < rows;
  for (int t = t0; t < t1; ++t) {
    const int64_t c0 = int64_t(t) * CN;
    __syncthreads();  // the tile before is no longer read
    if constexpr (kRowsAreQueries) {
      stage<T, W, CN, S::LC>(sc, p.k, p.sk, b, hk, 1, c0, cols, p.D);
      stage<T, W, CN, S::LC>(sc2, p.v, p.sv, b, hk, 1, c0, cols, p.Dv);
    } else {
      stage<T, W, CN, S::LC>(sc, p.q, p.sq, b, h0, p.G, c0, cols, p.D);
      stage<T, W, CN, S::LC>(sc2, p.dout, p.se, b, h0, p.G, c0, cols, p.Dv);
      for (int c = threadIdx.x; c < CN; c += kThreads) {
        const int64_t r = c0 + c;
        float x = INFINITY, y = 0.f, g = 0.f;  // weighs nothing
        if (r < cols) {
          const int64_t n = r / p.G, h = h0 + r - n * p.G;
          x = p.lse[(b * p.H + h) * p.Nq + n];
          y = p.delta[(b * p.H + h) * p.Nq + n];
          g = cross_scale(p, b, h);
        }
        col_lse[c] = x;
        col_delta[c] = y;
        col_g[c] = g;
      }
    }
    __syncthreads();
    if constexpr (kLeaveOut<T> && !kRowsAreQueries) {
      // Four threads a column.
      for (int c = threadIdx.x / 4; c < CN; c += kThreads / 4) {
        float sq = 0.f;
        for (int d = threadIdx.x % 4; d < p.D; d += 4) {
          const float x = sc[d * S::LC + c];
          sq = fmaf(x, x, sq);
        }
        sq += __shfl_xor_sync(0xffffffffu, sq, 1);
        sq += __shfl_xor_sync(0xffffffffu, sq, 2);
        if (threadIdx.x % 4 == 0) col_lse[c] -= col_g[c] * kLog2e * sq;
      }
      __syncthreads();
    }

    // A warp none of whose rows lives only stages the others' operands.
    if (!works) continue;

    // Sums of eight components at a time: a sum of D terms one by one would
    // be off by twice as much, and the weights' exponents with it. Two columns
    // in one instruction.
    uint64_t s2[RT][CT / 2], u2[RT][CT / 2];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT / 2; ++j) s2[i][j] = u2[i][j] = 0;
    const uint64_t minus = f2pk(-1.f, -1.f);
#pragma unroll 1
    for (int d0 = 0; d0 < p.D; d0 += 8) {
      uint64_t eight[RT][CT / 2];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT / 2; ++j) eight[i][j] = 0;
#pragma unroll
      for (int d = d0; d < d0 + 8; ++d) {  // zeros past the width
        uint64_t r[RT], c[CT / 2];
        load_pairs<RT, CT>(sr + d * S::LR + ty * RT, sc + d * S::LC + tx * CT,
                           r, c);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < CT / 2; ++j) {
            const uint64_t x = ffma2(c[j], minus, r[i]);
            eight[i][j] = ffma2(x, x, eight[i][j]);
          }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT / 2; ++j)
          s2[i][j] = fadd2(s2[i][j], eight[i][j]);
    }
    if constexpr (S::kBack) {
#pragma unroll 4
      for (int d = 0; d < p.Dv; ++d) {
        uint64_t r[RT], c[CT / 2];
        load_pairs<RT, CT>(sr2 + d * S::LR + ty * RT,
                           sc2 + d * S::LC + tx * CT, r, c);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < CT / 2; ++j)
            u2[i][j] = ffma2(r[i], c[j], u2[i][j]);
      }
    }
    float s[RT][CT], u[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; j += 2) {
        const float2 x = f2upk(s2[i][j / 2]), y = f2upk(u2[i][j / 2]);
        s[i][j] = x.x, s[i][j + 1] = x.y;
        u[i][j] = y.x, u[i][j + 1] = y.y;
      }

    if constexpr (PASS == kForward) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float top = kNegInf;
        bool nan = false;
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          s[i][j] = c0 + tx * CT + j < cols ? logit(g2[i], s[i][j]) : kNegInf;
          top = fmaxf(top, s[i][j]);
          nan = nan || s[i][j] != s[i][j];
        }
        if (nan) top = NAN;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          const float x = __shfl_xor_sync(0xffffffffu, top, o);
          top = x != x || top != top ? NAN : fmaxf(top, x);
        }
        // A maximum that stays at -inf: no weight yet, and no difference of
        // infinities.
        const float next = top != top || m[i] != m[i] ? NAN : fmaxf(m[i], top);
        const float ref = next == kNegInf ? 0.f : next;
        const float f = m[i] == kNegInf ? 0.f : exp2f(m[i] - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          s[i][j] = exp2f(s[i][j] - ref);
          sum += s[i][j];
        }
        m[i] = next;
        l[i] = l[i] * f + sum;
#pragma unroll
        for (int j = 0; j < WT; ++j) acc2[i][j] *= f;
#pragma unroll
        for (int j = 0; j < CT; ++j)
          sp[(ty * RT + i) * S::LC + tx * CT + j] = s[i][j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          const int c = tx * CT + j;
          const bool live = kRowsAreQueries
                                ? c0 + c < cols && qrow[i] >= 0
                                : c0 + c < cols && first + ty * RT + i < rows;
          const float g = kRowsAreQueries ? g2[i] : col_g[c];
          const float from = kRowsAreQueries ? lse[i] : col_lse[c];
          const float ci = kRowsAreQueries ? delta[i] : col_delta[c];
          const float w = live ? exp2f(logit(g, s[i][j]) - from) : 0.f;
          float z = live ? w * (u[i][j] - ci) : 0.f;
          if constexpr (PASS == kQueries) {
            xs[i] = live ? fmaf(z, s[i][j], xs[i]) : xs[i];
            ys[i] = live ? fmaf(w, s[i][j], ys[i]) : ys[i];
          } else {
            z *= 2.f * g;
            sp[(ty * RT + i) * S::LC + c] = w;
          }
          zs[i] += z;
          sz[(ty * RT + i) * S::LC + c] = z;
        }
      }
    }
    __syncwarp();  // a row's P and z are its own warp's

    // acc += z c, acc' += P c', four columns of the tile at a time.
#pragma unroll 1
    for (int c = 0; c < CN; c += 4) {
      if constexpr (S::kBack) {
        float4 z[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i)
          z[i] = *reinterpret_cast<const float4*>(
              &sz[(ty * RT + i) * S::LC + c]);
#pragma unroll
        for (int j = 0; j < WT; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(
              &sc[(tx + 16 * j) * S::LC + c]);
#pragma unroll
          for (int i = 0; i < RT; ++i)
            acc[i][j] = fmaf(z[i].x, x.x,
                             fmaf(z[i].y, x.y,
                                  fmaf(z[i].z, x.z,
                                       fmaf(z[i].w, x.w, acc[i][j]))));
        }
      }
      if constexpr (PASS != kQueries) {
        float4 w[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i)
          w[i] = *reinterpret_cast<const float4*>(
              &sp[(ty * RT + i) * S::LC + c]);
#pragma unroll
        for (int j = 0; j < WT; ++j) {
          const float4 x = *reinterpret_cast<const float4*>(
              &sc2[(tx + 16 * j) * S::LC + c]);
#pragma unroll
          for (int i = 0; i < RT; ++i)
            acc2[i][j] = fmaf(w[i].x, x.x,
                              fmaf(w[i].y, x.y,
                                   fmaf(w[i].z, x.z,
                                        fmaf(w[i].w, x.w, acc2[i][j]))));
        }
      }
    }
  }

  // Row sums over the 16 threads of a row.
#pragma unroll
  for (int i = 0; i < RT; ++i) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
      zs[i] += __shfl_xor_sync(0xffffffffu, zs[i], o);
      xs[i] += __shfl_xor_sync(0xffffffffu, xs[i], o);
      ys[i] += __shfl_xor_sync(0xffffffffu, ys[i], o);
    }
  }

  const bool whole = p.splits == 1;
  if constexpr (kRowsAreQueries) {
    const int64_t all = p.B * p.H * p.Nq;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (qrow[i] < 0) continue;
      const int64_t bh = qrow[i] / p.Nq, n = qrow[i] - bh * p.Nq;
      const int64_t h = bh - b * p.H;
      const int64_t at = part * all + qrow[i];
      if constexpr (PASS == kForward) {
        T* out = static_cast<T*>(p.out) + b * p.so[0] + h * p.so[1] +
                 n * p.so[2];
#pragma unroll
        for (int j = 0; j < WT; ++j) {
          const int d = tx + 16 * j;
          if (d >= p.Dv) continue;
          if (whole)
            store_with_rest<T>(
                out + d,
                p.rest ? static_cast<T*>(p.rest) + qrow[i] * p.Dv + d : nullptr,
                len > 0 ? acc2[i][j] / l[i] : 0.f);
          else
            p.part[at * p.Dv + d] = acc2[i][j];
        }
        if (tx == 0) {
          if (!whole) {
            p.part_ml[at * 2] = m[i] + left_out[i];
            p.part_ml[at * 2 + 1] = l[i];
          } else if (p.lse) {
            p.lse[qrow[i]] =
                len > 0 ? m[i] + left_out[i] + log2f(l[i]) : INFINITY;
          }
        }
      } else {
        const float g = 2.f * g2[i];
        T* out = static_cast<T*>(p.dq) + b * p.sdq[0] + h * p.sdq[1] +
                 n * p.sdq[2];
#pragma unroll
        for (int j = 0; j < WT; ++j) {
          const int d = tx + 16 * j;
          if (d >= p.D || !p.dq) continue;
          const float x =
              t0 < t1 ? g * (acc[i][j] -
                             sr[d * S::LR + ty * RT + i] * zs[i])
                      : 0.f;
          if (whole)
            out[d] = from_f32<T>(x);
          else
            p.part[at * p.D + d] = x;
        }
        if (tx == 0 && p.dscale_rows) {
          p.dscale_rows[at * 3] = xs[i];
          p.dscale_rows[at * 3 + 1] = ys[i];
          p.dscale_rows[at * 3 + 2] = zs[i];
        }
      }
    }
  } else {
    const int64_t all = p.B * p.Hk * p.Nk;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t key = first + ty * RT + i;
      if (key >= p.Nk) continue;
      const int64_t at = part * all + plane * p.Nk + key;
      const bool live = key < rows && t0 < t1;
#pragma unroll
      for (int j = 0; j < WT; ++j) {
        const int d = tx + 16 * j;
        if (d < p.D) {
          const float x =
              live ? acc[i][j] - sr[d * S::LR + ty * RT + i] * zs[i] : 0.f;
          if (whole)
            static_cast<T*>(p.dk)[b * p.sdk[0] + hk * p.sdk[1] +
                                  key * p.sdk[2] + d] = from_f32<T>(x);
          else
            p.part[at * p.D + d] = x;
        }
        if (d < p.Dv) {
          const float x = live ? acc2[i][j] : 0.f;
          if (whole)
            static_cast<T*>(p.dv)[b * p.sdv[0] + hk * p.sdv[1] +
                                  key * p.sdv[2] + d] = from_f32<T>(x);
          else
            p.part_v[at * p.Dv + d] = x;
        }
      }
    }
  }
}

template <typename T, int W, int R, int CN, int PASS>
__global__ void __launch_bounds__(kThreads)
    cross_simple_kernel(const __grid_constant__ CrossProblem p) {
  extern __shared__ __align__(16) float smem[];
  allow_dependents();
  grid_dependency_wait();
  cross_pass<T, W, R, CN, PASS>(p, blockIdx.x, blockIdx.y, smem);
}

// Both backward passes in one grid, the keys' blocks, which are longer, first:
// the last wave of blocks, of two an SM and more, is left half empty once.
template <typename T, int W, int R, int CN>
__global__ void __launch_bounds__(kThreads)
    cross_backward_kernel(const __grid_constant__ CrossProblem keys,
                          const __grid_constant__ CrossProblem queries,
                          uint32_t key_part, uint32_t key_blocks,
                          uint32_t query_part) {
  extern __shared__ __align__(16) float smem[];
  allow_dependents();
  grid_dependency_wait();
  if (blockIdx.x < key_blocks) {
    const uint32_t part = blockIdx.x / key_part;
    cross_pass<T, W, R, CN, kKeys>(keys, blockIdx.x - part * key_part,
                                   int(part), smem);
  } else {
    const uint32_t at = blockIdx.x - key_blocks, part = at / query_part;
    cross_pass<T, W, R, CN, kQueries>(queries, at - part * query_part,
                                      int(part), smem);
  }
}

template <typename K, typename... A>
cudaError_t start(K kern, dim3 grid, int bytes, cudaStream_t stream,
                  const A&... args) {
  const cudaError_t e = cudaFuncSetAttribute(
      kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  count_launches(1);
  return launch_pdl(kern, grid, dim3(kThreads), bytes, stream, args...);
}

// Blocks of a part of a pass.
int64_t set_blocks(CrossProblem* p, int64_t rows, int R) {
  p->row_blocks = (rows + R - 1) / R;
  return p->row_blocks * p->B * p->Hk;
}

template <typename T, int W, int R, int CN, int PASS>
cudaError_t launch(CrossProblem p, int64_t rows, cudaStream_t stream) {
  const int64_t blocks = set_blocks(&p, rows, R);
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  return start(cross_simple_kernel<T, W, R, CN, PASS>,
               dim3(unsigned(blocks), unsigned(p.splits)),
               Shape<W, R, CN, PASS>::BYTES, stream, p);
}

template <typename T, int W, int R, int CN>
cudaError_t launch_both(CrossProblem keys, CrossProblem queries, bool want_k,
                        bool want_q, cudaStream_t stream) {
  const int64_t k = set_blocks(&keys, keys.Nk, R);
  const int64_t q = set_blocks(&queries, queries.Nq * queries.G, R);
  const int64_t k_all = want_k ? k * keys.splits : 0;
  const int64_t all = k_all + (want_q ? q * queries.splits : 0);
  if (all > 0x7fffffff) return cudaErrorInvalidValue;
  constexpr int k_bytes = Shape<W, R, CN, kKeys>::BYTES;
  constexpr int q_bytes = Shape<W, R, CN, kQueries>::BYTES;
  return start(cross_backward_kernel<T, W, R, CN>, dim3(unsigned(all)),
               k_bytes > q_bytes ? k_bytes : q_bytes, stream, keys, queries,
               uint32_t(k), uint32_t(k_all), uint32_t(q));
}

int width_of(const CrossProblem& p) {
  const int w = p.D > p.Dv ? p.D : p.Dv;
  return w <= 32 ? 32 : (w <= 64 ? 64 : (w <= 128 ? 128 : 256));
}

// Rows and columns of a tile: 16 rows where there are no more, else 64 (32 of
// the widest vectors, whose operands would not fit).
void tile_of(const CrossProblem& p, int64_t rows, int* r, int* c) {
  const bool wide = width_of(p) == 256;
  *r = rows <= 16 ? 16 : (wide ? 32 : 64);
  *c = wide ? 32 : 64;
}

// f(the type, the padded width, and a tile's columns, as tile_of has them).
template <typename F>
cudaError_t with_shape(const CrossProblem& p, F&& f) {
  return with_dtype(p.dtype, [&](auto* t) {
    using C32 = std::integral_constant<int, 32>;
    using C64 = std::integral_constant<int, 64>;
    switch (width_of(p)) {
      case 32:
        return f(t, C32{}, C64{});
      case 64:
        return f(t, C64{}, C64{});
      case 128:
        return f(t, std::integral_constant<int, 128>{}, C64{});
      default:
        return f(t, std::integral_constant<int, 256>{}, C32{});
    }
  });
}

cudaError_t launch_forward(const CrossProblem& p, cudaStream_t stream) {
  const int64_t rows = p.Nq * p.G;
  return with_shape(p, [&](auto* t, auto width, auto cols) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int W = decltype(width)::value, CN = decltype(cols)::value;
    return rows <= 16 ? launch<T, W, 16, CN, kForward>(p, rows, stream)
                      : launch<T, W, CN, CN, kForward>(p, rows, stream);
  });
}

// The passes over 16 rows or fewer by themselves, the others in one grid.
cudaError_t launch_backward(const CrossProblem& keys,
                            const CrossProblem& queries, bool want_k,
                            bool want_q, cudaStream_t stream) {
  const int64_t n_k = keys.Nk, n_q = queries.Nq * queries.G;
  return with_shape(keys, [&](auto* t, auto width, auto cols) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int W = decltype(width)::value, CN = decltype(cols)::value;
    cudaError_t e = cudaSuccess;
    if (want_k && n_k <= 16)
      e = launch<T, W, 16, CN, kKeys>(keys, n_k, stream);
    if (e == cudaSuccess && want_q && n_q <= 16)
      e = launch<T, W, 16, CN, kQueries>(queries, n_q, stream);
    const bool k = want_k && n_k > 16, q = want_q && n_q > 16;
    if (e == cudaSuccess && (k || q))
      e = launch_both<T, W, CN, CN>(keys, queries, k, q, stream);
    return e;
  });
}

// Parts of the axis that a block walks: enough for twice the blocks that the
// SMs hold (`per_sm` by their shared memory), each of two tiles at least.
int splits_for(const CrossProblem& p, int64_t rows, int64_t cols,
               bool backward) {
  int r, c;
  tile_of(p, rows, &r, &c);
  const int64_t blocks = (rows + r - 1) / r * p.B * p.Hk;
  const int64_t tiles = (cols + c - 1) / c;
  if (blocks == 0) return 1;
  const int64_t w = width_of(p);
  const int64_t bytes =
      4 * (backward ? 2 * w * (r + c + 8) + 2 * r * (c + 4)
                    : w * (r + 2 * c + 12) + r * (c + 4));
  int64_t per_sm = 227 * 1024 / (bytes + 1024);
  if (per_sm > 4) per_sm = 4;
  int64_t s = 2 * per_sm * device_sm_count() / blocks;
  if (s > tiles / 2) s = tiles / 2;
  if (s > 64) s = 64;
  return s < 1 ? 1 : int(s);
}

float* take_floats(Workspace& ws, int64_t n) {
  return static_cast<float*>(ws.take(size_t(n) * sizeof(float)));
}

}  // namespace

cudaError_t run_cross_simple_forward(const CrossProblem& problem,
                                     Workspace& ws, cudaStream_t stream) {
  CrossProblem p = problem;
  const int64_t rows = p.B * p.H * p.Nq;
  p.splits = splits_for(p, p.Nq * p.G, p.Nk, false);
  if (p.splits > 1) {
    p.part = take_floats(ws, p.splits * rows * p.Dv);
    p.part_ml = take_floats(ws, p.splits * rows * 2);
  }
  if (ws.dry || ws.overflow || rows == 0) return cudaSuccess;
  const cudaError_t e = launch_forward(p, stream);
  return e != cudaSuccess || p.splits == 1 ? e : launch_cross_join(p, stream);
}

cudaError_t run_cross_simple_backward(const CrossProblem& problem,
                                      Workspace& ws, cudaStream_t stream) {
  CrossProblem p = problem;
  const int64_t rows = p.B * p.H * p.Nq, keys = p.B * p.Hk * p.Nk;
  float* delta = take_floats(ws, rows);
  p.delta = delta;
  CrossProblem pq = p, pk = p;
  const bool want_q = p.dq || p.dscale;
  if (want_q) {
    pq.splits = splits_for(p, p.Nq * p.G, p.Nk, true);
    if (p.dscale) pq.dscale_rows = take_floats(ws, pq.splits * rows * 3);
    if (pq.splits > 1 && p.dq) pq.part = take_floats(ws, pq.splits * rows * p.D);
  }
  if (p.dk) {
    pk.splits = splits_for(p, p.Nk, p.Nq * p.G, true);
    if (pk.splits > 1) {
      pk.part = take_floats(ws, pk.splits * keys * p.D);
      pk.part_v = take_floats(ws, pk.splits * keys * p.Dv);
    }
  }
  if (ws.dry || ws.overflow) return cudaSuccess;
  cudaError_t e = launch_cross_delta(p, delta, stream);
  if (e == cudaSuccess)
    e = launch_backward(pk, pq, p.dk && keys > 0, want_q && rows > 0, stream);
  if (e == cudaSuccess && pq.part && rows > 0)
    e = launch_cross_sum(p.dtype, pq.part, pq.splits, p.B, p.H, p.Nq, p.D,
                         p.dq, p.sdq, stream);
  if (e == cudaSuccess && p.dscale)
    e = launch_cross_dscale(pq, pq.splits, stream);
  if (e == cudaSuccess && pk.part && keys > 0)
    e = launch_cross_sum(p.dtype, pk.part, pk.splits, p.B, p.Hk, p.Nk, p.D,
                         p.dk, p.sdk, stream);
  if (e == cudaSuccess && pk.part && keys > 0)
    e = launch_cross_sum(p.dtype, pk.part_v, pk.splits, p.B, p.Hk, p.Nk, p.Dv,
                         p.dv, p.sdv, stream);
  return e;
}

}  // namespace vectra
