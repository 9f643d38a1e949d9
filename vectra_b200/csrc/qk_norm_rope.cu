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
// Memory-bound: each vector is read once and written once. Measured on a B200:
// 65 us for the 16,384 tokens of 32 + 8 heads of 128, bf16, views of one
// projection (344 MB: 5.3 TB/s, 0.81 of the copy rate; writes alone reach
// 3.7 TB/s here, so their half takes 46 us); 2.9 us for 64 single tokens;
// forward and backward of 6,147 tokens of 16 + 16 heads of 64, f16, half
// rotated, 47 us for 101 MB. There the backward kernel is bound by latency: its
// 146 registers leave one block of eight warps an SM (12 % occupancy, DRAM
// 10 %, issue 0.32 per scheduler), in waves of load, compute and store. float32,
// 8,192 tokens of 32 + 8 heads of 128: forward 58.7 us (336 MB), forward and
// backward 150.6 (671 MB).
#include "block_common.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

using tc::f2pk;
using tc::f2upk;
using tc::ffma2;

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

// ---------------------------------------------------------------------------
// The vector kernels: 16-byte loads and stores.
//
// A group of G lanes (the power of two from 1 to 32 that covers the vector's
// chunk pairs) owns a head vector; each lane holds two 16-byte chunks of VE
// elements, chosen so that no rotated pair spans lanes: chunks j and
// j + R2 / VE when pairs are (i, i + R2), so both members sit at the same
// place of the two chunks, and any two chunks when pairs are neighbours.
// Unrotated chunks pair up behind them and turn by cos = 1, sin = 0. The
// norm is a butterfly over the group. A group walks several heads of one
// token, so the token's cosines and sines (which a vector would otherwise
// re-read at twice its own size) are loaded once into registers, and the
// heads' loads are issued kBatch at a time before any is used.
// ---------------------------------------------------------------------------
template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

template <typename T>
union Chunk {
  uint4 u;
  T e[kVec<T>];
};

struct QkVecArgs {
  QkProblem p;
  float* partial;
  int heads_per_group;
  int groups_per_token[2];  // of the queries, of the keys
  int64_t groups[2];
  int blocks[2];            // backward: blocks of each side
  bool w_vec[2];            // weights in 16-byte pieces
};

// The two chunks of lane j's slot; -1: none.
__device__ __forceinline__ void slot_chunks(int j, int slots, int chunks,
                                            int r_chunks, int interleaved,
                                            int* c0, int* c1) {
  if (interleaved) {
    *c0 = j;
    *c1 = j + slots;
  } else if (j < r_chunks) {
    *c0 = j;
    *c1 = j + r_chunks;
  } else {
    *c0 = 2 * j;
    *c1 = 2 * j + 1;
  }
  if (j >= slots || *c0 >= chunks) *c0 = -1;
  if (j >= slots || *c1 >= chunks) *c1 = -1;
}

// VE cosines and sines of a slot. Pairs (i, i + R2): element e of both
// chunks. Neighbours: pair e / 2 of chunk 0, then of chunk 1.
template <typename T>
struct Angles {
  float c[kVec<T>], s[kVec<T>];
};

template <typename T, bool INTER>
__device__ __forceinline__ void load_angles(const QkProblem& p, int64_t pos,
                                            bool known, int c0, int c1,
                                            Angles<T>* a) {
  constexpr int VE = kVec<T>;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    a->c[i] = 1.f;
    a->s[i] = 0.f;
  }
  if (!known) return;
  const float* cr = p.cos + pos * p.cos_ld;
  const float* sr = p.sin + pos * p.sin_ld;
  if constexpr (!INTER) {
    if (c0 >= 0 && c0 * VE < p.R2) {
#pragma unroll
      for (int i = 0; i < VE; i += 4) {
        *reinterpret_cast<float4*>(a->c + i) =
            __ldg(reinterpret_cast<const float4*>(cr + c0 * VE + i));
        *reinterpret_cast<float4*>(a->s + i) =
            __ldg(reinterpret_cast<const float4*>(sr + c0 * VE + i));
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = h ? c1 : c0;
      if (c < 0 || c * VE >= 2 * p.R2) continue;
#pragma unroll
      for (int i = 0; i < VE / 2; i += 2) {
        *reinterpret_cast<float2*>(a->c + h * (VE / 2) + i) =
            __ldg(reinterpret_cast<const float2*>(cr + c * VE / 2 + i));
        *reinterpret_cast<float2*>(a->s + h * (VE / 2) + i) =
            __ldg(reinterpret_cast<const float2*>(sr + c * VE / 2 + i));
      }
    }
  }
}

// One chunk's weights; `w_vec`: they can be read 16 bytes at a time.
template <typename T>
__device__ __forceinline__ void load_weight(const QkSide& s, bool w_vec,
                                            int chunk, float* w) {
  constexpr int VE = kVec<T>;
#pragma unroll
  for (int i = 0; i < VE; ++i) w[i] = 1.f;
  if (s.w == nullptr || chunk < 0) return;
  if (w_vec && s.w_dtype == VECTRA_F32) {
#pragma unroll
    for (int i = 0; i < VE; i += 4)
      *reinterpret_cast<float4*>(w + i) = __ldg(reinterpret_cast<const float4*>(
          static_cast<const float*>(s.w) + chunk * VE + i));
  } else if (w_vec) {
    Chunk<T> c;
    c.u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(s.w) +
                                               chunk * VE));
#pragma unroll
    for (int i = 0; i < VE; ++i) w[i] = to_f32(c.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i)
      w[i] = load_any(s.w, s.w_dtype, int64_t(chunk * VE + i) * s.sw);
  }
}

template <int G>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1)
    x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// A chunk as pairs of neighbours for the packed float pipe.
template <typename T>
__device__ __forceinline__ void unpack_chunk(const Chunk<T>& c, uint64_t* x) {
  const uint32_t w[4] = {c.u.x, c.u.y, c.u.z, c.u.w};
  if constexpr (std::is_same<T, float>::value) {
    x[0] = f2pk(__uint_as_float(w[0]), __uint_as_float(w[1]));
    x[1] = f2pk(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[i] = f2pk(__uint_as_float(w[i] << 16),
                    __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 f =
            __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[i] = f2pk(f.x, f.y);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const uint64_t* x) {
  uint32_t w[4];
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = f2upk(x[i]);
      w[2 * i] = __float_as_uint(f.x);
      w[2 * i + 1] = __float_as_uint(f.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = f2upk(x[i]);
      w[i] = tc::pack2<T>(f.x, f.y);
    }
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return f2pk(x, x); }
__device__ __forceinline__ uint64_t swap2(uint64_t x) {
  const float2 f = f2upk(x);
  return f2pk(f.y, f.x);
}
__device__ __forceinline__ float add_halves(uint64_t x) {
  const float2 f = f2upk(x);
  return f.x + f.y;
}

// A slot's rotation as products: out = direct * x + cross * (the pair's other
// member), for VE packed neighbours (VE / 2 of each chunk). The other member
// sits at the same place of the other chunk, or (INTER) beside it. `sign`
// -1 turns back; w scales the components before the rotation. `mask` is 0
// for a chunk that is not rotated (for both, unless INTER): its zero factor
// alone would make an infinite other member NaN here. Where every component
// turns the masks are compiled out: their two ANDs a pair took the 16,384
// tokens from 64.8 to 67.3 us, and the half-rotated training case from 45.7 to
// 46.9.
template <typename T>
struct Turn {
  static constexpr int P = kVec<T>;
  uint64_t direct[P], cross[P];
  uint64_t mask[2];
};
template <typename T, bool INTER>
__device__ __forceinline__ void make_turn(Turn<T>* t, const Angles<T>& a,
                                          const float* w, float sign, int c0,
                                          int c1, int r2) {
  constexpr int VE = kVec<T>, H = VE / 2;
  const int end = (INTER ? 2 * r2 : r2) / VE;  // chunks (INTER: of both) turned
  t->mask[0] = c0 < end ? ~uint64_t(0) : 0;
  t->mask[1] = c1 < end ? ~uint64_t(0) : 0;
#pragma unroll
  for (int i = 0; i < H; ++i) {
    if constexpr (INTER) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = h * VE + 2 * i;          // the pair's first component
        const float c = a.c[h * H + i], s = sign * a.s[h * H + i];
        t->direct[h * H + i] = f2pk(c * w[e], c * w[e + 1]);
        t->cross[h * H + i] = f2pk(-s * w[e + 1], s * w[e]);
      }
    } else {
      const float c0 = a.c[2 * i], c1 = a.c[2 * i + 1];
      const float s0 = sign * a.s[2 * i], s1 = sign * a.s[2 * i + 1];
      const float* v = w + VE;
      t->direct[i] = f2pk(c0 * w[2 * i], c1 * w[2 * i + 1]);
      t->cross[i] = f2pk(-s0 * v[2 * i], -s1 * v[2 * i + 1]);
      t->direct[H + i] = f2pk(c0 * v[2 * i], c1 * v[2 * i + 1]);
      t->cross[H + i] = f2pk(s0 * w[2 * i], s1 * w[2 * i + 1]);
    }
  }
}
template <typename T, bool INTER, bool MASKED>
__device__ __forceinline__ uint64_t turned(const Turn<T>& t,
                                           const uint64_t* x, int i) {
  constexpr int H = kVec<T> / 2;
  uint64_t other = INTER ? swap2(x[i]) : x[i < H ? i + H : i - H];
  if constexpr (MASKED) other &= t.mask[INTER ? i / H : 0];
  return ffma2(x[i], t.direct[i], fmul2(other, t.cross[i]));
}

template <typename T, int G, bool INTER, bool MASKED, int BATCH>
__global__ void __launch_bounds__(kWarps * 32)
    qk_vec_forward_kernel(const __grid_constant__ QkVecArgs a) {
  constexpr int VE = kVec<T>;
  const QkProblem& p = a.p;
  allow_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x % 32, j = lane % G;
  int64_t g = (int64_t(blockIdx.x) * kWarps + threadIdx.x / 32) * (32 / G) +
              lane / G;
  const int side = g >= a.groups[0];
  if (side) g -= a.groups[0];
  const QkSide& s = p.side[side];
  const bool live = g < a.groups[side];
  if (!live) g = 0;
  const int per = a.groups_per_token[side];
  const int64_t token = per > 0 ? g / per : 0;
  const int h0 = per > 0 ? int(g - token * per) * a.heads_per_group : 0;
  const int h1 = !live ? h0
                       : (h0 + a.heads_per_group < s.H ? h0 + a.heads_per_group
                                                       : s.H);
  const int64_t b = token / p.N, n = token - b * p.N;
  const int chunks = p.D / VE, slots = (chunks + 1) / 2;
  int c0, c1;
  slot_chunks(j, slots, chunks, p.R2 / VE, INTER, &c0, &c1);
  const int64_t pos = live ? load_pos(p, b, n) : 0;
  const bool known = pos >= 0 && pos < p.P;
  const T* x = static_cast<const T*>(s.x) + b * s.sx[0] + n * s.sx[2];
  T* out = static_cast<T*>(s.out) + b * s.so[0] + n * s.so[2];
  Turn<T> rot;
  const float inv_d = 1.f / float(p.D);
  bool first = true;
  // Groups of one warp may have different head counts: the butterflies need
  // every lane, so the loop runs to the longest.
  const int most = __reduce_max_sync(0xffffffffu, h1 - h0);
  for (int hb = 0; hb < most; hb += BATCH) {
    Chunk<T> raw[BATCH][2];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      raw[i][0].u = raw[i][1].u = make_uint4(0, 0, 0, 0);
      const int h = h0 + hb + i;
      if (h < h1) {
        if (c0 >= 0)
          raw[i][0].u = __ldg(
              reinterpret_cast<const uint4*>(x + h * s.sx[1] + c0 * VE));
        if (c1 >= 0)
          raw[i][1].u = __ldg(
              reinterpret_cast<const uint4*>(x + h * s.sx[1] + c1 * VE));
      }
    }
    if (first) {
      // Weight and rotation of a component in one pair of factors, once per
      // token.
      Angles<T> ang;
      float w[2 * VE];
      load_angles<T, INTER>(p, pos, known, c0, c1, &ang);
      load_weight<T>(s, a.w_vec[side], c0, w);
      load_weight<T>(s, a.w_vec[side], c1, w + VE);
      make_turn<T, INTER>(&rot, ang, w, 1.f, c0, c1, p.R2);
      first = false;
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      uint64_t v[VE];
      unpack_chunk<T>(raw[i][0], v);
      unpack_chunk<T>(raw[i][1], v + VE / 2);
      uint64_t ss = 0;
#pragma unroll
      for (int e = 0; e < VE; ++e) ss = ffma2(v[e], v[e], ss);
      float r = rsqrtf(group_sum<G>(add_halves(ss)) * inv_d + p.eps);
      if (!known) r = NAN;
      const int h = h0 + hb + i;
      if (h >= h1) continue;
      const uint64_t r2 = both(r);
      uint64_t o[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e)
        o[e] = fmul2(turned<T, INTER, MASKED>(rot, v, e), r2);
      if (c0 >= 0) store_chunk<T>(out + h * s.so[1] + c0 * VE, o);
      if (c1 >= 0) store_chunk<T>(out + h * s.so[1] + c1 * VE, o + VE / 2);
    }
  }
}

// Backward: blocks 0 .. blocks[0] - 1 walk the queries' groups, the others
// the keys', so a lane's weight-gradient sums belong to one side.
template <typename T, int G, bool INTER, bool MASKED, int BATCH>
__global__ void __launch_bounds__(kWarps * 32)
    qk_vec_backward_kernel(const __grid_constant__ QkVecArgs a) {
  constexpr int VE = kVec<T>;
  __shared__ float sums[kWarps][G * 2 * VE];
  const QkProblem& p = a.p;
  allow_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, j = lane % G;
  const int side = int(blockIdx.x) >= a.blocks[0];
  const int block = int(blockIdx.x) - (side ? a.blocks[0] : 0);
  const QkSide& s = p.side[side];
  const int per = a.groups_per_token[side];
  const int chunks = p.D / VE, slots = (chunks + 1) / 2;
  int c0, c1;
  slot_chunks(j, slots, chunks, p.R2 / VE, INTER, &c0, &c1);
  uint64_t w2[VE], dw2[VE];
  {
    float w[2 * VE];
    load_weight<T>(s, a.w_vec[side], c0, w);
    load_weight<T>(s, a.w_vec[side], c1, w + VE);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      w2[e] = f2pk(w[2 * e], w[2 * e + 1]);
      dw2[e] = 0;
    }
  }
  const float inv_d = 1.f / float(p.D);
  const int64_t step = int64_t(a.blocks[side]) * kWarps * (32 / G);
  for (int64_t base = (int64_t(block) * kWarps + warp) * (32 / G);
       base < a.groups[side]; base += step) {
    int64_t g = base + lane / G;
    const bool live = g < a.groups[side];
    if (!live) g = 0;
    const int64_t token = g / per;
    const int h0 = int(g - token * per) * a.heads_per_group;
    const int h1 = !live
                       ? h0
                       : (h0 + a.heads_per_group < s.H ? h0 + a.heads_per_group
                                                       : s.H);
    const int64_t b = token / p.N, n = token - b * p.N;
    const int64_t pos = load_pos(p, b, n);
    const bool known = pos >= 0 && pos < p.P;
    Turn<T> rot;
    {
      Angles<T> ang;
      load_angles<T, INTER>(p, pos, known, c0, c1, &ang);
      float one[2 * VE];
#pragma unroll
      for (int e = 0; e < 2 * VE; ++e) one[e] = 1.f;
      make_turn<T, INTER>(&rot, ang, one, -1.f, c0, c1, p.R2);
    }
    const T* x = static_cast<const T*>(s.x) + b * s.sx[0] + n * s.sx[2];
    const T* dy = static_cast<const T*>(s.dy) + b * s.sy[0] + n * s.sy[2];
    T* out = static_cast<T*>(s.out) + b * s.so[0] + n * s.so[2];
    const int most = __reduce_max_sync(0xffffffffu, h1 - h0);
    for (int hb = 0; hb < most; hb += BATCH) {
      Chunk<T> rx[BATCH][2], ry[BATCH][2];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int h = h0 + hb + i;
        rx[i][0].u = rx[i][1].u = ry[i][0].u = ry[i][1].u =
            make_uint4(0, 0, 0, 0);
        if (h < h1) {
          if (c0 >= 0) {
            rx[i][0].u = __ldg(
                reinterpret_cast<const uint4*>(x + h * s.sx[1] + c0 * VE));
            ry[i][0].u = __ldg(
                reinterpret_cast<const uint4*>(dy + h * s.sy[1] + c0 * VE));
          }
          if (c1 >= 0) {
            rx[i][1].u = __ldg(
                reinterpret_cast<const uint4*>(x + h * s.sx[1] + c1 * VE));
            ry[i][1].u = __ldg(
                reinterpret_cast<const uint4*>(dy + h * s.sy[1] + c1 * VE));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        uint64_t v[VE], d[VE], t[VE];
        unpack_chunk<T>(rx[i][0], v);
        unpack_chunk<T>(rx[i][1], v + VE / 2);
        unpack_chunk<T>(ry[i][0], d);
        unpack_chunk<T>(ry[i][1], d + VE / 2);
        // t = g' v: the weight gradient's summand is t r, the dot product's
        // w t.
        uint64_t ss = 0, dot = 0, g2[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          g2[e] = turned<T, INTER, MASKED>(rot, d, e);
          ss = ffma2(v[e], v[e], ss);
          t[e] = fmul2(g2[e], v[e]);
          dot = ffma2(w2[e], t[e], dot);
        }
        float r = rsqrtf(group_sum<G>(add_halves(ss)) * inv_d + p.eps);
        const float c = group_sum<G>(add_halves(dot)) * r * r * inv_d;
        const int h = h0 + hb + i;
        if (h >= h1) continue;
        if (!known) r = NAN;
        const uint64_t r2 = both(r), rc = both(-r * c);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          dw2[e] = ffma2(t[e], r2, dw2[e]);
          g2[e] = ffma2(fmul2(g2[e], w2[e]), r2, fmul2(v[e], rc));
        }
        if (c0 >= 0) store_chunk<T>(out + h * s.so[1] + c0 * VE, g2);
        if (c1 >= 0)
          store_chunk<T>(out + h * s.so[1] + c1 * VE, g2 + VE / 2);
      }
    }
  }
  if (s.dw == nullptr) return;
  // The warp's groups, then the warps, in a fixed order.
  float dw[2 * VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const float2 f = f2upk(dw2[e]);
    dw[2 * e] = f.x;
    dw[2 * e + 1] = f.y;
  }
#pragma unroll
  for (int e = 0; e < 2 * VE; ++e) {
#pragma unroll
    for (int o = 16; o >= G; o >>= 1)
      dw[e] += __shfl_xor_sync(0xffffffffu, dw[e], o);
    if (lane < G) sums[warp][j * 2 * VE + e] = dw[e];
  }
  __syncthreads();
  float* part = a.partial + int64_t(blockIdx.x) * p.D;
  for (int q = threadIdx.x; q < G * 2 * VE; q += kWarps * 32) {
    int k0, k1;
    slot_chunks(q / (2 * VE), slots, chunks, p.R2 / VE, INTER, &k0, &k1);
    const int e = q % (2 * VE);
    const int chunk = e < VE ? k0 : k1;
    if (chunk < 0) continue;
    float t = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) t += sums[v][q];
    part[chunk * VE + e % VE] = t;
  }
}

// Adds the blocks' weight-gradient sums in order: blocks first[i] ..
// first[i] + count[i] - 1 hold side i.
struct QkFinish {
  QkProblem p;
  const float* partial;
  int first[2], count[2];
};
__global__ void __launch_bounds__(1024)
    qk_weight_finish_kernel(const QkFinish f) {
  __shared__ float sums[32][32];
  allow_dependents();
  grid_dependency_wait();
  const QkProblem& p = f.p;
  const QkSide& s = p.side[blockIdx.y];
  if (s.dw == nullptr) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int d = blockIdx.x * 32 + lane;
  const float* src = f.partial + int64_t(f.first[blockIdx.y]) * p.D;
  float t = 0.f;
  if (d < p.D) {
#pragma unroll 4
    for (int c = warp; c < f.count[blockIdx.y]; c += 32)
      t += __ldg(src + int64_t(c) * p.D + d);
  }
  sums[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && d < p.D) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) total += sums[w][lane];
    const int64_t i = d * s.sdw;
    if (s.w_dtype == VECTRA_F32)
      static_cast<float*>(s.dw)[i] = total;
    else if (s.w_dtype == VECTRA_F16)
      static_cast<__half*>(s.dw)[i] = from_f32<__half>(total);
    else
      static_cast<__nv_bfloat16*>(s.dw)[i] = from_f32<__nv_bfloat16>(total);
  }
}

bool lines_ok(const void* p, const int64_t* s, const int64_t* sizes, int es) {
  if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && (s[i] * es) % 16 != 0) return false;
  return sizes[3] <= 1 || s[3] == 1;
}

// Whether the vector kernels can run: whole 16-byte chunks everywhere, in
// the tables too, and at most 32 chunk pairs.
bool vec_ok(const QkProblem& p, bool backward) {
  const int es = p.dtype == VECTRA_F32 ? 4 : 2;
  const int ve = 16 / es;
  if (p.D % ve || p.D / ve > 64) return false;
  if ((p.interleaved ? 2 * p.R2 : p.R2) % ve) return false;
  if (p.R2 > 0 && ((reinterpret_cast<uintptr_t>(p.cos) & 15) ||
                   (reinterpret_cast<uintptr_t>(p.sin) & 15) ||
                   p.cos_ld % 4 || p.sin_ld % 4))
    return false;
  for (const QkSide& s : p.side) {
    const int64_t sizes[4] = {p.B, s.H, p.N, p.D};
    if (p.B * p.N * s.H == 0) continue;
    if (!lines_ok(s.x, s.sx, sizes, es) || !lines_ok(s.out, s.so, sizes, es))
      return false;
    if (backward && !lines_ok(s.dy, s.sy, sizes, es)) return false;
  }
  return true;
}

int lanes_of(const QkProblem& p) {
  const int slots = (p.D / (p.dtype == VECTRA_F32 ? 4 : 8) + 1) / 2;
  int g = 1;
  while (g < slots) g *= 2;
  return g;
}

// Heads per group: as many as still leave two groups for every lane group
// that the SMs hold at eight warps each, up to 16, so that a token's angles
// are read once for as many vectors as can be.
QkVecArgs vec_args(const QkProblem& p, int g) {
  QkVecArgs a{};
  a.p = p;
  const int64_t vectors = p.B * p.N * (p.side[0].H + p.side[1].H);
  const int64_t slots = int64_t(device_sm_count()) * 8 * (32 / g) * 2;
  a.heads_per_group = 16;
  while (a.heads_per_group > 1 && vectors / a.heads_per_group < slots)
    a.heads_per_group /= 2;
  for (int i = 0; i < 2; ++i) {
    a.groups_per_token[i] =
        (p.side[i].H + a.heads_per_group - 1) / a.heads_per_group;
    a.groups[i] = p.B * p.N * a.groups_per_token[i];
    a.w_vec[i] = (reinterpret_cast<uintptr_t>(p.side[i].w) & 15) == 0 &&
                 (p.side[i].sw == 1 || p.D == 1);
  }
  return a;
}

// Calls f with the lanes of a group, whether pairs are neighbours, and whether
// some components are not rotated, as compile-time constants.
template <typename T, typename F>
cudaError_t with_lanes(int g, const QkProblem& p, F&& f) {
  auto masked = [&](auto lanes, auto inter) {
    return p.D != 2 * p.R2 ? f(lanes, inter, std::true_type{})
                           : f(lanes, inter, std::false_type{});
  };
  auto inner = [&](auto lanes) {
    return p.interleaved ? masked(lanes, std::true_type{})
                         : masked(lanes, std::false_type{});
  };
  switch (g) {
    case 1:
      return inner(std::integral_constant<int, 1>{});
    case 2:
      return inner(std::integral_constant<int, 2>{});
    case 4:
      return inner(std::integral_constant<int, 4>{});
    case 8:
      return inner(std::integral_constant<int, 8>{});
    case 16:
      return inner(std::integral_constant<int, 16>{});
    default:
      return inner(std::integral_constant<int, 32>{});
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
  const cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (!vec_ok(p, false)) {
      const QkArgs a{p, nullptr};
      return launch_pdl(qk_general_kernel<T, false>,
                        dim3(unsigned(general_blocks(p)), 2),
                        dim3(kWarps * 32), 0, stream, a);
    }
    const int g = lanes_of(p);
    const QkVecArgs a = vec_args(p, g);
    const int64_t per_block = kWarps * (32 / g);
    const int64_t blocks =
        (a.groups[0] + a.groups[1] + per_block - 1) / per_block;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    return with_lanes<T>(g, p, [&](auto lanes, auto inter, auto masked) {
      constexpr int G = decltype(lanes)::value;
      constexpr bool I = decltype(inter)::value;
      constexpr bool K = decltype(masked)::value;
      return launch_pdl(a.heads_per_group == 1
                            ? qk_vec_forward_kernel<T, G, I, K, 1>
                            : qk_vec_forward_kernel<T, G, I, K, 4>,
                        dim3(unsigned(blocks)), dim3(kWarps * 32), 0, stream,
                        a);
    });
  });
  if (e == cudaSuccess) count_launches(1);
  return e;
}

cudaError_t run_qk_backward(const QkProblem& p, Workspace& ws,
                            cudaStream_t stream) {
  if (p.D == 0) return cudaSuccess;
  const bool weights = p.side[0].dw || p.side[1].dw;
  const bool vec = vec_ok(p, true) && p.B * p.N > 0 && p.side[0].H > 0 &&
                   p.side[1].H > 0;
  const int g = lanes_of(p);
  QkVecArgs a{};
  QkFinish f{p, nullptr, {0, 0}, {0, 0}};
  const int general = general_blocks(p);
  if (vec) {
    a = vec_args(p, g);
    // Blocks of each side in proportion to its vectors, four per SM in all.
    const int64_t per_block = kWarps * (32 / g);
    const int64_t all = a.groups[0] + a.groups[1];
    const int64_t most = int64_t(device_sm_count()) * 4;
    for (int i = 0; i < 2; ++i) {
      int64_t n = (a.groups[i] + per_block - 1) / per_block;
      const int64_t share = (most * a.groups[i] + all - 1) / all;
      if (n > share) n = share;
      a.blocks[i] = int(n < 1 ? 1 : n);
    }
    f.count[0] = a.blocks[0];
    f.first[1] = a.blocks[0];
    f.count[1] = a.blocks[1];
  } else {
    f.count[0] = f.count[1] = f.first[1] = general;
  }
  const int blocks = f.count[0] + f.count[1];
  float* partial = nullptr;
  if (weights)
    partial = static_cast<float*>(
        ws.take(size_t(blocks) * p.D * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;
  f.partial = a.partial = partial;
  cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (!vec) {
      const QkArgs ga{p, partial};
      return launch_pdl(qk_general_kernel<T, true>,
                        dim3(unsigned(general), 2), dim3(kWarps * 32), 0,
                        stream, ga);
    }
    return with_lanes<T>(g, p, [&](auto lanes, auto inter, auto masked) {
      constexpr int G = decltype(lanes)::value;
      constexpr bool I = decltype(inter)::value;
      constexpr bool K = decltype(masked)::value;
      return launch_pdl(qk_vec_backward_kernel<T, G, I, K, 2>,
                        dim3(unsigned(blocks)), dim3(kWarps * 32), 0, stream,
                        a);
    });
  });
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (!weights) return cudaSuccess;
  e = launch_pdl(qk_weight_finish_kernel,
                 dim3(unsigned((p.D + 31) / 32), 2), dim3(1024), 0, stream,
                 f);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace vectra
