// cross_rows.cu: attention to an encoder's states (cross.cuh) for few queries:
// up to 16 packed rows of a key head (single tokens, the subject of a price),
// bf16 and f16, head widths up to 128.
//
// Memory-bound: every key and value is read once, and in the backward pass
// every dk and dv is written once, by the one warp that also adds to dq. A
// warp owns all rows of a key head and walks 16 keys at a time, on warp-level
// matrix instructions (m16n8k16), whose 16 rows are the packed rows.
//
// A product over d may take d in any order, so that thread t of a quad loads 16
// neighbouring bytes of a key (8 components of every 32) and uses them as they
// are: word w of its piece stands for the fragment's pair. The loads are
// asynchronous copies into shared memory, several steps ahead, but a thread
// reads only what it copied itself: no barrier, no conflict. (With the next
// step's loads in registers instead, a step of 4,001 keys of 128 took a load's
// latency: 129 us for 32 decoding sequences.)
// Products that sum over keys or rows need fragments of the transposed matrix:
// one movmatrix an 8 x 8 block turns a word w of all threads into them, and the
// result's columns then lie in the same order as the loaded words, so results
// are stored, and a key is subtracted from its dk, in 16-byte pieces too.
//
//   S = q k^T, T = e v^T            operands as loaded
//   out += P v, dq += z k           v and k turned
//   dv = P^T e, dk = z^T q          P, z (and, once, e and q) turned
// float16 (cross.cuh): forward weights are multiplied by 2^14, P of dv too; z
// of dk by what its step's largest needs, z of dq by what its row's largest so
// far does, and dq's sums are brought along when that grows.
// What the rounding of P and z to an operand leaves is multiplied as well, as on
// the tensor cores (cross_tc.cu): the time goes to memory. z's sums over rows
// are products with ones.
//
// Measured against tcgen05 tiles, which are 128 rows high: one query of 32
// heads on up to 4,001 keys of 8 heads of 128, 32 sequences: 67 us (61 of them
// the keys, at 5.3 TB/s), with tiles 81; training of 1,024 subjects of 8 heads
// on 64 keys of 32: forward 18 and backward 45 us (41.5 without the second
// products of dk and dv), with tiles 1,050 together.
// Above 16 packed rows a fragment would no longer hold them.
#include <type_traits>

#include "cross.cuh"
#include "mma_sync.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 16;  // a step

__device__ __forceinline__ uint32_t turn(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ float2 pair(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(w << 16),
                       __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// log2 of what forward weights, 1 at most, are multiplied by, and that of P.
template <typename T>
constexpr float kLog2Lift = std::is_same<T, __half>::value ? 14.f : 0.f;
template <typename T>
constexpr float kLiftOf = std::is_same<T, __half>::value ? kLift : 1.f;

// One of T in both halves.
template <typename T>
__device__ __forceinline__ uint32_t ones() {
  return pack_pair<T>(1.f, 1.f);
}

// Two values as a pair of T, and what rounding left.
template <typename T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t* near,
                                           uint32_t* rest) {
  *near = pack_pair<T>(x, y);
  const float2 f = pair<T>(*near);
  *rest = pack_pair<T>(x - f.x, y - f.y);
}

// Sum over the four threads of a quad.
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}

// Thread t's 16 bytes of every 32 components of a row; zeros past `width` (a
// multiple of 8) and for rows that are not there.
template <int NB>
__device__ __forceinline__ void load_row(uint32_t (*w)[4], const void* row,
                                         bool live, int width, int t) {
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    uint4 x = make_uint4(0, 0, 0, 0);
    const int d = b * 32 + t * 8;
    if (live && d < width)
      x = __ldg(reinterpret_cast<const uint4*>(
          static_cast<const uint16_t*>(row) + d));
    w[b][0] = x.x;
    w[b][1] = x.y;
    w[b][2] = x.z;
    w[b][3] = x.w;
  }
}

// The rows of a fragment: g and g + 8 of the packed rows.
struct Row {
  bool live;
  int64_t at;   // of [B, H, Nq]
  int64_t h, i;
};
__device__ __forceinline__ Row packed_row(const CrossProblem& p, int64_t b,
                                          int64_t hk, int r) {
  Row w;
  w.live = r < p.Nq * p.G;
  w.i = r / int(p.G);
  w.h = hk * p.G + r % int(p.G);
  w.at = (b * p.H + w.h) * p.Nq + w.i;
  return w;
}
template <typename T>
__device__ __forceinline__ const T* row_of(const void* base, const int64_t* s,
                                           int64_t b, int64_t h, int64_t i) {
  return static_cast<const T*>(base) + b * s[0] + h * s[1] + i * s[2];
}
template <typename T>
__device__ __forceinline__ T* row_of(void* base, const int64_t* s, int64_t b,
                                     int64_t h, int64_t i) {
  return static_cast<T*>(base) + b * s[0] + h * s[1] + i * s[2];
}

// acc[8 n][.] += a b over the 32 components of every loaded word: S or T of 8
// keys. `a`: [row group][block][word].
template <typename T, int NB, int NR>
__device__ __forceinline__ void inner(float* c, const uint32_t (*a)[NB][4],
                                      const uint32_t (*b)[4]) {
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t f[4] = {a[0][n][2 * s], NR == 2 ? a[NR - 1][n][2 * s] : 0u,
                             a[0][n][2 * s + 1],
                             NR == 2 ? a[NR - 1][n][2 * s + 1] : 0u};
      mma16816<T>(c, f, b[n][2 * s], b[n][2 * s + 1]);
    }
}

// |k|^2 of 8 keys, of key g in every thread of quad g, as the pair of keys
// that the thread's columns are.
template <typename T, int NB>
__device__ __forceinline__ float2 squares(const uint32_t (*k)[4], int lane) {
  float s = 0.f;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 f = pair<T>(k[n][w]);
      s = fmaf(f.x, f.x, s);
      s = fmaf(f.y, f.y, s);
    }
  s = quad_sum(s);
  const int t = lane & 3;
  return make_float2(__shfl_sync(0xffffffffu, s, 8 * t),
                     __shfl_sync(0xffffffffu, s, 8 * t + 4));
}

__device__ __forceinline__ void copy16(void* dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   smem_addr(dst)),
               "l"(src), "r"(live ? 16 : 0)
               : "memory");
}

// The keys and values of the steps ahead: [step][k or v][half][block][thread].
template <typename T, int NB, int STAGES>
struct Ring {
  static constexpr int PIECES = 4 * NB;  // of a thread and step
  static constexpr int BYTES = STAGES * PIECES * kWarps * 32 * 16;
  uint4* mine;  // + piece * (kWarps * 32)

  __device__ __forceinline__ uint4* piece(int step, int which, int h, int n) {
    return mine + (((step % STAGES) * 2 + which) * 2 * NB + h * NB + n) *
                      (kWarps * 32);
  }
  // Step `step`, of which nothing at or past `end` or `len` is copied: zeros.
  __device__ __forceinline__ void fetch(const CrossProblem& p, int64_t b,
                                        int64_t hk, int step, int end, int len,
                                        int lane) {
    const int t = lane % 4;
    if (step < end) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = step * kKeys + 8 * h + lane / 4;
        const T* k = row_of<T>(p.k, p.sk, b, hk, key);
        const T* v = row_of<T>(p.v, p.sv, b, hk, key);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int d = n * 32 + t * 8;
          const bool live = key < len;
          copy16(piece(step, 0, h, n), live && d < p.D ? k + d : p.k,
                 live && d < p.D);
          copy16(piece(step, 1, h, n), live && d < p.Dv ? v + d : p.v,
                 live && d < p.Dv);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Waits until the oldest step but STAGES - 1 has landed.
  __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
  }
  __device__ __forceinline__ void read(int step, int which, int h,
                                       uint32_t (*w)[4]) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const uint4 x = *piece(step, which, h, n);
      w[n][0] = x.x;
      w[n][1] = x.y;
      w[n][2] = x.z;
      w[n][3] = x.w;
    }
  }
};

// Steps in flight: 128 to 192 KB an SM of the widest vectors.
template <int NB>
constexpr int kForwardStages = NB > 2 ? 3 : 4;
template <int NB>
constexpr int kBackwardStages = NB > 2 ? 2 : 3;

template <typename T, int NB, int NR>
__global__ void __launch_bounds__(kWarps * 32)
    rows_forward_kernel(const __grid_constant__ CrossProblem p) {
  allow_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int64_t unit = int64_t(blockIdx.x) * kWarps + threadIdx.x / 32;
  const int64_t plane = unit / p.splits;
  if (plane >= p.B * p.Hk) return;
  const int part = int(unit - plane * p.splits);
  const int64_t b = plane / p.Hk, hk = plane - b * p.Hk;
  const int len = cross_length(p, b);
  int t0, t1;
  split_range((len + kKeys - 1) / kKeys, part, p.splits, &t0, &t1);

  Row row[NR];
  uint32_t q[NR][NB][4];
  float gl[NR], m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    row[r] = packed_row(p, b, hk, g + 8 * r);
    load_row<NB>(q[r], row_of<T>(p.q, p.sq, b, row[r].h, row[r].i),
                 row[r].live, p.D, t);
    gl[r] = row[r].live ? cross_scale(p, b, row[r].h) * kLog2e : 0.f;
    m[r] = kNegInf;
    l[r] = 0.f;
  }
  float acc[NB * 4][4];
#pragma unroll
  for (int n = 0; n < NB * 4; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  extern __shared__ uint4 ring_memory[];
  constexpr int STAGES = kForwardStages<NB>;
  Ring<T, NB, STAGES> ring{ring_memory + threadIdx.x};
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
    ring.fetch(p, b, hk, t0 + i, t1, len, lane);
  for (int step = t0; step < t1; ++step) {
    ring.fetch(p, b, hk, step + STAGES - 1, t1, len, lane);
    ring.wait();
    float s[2][4];
    float2 nk[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t k[NB][4];
      ring.read(step, 0, h, k);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[h][i] = 0.f;
      inner<T, NB, NR>(s[h], q, k);
      nk[h] = squares<T, NB>(k, lane);
    }
    uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
    const int first = step * kKeys + 2 * t;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float x[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[2 * h] = gl[r] * fmaf(2.f, s[h][2 * r], -nk[h].x);
        x[2 * h + 1] = gl[r] * fmaf(2.f, s[h][2 * r + 1], -nk[h].y);
        if (first + 8 * h >= len) x[2 * h] = kNegInf;
        if (first + 8 * h + 1 >= len) x[2 * h + 1] = kNegInf;
      }
      const float top =
          quad_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
      const bool grows = top > m[r];
      if (__any_sync(0xffffffffu, grows)) {
        const float next = fmaxf(m[r], top);
        const float f = m[r] == kNegInf ? 0.f : fast_exp2(m[r] - next);
        m[r] = next;
        l[r] *= f;
#pragma unroll
        for (int n = 0; n < NB * 4; ++n) {
          acc[n][2 * r] *= f;
          acc[n][2 * r + 1] *= f;
        }
      }
      const float ref = m[r] == kNegInf ? 0.f : m[r] - kLog2Lift<T>;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = fast_exp2(x[i] - ref);
        l[r] += x[i];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        hi[2 * h + r] = pack_pair<T>(x[2 * h], x[2 * h + 1]);
        const float2 f = pair<T>(hi[2 * h + r]);
        lo[2 * h + r] = pack_pair<T>(x[2 * h] - f.x, x[2 * h + 1] - f.y);
      }
    }
    uint32_t v[2][NB][4];
    ring.read(step, 1, 0, v[0]);
    ring.read(step, 1, 1, v[1]);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t v0 = turn(v[0][n][w]), v1 = turn(v[1][n][w]);
        mma16816<T>(acc[n * 4 + w], hi, v0, v1);
        mma16816<T>(acc[n * 4 + w], lo, v0, v1);
      }
  }

  const int64_t rows = p.B * p.H * p.Nq;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    l[r] = quad_sum(l[r]);
    m[r] -= kLog2Lift<T>;
    if (!row[r].live) continue;
    const int64_t k_part = part * rows + row[r].at;
    const bool whole = p.splits == 1;
    const float inv = whole ? (len > 0 ? 1.f / l[r] : 0.f) : 1.f;
    if (t == 0) {
      if (!whole) {
        p.part_ml[2 * k_part] = m[r];
        p.part_ml[2 * k_part + 1] = l[r];
      } else if (p.lse) {
        p.lse[row[r].at] = len > 0 ? m[r] + log2f(l[r]) : INFINITY;
      }
    }
    T* out = row_of<T>(p.out, p.so, b, row[r].h, row[r].i);
    T* rest = p.rest ? static_cast<T*>(p.rest) + row[r].at * p.Dv : nullptr;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int d = n * 32 + t * 8;
      if (d >= p.Dv) continue;
      uint32_t w[4], x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a0 = acc[n * 4 + i][2 * r] * inv;
        const float a1 = acc[n * 4 + i][2 * r + 1] * inv;
        if (!whole) {
          *reinterpret_cast<float2*>(p.part + k_part * p.Dv + d + 2 * i) =
              make_float2(a0, a1);
          continue;
        }
        w[i] = pack_pair<T>(a0, a1);
        const float2 f = pair<T>(w[i]);
        x[i] = pack_pair<T>((a0 - f.x) * kRestLift<T>,
                            (a1 - f.y) * kRestLift<T>);
      }
      if (!whole) continue;
      *reinterpret_cast<uint4*>(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
      if (rest)
        *reinterpret_cast<uint4*>(rest + d) =
            make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
}

// Up to 8 rows: the rows are the fragments' 8 columns and the keys, or the
// components of out, their 16 rows, which takes half as many instructions on
// the tensor cores (whose warp-level form set the pace of a decoding step: 48 a
// step of 16 keys of 128 with the rows as rows, 79 us for 32 sequences over up
// to 4,001 keys).
//   S^T = k q^T, out^T += v^T P^T
template <typename T, int NB>
__global__ void __launch_bounds__(kWarps * 32)
    few_rows_forward_kernel(const __grid_constant__ CrossProblem p) {
  allow_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int64_t unit = int64_t(blockIdx.x) * kWarps + threadIdx.x / 32;
  const int64_t plane = unit / p.splits;
  if (plane >= p.B * p.Hk) return;
  const int part = int(unit - plane * p.splits);
  const int64_t b = plane / p.Hk, hk = plane - b * p.Hk;
  const int len = cross_length(p, b);
  int t0, t1;
  split_range((len + kKeys - 1) / kKeys, part, p.splits, &t0, &t1);

  extern __shared__ uint4 ring_memory[];
  constexpr int STAGES = kForwardStages<NB>;
  Ring<T, NB, STAGES> ring{ring_memory + threadIdx.x};
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
    ring.fetch(p, b, hk, t0 + i, t1, len, lane);

  const Row own = packed_row(p, b, hk, g);
  uint32_t q[NB][4];
  load_row<NB>(q, row_of<T>(p.q, p.sq, b, own.h, own.i), own.live, p.D, t);
  // Rows 2 t and 2 t + 1, the columns of this thread's fragments.
  float gl[2], m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const Row r = packed_row(p, b, hk, 2 * t + c);
    gl[c] = r.live ? cross_scale(p, b, r.h) * kLog2e : 0.f;
  }
  float acc[NB * 2][4];
#pragma unroll
  for (int n = 0; n < NB * 2; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  for (int step = t0; step < t1; ++step) {
    ring.fetch(p, b, hk, step + STAGES - 1, t1, len, lane);
    ring.wait();
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    float nk[2];
    {
      uint32_t k[2][NB][4];
      ring.read(step, 0, 0, k[0]);
      ring.read(step, 0, 1, k[1]);
      float sq[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int w = 0; w < 4; w += 2) {
          const uint32_t f[4] = {k[0][n][w], k[1][n][w], k[0][n][w + 1],
                                 k[1][n][w + 1]};
          mma16816<T>(s, f, q[n][w], q[n][w + 1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 f = pair<T>(k[h][n][w]);
            sq[h] = fmaf(f.x, f.x, sq[h]);
            sq[h] = fmaf(f.y, f.y, sq[h]);
          }
      }
      nk[0] = quad_sum(sq[0]);
      nk[1] = quad_sum(sq[1]);
    }
    // s[2 h + c]: key g + 8 h, row 2 t + c.
    float x[4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool in = step * kKeys + 8 * h + g < len;
        x[2 * h + c] =
            in ? gl[c] * fmaf(2.f, s[2 * h + c], -nk[h]) : kNegInf;
      }
    bool grows = false;
    float top[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      top[c] = fmaxf(x[c], x[2 + c]);
#pragma unroll
      for (int o = 4; o < 32; o *= 2)
        top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
      grows = grows || top[c] > m[c];
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float next = fmaxf(m[c], top[c]);
        const float f = m[c] == kNegInf ? 0.f : fast_exp2(m[c] - next);
        m[c] = next;
        l[c] *= f;
#pragma unroll
        for (int n = 0; n < NB * 2; ++n) {
          acc[n][c] *= f;
          acc[n][2 + c] *= f;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float ref = m[c] == kNegInf ? 0.f : m[c] - kLog2Lift<T>;
        x[2 * h + c] = fast_exp2(x[2 * h + c] - ref);
        l[c] += x[2 * h + c];
      }
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = pack_pair<T>(x[2 * h], x[2 * h + 1]);
      hi[h] = turn(w);
      const float2 f = pair<T>(w);
      lo[h] = turn(pack_pair<T>(x[2 * h] - f.x, x[2 * h + 1] - f.y));
    }
    uint32_t v[2][NB][4];
    ring.read(step, 1, 0, v[0]);
    ring.read(step, 1, 1, v[1]);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int w = 0; w < 4; w += 2) {
        const uint32_t f[4] = {turn(v[0][n][w]), turn(v[0][n][w + 1]),
                               turn(v[1][n][w]), turn(v[1][n][w + 1])};
        mma16816<T>(acc[n * 2 + w / 2], f, hi[0], hi[1]);
        mma16816<T>(acc[n * 2 + w / 2], f, lo[0], lo[1]);
      }
  }

  const int64_t rows = p.B * p.H * p.Nq;
  const bool whole = p.splits == 1;
  float inv[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int o = 4; o < 32; o *= 2)
      l[c] += __shfl_xor_sync(0xffffffffu, l[c], o);
    inv[c] = whole ? (len > 0 ? 1.f / l[c] : 0.f) : 1.f;
    m[c] -= kLog2Lift<T>;
    const Row r = packed_row(p, b, hk, 2 * t + c);
    if (g != 0 || !r.live) continue;
    if (!whole) {
      const int64_t at = part * rows + r.at;
      p.part_ml[2 * at] = m[c];
      p.part_ml[2 * at + 1] = l[c];
    } else if (p.lse) {
      p.lse[r.at] = len > 0 ? m[c] + log2f(l[c]) : INFINITY;
    }
  }
  if (!whole) {
    // acc[2 n + w / 2][2 (w % 2) + c]: row 2 t + c, component
    // 32 n + 8 (g / 2) + 2 w + g % 2.
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Row r = packed_row(p, b, hk, 2 * t + c);
      if (!r.live) continue;
      float* out = p.part + (part * rows + r.at) * p.Dv;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int d = n * 32 + 8 * (g / 2) + 2 * w + g % 2;
          if (d < p.Dv) out[d] = acc[n * 2 + w / 2][2 * (w % 2) + c];
        }
    }
    return;
  }
  T* out = row_of<T>(p.out, p.so, b, own.h, own.i);
  T* rest = p.rest ? static_cast<T*>(p.rest) + own.at * p.Dv : nullptr;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int d = n * 32 + t * 8;
    uint32_t w[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a0 = acc[n * 2 + i / 2][2 * (i % 2)] * inv[0];
      const float a1 = acc[n * 2 + i / 2][2 * (i % 2) + 1] * inv[1];
      const uint32_t pr = pack_pair<T>(a0, a1);
      w[i] = turn(pr);
      const float2 f = pair<T>(pr);
      x[i] = turn(pack_pair<T>((a0 - f.x) * kRestLift<T>,
                               (a1 - f.y) * kRestLift<T>));
    }
    if (!own.live || d >= p.Dv) continue;
    *reinterpret_cast<uint4*>(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
    if (rest)
      *reinterpret_cast<uint4*>(rest + d) = make_uint4(x[0], x[1], x[2], x[3]);
  }
}

// The turned q and e of dk and dv, [warp][q or e][block][row group and word]:
// in shared memory for widths whose registers they would take.
template <int NB>
constexpr bool kTurnedInShared = NB > 2;

template <typename T, int NB, int NR>
__global__ void __launch_bounds__(kWarps * 32, NB > 2 ? 2 : 3)
    rows_backward_kernel(const __grid_constant__ CrossProblem p) {
  constexpr bool kShared = kTurnedInShared<NB>;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  constexpr int STAGES = kBackwardStages<NB>;
  extern __shared__ uint4 ring_memory[];
  // Behind the ring.
  uint4(*turned)[32] = reinterpret_cast<uint4(*)[32]>(
      ring_memory + Ring<T, NB, STAGES>::BYTES / 16);
  allow_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int64_t unit = int64_t(blockIdx.x) * kWarps + warp;
  const int64_t plane = unit / p.splits;
  if (plane >= p.B * p.Hk) return;
  const int part = int(unit - plane * p.splits);
  const int64_t b = plane / p.Hk, hk = plane - b * p.Hk;
  const int len = cross_length(p, b);
  // Steps of all keys: those that are not seen have zero gradients.
  int t0, t1;
  split_range(int((p.Nk + kKeys - 1) / kKeys), part, p.splits, &t0, &t1);

  Row row[NR];
  uint32_t q[NR][NB][4], e[NR][NB][4];
  float gl[NR], g2[NR], lse[NR], ci[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    row[r] = packed_row(p, b, hk, g + 8 * r);
    const bool live = row[r].live && len > 0;
    load_row<NB>(q[r], row_of<T>(p.q, p.sq, b, row[r].h, row[r].i), live, p.D,
                 t);
    load_row<NB>(e[r], row_of<T>(p.dout, p.se, b, row[r].h, row[r].i), live,
                 p.Dv, t);
    const float scale = live ? cross_scale(p, b, row[r].h) : 0.f;
    gl[r] = scale * kLog2e;
    g2[r] = 2.f * scale;
    lse[r] = live ? p.lse[row[r].at] : INFINITY;  // weighs nothing
    // c_i = e_i . out_i, with what out's rounding left.
    float c = 0.f;
    const T* out = row_of<T>(p.out, p.so, b, row[r].h, row[r].i);
    const T* rest = static_cast<const T*>(p.rest) + row[r].at * p.Dv;
    uint32_t o[NB][4], x[NB][4];
    load_row<NB>(o, out, live, p.Dv, t);
    load_row<NB>(x, rest, live, p.Dv, t);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 a = pair<T>(o[n][w]), d = pair<T>(x[n][w]),
                     f = pair<T>(e[r][n][w]);
        c = fmaf(fmaf(d.x, 1.f / kRestLift<T>, a.x), f.x, c);
        c = fmaf(fmaf(d.y, 1.f / kRestLift<T>, a.y), f.y, c);
      }
    ci[r] = quad_sum(c);
  }
  uint32_t qt[kShared ? 1 : NR][NB][4], et[kShared ? 1 : NR][NB][4];
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      uint32_t a[4], c[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        a[w] = turn(q[r][n][w]);
        c[w] = turn(e[r][n][w]);
        if constexpr (!kShared) {
          qt[r][n][w] = a[w];
          et[r][n][w] = c[w];
        }
      }
      if constexpr (kShared) {
        turned[((warp * 2 + 0) * NB + n) * NR + r][lane] =
            make_uint4(a[0], a[1], a[2], a[3]);
        turned[((warp * 2 + 1) * NB + n) * NR + r][lane] =
            make_uint4(c[0], c[1], c[2], c[3]);
      }
    }
  __syncwarp();

  float dq[NB * 4][4];
#pragma unroll
  for (int n = 0; n < NB * 4; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) dq[n][i] = 0.f;
  float xs[NR], ys[NR], zx[NR];
  float up[NR];  // float16: what z of dq is multiplied by
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    xs[r] = ys[r] = zx[r] = 0.f;
    up[r] = kScaled ? scale_up_to(0.f, 0) : 1.f;
  }

  Ring<T, NB, STAGES> ring{ring_memory + threadIdx.x};
  const int t_seen = min(t1, (len + kKeys - 1) / kKeys);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
    ring.fetch(p, b, hk, t0 + i, t_seen, len, lane);
  for (int step = t0; step < t1; ++step) {
    ring.fetch(p, b, hk, step + STAGES - 1, t_seen, len, lane);
    ring.wait();
    T* dk[2];
    T* dv[2];
    bool live_key[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = step * kKeys + 8 * h + g;
      live_key[h] = key < p.Nk;
      dk[h] = row_of<T>(p.dk, p.sdk, b, hk, key);
      dv[h] = row_of<T>(p.dv, p.sdv, b, hk, key);
    }
    if (step * kKeys >= len) {
      if (!p.dk) break;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int d = n * 32 + t * 8;
          const uint4 zero = make_uint4(0, 0, 0, 0);
          if (live_key[h] && d < p.D)
            *reinterpret_cast<uint4*>(dk[h] + d) = zero;
          if (live_key[h] && d < p.Dv)
            *reinterpret_cast<uint4*>(dv[h] + d) = zero;
        }
      continue;
    }
    uint32_t k[2][NB][4];
    float s[2][4], u[2][4];
    float2 nk[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[NB][4];
      ring.read(step, 0, h, k[h]);
      ring.read(step, 1, h, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[h][i] = u[h][i] = 0.f;
      inner<T, NB, NR>(s[h], q, k[h]);
      inner<T, NB, NR>(u[h], e, v);
      nk[h] = squares<T, NB>(k[h], lane);
    }
    // P and z of the 16 keys, and what rounding left of them; z for dk has its
    // row's scale before rounding.
    uint32_t pw[4] = {0, 0, 0, 0}, zw[4] = {0, 0, 0, 0}, zk[4] = {0, 0, 0, 0};
    uint32_t pl[4] = {0, 0, 0, 0}, zl[4] = {0, 0, 0, 0}, kl[4] = {0, 0, 0, 0};
    const int first = step * kKeys + 2 * t;
    float z[NR][2][2];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a = fmaf(2.f, s[h][2 * r + i], i ? -nk[h].y : -nk[h].x);
          const bool in = first + 8 * h + i < len;
          w[i] = in ? fast_exp2(fmaf(gl[r], a, -lse[r])) : 0.f;
          z[r][h][i] = in ? w[i] * (u[h][2 * r + i] - ci[r]) : 0.f;
          if (in) {
            xs[r] = fmaf(z[r][h][i], a, xs[r]);
            ys[r] = fmaf(w[i], a, ys[r]);
            zx[r] += z[r][h][i];
          }
        }
        split_pair<T>(w[0] * kLiftOf<T>, w[1] * kLiftOf<T>, &pw[2 * h + r],
                      &pl[2 * h + r]);
      }
    float up_k = 1.f;  // what z of dk is multiplied by
    if constexpr (kScaled) {
      float all = 0.f;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float top = quad_max(
            fmaxf(fmaxf(fabsf(z[r][0][0]), fabsf(z[r][0][1])),
                  fmaxf(fabsf(z[r][1][0]), fabsf(z[r][1][1]))));
        all = fmaxf(all, fabsf(g2[r]) * top);
        // To 2^10, until one reaches 2^14.
        const bool grows = top * up[r] > 0x1p14f;
        if (__any_sync(0xffffffffu, grows)) {
          const float next = grows ? scale_up_to(top, 10) : up[r];
          const float f = next * inverse_of(up[r]);
          up[r] = next;
#pragma unroll
          for (int n = 0; n < NB * 4; ++n) {
            dq[n][2 * r] *= f;
            dq[n][2 * r + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int o = 4; o < 32; o *= 2)
        all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
      up_k = scale_up_to(all, 13);
    }
    const float down_k = inverse_of(up_k);
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        split_pair<T>(z[r][h][0] * up[r], z[r][h][1] * up[r], &zw[2 * h + r],
                      &zl[2 * h + r]);
        split_pair<T>(g2[r] * z[r][h][0] * up_k, g2[r] * z[r][h][1] * up_k,
                      &zk[2 * h + r], &kl[2 * h + r]);
      }
    // dq += z k.
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int w = 0; w < 4; ++w)
      {
        const uint32_t k0 = turn(k[0][n][w]), k1 = turn(k[1][n][w]);
        mma16816<T>(dq[n * 4 + w], zw, k0, k1);
        mma16816<T>(dq[n * 4 + w], zl, k0, k1);
      }
    if (!p.dk) continue;
    // P^T and z^T: fragments of 16 keys by 16 rows.
    const uint32_t pt[4] = {turn(pw[0]), turn(pw[2]), turn(pw[1]),
                            turn(pw[3])};
    const uint32_t zt[4] = {turn(zk[0]), turn(zk[2]), turn(zk[1]),
                            turn(zk[3])};
    const uint32_t ptl[4] = {turn(pl[0]), turn(pl[2]), turn(pl[1]),
                             turn(pl[3])};
    const uint32_t ztl[4] = {turn(kl[0]), turn(kl[2]), turn(kl[1]),
                             turn(kl[3])};
    float ksum[4] = {0.f, 0.f, 0.f, 0.f};
    mma16816<T>(ksum, zt, ones<T>(), ones<T>());
    mma16816<T>(ksum, ztl, ones<T>(), ones<T>());
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      uint32_t qb[2][4], eb[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int w = 0; w < 4; ++w) qb[r][w] = eb[r][w] = 0;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if constexpr (kShared) {
          const uint4 a = turned[((warp * 2 + 0) * NB + n) * NR + r][lane];
          const uint4 c = turned[((warp * 2 + 1) * NB + n) * NR + r][lane];
          qb[r][0] = a.x, qb[r][1] = a.y, qb[r][2] = a.z, qb[r][3] = a.w;
          eb[r][0] = c.x, eb[r][1] = c.y, eb[r][2] = c.z, eb[r][3] = c.w;
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            qb[r][w] = qt[r][n][w];
            eb[r][w] = et[r][n][w];
          }
        }
      }
      float a[4][4], c[4][4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[w][i] = c[w][i] = 0.f;
        mma16816<T>(a[w], zt, qb[0][w], qb[1][w]);
        mma16816<T>(a[w], ztl, qb[0][w], qb[1][w]);
        mma16816<T>(c[w], pt, eb[0][w], eb[1][w]);
        mma16816<T>(c[w], ptl, eb[0][w], eb[1][w]);
      }
      const int d = n * 32 + t * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!live_key[h]) continue;
        uint32_t x[4], y[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 f = pair<T>(k[h][n][w]);  // 0 where not seen
          x[w] = pack_pair<T>((a[w][2 * h] - f.x * ksum[2 * h]) * down_k,
                              (a[w][2 * h + 1] - f.y * ksum[2 * h]) * down_k);
          y[w] = pack_pair<T>(c[w][2 * h] * (1.f / kLiftOf<T>),
                              c[w][2 * h + 1] * (1.f / kLiftOf<T>));
        }
        if (d < p.D)
          *reinterpret_cast<uint4*>(dk[h] + d) =
              make_uint4(x[0], x[1], x[2], x[3]);
        if (d < p.Dv)
          *reinterpret_cast<uint4*>(dv[h] + d) =
              make_uint4(y[0], y[1], y[2], y[3]);
      }
    }
  }

  const int64_t rows = p.B * p.H * p.Nq;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    xs[r] = quad_sum(xs[r]);
    ys[r] = quad_sum(ys[r]);
    zx[r] = quad_sum(zx[r]);
    if (!row[r].live) continue;
    const int64_t k_part = part * rows + row[r].at;
    if (p.dscale_rows && t == 0) {
      // Minus: the finish kernel takes sums of distances (cross_tc.cu).
      p.dscale_rows[k_part * 3] = -xs[r];
      p.dscale_rows[k_part * 3 + 1] = -ys[r];
      p.dscale_rows[k_part * 3 + 2] = zx[r];
    }
    if (!p.dq) continue;
    T* out = row_of<T>(p.dq, p.sdq, b, row[r].h, row[r].i);
    const float down = inverse_of(up[r]);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int d = n * 32 + t * 8;
      if (d >= p.D) continue;
      uint32_t x[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 f = pair<T>(q[r][n][w]);
        const float a0 = g2[r] * (dq[n * 4 + w][2 * r] * down - f.x * zx[r]);
        const float a1 =
            g2[r] * (dq[n * 4 + w][2 * r + 1] * down - f.y * zx[r]);
        if (p.splits > 1)
          *reinterpret_cast<float2*>(p.part + k_part * p.D + d + 2 * w) =
              make_float2(a0, a1);
        x[w] = pack_pair<T>(a0, a1);
      }
      if (p.splits == 1)
        *reinterpret_cast<uint4*>(out + d) =
            make_uint4(x[0], x[1], x[2], x[3]);
    }
  }
}

template <typename F>
cudaError_t with_shape(const CrossProblem& p, F&& f) {
  const int w = p.D > p.Dv ? p.D : p.Dv;
  const bool two = p.Nq * p.G > 8;
  const auto typed = [&](auto* type) {
    const auto groups = [&](auto nb) {
      return two ? f(type, nb, std::integral_constant<int, 2>{})
                 : f(type, nb, std::integral_constant<int, 1>{});
    };
    return w <= 32   ? groups(std::integral_constant<int, 1>{})
           : w <= 64 ? groups(std::integral_constant<int, 2>{})
                     : groups(std::integral_constant<int, 4>{});
  };
  return p.dtype == VECTRA_BF16 ? typed(static_cast<__nv_bfloat16*>(nullptr))
                                : typed(static_cast<__half*>(nullptr));
}

// Warps a key head's keys are split over: three times what the SMs hold, so
// that sequences of different lengths even out, of eight steps at least; where
// there are few key heads, what the SMs hold, of two steps at least.
int splits_for(const CrossProblem& p) {
  const int64_t planes = p.B * p.Hk, steps = (p.Nk + kKeys - 1) / kKeys;
  const int w = p.D > p.Dv ? p.D : p.Dv;
  const int64_t hold = int64_t(device_sm_count()) * (w > 64 ? 8 : 16);
  if (planes == 0) return 1;
  int64_t s = 3 * hold / planes;
  if (s > steps / 8) s = steps / 8;
  if (s * planes < hold) {
    s = hold / planes;
    if (s > steps / 2) s = steps / 2;
  }
  if (s > 64) s = 64;
  return s < 1 ? 1 : int(s);
}

float* take_floats(Workspace& ws, int64_t n) {
  return static_cast<float*>(ws.take(size_t(n) * sizeof(float)));
}

bool rows_ok(const void* base, const int64_t* s, const int64_t* sizes) {
  if (base == nullptr) return true;
  if (reinterpret_cast<uintptr_t>(base) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && s[i] % 8 != 0) return false;
  return s[3] == 1;
}

}  // namespace

bool cross_rows_supports(const CrossProblem& p, bool backward) {
  if (p.dtype != VECTRA_BF16 && p.dtype != VECTRA_F16) return false;
  if (p.Nq * p.G > 16 || p.D > 128 || p.Dv > 128 || p.D % 8 || p.Dv % 8)
    return false;
  const int64_t q[3] = {p.B, p.H, p.Nq}, k[3] = {p.B, p.Hk, p.Nk};
  if (!rows_ok(p.q, p.sq, q) || !rows_ok(p.k, p.sk, k) ||
      !rows_ok(p.v, p.sv, k) || !rows_ok(p.out, p.so, q) ||
      (reinterpret_cast<uintptr_t>(p.rest) & 15))
    return false;
  return !backward ||
         (rows_ok(p.dout, p.se, q) && rows_ok(p.dq, p.sdq, q) &&
          rows_ok(p.dk, p.sdk, k) && rows_ok(p.dv, p.sdv, k));
}

cudaError_t run_cross_rows_forward(const CrossProblem& problem, Workspace& ws,
                                   cudaStream_t stream) {
  CrossProblem p = problem;
  const int64_t rows = p.B * p.H * p.Nq;
  p.splits = splits_for(p);
  if (p.splits > 1) {
    p.part = take_floats(ws, p.splits * rows * p.Dv);
    p.part_ml = take_floats(ws, p.splits * rows * 2);
  }
  if (ws.dry || ws.overflow || rows == 0) return cudaSuccess;
  const int64_t blocks = (p.B * p.Hk * p.splits + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const cudaError_t e = with_shape(p, [&](auto* t, auto nb, auto nr) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int NB = decltype(nb)::value;
    constexpr int bytes = Ring<T, NB, kForwardStages<NB>>::BYTES;
    auto kern = rows_forward_kernel<T, NB, 2>;
    if (decltype(nr)::value == 1)
      kern = few_rows_forward_kernel<T, NB>;
    const cudaError_t st = cudaFuncSetAttribute(
        kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (st != cudaSuccess) return st;
    return launch_pdl(kern, dim3(unsigned(blocks)), dim3(kWarps * 32), bytes,
                      stream, p);
  });
  if (e != cudaSuccess) return e;
  count_launches(1);
  return p.splits == 1 ? e : launch_cross_join(p, stream);
}

cudaError_t run_cross_rows_backward(const CrossProblem& problem, Workspace& ws,
                                    cudaStream_t stream) {
  CrossProblem p = problem;
  const int64_t rows = p.B * p.H * p.Nq;
  p.splits = splits_for(p);
  if (p.dscale) p.dscale_rows = take_floats(ws, p.splits * rows * 3);
  if (p.splits > 1 && p.dq) p.part = take_floats(ws, p.splits * rows * p.D);
  if (ws.dry || ws.overflow) return cudaSuccess;
  const int64_t blocks = (p.B * p.Hk * p.splits + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  cudaError_t e = cudaSuccess;
  if (blocks > 0) {
    e = with_shape(p, [&](auto* t, auto nb, auto nr) {
      using T = std::remove_pointer_t<decltype(t)>;
      constexpr int NB = decltype(nb)::value, NR = decltype(nr)::value;
      constexpr int bytes =
          Ring<T, NB, kBackwardStages<NB>>::BYTES +
          (kTurnedInShared<NB> ? kWarps * 2 * NB * NR * 32 * 16 : 0);
      auto kern = rows_backward_kernel<T, NB, NR>;
      const cudaError_t st = cudaFuncSetAttribute(
          kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (st != cudaSuccess) return st;
      return launch_pdl(kern, dim3(unsigned(blocks)), dim3(kWarps * 32), bytes,
                        stream, p);
    });
    if (e == cudaSuccess) count_launches(1);
  }
  if (e == cudaSuccess && p.dq && p.splits > 1)
    e = launch_cross_sum(p.dtype, p.part, p.splits, p.B, p.H, p.Nq, p.D, p.dq,
                         p.sdq, stream);
  if (e == cudaSuccess && p.dscale)
    e = launch_cross_dscale(p, p.splits, stream);
  return e;
}

}  // namespace vectra
