// cross_tc.cu: attention to an encoder's states (cross.cuh) on the 5th
// generation tensor cores: bf16 and f16, head widths up to 128, tensors that
// tensor maps describe.
//
// One block owns 128 rows and walks tiles of columns: packed queries over keys
// (forward, dq), or keys over packed queries (dk and dv). With row operands
// r, r' and column operands c, c' (q, e and k, v, or the other way round) a
// tile of the
//   forward pass is  S = r c^T, P = 2^(logit - max), O += P c'
//   backward passes  S = r c^T, T = r' c'^T, P and z from both,
//                    acc += z c, and for keys acc' += P c'.
// |q_i - k_j|^2 = |q_i|^2 - (2 S - |k_j|^2), and |q_i|^2 cancels in a softmax
// over j, so a logit is g (2 S - |k_j|^2). Products with P and z take them
// from TMEM, rounded to 16 bits, where they lie as the first operand has to:
// the transposed form of the keys' pass needs no transposition.
//
// Warps: two warpgroups form P and z, one thread a row, each of one half of a
// tile's columns, while the tensor cores work on the next tile's S and T (two
// tiles are in TMEM); a TMA producer; an MMA issuer; a warpgroup for the
// columns' terms, which are |k_j|^2, or a query's lse, c_i and scale. Where
// several blocks walk the same keys their |k_j|^2 are formed once beforehand; a
// lone block (a decoding step) forms them from the tile in shared memory (two
// warps doing that in every block set the pace: 627 us of 4,096 queries on
// 5,003 keys, 32 heads of 128, against 432 without). In the forward pass every
// warpgroup has its own accumulator, maximum and sum, joined once at the end:
// nothing is exchanged on the way.
//
// Lengths: tiles past a sequence's length are not walked. In the last tile the
// unseen rows of the operand that a product sums over are overwritten with
// zeros in shared memory, so that what they held (NaN included) meets no
// weight.
//
// P and z enter their products as two 16-bit numbers, the second what the
// first's rounding left, so that each result is off by its own rounding (bf16
// 1.7e-3) alone. With the first numbers only it were 1.8e-3 of out, 2.35e-3 of
// dk and dv, and 3.2e-3 of dq, whose errors meet the distances between q_i and
// the keys, c_i's too.
//
// float16 (cross.cuh): forward weights, at most 2^8, are multiplied by 2^7, P
// of dv by 2^14, z of dq by what a bound of its row needs and z of dk by what
// that of its key head does: |z_ij| <= P_ij |e_i| (|v_j| + |out_i|), at most
// 2 |e_i| max |v_j|. (A query's share of dk loses bits where its weight times its
// gradient over the largest of its key head is below 2^-23.) The bounds' kernel
// takes 27 us of all gradients of the training below in f16, their use 50.
//
// Measured: 4,096 queries of 32 heads on 5,003 keys of 8 heads of 128, f16:
// 452 us by itself and 524 call after call, 640 TFLOP/s of the formula's; bound
// by the latency of the row warps, two a scheduler (tensor pipe 51 %, issue
// 43 %). (396 and 441 us without the second products.) Training of 2,048 queries
// of 16 heads on up to 4,500 keys of 4 heads of 128, batch 4, bf16: forward 305,
// all gradients 855 us (775 without the second products of dk and dv; tensor
// pipe 54 %, issue 43 %).
#include <atomic>
#include <type_traits>

#include "cross.cuh"
#include "tcgen05.cuh"

namespace vectra {
namespace {

using namespace tc;

enum Pass { kForward = 0, kQueries = 1, kKeys = 2 };

constexpr int kRows = 128;
constexpr int kThreads = 512;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kTermWarp = 12;
constexpr int kTermThreads = 128;
constexpr float kRescaleThreshold = 8.f;  // log2 of the lazy-rescale factor
// log2 of what forward weights, at most 2^8, are multiplied by.
template <typename T>
constexpr float kLog2Lift = std::is_same<T, __half>::value ? 7.f : 0.f;
// Registers after the launch's equal share: the warpgroups that hold a row of
// a tile, and the others (checked against the launch's total on the host).
constexpr int kRowRegs = 200;
constexpr int kOtherRegs = 56;

template <int W, int PASS>
struct Cfg {
  static_assert(W == 64 || W == 128, "width");
  static constexpr bool kBack = PASS != kForward;
  static constexpr int CN = kBack ? 64 : 128;  // columns of a tile
  static constexpr int KB = W / 64;            // 128-byte pieces of a vector
  static constexpr int RBLOCK = kRows * 128;
  static constexpr int CBLOCK = CN * 128;
  static constexpr int RTILE = RBLOCK * KB;
  static constexpr int CTILE = CBLOCK * KB;
  static constexpr int STAGE = 2 * CTILE;      // c then c'
  static constexpr int NS = kBack || W == 64 ? 4 : 3;
  static constexpr int OFF_R = 0;
  static constexpr int OFF_C = OFF_R + RTILE * (kBack ? 2 : 1);
  // Column terms: |k|^2, or lse, c_i, g log2e and 2 g.
  static constexpr int TERMS = PASS == kKeys ? 4 : 1;
  static constexpr int OFF_TERM = OFF_C + NS * STAGE;
  static constexpr int OFF_JOIN = OFF_TERM + NS * TERMS * CN * 4;
  static constexpr int JOIN = 4;               // floats a row and warpgroup
  static constexpr int OFF_BAR = OFF_JOIN + (kBack ? 2 * kRows * JOIN * 4 : 0);
  static constexpr int NBAR = 6 + 3 * NS;
  static constexpr int OFF_TMEM = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_TMEM + 16;
  static constexpr int SMEM_ALLOC = SMEM + 1024;  // for 1024-byte alignment
  static_assert(SMEM_ALLOC <= 232448, "shared memory");
  // TMEM columns: S of two tiles, T of two (backward), accumulators. Each
  // warpgroup's P overlays its half of S, z that of T.
  static constexpr int S0 = 0, T0 = 2 * CN, A0 = kBack ? 4 * CN : 2 * CN;
  static constexpr int TMEM_COLS = 512;
  static_assert(A0 + 2 * W <= TMEM_COLS, "TMEM");
};

struct TcArgs {
  CrossProblem p;
  int32_t rows_i;   // queries in a row tile (kRows / G), or kRows keys
  int32_t cols_i;   // queries in a column tile, or CN keys
  int32_t row_bytes, col_bytes;  // of one 128-byte piece's box
};

// Loads that have landed when the statement ends (tcgen05.cuh, tmem_load32):
// 64 columns at one address, or 32 at each of two.
#define VECTRA_R8(a, i) "=&r"(a[i]), "=&r"(a[i + 1]), "=&r"(a[i + 2]), \
      "=&r"(a[i + 3]), "=&r"(a[i + 4]), "=&r"(a[i + 5]), "=&r"(a[i + 6]), \
      "=&r"(a[i + 7])
__device__ __forceinline__ void tmem_load64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, "
      "%7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, "
      "%35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, "
      "%49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, "
      "%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : VECTRA_R8(r, 0), VECTRA_R8(r, 8), VECTRA_R8(r, 16), VECTRA_R8(r, 24),
        VECTRA_R8(r, 32), VECTRA_R8(r, 40), VECTRA_R8(r, 48), VECTRA_R8(r, 56)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_load32x2(uint32_t t0, uint32_t* r,
                                              uint32_t t1, uint32_t* q) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, "
      "%7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, "
      "%38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, "
      "%52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];"
      "\n\ttcgen05.wait::ld.sync.aligned;"
      : VECTRA_R8(r, 0), VECTRA_R8(r, 8), VECTRA_R8(r, 16), VECTRA_R8(r, 24),
        VECTRA_R8(q, 0), VECTRA_R8(q, 8), VECTRA_R8(q, 16), VECTRA_R8(q, 24)
      : "r"(t0), "r"(t1)
      : "memory");
}
#undef VECTRA_R8

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void* tmap,
                                            uint32_t bar, int c0, int c1,
                                            int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1),
      "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return f2pk(x, x); }
__device__ __forceinline__ uint64_t bits2(const uint32_t* r) {
  return f2pk(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves(uint64_t x) {
  const float2 f = f2upk(x);
  return f.x + f.y;
}
// A packed pair as floats.
template <typename T>
__device__ __forceinline__ uint64_t unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return f2pk(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2pk(f.x, f.y);
  }
}

// What rounding the pair v to `rounded` left, rounded itself.
template <typename T>
__device__ __forceinline__ uint32_t rest_of(uint32_t rounded, uint64_t v) {
  const float2 f = f2upk(ffma2(unpack2<T>(rounded), both(-1.f), v));
  return pack2<T>(f.x, f.y);
}

// Row r's vector in a 128-byte swizzled tile whose pieces are `block` bytes
// apart: 16-byte chunk c of piece kb.
__device__ __forceinline__ uint32_t chunk_at(int block, int r, int kb, int c) {
  return uint32_t(kb * block + r * 128 + ((c ^ (r & 7)) << 4));
}

// The sum of squares of chunks [from, from + N) of row r.
template <typename T, int N>
__device__ __forceinline__ float row_square(const uint8_t* tile, int block,
                                            int r, int from) {
  uint64_t a = 0, b = 0;
#pragma unroll 4
  for (int i = from; i < from + N; ++i) {
    const uint4 raw = *reinterpret_cast<const uint4*>(
        tile + chunk_at(block, r, i / 8, i % 8));
    const uint64_t x = unpack2<T>(raw.x), y = unpack2<T>(raw.y),
                   z = unpack2<T>(raw.z), w = unpack2<T>(raw.w);
    a = ffma2(x, x, a);
    b = ffma2(y, y, b);
    a = ffma2(z, z, a);
    b = ffma2(w, w, b);
  }
  return halves(fadd2(a, b));
}

__device__ __forceinline__ void sync_rows() {  // the two row warpgroups
  asm volatile("bar.sync 1, 256;" ::: "memory");
}

// Eight values of a row: 16 bytes of T with what rounding left, or floats.
template <typename T>
__device__ __forceinline__ void store8(T* out, T* rest, const float* v,
                                       int live) {
  union {
    T e[8];
    uint4 u;
  } a, b;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a.e[i] = from_f32<T>(v[i]);
    b.e[i] = from_f32<T>((v[i] - to_f32(a.e[i])) * kRestLift<T>);
  }
  const bool whole =
      live >= 8 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  if (whole) {
    *reinterpret_cast<uint4*>(out) = a.u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < live) out[i] = a.e[i];
  }
  if (rest == nullptr) return;
  if (live >= 8 && (reinterpret_cast<uintptr_t>(rest) & 15) == 0) {
    *reinterpret_cast<uint4*>(rest) = b.u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < live) rest[i] = b.e[i];
  }
}
__device__ __forceinline__ void store8f(float* out, const float* v, int live) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < live) out[i] = v[i];
}

// One pass' work of one block: rows `block`, part `part` of the columns.
template <typename T, int W, int PASS>
__device__ __forceinline__ void cross_pass(const CUtensorMap& tr,
                                           const CUtensorMap& tr2,
                                           const CUtensorMap& tcol,
                                           const CUtensorMap& tcol2,
                                           const TcArgs& a, uint32_t block,
                                           int part, uint8_t* smem_raw) {
  using C = Cfg<W, PASS>;
  constexpr bool kBack = C::kBack;
  constexpr bool kScaled = std::is_same<T, __half>::value;
  constexpr bool kRowsAreQueries = PASS != kKeys;
  constexpr int CN = C::CN, NS = C::NS;
  constexpr int FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  const CrossProblem& p = a.p;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_addr(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  // 0 rows loaded; 1, 2 S (and T) of a buffer formed; 3, 4 its P (and z)
  // written; 5 accumulators final; then per stage loaded, free, terms written.
  const uint32_t bar_r = smem_addr(&bars[0]);
  auto bar_s = [&](int x) { return smem_addr(&bars[1 + x]); };
  auto bar_p = [&](int x) { return smem_addr(&bars[3 + x]); };
  const uint32_t bar_end = smem_addr(&bars[5]);
  auto bar_full = [&](int s) { return smem_addr(&bars[6 + s]); };
  auto bar_free = [&](int s) { return smem_addr(&bars[6 + NS + s]); };
  auto bar_term = [&](int s) { return smem_addr(&bars[6 + 2 * NS + s]); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_TMEM);
  float* term = reinterpret_cast<float*>(smem + C::OFF_TERM);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t plane = block / p.row_blocks;
  const int tile = int(block - plane * p.row_blocks);
  const int b = int(plane / p.Hk), hk = int(plane - int64_t(b) * p.Hk);
  const int G = int(p.G);

  const int len = cross_length(p, b);
  const int nq = int(p.Nq);
  const int row0 = tile * a.rows_i;    // first query, or first key
  int t0, t1;
  {
    const int cols = kRowsAreQueries ? len : nq;
    const int rows = kRowsAreQueries ? nq : len;
    const int tiles = row0 < rows ? (cols + a.cols_i - 1) / a.cols_i : 0;
    split_range(tiles, part, p.splits, &t0, &t1);
  }
  const int n = t1 - t0;
  // What z of dk is multiplied by.
  float up_k = 1.f;
  if (kScaled && PASS == kKeys && n > 0)
    up_k = scale_up_to(
        __ldg(p.bounds + 2 * plane) * (2.f * __ldg(p.bounds + 2 * plane + 1)),
        13);

  // This thread's row, and its place among the results' rows.
  const int r = threadIdx.x & 127;
  const int qi = row0 + r / G, qh = hk * G + r % G;     // as a query
  const int key = row0 + r;                             // as a key
  const bool row_live = kRowsAreQueries ? r < a.rows_i * G && qi < nq
                                        : key < int(p.Nk);
  const int64_t at = kRowsAreQueries
                         ? (int64_t(b) * p.H + qh) * p.Nq + qi
                         : (int64_t(b) * p.Hk + hk) * p.Nk + key;
  const int64_t all_rows =
      kRowsAreQueries ? p.B * p.H * p.Nq : p.B * p.Hk * p.Nk;
  const bool whole = p.splits == 1;

  bool ok = true;
  uint32_t tmem = 0;
  if (n > 0) {
    if (threadIdx.x == 0) {
      mbar_init(bar_r, 1);
      mbar_init(bar_end, 1);
      for (int x = 0; x < 2; ++x) {
        mbar_init(bar_s(x), 1);
        mbar_init(bar_p(x), 8);
      }
      for (int s = 0; s < NS; ++s) {
        mbar_init(bar_full(s), 1);
        mbar_init(bar_free(s), 1);
        mbar_init(bar_term(s), kTermThreads / 32);
      }
      fence_barrier_init();
    }
    if (warp == kMmaWarp) {
      tmem_alloc(smem_addr(tmem_slot), C::TMEM_COLS);
      tmem_relinquish();
    }
    // Column rows that no box fills (64 is not a multiple of G) stay zero.
    if (PASS == kKeys && a.cols_i * G < CN) {
      for (int i = threadIdx.x; i < NS * C::STAGE / 16; i += kThreads)
        reinterpret_cast<uint4*>(smem + C::OFF_C)[i] = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    tmem = *tmem_slot;
  }

  if (n > 0 && warp >= kProducerWarp) {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == kProducerWarp) {
      // ----------------------------------------------------------- producer
      if (elect_one()) {
        const auto load = [&](uint32_t dst, const CUtensorMap* map,
                              uint32_t bar, bool queries, int kb, int first) {
          if (queries)
            tma_load_5d(dst, map, bar, kb * 64, 0, first, hk, b);
          else
            tma_load_4d(dst, map, bar, kb * 64, first, hk, b);
        };
        mbar_arrive_expect_tx(bar_r,
                              uint32_t(a.row_bytes * C::KB * (kBack ? 2 : 1)));
        for (int kb = 0; kb < C::KB; ++kb) {
          const uint32_t dst = sbase + C::OFF_R + kb * C::RBLOCK;
          load(dst, &tr, bar_r, kRowsAreQueries, kb, row0);
          if (kBack)
            load(dst + C::RTILE, &tr2, bar_r, kRowsAreQueries, kb, row0);
        }
        for (int t = 0; t < n && ok; ++t) {
          const int s = t % NS;
          ok = mbar_wait(bar_free(s), uint32_t(((t / NS) & 1) ^ 1), p.err);
          if (!ok) break;
          mbar_arrive_expect_tx(bar_full(s), uint32_t(a.col_bytes * C::KB * 2));
          const int first = (t0 + t) * a.cols_i;
          for (int kb = 0; kb < C::KB; ++kb) {
            const uint32_t dst =
                sbase + C::OFF_C + s * C::STAGE + kb * C::CBLOCK;
            load(dst, &tcol, bar_full(s), !kRowsAreQueries, kb, first);
            load(dst + C::CTILE, &tcol2, bar_full(s), !kRowsAreQueries, kb,
                 first);
          }
        }
      }
    } else if (warp == kMmaWarp) {
      // --------------------------------------------------------- MMA issuer
      if (elect_one()) {
        const uint32_t idesc_s = f16_idesc(FMT, kRows, CN, 0);
        // Widths in steps of 16, which the products' sizes come in.
        const int d16 = (p.D + 15) / 16, dv16 = (p.Dv + 15) / 16;
        const uint32_t idesc_a = f16_idesc(FMT, kRows, d16 * 16, 1);
        const uint32_t idesc_a2 = f16_idesc(FMT, kRows, dv16 * 16, 1);
        const uint64_t dr = sw128_desc(sbase + C::OFF_R, 16, 1024);
        const uint64_t dr2 = dr + uint64_t(C::RTILE >> 4);
        const uint64_t dc = sw128_desc(sbase + C::OFF_C, 16, 1024);
        const uint64_t dcm =
            sw128_desc(sbase + C::OFF_C, C::CBLOCK, 1024);
        // Unrolled: with a counted loop the issuing thread's address
        // arithmetic, about 100 cycles an MMA, set the pace.
        auto inner = [&](uint32_t dst, uint64_t da, uint64_t db, int steps) {
#pragma unroll
          for (int k = 0; k < W / 16; ++k)
            if (k < steps)
              tc_mma(tmem + dst,
                     da + uint64_t(((k >> 2) * C::RBLOCK + (k & 3) * 32) >> 4),
                     db + uint64_t(((k >> 2) * C::CBLOCK + (k & 3) * 32) >> 4),
                     idesc_s, k > 0);
        };
        auto form = [&](int t) {  // S (and T) of tile t
          const int x = t & 1, s = t % NS;
          const uint64_t col = dc + uint64_t((s * C::STAGE) >> 4);
          inner(C::S0 + x * CN, dr, col, d16);
          if (kBack)
            inner(C::T0 + x * CN, dr2, col + uint64_t(C::CTILE >> 4), dv16);
          tc_commit(bar_s(x));
        };
        // acc += A B of warpgroup x's columns, A its 16-bit pairs in TMEM.
        auto sum = [&](uint32_t dst, uint32_t src, uint64_t db, uint32_t idesc,
                       int x, bool first) {
#pragma unroll
          for (int k = 0; k < CN / 32; ++k)
            tc_mma_ts(tmem + dst, tmem + src + x * (CN / 2) + k * 8,
                      db + uint64_t(((x * (CN / 2) + k * 16) * 128) >> 4),
                      idesc, !first || k > 0);
        };
        ok = mbar_wait(bar_r, 0, p.err);
        for (int t = 0; t < 2 && t < n && ok; ++t) {
          ok = mbar_wait(bar_full(t % NS), 0, p.err);
          if (!ok) break;
          tc_fence_after();
          form(t);
        }
        for (int t = 0; t < n && ok; ++t) {
          const int x = t & 1, s = t % NS;
          ok = mbar_wait(bar_p(x), uint32_t((t >> 1) & 1), p.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t col = dcm + uint64_t((s * C::STAGE) >> 4);
          const uint64_t col2 = col + uint64_t(C::CTILE >> 4);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (PASS == kForward) {
              const uint32_t src = C::S0 + x * CN;
              sum(C::A0 + g * W, src, col2, idesc_a2, g, t == 0);
              sum(C::A0 + g * W, src + CN / 4, col2, idesc_a2, g, false);
            } else {
              const uint32_t z = C::T0 + x * CN, w = C::S0 + x * CN;
              sum(C::A0, z, col, idesc_a, g, t == 0 && g == 0);
              sum(C::A0, z + CN / 4, col, idesc_a, g, false);
              if (PASS == kKeys) {
                sum(C::A0 + W, w, col2, idesc_a2, g, t == 0 && g == 0);
                sum(C::A0 + W, w + CN / 4, col2, idesc_a2, g, false);
              }
            }
          }
          tc_commit(bar_free(s));
          if (t + 2 < n) {
            ok = mbar_wait(bar_full((t + 2) % NS),
                           uint32_t(((t + 2) / NS) & 1), p.err);
            if (!ok) break;
            tc_fence_after();
            form(t + 2);
          }
        }
        if (ok) tc_commit(bar_end);
      }
    } else if (warp >= kTermWarp) {
      // ------------------------------------------------------- column terms
      const int th = threadIdx.x - kTermWarp * 32;  // 0 .. 127
      for (int t = 0; t < n && ok; ++t) {
        const int s = t % NS;
        float* out = term + s * C::TERMS * CN;
        if constexpr (kRowsAreQueries) {
          // Threads of a column, which are neighbours, and this one's part.
          constexpr int PER = kTermThreads / CN, CHUNKS = 8 * C::KB / PER;
          const int c = th / PER, part_of = th % PER;
          const int first = (t0 + t) * CN;
          const bool known = p.key_squares != nullptr;
          const bool last = first + CN > len;
          ok = known ? mbar_wait(bar_free(s), uint32_t(((t / NS) & 1) ^ 1),
                                 p.err)
                     : true;
          float sq = 0.f;
          if (known && ok && first + c < len)
            sq = __ldg(p.key_squares + plane * p.Nk + first + c);
          if (ok && (!known || last))
            ok = mbar_wait(bar_full(s), uint32_t((t / NS) & 1), p.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint8_t* k_tile = smem + C::OFF_C + s * C::STAGE;
          if (!known) {
            sq = row_square<T, CHUNKS>(k_tile, C::CBLOCK, c, part_of * CHUNKS);
            if (PER == 2) sq += __shfl_xor_sync(0xffffffffu, sq, 1);
          }
          if (last) {
            // Unseen rows of the operand that a product sums.
            uint8_t* summed = k_tile + (PASS == kForward ? C::CTILE : 0);
            if (first + c >= len) {
              sq = 0.f;
              for (int i = part_of * CHUNKS; i < (part_of + 1) * CHUNKS; ++i)
                *reinterpret_cast<uint4*>(
                    summed + chunk_at(C::CBLOCK, c, i / 8, i % 8)) =
                    make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          if (part_of == 0) out[c] = -sq;
        } else {
          ok = mbar_wait(bar_free(s), uint32_t(((t / NS) & 1) ^ 1), p.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int i = (t0 + t) * a.cols_i + th / G, h = hk * G + th % G;
          if (th < CN) {
            float lse = INFINITY, ci = 0.f, g = 0.f;  // weighs nothing
            if (th < a.cols_i * G && i < nq) {
              const int64_t q = (int64_t(b) * p.H + h) * p.Nq + i;
              lse = __ldg(p.lse + q);
              ci = __ldg(p.delta + q);
              g = cross_scale(p, b, h);
            }
            // P is formed times kLift, z times up_k.
            out[th] = kScaled ? 14.f - lse : -lse;
            out[CN + th] = -ci;
            out[2 * CN + th] = g * kLog2e;
            out[3 * CN + th] = kScaled ? 2.f * g * (up_k / kLift) : 2.f * g;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_term(s));
      }
    }
  } else if (n > 0) {
    // -------------------------------------------------- rows: P, z, results
    setmaxnreg_inc<kRowRegs>();
    const int x = warp >> 2;
    const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
    constexpr int HALF = CN / 2;  // columns of this warpgroup
    const uint32_t s_base = tmem + lane_base + C::S0 + x * HALF;
    const uint32_t t_base = tmem + lane_base + C::T0 + x * HALF;
    const uint32_t acc = tmem + lane_base + C::A0;
    // A warp none of whose rows lives only keeps step.
    const bool warp_live = __any_sync(0xffffffffu, row_live);
    const float scale =
        kRowsAreQueries && row_live ? cross_scale(p, b, qh) : 0.f;
    const float gl = scale * kLog2e;

    if constexpr (PASS == kForward) {
      const uint32_t o_col = acc + x * W;
      const uint64_t two = both(2.f);
      const bool warp_negative = __any_sync(0xffffffffu, gl < 0.f);
      // A scale of 0 keeps masked columns at weight 0 through a tiny one.
      const float gle = warp_negative ? 1.f : (gl == 0.f ? 1e-37f : gl);
      const uint64_t gl2 = both(gle);
      float m_used = kNegInf, l = 0.f;
      for (int t = 0; t < n && ok; ++t) {
        const int s = t % NS, buf = t & 1;
        const float* nk = term + s * CN + x * HALF;
        const uint32_t s_col = s_base + buf * CN;
        ok = mbar_wait(bar_s(buf), uint32_t((t >> 1) & 1), p.err) &&
             mbar_wait(bar_term(s), uint32_t((t / NS) & 1), p.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          uint32_t v[HALF];
          tmem_load64(s_col, v);
          float mx[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
          // u = 2 S - |k|^2; the logit is gl u.
#pragma unroll
          for (int j = 0; j < HALF; j += 4) {
            const float4 n4 = *reinterpret_cast<const float4*>(nk + j);
            const float2 lo = f2upk(ffma2(two, bits2(v + j), f2pk(n4.x, n4.y)));
            const float2 hi =
                f2upk(ffma2(two, bits2(v + j + 2), f2pk(n4.z, n4.w)));
            v[j] = __float_as_uint(lo.x);
            v[j + 1] = __float_as_uint(lo.y);
            v[j + 2] = __float_as_uint(hi.x);
            v[j + 3] = __float_as_uint(hi.y);
          }
          if (warp_negative) {  // the largest logit is not that of the largest u
#pragma unroll
            for (int j = 0; j < HALF; ++j)
              v[j] = __float_as_uint(gl * __uint_as_float(v[j]));
          }
          const int live = len - (t0 + t) * CN - x * HALF;
          if (live < HALF) {
#pragma unroll
            for (int j = 0; j < HALF; ++j)
              if (j >= live) v[j] = __float_as_uint(kNegInf);
          }
#pragma unroll
          for (int j = 0; j < HALF; j += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mx[q] = fmax3(mx[q], __uint_as_float(v[j + 2 * q]),
                            __uint_as_float(v[j + 2 * q + 1]));
          const float u_top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          // (A scale of 0 has logits 0; 0 * -inf only where nothing is live.)
          const float top = u_top == kNegInf ? kNegInf : gle * u_top;
          // The reference maximum moves when the new one is more than 2^8
          // larger; the warp rescales O if any of its rows moved.
          const bool need = top > m_used + kRescaleThreshold ||
                            (m_used == kNegInf && top != kNegInf);
          float factor = 1.f;
          if (need) {
            factor = m_used == kNegInf ? 0.f : fast_exp2(m_used - top);
            m_used = top;
            l *= factor;
          }
          if (t > 0 && __any_sync(0xffffffffu, need)) {
            // The tile before's product into O, which may still run: this
            // tile's S was issued ahead of it. Its stage is free behind it.
            ok = mbar_wait(bar_free((t - 1) % NS),
                           uint32_t(((t - 1) / NS) & 1), p.err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < W / 32; ++c) {
              uint32_t o[32];
              tmem_load32(o_col + c * 32, o);
              float f[32];
#pragma unroll
              for (int i = 0; i < 32; ++i)
                f[i] = __uint_as_float(o[i]) * factor;
              tmem_st32(o_col + c * 32, f);
            }
          }
          const float ref = m_used == kNegInf ? 0.f : m_used - kLog2Lift<T>;
          const uint64_t neg = both(-ref);
          uint64_t sa = 0, sb = 0;
#pragma unroll
          for (int c = 0; c < HALF / 32; ++c) {
            uint32_t w[16], rest[16];
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const int k = c * 32 + 2 * j;
              const float2 e0 = f2upk(ffma2(gl2, bits2(v + k), neg));
              const float2 e1 = f2upk(ffma2(gl2, bits2(v + k + 2), neg));
              const uint64_t p0 = f2pk(fast_exp2(e0.x), fast_exp2(e0.y));
              const uint64_t p1 = f2pk(fast_exp2(e1.x), fast_exp2(e1.y));
              w[j] = pack2<T>(f2upk(p0).x, f2upk(p0).y);
              w[j + 1] = pack2<T>(f2upk(p1).x, f2upk(p1).y);
              sa = fadd2(sa, p0);
              sb = fadd2(sb, p1);
              rest[j] = rest_of<T>(w[j], p0);
              rest[j + 1] = rest_of<T>(w[j + 1], p1);
            }
            tmem_st16(s_col + c * 16, w);
            tmem_st16(s_col + HALF / 2 + c * 16, rest);
          }
          l += halves(fadd2(sa, sb));
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p(buf));
      }
      if (ok) ok = mbar_wait(bar_end, 0, p.err);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      // The warpgroups' maxima and sums, through the row operand's memory
      // (every product has read it by now).
      float2* join = reinterpret_cast<float2*>(smem + C::OFF_R);
      join[x * kRows + r] = make_float2(m_used - kLog2Lift<T>, l);
      sync_rows();
      const float2 j0 = join[r], j1 = join[kRows + r];
      const float m = fmaxf(j0.x, j1.x);
      const float f0 = j0.x == kNegInf ? 0.f : fast_exp2(j0.x - m);
      const float f1 = j1.x == kNegInf ? 0.f : fast_exp2(j1.x - m);
      // Without a finite maximum nothing was weighed: 0 / 0.
      const float sum = f0 * j0.y + f1 * j1.y;
      const float inv = whole ? 1.f / sum : 1.f;
      const float lse = m + log2f(sum);
      if (ok && warp_live) {
        if (row_live && x == 0) {
          const int64_t k = part * all_rows + at;
          if (!whole) {
            p.part_ml[2 * k] = m;
            p.part_ml[2 * k + 1] = sum;
          } else if (p.lse) {
            p.lse[at] = lse;
          }
        }
        T* out = static_cast<T*>(p.out) + b * p.so[0] + qh * p.so[1] +
                 int64_t(qi) * p.so[2];
        T* rest = p.rest ? static_cast<T*>(p.rest) + at * p.Dv : nullptr;
        float* part_out =
            whole ? nullptr : p.part + (part * all_rows + at) * p.Dv;
#pragma unroll
        for (int c = 0; c < W / 64; ++c) {
          const int d0 = (x * (W / 64) + c) * 32;
          if (d0 >= p.Dv) break;
          uint32_t o0[32], o1[32];
          tmem_load32x2(acc + d0, o0, acc + W + d0, o1);
          if (!row_live) continue;
#pragma unroll
          for (int q = 0; q < 32; q += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              v[i] = (__uint_as_float(o0[q + i]) * f0 +
                      __uint_as_float(o1[q + i]) * f1) * inv;
            }
            const int d = d0 + q, live = p.Dv - d;
            if (live <= 0) break;
            if (whole)
              store8<T>(out + d, rest ? rest + d : nullptr, v, live);
            else
              store8f(part_out + d, v, live);
          }
        }
      }
    } else {
      const uint64_t two = both(2.f);
      float nkr = 0.f, lse = 0.f, ci = 0.f;
      if (kRowsAreQueries && row_live) {
        lse = __ldg(p.lse + at);
        ci = __ldg(p.delta + at);
      }
      ok = mbar_wait(bar_r, 0, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!kRowsAreQueries && ok)
        nkr = -row_square<T, 8 * C::KB>(smem + C::OFF_R, C::RBLOCK, r, 0);
      // What z of dq is multiplied by.
      float up = 1.f;
      if (kScaled && kRowsAreQueries && ok)
        up = scale_up_to(
            sqrtf(row_square<T, 8 * C::KB>(smem + C::OFF_R + C::RTILE,
                                           C::RBLOCK, r, 0)) *
                (2.f * __ldg(p.bounds + 2 * plane + 1)),
            13);
      const uint64_t nkr2 = both(nkr), gl2 = both(gl), lse2 = both(-lse),
                     ci2 = both(-ci * up), up2 = both(up);
      uint64_t zs = 0, xs = 0, ys = 0;  // sums of z; for dscale
      static_assert(!kBack || HALF == 32, "a tile is read before z is written");
      const bool want_scale = PASS == kQueries && p.dscale_rows != nullptr;
      for (int t = 0; t < n && ok; ++t) {
        const int s = t % NS, buf = t & 1;
        const float* col = term + s * C::TERMS * CN + x * HALF;
        const uint32_t s_col = s_base + buf * CN, t_col = t_base + buf * CN;
        ok = mbar_wait(bar_s(buf), uint32_t((t >> 1) & 1), p.err) &&
             mbar_wait(bar_term(s), uint32_t((t / NS) & 1), p.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          const int live =
              kRowsAreQueries ? len - (t0 + t) * CN - x * HALF : HALF;
#pragma unroll
          for (int c = 0; c < HALF; c += 32) {
            uint32_t sv[32], tv[32];
            tmem_load32x2(s_col + c, sv, t_col + c, tv);
            uint32_t zw[16], zl[16];  // z and what its rounding left
            uint32_t pw[16], pl[16];  // keys: P
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              uint64_t lg[2], zc[2], u2[2];
              if constexpr (kRowsAreQueries) {
                const float4 n4 =
                    *reinterpret_cast<const float4*>(col + c + j);
                u2[0] = ffma2(two, bits2(sv + j), f2pk(n4.x, n4.y));
                u2[1] = ffma2(two, bits2(sv + j + 2), f2pk(n4.z, n4.w));
                lg[0] = ffma2(gl2, u2[0], lse2);
                lg[1] = ffma2(gl2, u2[1], lse2);
                zc[0] = kScaled ? ffma2(bits2(tv + j), up2, ci2)
                                : fadd2(bits2(tv + j), ci2);
                zc[1] = kScaled ? ffma2(bits2(tv + j + 2), up2, ci2)
                                : fadd2(bits2(tv + j + 2), ci2);
              } else {
                const float4 l4 =
                    *reinterpret_cast<const float4*>(col + c + j);
                const float4 c4 =
                    *reinterpret_cast<const float4*>(col + CN + c + j);
                const float4 g4 =
                    *reinterpret_cast<const float4*>(col + 2 * CN + c + j);
                const float4 h4 =
                    *reinterpret_cast<const float4*>(col + 3 * CN + c + j);
                u2[0] = ffma2(two, bits2(sv + j), nkr2);
                u2[1] = ffma2(two, bits2(sv + j + 2), nkr2);
                lg[0] = ffma2(f2pk(g4.x, g4.y), u2[0], f2pk(l4.x, l4.y));
                lg[1] = ffma2(f2pk(g4.z, g4.w), u2[1], f2pk(l4.z, l4.w));
                zc[0] = mul2(fadd2(bits2(tv + j), f2pk(c4.x, c4.y)),
                             f2pk(h4.x, h4.y));
                zc[1] = mul2(fadd2(bits2(tv + j + 2), f2pk(c4.z, c4.w)),
                             f2pk(h4.z, h4.w));
              }
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float2 e = f2upk(lg[q]);
                float w0 = fast_exp2(e.x), w1 = fast_exp2(e.y);
                float2 z = f2upk(mul2(f2pk(w0, w1), zc[q]));
                if (kRowsAreQueries && live < HALF) {
                  const int k = c + j + 2 * q;
                  if (k >= live) w0 = z.x = 0.f;
                  if (k + 1 >= live) w1 = z.y = 0.f;
                  float2 f = f2upk(u2[q]);
                  if (k >= live) f.x = 0.f;
                  if (k + 1 >= live) f.y = 0.f;
                  u2[q] = f2pk(f.x, f.y);
                }
                const uint32_t zp = pack2<T>(z.x, z.y);
                const uint64_t z2 = f2pk(z.x, z.y);
                zw[j / 2 + q] = zp;
                zl[j / 2 + q] = rest_of<T>(zp, z2);
                zs = fadd2(zs, z2);
                if constexpr (PASS == kKeys) {
                  const uint32_t pp = pack2<T>(w0, w1);
                  pw[j / 2 + q] = pp;
                  pl[j / 2 + q] = rest_of<T>(pp, f2pk(w0, w1));
                } else if (want_scale) {
                  xs = ffma2(z2, u2[q], xs);
                  ys = ffma2(f2pk(w0, w1), u2[q], ys);
                }
              }
            }
            tmem_st16(t_col + c / 2, zw);
            tmem_st16(t_col + HALF / 2, zl);
            if constexpr (PASS == kKeys) {
              tmem_st16(s_col + c / 2, pw);
              tmem_st16(s_col + HALF / 2, pl);
            }
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p(buf));
      }
      if (ok) ok = mbar_wait(bar_end, 0, p.err);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      float4* join = reinterpret_cast<float4*>(smem + C::OFF_JOIN);
      join[x * kRows + r] =
          make_float4(halves(zs), halves(xs), halves(ys), 0.f);
      sync_rows();
      const float4 j0 = join[r], j1 = join[kRows + r];
      const float z_sum = j0.x + j1.x;
      const float down = inverse_of(PASS == kKeys ? up_k : up);
      if (ok && warp_live) {
        if (want_scale && row_live && x == 0) {
          // Minus: the finish kernel takes sums of distances, and u is
          // |q|^2 less one.
          float* w = p.dscale_rows + (part * all_rows + at) * 3;
          w[0] = -(j0.y + j1.y) * down;
          w[1] = -(j0.z + j1.z);
          w[2] = z_sum * down;
        }
        // acc less the row's own vector times its sum: dq by columns between
        // the warpgroups; of the keys' two results one each.
        const float g = (kRowsAreQueries ? 2.f * scale : 1.f) * down;
        const bool live = kRowsAreQueries ? row_live : key < len;
        const bool second = PASS == kKeys && x == 1;
        const int width = second ? p.Dv : p.D;
        const int c0 = PASS == kKeys ? 0 : x * (W / 2);
        const int c1 = PASS == kKeys ? W : c0 + W / 2;
        void* base = PASS == kQueries ? p.dq : (second ? p.dv : p.dk);
        const int64_t* st =
            PASS == kQueries ? p.sdq : (second ? p.sdv : p.sdk);
        float* part_base = second ? p.part_v : p.part;
        if (base) {
          T* out = static_cast<T*>(base) + b * st[0] +
                   (kRowsAreQueries ? qh : hk) * st[1] +
                   int64_t(kRowsAreQueries ? qi : key) * st[2];
          float* part_out =
              whole ? nullptr : part_base + (part * all_rows + at) * width;
          const uint32_t src = acc + (second ? W : 0);
          const uint8_t* own = smem + C::OFF_R;
          for (int d0 = c0; d0 < c1 && d0 < width; d0 += 32) {
            uint32_t o[32];
            tmem_load32(src + d0, o);
            if (!row_live) continue;
#pragma unroll
            for (int q = 0; q < 32; q += 8) {
              const int d = d0 + q, left = width - d;
              if (left <= 0) break;
              float v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(o[q + i]);
              if (!second) {
                const uint4 raw = *reinterpret_cast<const uint4*>(
                    own + chunk_at(C::RBLOCK, r, d / 64, (d % 64) / 8));
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = f2upk(unpack2<T>(w[i]));
                  v[2 * i] = g * (v[2 * i] - f.x * z_sum);
                  v[2 * i + 1] = g * (v[2 * i + 1] - f.y * z_sum);
                }
              }
              if (kScaled && second) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= 1.f / kLift;
              }
              if (!live) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.f;
              }
              if (whole)
                store8<T>(out + d, nullptr, v, left);
              else
                store8f(part_out + d, v, left);
            }
          }
        }
      }
    }
  }

  if (n > 0) {
    // Every TMEM access is done before the allocating warp frees it.
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
      tc_fence_after();
      tmem_dealloc(tmem, C::TMEM_COLS);
    }
    return;
  }
  // Nothing to walk: no key is seen, these keys are not, or this part of the
  // axis is empty. Zero results, and parts that weigh nothing.
  if (warp >= kProducerWarp || !row_live) return;
  const int x = warp >> 2;
  const int64_t k = part * all_rows + at;
  const float zero[8] = {0.f};
  const auto clear = [&](void* base, const int64_t* st, T* rest, float* part_to,
                         int width, int h, int64_t i) {
    if (base == nullptr) return;
    T* out = static_cast<T*>(base) + b * st[0] + h * st[1] + i * st[2];
    for (int d = 0; d < width; d += 8) {
      if (whole)
        store8<T>(out + d, rest ? rest + d : nullptr, zero, width - d);
      else
        store8f(part_to + k * width + d, zero, width - d);
    }
  };
  if constexpr (PASS == kForward) {
    if (x != 0) return;
    T* rest = p.rest ? static_cast<T*>(p.rest) + at * p.Dv : nullptr;
    clear(p.out, p.so, rest, p.part, p.Dv, qh, qi);
    if (!whole) {
      p.part_ml[2 * k] = kNegInf;
      p.part_ml[2 * k + 1] = 0.f;
    } else if (p.lse) {
      p.lse[at] = INFINITY;
    }
  } else if constexpr (PASS == kQueries) {
    if (x != 0) return;
    clear(p.dq, p.sdq, nullptr, p.part, p.D, qh, qi);
    if (p.dscale_rows)
      for (int i = 0; i < 3; ++i) p.dscale_rows[k * 3 + i] = 0.f;
  } else {
    if (x == 0)
      clear(p.dk, p.sdk, nullptr, p.part, p.D, hk, key);
    else
      clear(p.dv, p.sdv, nullptr, p.part_v, p.Dv, hk, key);
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(kThreads, 1)
    cross_tc_forward_kernel(const __grid_constant__ CUtensorMap q,
                            const __grid_constant__ CUtensorMap k,
                            const __grid_constant__ CUtensorMap v,
                            const __grid_constant__ TcArgs a) {
  extern __shared__ uint8_t smem_raw[];
  allow_dependents();
  grid_dependency_wait();
  cross_pass<T, W, kForward>(q, q, k, v, a, blockIdx.x, blockIdx.y, smem_raw);
}

// Both backward passes in one grid: the keys' blocks, which are longer, first,
// and the queries' behind them fill the SMs that they leave. All gradients of 2048
// queries x 16 heads over 4500 keys x 4 heads, width 128, batch 4: 726 us, as
// two launches 838.
struct BackwardArgs {
  CUtensorMap keys[4];     // k, v, q, e
  CUtensorMap queries[4];  // q, e, k, v
  TcArgs a[2];             // of the keys' and the queries' pass
  uint32_t blocks[2];      // of a part of each
  uint32_t key_blocks;     // of all parts
};
template <typename T, int W>
__global__ void __launch_bounds__(kThreads, 1)
    cross_tc_backward_kernel(const __grid_constant__ BackwardArgs x) {
  extern __shared__ uint8_t smem_raw[];
  allow_dependents();
  grid_dependency_wait();
  if (blockIdx.x < x.key_blocks) {
    const uint32_t part = blockIdx.x / x.blocks[0];
    cross_pass<T, W, kKeys>(x.keys[0], x.keys[1], x.keys[2], x.keys[3], x.a[0],
                            blockIdx.x - part * x.blocks[0], int(part),
                            smem_raw);
  } else {
    const uint32_t at = blockIdx.x - x.key_blocks;
    const uint32_t part = at / x.blocks[1];
    cross_pass<T, W, kQueries>(x.queries[0], x.queries[1], x.queries[2],
                               x.queries[3], x.a[1], at - part * x.blocks[1],
                               int(part), smem_raw);
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// A pass' tiles and blocks; false: too many blocks.
template <int W, int PASS>
bool describe_pass(const CrossProblem& problem, TcArgs* a) {
  using C = Cfg<W, PASS>;
  a->p = problem;
  CrossProblem& p = a->p;
  const int G = int(p.G);
  const bool rows_q = PASS != kKeys;
  a->rows_i = rows_q ? kRows / G : kRows;
  a->cols_i = rows_q ? C::CN : C::CN / G;
  a->row_bytes = 128 * a->rows_i * (rows_q ? G : 1);
  a->col_bytes = 128 * a->cols_i * (rows_q ? 1 : G);
  p.row_blocks = ((rows_q ? p.Nq : p.Nk) + a->rows_i - 1) / a->rows_i;
  return p.row_blocks * p.B * p.Hk * p.splits <= 0x7fffffff;
}
uint32_t blocks_of(const TcArgs& a) {
  return uint32_t(a.p.row_blocks * a.p.B * a.p.Hk);
}

// Maps of q, e (backward), k and v with boxes of `queries` and `keys` rows.
bool make_maps(const CrossProblem& p, int queries, int keys, CUtensorMap* q,
               CUtensorMap* e, CUtensorMap* k, CUtensorMap* v) {
  return make_group_map(q, p.q, p.dtype, p.B, p.Hk, p.G, p.Nq, p.D, p.sq,
                        queries) &&
         (e == nullptr ||
          make_group_map(e, p.dout, p.dtype, p.B, p.Hk, p.G, p.Nq, p.Dv, p.se,
                         queries)) &&
         make_tile_map(k, p.k, p.dtype, p.B, p.Hk, p.Nk, p.D, p.sk, keys) &&
         make_tile_map(v, p.v, p.dtype, p.B, p.Hk, p.Nk, p.Dv, p.sv, keys);
}

// Once a kernel and device: its shared memory, and that the setmaxnreg split
// fits in the registers the block is launched with; a deficit would leave
// setmaxnreg.inc waiting forever.
template <typename K>
cudaError_t configure(K kern, int bytes, std::atomic<int>* configured) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev >= 0 && dev < 64 && configured[dev].load()) return cudaSuccess;
  cudaFuncAttributes attr;
  err = cudaFuncGetAttributes(&attr, kern);
  if (err != cudaSuccess) return err;
  if (int64_t(attr.numRegs) * kThreads <
      int64_t(256) * (kRowRegs + kOtherRegs))
    return cudaErrorInvalidConfiguration;
  err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             bytes);
  if (err == cudaSuccess && dev >= 0 && dev < 64) configured[dev].store(1);
  return err;
}

template <typename T, int W>
cudaError_t launch_forward(const CrossProblem& p, cudaStream_t stream) {
  TcArgs a{};
  if (!describe_pass<W, kForward>(p, &a)) return cudaErrorInvalidValue;
  CUtensorMap q, k, v;
  if (!tensor_maps_available()) return cudaErrorNotSupported;
  if (!make_maps(p, a.rows_i, a.cols_i, &q, nullptr, &k, &v))
    return cudaErrorInvalidValue;
  constexpr int bytes = Cfg<W, kForward>::SMEM_ALLOC;
  auto kern = cross_tc_forward_kernel<T, W>;
  static std::atomic<int> configured[64];
  const cudaError_t err = configure(kern, bytes, configured);
  if (err != cudaSuccess) return err;
  count_launches(1);
  return launch_pdl(kern, dim3(blocks_of(a), unsigned(p.splits)),
                    dim3(kThreads), bytes, stream, q, k, v, a);
}

// The keys' pass where it has dk, the queries' where `want_q`.
template <typename T, int W>
cudaError_t launch_backward(const CrossProblem& keys,
                            const CrossProblem& queries, bool want_q,
                            cudaStream_t stream) {
  BackwardArgs x{};
  if (!describe_pass<W, kKeys>(keys, &x.a[0]) ||
      !describe_pass<W, kQueries>(queries, &x.a[1]))
    return cudaErrorInvalidValue;
  if (!tensor_maps_available()) return cudaErrorNotSupported;
  if (!make_maps(keys, x.a[0].cols_i, x.a[0].rows_i, &x.keys[2], &x.keys[3],
                 &x.keys[0], &x.keys[1]) ||
      !make_maps(queries, x.a[1].rows_i, x.a[1].cols_i, &x.queries[0],
                 &x.queries[1], &x.queries[2], &x.queries[3]))
    return cudaErrorInvalidValue;
  for (int i = 0; i < 2; ++i) x.blocks[i] = blocks_of(x.a[i]);
  const int64_t key_blocks =
      keys.dk ? int64_t(x.blocks[0]) * keys.splits : 0;
  const int64_t all =
      key_blocks + (want_q ? int64_t(x.blocks[1]) * queries.splits : 0);
  if (all > 0x7fffffff) return cudaErrorInvalidValue;
  if (all == 0) return cudaSuccess;
  x.key_blocks = uint32_t(key_blocks);
  constexpr int k_bytes = Cfg<W, kKeys>::SMEM_ALLOC;
  constexpr int q_bytes = Cfg<W, kQueries>::SMEM_ALLOC;
  constexpr int bytes = k_bytes > q_bytes ? k_bytes : q_bytes;
  auto kern = cross_tc_backward_kernel<T, W>;
  static std::atomic<int> configured[64];
  const cudaError_t err = configure(kern, bytes, configured);
  if (err != cudaSuccess) return err;
  count_launches(1);
  return launch_pdl(kern, dim3(unsigned(all)), dim3(kThreads), bytes, stream,
                    x);
}

// Calls f with the type and the padded width.
template <typename F>
cudaError_t with_width(const CrossProblem& p, F&& f) {
  const bool wide = p.D > 64 || p.Dv > 64;
  const auto typed = [&](auto* t) {
    return wide ? f(t, std::integral_constant<int, 128>{})
                : f(t, std::integral_constant<int, 64>{});
  };
  return p.dtype == VECTRA_BF16 ? typed(static_cast<__nv_bfloat16*>(nullptr))
                                : typed(static_cast<__half*>(nullptr));
}

// Parts of the axis that a block walks, where the rows alone leave SMs
// without a block: one block an SM, each of four tiles at least.
int splits_for(const CrossProblem& p, int pass) {
  const int64_t cn = pass == kForward ? 128 : 64;
  const int64_t rows = pass == kKeys ? p.Nk : p.Nq;
  const int64_t rows_i = pass == kKeys ? kRows : kRows / p.G;
  const int64_t blocks = (rows + rows_i - 1) / rows_i * p.B * p.Hk;
  const int64_t cols = pass == kKeys ? p.Nq : p.Nk;
  const int64_t cols_i = pass == kKeys ? cn / p.G : cn;
  const int64_t tiles = (cols + cols_i - 1) / cols_i;
  if (blocks == 0) return 1;
  int64_t s = int64_t(device_sm_count()) / blocks;
  if (s > tiles / 4) s = tiles / 4;
  if (s > 64) s = 64;
  return s < 1 ? 1 : int(s);
}

float* take_floats(Workspace& ws, int64_t n) {
  return static_cast<float*>(ws.take(size_t(n) * sizeof(float)));
}

// |k_j|^2 of every key, where more than one block of a pass would form it.
bool want_squares(const CrossProblem& p) {
  return p.Nq > kRows / p.G && p.Nk > 0;
}

bool map_ok(const void* base, const int64_t* s, const int64_t* sizes) {
  if (reinterpret_cast<uintptr_t>(base) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && (s[i] < 0 || s[i] % 8 != 0)) return false;
  return s[3] == 1 || sizes[3] == 1;
}

}  // namespace

bool cross_tc_supports(const CrossProblem& p, bool backward) {
  if (p.dtype != VECTRA_BF16 && p.dtype != VECTRA_F16) return false;
  if (p.D > 128 || p.Dv > 128 || p.G > 64 || p.G < 1) return false;
  // A tensor map has no empty dimension.
  if (p.B * p.H * p.Nq == 0 || p.Nk == 0) return false;
  const int64_t q[4] = {p.B, p.H, p.Nq, p.D}, e[4] = {p.B, p.H, p.Nq, p.Dv};
  const int64_t k[4] = {p.B, p.Hk, p.Nk, p.D}, v[4] = {p.B, p.Hk, p.Nk, p.Dv};
  return map_ok(p.q, p.sq, q) && map_ok(p.k, p.sk, k) &&
         map_ok(p.v, p.sv, v) && (!backward || map_ok(p.dout, p.se, e));
}

cudaError_t run_cross_tc_forward(const CrossProblem& problem, Workspace& ws,
                                 cudaStream_t stream) {
  CrossProblem p = problem;
  const int64_t rows = p.B * p.H * p.Nq;
  p.splits = splits_for(p, kForward);
  if (p.splits > 1) {
    p.part = take_floats(ws, p.splits * rows * p.Dv);
    p.part_ml = take_floats(ws, p.splits * rows * 2);
  }
  float* squares =
      want_squares(p) ? take_floats(ws, p.B * p.Hk * p.Nk) : nullptr;
  p.key_squares = squares;
  if (ws.dry || ws.overflow || rows == 0) return cudaSuccess;
  if (squares) {
    const cudaError_t st = launch_cross_squares(p, squares, stream);
    if (st != cudaSuccess) return st;
  }
  const cudaError_t e = with_width(p, [&](auto* t, auto width) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_forward<T, decltype(width)::value>(p, stream);
  });
  return e != cudaSuccess || p.splits == 1 ? e : launch_cross_join(p, stream);
}

cudaError_t run_cross_tc_backward(const CrossProblem& problem, Workspace& ws,
                                  cudaStream_t stream) {
  CrossProblem p = problem;
  const int64_t rows = p.B * p.H * p.Nq, keys = p.B * p.Hk * p.Nk;
  float* delta = take_floats(ws, rows);
  p.delta = delta;
  float* squares = (p.dq || p.dscale) && want_squares(p)
                       ? take_floats(ws, p.B * p.Hk * p.Nk)
                       : nullptr;
  p.key_squares = squares;
  float* bounds =
      p.dtype == VECTRA_F16 ? take_floats(ws, p.B * p.Hk * 2) : nullptr;
  p.bounds = bounds;
  CrossProblem pq = p, pk = p;
  const bool want_q = p.dq || p.dscale;
  if (want_q) {
    pq.splits = splits_for(p, kQueries);
    if (p.dscale) pq.dscale_rows = take_floats(ws, pq.splits * rows * 3);
    if (pq.splits > 1 && p.dq)
      pq.part = take_floats(ws, pq.splits * rows * p.D);
  }
  if (p.dk) {
    pk.splits = splits_for(p, kKeys);
    if (pk.splits > 1) {
      pk.part = take_floats(ws, pk.splits * keys * p.D);
      pk.part_v = take_floats(ws, pk.splits * keys * p.Dv);
    }
  }
  if (ws.dry || ws.overflow) return cudaSuccess;
  cudaError_t e = launch_cross_delta(p, delta, stream);
  if (e == cudaSuccess && squares)
    e = launch_cross_squares(p, squares, stream);
  if (e == cudaSuccess && bounds) e = launch_cross_bounds(p, bounds, stream);
  if (e == cudaSuccess)
    e = with_width(p, [&](auto* t, auto width) {
      return launch_backward<std::remove_pointer_t<decltype(t)>,
                             decltype(width)::value>(pk, pq, want_q, stream);
    });
  if (e == cudaSuccess && pq.part)
    e = launch_cross_sum(p.dtype, pq.part, pq.splits, p.B, p.H, p.Nq, p.D,
                         p.dq, p.sdq, stream);
  if (e == cudaSuccess && p.dscale)
    e = launch_cross_dscale(pq, pq.splits, stream);
  if (e == cudaSuccess && pk.part)
    e = launch_cross_sum(p.dtype, pk.part, pk.splits, p.B, p.Hk, p.Nk, p.D,
                         p.dk, p.sdk, stream);
  if (e == cudaSuccess && pk.part)
    e = launch_cross_sum(p.dtype, pk.part_v, pk.splits, p.B, p.Hk, p.Nk, p.Dv,
                         p.dv, p.sdv, stream);
  return e;
}

}  // namespace vectra
