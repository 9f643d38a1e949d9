// gemm_tc.cu: host side of the tensor-core products (gemm_tc_kernel.cuh):
// operand forms, packing, tensor maps and launch arguments.
#include "block_common.cuh"
#include "gemm_tc.cuh"

namespace vectra {
namespace {

// ---------------------------------------------------------------------------
// Packing: operands the tensor maps cannot describe (odd strides, unaligned
// rows) are first copied to rows of a multiple of 16 bytes.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    pack_kernel(const uint16_t* src, int64_t s_outer, int64_t s_inner,
                uint16_t* dst, int64_t ld, int64_t outer, int64_t inner) {
  allow_dependents();
  grid_dependency_wait();
  const int64_t total = outer * inner;
  const int64_t step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += step) {
    const int64_t o = e / inner, i = e - o * inner;
    dst[o * ld + i] = src[o * s_outer + i * s_inner];
  }
}

// Splits float32 into three bf16 planes: hi the nearest bf16, mid the
// nearest to the rest, lo the rest's rest (exact: 8 + 8 + 8 bits). A value
// that would round up to infinity is truncated instead; NaN stands in hi
// alone. An infinity is (1, 0, infinity) with its sign: lo meets nothing but
// the other operand's hi, so one product of the pair is infinite (NaN where
// that hi is 0: a zero, or a number below 2^-134), the finite others change
// nothing, and infinity times infinity is hi times lo.
__device__ __forceinline__ void split3(float x, __nv_bfloat16* hi,
                                       __nv_bfloat16* mid,
                                       __nv_bfloat16* lo) {
  __nv_bfloat16 h = __float2bfloat16_rn(x);
  const bool finite = fabsf(x) <= 3.402823466e38f;
  if (finite && fabsf(x) >= 3.39e38f) h = __float2bfloat16_rz(x);
  const float r = finite ? x - __bfloat162float(h) : 0.f;
  const __nv_bfloat16 m = __float2bfloat16_rn(r);
  const bool inf = fabsf(x) > 3.402823466e38f;  // not NaN
  *hi = inf ? __float2bfloat16_rn(copysignf(1.f, x)) : h;
  *mid = m;
  *lo = __float2bfloat16_rn(inf ? x : r - __bfloat162float(m));
}

// One operand's splitting: dst[plane][line][i], lines past `outer` zero.
struct SplitJob {
  const float* src;
  int64_t s_outer, s_inner;
  __nv_bfloat16* dst;
  int64_t ld, outer, lines, inner;
  int vec;  // eight elements per thread, else one
};
struct SplitJobs {
  SplitJob job[4];
};

template <int VEC>
__device__ __forceinline__ void split_operand(const SplitJob& j) {
  const int64_t per_line = (j.inner + VEC - 1) / VEC;
  const int64_t total = j.lines * per_line;
  const int64_t plane = j.lines * j.ld;
  const int64_t step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += step) {
    const int64_t o = e / per_line, i = (e - o * per_line) * VEC;
    union {
      __nv_bfloat16 e[VEC];
      uint4 u[VEC / 8 > 0 ? VEC / 8 : 1];
    } q[3];
    float x[VEC];
    if constexpr (VEC == 8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (o < j.outer)
          f = __ldg(
              reinterpret_cast<const float4*>(j.src + o * j.s_outer + i) + h);
        x[4 * h] = f.x;
        x[4 * h + 1] = f.y;
        x[4 * h + 2] = f.z;
        x[4 * h + 3] = f.w;
      }
    } else {
      x[0] = o < j.outer ? j.src[o * j.s_outer + i * j.s_inner] : 0.f;
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      split3(x[v], &q[0].e[v], &q[1].e[v], &q[2].e[v]);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      __nv_bfloat16* d = j.dst + s * plane + o * j.ld + i;
      if constexpr (VEC == 8)
        *reinterpret_cast<uint4*>(d) = q[s].u[0];
      else
        *d = q[s].e[0];
    }
  }
}

// Memory-bound: reads 4 bytes and writes 6 per element; all operands of a
// product in one launch (blockIdx.y). 33 MB of x and a small weight take 12
// us of the 51 of 65,536 x 128 x 256.
__global__ void __launch_bounds__(256)
    split_planes_kernel(const __grid_constant__ SplitJobs jobs) {
  allow_dependents();
  grid_dependency_wait();
  const SplitJob& j = jobs.job[blockIdx.y];
  if (j.vec)
    split_operand<8>(j);
  else
    split_operand<1>(j);
}

bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// An operand as the tensor maps see it.
struct TmaOperand {
  const void* p;
  bool mn;         // rows contiguous
  int64_t ld;      // elements between lines of the other direction
  int64_t lines;   // lines of one plane
  int planes;
};

bool describable(const MatView& m, int64_t rows, int64_t k, bool mn) {
  const int64_t inner = mn ? m.sr : m.sk, outer = mn ? m.sk : m.sr;
  const int64_t lines = mn ? k : rows;
  if (!aligned16(m.p) || (inner != 1 && (mn ? rows : k) > 1)) return false;
  return lines <= 1 || (outer > 0 && outer % 8 == 0 &&
                        outer < (int64_t(1) << 36));
}

// Which form an operand is staged in, or -1: it has to be packed.
int form_of(const MatView& m, int64_t rows, int64_t k) {
  if (describable(m, rows, k, false)) return 0;
  if (describable(m, rows, k, true)) return 1;
  return -1;
}

cudaError_t pack(const MatView& m, int64_t rows, int64_t k, bool mn,
                 Workspace& ws, TmaOperand* out, cudaStream_t stream) {
  const int64_t outer = mn ? k : rows, inner = mn ? rows : k;
  const int64_t ld = (inner + 7) / 8 * 8;
  uint16_t* dst = static_cast<uint16_t*>(ws.take(size_t(outer) * ld * 2));
  *out = {dst, mn, ld, outer, 1};
  if (ws.dry || ws.overflow) return cudaSuccess;
  const int64_t blocks = (outer * inner + 255) / 256;
  const int64_t most = int64_t(device_sm_count()) * 16;
  const cudaError_t e = launch_pdl(
      pack_kernel, dim3(unsigned(blocks < most ? blocks : most)), dim3(256),
      0, stream, static_cast<const uint16_t*>(m.p), mn ? m.sk : m.sr,
      mn ? m.sr : m.sk, dst, ld, outer, inner);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

// float32 to planes. The lines of a reduction are padded with zeros to whole
// stages: a stage that ran past one plane would read the next.
SplitJob split_planes(const MatView& m, int64_t rows, int64_t k, bool mn,
                      Workspace& ws, TmaOperand* out) {
  SplitJob j{};
  j.outer = mn ? k : rows;
  j.inner = mn ? rows : k;
  j.lines = mn ? (k + kTcStep - 1) / kTcStep * kTcStep : rows;
  j.ld = (j.inner + 7) / 8 * 8;
  j.dst = static_cast<__nv_bfloat16*>(
      ws.take(size_t(3) * j.lines * j.ld * 2));
  j.src = static_cast<const float*>(m.p);
  j.s_outer = mn ? m.sk : m.sr;
  j.s_inner = mn ? m.sr : m.sk;
  j.vec = j.inner % 8 == 0 && j.s_inner == 1 && aligned16(m.p) &&
          (j.outer <= 1 || j.s_outer % 4 == 0);
  *out = {j.dst, mn, j.ld, j.lines, 3};
  return j;
}

cudaError_t launch_splits(const SplitJobs& jobs, int n, cudaStream_t stream) {
  int64_t blocks = 1;
  for (int i = 0; i < n; ++i) {
    const SplitJob& j = jobs.job[i];
    const int64_t need =
        (j.lines * (j.inner / (j.vec ? 8 : 1) + 1) + 255) / 256;
    if (need > blocks) blocks = need;
  }
  const int64_t most = int64_t(device_sm_count()) * 16;
  const cudaError_t e = launch_pdl(
      split_planes_kernel,
      dim3(unsigned(blocks < most ? blocks : most), unsigned(n)), dim3(256),
      0, stream, jobs);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace

cudaError_t split_for_products(const void* p, int64_t lines, int64_t inner,
                               int64_t s_line, int64_t s_inner, Workspace& ws,
                               MatView* rows, MatView* cols,
                               cudaStream_t stream) {
  SplitJobs jobs{};
  TmaOperand o;
  // As an operand reduced over the lines, whose padding both uses can share.
  jobs.job[0] =
      split_planes({p, s_inner, s_line}, inner, lines, true, ws, &o);
  *rows = {o.p, o.ld, 1, o.lines};
  *cols = {o.p, 1, o.ld, o.lines};
  if (ws.dry || ws.overflow) return cudaSuccess;
  return launch_splits(jobs, 1, stream);
}

cudaError_t run_gemm_tc(const GemmProblem& p, const TcShape& shape,
                        Workspace& ws, cudaStream_t stream) {
  const bool gated =
      p.epilogue == kEpiGated || p.epilogue == kEpiGatedGrad;
  const int tile_n = gated ? shape.bn / 2 : shape.bn;
  if (tile_n < 64 || (shape.bn == 256) != (shape.cg == 2) ||
      (shape.cg == 2 && p.dtype == VECTRA_F32))
    return cudaErrorInvalidValue;
  TcArgs g{};
  g.p = p;
  g.tiles_m = int((p.M + kTcRows * shape.cg - 1) / (kTcRows * shape.cg));
  g.tiles_n = int((p.N + tile_n - 1) / tile_n);
  g.steps_seg = int((p.K + kTcStep - 1) / kTcStep);
  const bool f32 = p.dtype == VECTRA_F32;
  g.steps = g.steps_seg * p.segments;
  g.split = shape.split;
  g.steps_part = (g.steps + g.split - 1) / g.split;
  g.split = (g.steps + g.steps_part - 1) / g.steps_part;  // no empty parts
  g.units = int64_t(g.tiles_m) * g.tiles_n * g.split;

  // Both A's (and both B's) of a call are staged in one form.
  const int n_a = p.segments, n_b = gated ? 2 : p.segments;
  TmaOperand op[4];
  SplitJobs jobs{};
  int n_jobs = 0;
  for (int side = 0; side < 2; ++side) {
    const MatView* v = side ? p.b : p.a;
    const int n = side ? n_b : n_a;
    const int64_t rows = side ? p.N : p.M;
    int form = f32 ? -1 : form_of(v[0], rows, p.K);
    if (form < 0) form = v[0].sr == 1 && v[0].sk != 1;
    const bool mn = form == 1;
    for (int i = 0; i < n; ++i) {
      TmaOperand* o = &op[2 * side + i];
      cudaError_t e = cudaSuccess;
      if (v[i].plane_lines)
        *o = {v[i].p, mn, mn ? v[i].sk : v[i].sr, v[i].plane_lines, 3};
      else if (f32)
        jobs.job[n_jobs++] = split_planes(v[i], rows, p.K, mn, ws, o);
      else if (describable(v[i], rows, p.K, mn))
        *o = {v[i].p, mn, mn ? v[i].sk : v[i].sr, mn ? p.K : rows, 1};
      else
        e = pack(v[i], rows, p.K, mn, ws, o, stream);
      if (e != cudaSuccess) return e;
    }
    if (n == 1) op[2 * side + 1] = op[2 * side];
    (side ? g.b_mn : g.a_mn) = uint8_t(mn);
  }
  g.a_lines = int(op[0].lines);
  g.b_lines = int(op[2].lines);
  if (g.split > 1)
    g.partial = static_cast<float*>(ws.take(
        size_t(g.split) * (gated ? 2 : 1) * p.M * p.N * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;
  if (n_jobs > 0) {
    const cudaError_t e = launch_splits(jobs, n_jobs, stream);
    if (e != cudaSuccess) return e;
  }
  g.p.err = device_error_ptr();
  if (g.p.err == nullptr) return cudaErrorNotSupported;

  const int64_t es = f32 ? 4 : 2;
  g.vec_res = p.N * es % 16 == 0 && p.res_sn == 1 && aligned16(p.res) &&
              p.res_sm * es % 16 == 0;

  CUtensorMap maps[7] = {};
  const int b_rows = gated && shape.cg == 1 ? shape.bn / 2
                                            : shape.bn / shape.cg;
  for (int i = 0; i < 4; ++i) {
    const int64_t rows = i < 2 ? p.M : p.N;
    const TmaOperand& o = op[i];
    const int box = o.mn ? kTcStep : (i < 2 ? kTcRows : b_rows);
    if (!make_line_map(&maps[i], o.p,
                       p.dtype == VECTRA_F16 ? VECTRA_F16 : VECTRA_BF16,
                       o.mn ? rows : p.K, o.lines * o.planes, o.ld, box))
      return cudaErrorInvalidValue;
  }
  // Results, 32 rows of 64 bytes at a time.
  const auto result = [&](CUtensorMap* map, const void* q, int dtype,
                          int64_t ld, int64_t planes) {
    return uint8_t(q != nullptr && make_result_map(map, q, dtype, p.N, p.M,
                                                   planes, ld));
  };
  if (g.split > 1) {
    g.tma_out = result(&maps[4], g.partial, VECTRA_F32, p.N,
                       int64_t(g.split) * (gated ? 2 : 1));
  } else {
    g.tma_out = result(&maps[4], p.out, p.dtype, p.out_ld, 1);
    if (p.pre)
      g.tma_pre = result(&maps[5], p.pre, p.dtype, p.pre_ld, 1);
    else if (p.epilogue == kEpiGated && p.gate)
      g.tma_pre = result(&maps[5], p.gate, VECTRA_F32, p.gate_ld, 1) &&
                  result(&maps[6], p.up, VECTRA_F32, p.up_ld, 1);
  }
  const int epilogue =
      g.split == 1 ? p.epilogue : (gated ? kEpiGatedPartial : kEpiPartial);
  const cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return epilogue == kEpiLinear
               ? launch_tc_linear<T>(shape.bn, shape.cg, maps, g, stream)
               : launch_tc_other<T>(epilogue, shape.bn, shape.cg, maps, g,
                                    stream);
  });
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (g.split > 1) {
    const cudaError_t f = launch_split_finish(p, g.split, g.partial, stream);
    if (f == cudaSuccess) count_launches(1);
    return f;
  }
  return cudaSuccess;
}

}  // namespace vectra
