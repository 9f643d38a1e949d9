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

bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// An operand as the tensor maps see it.
struct TmaOperand {
  const void* p;
  bool mn;        // rows contiguous
  int64_t ld;     // elements between lines of the other direction
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
  *out = {dst, mn, ld};
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

}  // namespace

bool gemm_tc_supports(const GemmProblem& p) {
  return (p.dtype == VECTRA_BF16 || p.dtype == VECTRA_F16) && p.K > 0 &&
         p.K < (int64_t(1) << 30);
}

cudaError_t run_gemm_tc(const GemmProblem& p, const TcShape& shape,
                        Workspace& ws, cudaStream_t stream) {
  const bool gated = p.epilogue == kEpiGated;
  const int tile_n = gated ? shape.bn / 2 : shape.bn;
  if (tile_n < 64 || (shape.bn == 256) != (shape.cg == 2))
    return cudaErrorInvalidValue;
  TcArgs g{};
  g.p = p;
  g.tiles_m = int((p.M + kTcRows * shape.cg - 1) / (kTcRows * shape.cg));
  g.tiles_n = int((p.N + tile_n - 1) / tile_n);
  g.steps_seg = int((p.K + kTcStep - 1) / kTcStep);
  g.steps = g.steps_seg * p.segments;
  g.split = shape.split;
  g.steps_part = (g.steps + g.split - 1) / g.split;
  g.split = (g.steps + g.steps_part - 1) / g.steps_part;  // no empty parts
  g.units = int64_t(g.tiles_m) * g.tiles_n * g.split;

  // Both A's (and both B's) of a call are staged in one form.
  const int n_a = p.segments, n_b = gated ? 2 : p.segments;
  TmaOperand op[4];
  for (int side = 0; side < 2; ++side) {
    const MatView* v = side ? p.b : p.a;
    const int n = side ? n_b : n_a;
    const int64_t rows = side ? p.N : p.M;
    int form = form_of(v[0], rows, p.K);
    if (form < 0) form = v[0].sr == 1 && v[0].sk != 1;
    for (int i = 0; i < n; ++i) {
      if (describable(v[i], rows, p.K, form == 1)) {
        op[2 * side + i] = {v[i].p, form == 1, form ? v[i].sk : v[i].sr};
      } else {
        const cudaError_t e =
            pack(v[i], rows, p.K, form == 1, ws, &op[2 * side + i], stream);
        if (e != cudaSuccess) return e;
      }
    }
    if (n == 1) op[2 * side + 1] = op[2 * side];
    (side ? g.b_mn : g.a_mn) = uint8_t(form == 1);
  }
  if (g.split > 1)
    g.partial = static_cast<float*>(ws.take(
        size_t(g.split) * (gated ? 2 : 1) * p.M * p.N * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;

  const auto vec = [](const void* q, int64_t ld, int64_t es) {
    return uint8_t(aligned16(q) && (ld * es) % 16 == 0);
  };
  const bool n8 = p.N % 8 == 0;
  g.vec_out = n8 && vec(p.out, p.out_ld, 2);
  g.vec_pre = n8 && vec(p.pre, p.pre_ld, 2);
  g.vec_res = n8 && p.res_sn == 1 && vec(p.res, p.res_sm, 2);
  g.vec_f32 = g.split > 1 ? p.N % 4 == 0
                          : p.N % 4 == 0 && vec(p.gate, p.gate_ld, 4) &&
                                vec(p.up, p.up_ld, 4);

  CUtensorMap maps[4];
  const int b_rows = gated && shape.cg == 1 ? shape.bn / 2
                                            : shape.bn / shape.cg;
  for (int i = 0; i < 4; ++i) {
    const int64_t rows = i < 2 ? p.M : p.N;
    const TmaOperand& o = op[i];
    const int64_t inner = o.mn ? rows : p.K, outer = o.mn ? p.K : rows;
    const int box = o.mn ? kTcStep : (i < 2 ? kTcRows : b_rows);
    if (!make_line_map(&maps[i], o.p, p.dtype, inner, outer, o.ld, box))
      return cudaErrorInvalidValue;
  }
  const int epilogue =
      g.split == 1 ? p.epilogue : (gated ? kEpiGatedPartial : kEpiPartial);
  const bool bf16 = p.dtype == VECTRA_BF16;
  const cudaError_t e =
      epilogue == kEpiLinear
          ? (bf16 ? launch_tc_linear<__nv_bfloat16>(shape.bn, shape.cg, maps,
                                                    g, stream)
                  : launch_tc_linear<__half>(shape.bn, shape.cg, maps, g,
                                             stream))
          : (bf16 ? launch_tc_other<__nv_bfloat16>(epilogue, shape.bn,
                                                   shape.cg, maps, g, stream)
                  : launch_tc_other<__half>(epilogue, shape.bn, shape.cg,
                                            maps, g, stream));
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
