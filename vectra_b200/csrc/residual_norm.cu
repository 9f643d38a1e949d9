// residual_norm.cu: how the kernels of dropout and of the norms, gate and
// residual between two sublayers (residual_norm_kernel.cuh) are launched.
#include <type_traits>

#include "residual_norm.cuh"

namespace vectra {
namespace {

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
         ptr_vec(p.dx) && ptr_vec(p.dbranch) && ptr_vec(p.dgate) &&
         ptr_vec(p.stats) && ptr_vec(p.rest);
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

// Rows that are under way: up to `most`, as many as let `blocks` blocks of
// this team have their copies on an SM beside their `kept` vectors, else one; 0:
// not one fits.
int stages_of(const NormProblem& p, const Team& team, int blocks, int most,
              int kept, size_t* bytes) {
  const size_t es = p.dtype == VECTRA_F32 ? 4 : 2;
  const size_t threads = size_t(team.block.x) * team.block.y;
  const size_t chunks = threads * team.nc * kChunk * es;
  const size_t one = threads * 16 + chunks * p.tensors, vectors = chunks * kept;
  const auto fit = [&](int n) {
    const size_t all = size_t(224 * 1024) / n;
    return all < vectors ? 0 : int((all - vectors) / one);
  };
  int stages = fit(blocks);
  if (stages > most) stages = most;
  if (stages == 0 && fit(1) > 0) stages = 1;
  *bytes = stages * one + vectors;
  return stages;
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
    return dropout_typed<std::remove_pointer_t<decltype(t)>>(
        a, vec, unsigned(blocks), stream);
  });
  if (e == cudaSuccess) count_launches(1);
  return e;
}

cudaError_t launch_norm_forward(const NormProblem& problem,
                                cudaStream_t stream) {
  NormProblem p = problem;
  if (p.M == 0 || p.C == 0) return cudaSuccess;
  const Team team = team_of(p.C);
  const int threads = int(team.block.x * team.block.y);
  int resident = 1024 / threads;  // blocks an SM, for 64 registers
  if (resident < 1) resident = 1;
  int64_t blocks = (p.M + team.block.y - 1) / team.block.y;
  const int64_t most = int64_t(device_sm_count()) * resident;
  // A block that has one row has nothing to fetch ahead.
  const int depth = blocks > most ? 3 : 1;
  if (blocks > most) blocks = most;
  size_t bytes = 0;
  p.tensors = p.gate.p && p.gate_rows == 1 ? 3 : 2;
  p.stages = stages_of(p, team, resident, depth, kNormVectors, &bytes);
  const bool vec = all_vec(p) && p.stages > 0;
  if (!vec) bytes = 0;
  const NormLaunch how{team.nc, team.block, unsigned(blocks), vec, false, bytes};
  const cudaError_t e = with_dtype(p.dtype, [&](auto* t) {
    return norm_forward_typed<std::remove_pointer_t<decltype(t)>>(p, how,
                                                                  stream);
  });
  if (e == cudaSuccess) count_launches(1);
  return e;
}

cudaError_t run_norm_backward(const NormProblem& problem, Workspace& ws,
                              cudaStream_t stream) {
  NormProblem p = problem;
  if (p.C == 0) return cudaSuccess;
  Team team = team_of(p.C);
  if (team.block.x > 512)
    team = {4, dim3((team.block.x / 32 + 1) / 2 * 32, 1)};
  const bool gate = p.gate.p != nullptr;
  const bool norm0 = p.branch_weight.p != nullptr;
  // Two resident blocks an SM (one of the widest rows), teams that each get a
  // unit at least. The limit, in us of two blocks an SM and of one, 8,193 bf16
  // rows, norms on both sides: 5,120 columns (320 threads) with a gate 232 and
  // 485, without 169 and 152; 5,632 (352 threads) 299 and 500, 207 and 156. Two
  // blocks of 352 threads have fewer registers: with that limit 5,120 columns
  // take 278 and 195.
  const int resident = team.block.x > 320 ? 1 : 2;
  int64_t blocks = int64_t(device_sm_count()) * resident;
  const int64_t groups = gate ? p.gate_count : 1;
  const int64_t group_rows = gate ? p.gate_rows : p.M;
  const int64_t teams = blocks * team.block.y;
  int64_t per_group = groups > 0 ? (teams + groups - 1) / groups : 1;
  // Units of eight rows or more, where a gate's sums are written for each.
  const int64_t most = (group_rows + 7) / 8;
  if (gate && groups > 1 && per_group > most) per_group = most;
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

  const bool one_gate = gate && p.gate_count == 1;
  void* outs[4] = {p.dweight, p.dbias, norm0 ? p.dbranch_weight : nullptr,
                   one_gate ? p.dgate : nullptr};
  bool sums = false;
  for (int k = 0; k < 4; ++k) {
    p.part[k] = nullptr;
    if (!outs[k]) continue;
    sums = true;
    p.part[k] = static_cast<float*>(
        ws.take(size_t(blocks) * p.C * sizeof(float)));
  }
  p.gate_part = nullptr;
  const bool gate_sums =
      gate && !one_gate && p.dgate && p.units_per_group > 1;
  if (gate_sums)
    p.gate_part =
        static_cast<float*>(ws.take(size_t(p.units) * p.C * sizeof(float)));
  if (ws.dry || ws.overflow) return cudaSuccess;
  if (p.M == 0 && p.dgate && !one_gate) {
    const size_t es = p.dtype == VECTRA_F32 ? 4 : 2;
    const cudaError_t st =
        cudaMemsetAsync(p.dgate, 0, size_t(p.gate_count) * p.C * es, stream);
    if (st != cudaSuccess) return st;
  }
  size_t bytes = 0;
  p.tensors = 4 + (gate && p.gate_rows == 1) + (p.rest != nullptr);
  // The bias, the last vector, is not read backward.
  p.stages = stages_of(p, team, resident, 3, kNormVectors - 1, &bytes);
  const bool vec = all_vec(p) && p.stages > 0;
  if (!vec) bytes = 0;
  // Teams of a warp join their sums in this memory.
  const size_t join = team.block.y > 1 ? 8 * (512 + 8) * sizeof(float) : 0;
  if (bytes < join) bytes = join;
  const NormLaunch how{team.nc, team.block, unsigned(blocks), vec,
                       resident == 2, bytes};
  return with_dtype(p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    cudaError_t st = norm_backward_typed<T>(p, how, stream);
    if (st == cudaSuccess) count_launches(1);
    const unsigned across = unsigned((p.C + 31) / 32);
    if (st == cudaSuccess && sums) {
      const FinishArgs f{{p.part[0], p.part[1], p.part[2], p.part[3]},
                         {outs[0], outs[1], outs[2], outs[3]}, blocks, 1, p.C};
      st = norm_finish_typed<T>(f, dim3(across, 1, 4), 1024, stream);
      if (st == cudaSuccess) count_launches(1);
    }
    if (st == cudaSuccess && gate_sums) {
      const FinishArgs f{{p.gate_part, nullptr, nullptr, nullptr},
                         {p.dgate, nullptr, nullptr, nullptr},
                         p.units_per_group, groups, p.C};
      const unsigned down = unsigned(groups < 32768 ? groups : 32768);
      st = norm_finish_typed<T>(f, dim3(across, down, 1),
                                p.units_per_group < 32 ? 128 : 1024, stream);
      if (st == cudaSuccess) count_launches(1);
    }
    return st;
  });
}

}  // namespace vectra
