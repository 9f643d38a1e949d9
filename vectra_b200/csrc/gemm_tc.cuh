// gemm_tc.cuh: interface of the tensor-core matrix products (gemm_tc.cu).
#pragma once

#include "block_common.cuh"

namespace vectra {

// A launch shape: tile columns (accumulator columns; a gated tile has half
// as many outputs), CTAs per tile, and parts of the reduction.
struct TcShape {
  int bn = 128;  // 64, 128, or with CTA pairs 256
  int cg = 1;
  int split = 1;
};

constexpr int kTcRows = 128;  // rows of a tile per CTA
constexpr int kTcStep = 64;   // reduction per stage: one 128-byte row

struct TcArgs {
  GemmProblem p;
  float* partial;     // split > 1: [split][planes][M][N]
  int tiles_m, tiles_n;
  int steps_seg;      // stages of one segment
  int steps;          // of all segments
  int split;
  int steps_part;     // steps of one part
  int64_t units;      // tiles * split
  uint8_t a_mn, b_mn;  // operand staged MN-major
  uint8_t tma_out, tma_pre;  // results, saved values: by tensor map
  uint8_t vec_res;           // residual in 16-byte pieces
  int32_t a_lines, b_lines;  // float32: lines of one plane
};

// Epilogues of the kernels beyond GemmEpilogue: float32 sums of one part.
enum { kEpiPartial = 4, kEpiGatedPartial = 5 };

template <typename T>
cudaError_t launch_tc_linear(int bn, int cg, const CUtensorMap* maps,
                             const TcArgs& g, cudaStream_t stream);
template <typename T>
cudaError_t launch_tc_other(int epilogue, int bn, int cg,
                            const CUtensorMap* maps, const TcArgs& g,
                            cudaStream_t stream);

// Any type and layout; the reduction is not empty.
cudaError_t run_gemm_tc(const GemmProblem& p, const TcShape& shape,
                        Workspace& ws, cudaStream_t stream);

}  // namespace vectra
