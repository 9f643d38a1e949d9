// gemm_select.cu: which kernel computes a matrix product of the
// transformer-block operators.
#include "block_common.cuh"
#include "gemm_rows.cuh"
#include "gemm_tc.cuh"

namespace vectra {
namespace {

// Tile shape and parts of a tensor-core product: the least estimated time
// over the shapes, each with one part or as many as fill the SMs.
//
// A stage of 64 of the reduction takes a CTA about kStep microseconds: for
// the pair's 256 x 256 tile the tensor cores bound it, for the narrow tiles
// the 24 or 32 KB that it brings in. A tile's start and epilogue that nothing
// overlaps take kTile. Parts write and re-read float32 sums and need a
// second launch.
TcShape tc_shape(const GemmProblem& p) {
  struct Option {
    int bn, cg;
    double step;
  };
  constexpr Option kOptions[] = {
      {256, 2, 0.28}, {128, 1, 0.25}, {64, 1, 0.19}};
  // float32 stages hold three planes and are multiplied six times.
  constexpr double kPlanes = 3.4;
  constexpr double kTile = 2.0, kSecondLaunch = 2.5, kBytesPerUs = 5.0e6;
  const bool gated =
      p.epilogue == kEpiGated || p.epilogue == kEpiGatedGrad;
  const double sms = device_sm_count();
  const bool f32 = p.dtype == VECTRA_F32;
  const int64_t steps = (p.K + 63) / 64 * p.segments;
  TcShape best;
  double least = 1e30;
  for (const Option& o : kOptions) {
    if (o.cg == 2 && (f32 || p.M <= 128)) continue;
    if (gated && o.bn < 128) continue;
    const int64_t cols = gated ? o.bn / 2 : o.bn;
    const int64_t rows = int64_t(kTcRows) * o.cg;
    const int64_t tiles =
        ((p.M + rows - 1) / rows) * ((p.N + cols - 1) / cols);
    const int64_t slots = int64_t(sms) / o.cg;
    int64_t most = slots / tiles;
    if (most > steps / 4) most = steps / 4;
    if (most > 64) most = 64;
    for (const int64_t split : {int64_t(1), most}) {
      if (split < 1 || (split > 1 && p.epilogue == kEpiGatedGrad)) continue;
      const int64_t per = (steps + split - 1) / split;
      const int64_t waves = (tiles * split + slots - 1) / slots;
      double t = double(waves) * double(per) * o.step * (f32 ? kPlanes : 1.0) +
                 kTile;
      if (split > 1)
        t += kSecondLaunch + 8.0 * double(split) * double(p.M) *
                                 double(p.N) * (gated ? 2 : 1) / kBytesPerUs;
      if (t < least) {
        least = t;
        best.bn = o.bn;
        best.cg = o.cg;
        best.split = int(split);
      }
    }
  }
  return best;
}

}  // namespace

cudaError_t run_gemm(const GemmProblem& p, Workspace& ws,
                     cudaStream_t stream) {
  if (p.M == 0 || p.N == 0) return cudaSuccess;
  if (p.K == 0) {
    if (ws.dry) return cudaSuccess;
    const cudaError_t e = launch_split_finish(p, 0, nullptr, stream);
    if (e == cudaSuccess) count_launches(1);
    return e;
  }
  if (p.epilogue != kEpiGatedGrad && gemm_rows_supports(p)) {
    if (ws.dry) return cudaSuccess;
    const cudaError_t e = launch_gemm_rows(p, stream);
    if (e == cudaSuccess) count_launches(1);
    return e;
  }
  return run_gemm_tc(p, tc_shape(p), ws, stream);
}

}  // namespace vectra
