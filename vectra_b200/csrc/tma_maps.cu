// tma_maps.cu: TMA tensor-map encoding for [B, H, N, D] operands, shared by
// the tensor-core kernels. cuTensorMapEncodeTiled is a driver entry point,
// fetched once through the runtime (no link-time dependency on libcuda).
#include <mutex>

#include "rbf_common.cuh"

namespace vectra {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr,
                                cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Encodes through `call`. A thread that has made no CUDA runtime call yet (an
// autograd worker, a serving thread) has no current context, which the
// encoder refuses: bind the device's and try once more.
template <typename F>
bool encode(F&& call) {
  if (call() == CUDA_SUCCESS) return true;
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess &&
         cudaSetDevice(dev) == cudaSuccess && call() == CUDA_SUCCESS;
}

}  // namespace

bool tensor_maps_available() { return encode_fn() != nullptr; }

bool make_tile_map(CUtensorMap* map, const void* base, int dtype, int64_t B,
                   int64_t H, int64_t N, int64_t D, const int64_t* s,
                   int box_rows, int box_cols) {
  auto fn = encode_fn();
  if (!fn) return false;
  const int64_t es = 2;
  cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(N), cuuint64_t(H),
                        cuuint64_t(B)};
  cuuint64_t strides[3] = {cuuint64_t(s[2] * es), cuuint64_t(s[1] * es),
                           cuuint64_t(s[0] * es)};
  // Strides of size-1 dimensions are never used; give them valid values.
  if (N == 1) strides[0] = cuuint64_t(D * es + 15) / 16 * 16;
  if (H == 1) strides[1] = strides[0] * N;
  if (B == 1) strides[2] = strides[1] * H;
  // The swizzle span is the box's row: 128, 64 or 32 bytes.
  const int row_bytes = box_cols * int(es);
  if (row_bytes != 128 && row_bytes != 64 && row_bytes != 32) return false;
  const CUtensorMapSwizzle swizzle =
      row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                       : (row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                          : CU_TENSOR_MAP_SWIZZLE_32B);
  cuuint32_t box[4] = {cuuint32_t(box_cols), cuuint32_t(box_rows), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return encode([&] {
    return fn(map,
              dtype == VECTRA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
              4, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

bool make_group_map(CUtensorMap* map, const void* base, int dtype, int64_t B,
                    int64_t Hk, int64_t G, int64_t N, int64_t D,
                    const int64_t* s, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[5] = {cuuint64_t(D), cuuint64_t(G), cuuint64_t(N),
                        cuuint64_t(Hk), cuuint64_t(B)};
  cuuint64_t strides[4] = {cuuint64_t(s[1] * 2), cuuint64_t(s[2] * 2),
                           cuuint64_t(s[1] * G * 2), cuuint64_t(s[0] * 2)};
  // Strides of size-1 dimensions are never used; give them valid values.
  const cuuint64_t line = cuuint64_t(D * 2 + 15) / 16 * 16;
  for (int i = 0; i < 4; ++i)
    if (dims[i + 1] == 1) strides[i] = line;
  cuuint32_t box[5] = {64, cuuint32_t(G), cuuint32_t(box_rows), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return encode([&] {
    return fn(map,
              dtype == VECTRA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
              5, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

bool make_line_map(CUtensorMap* map, const void* base, int dtype,
                   int64_t inner, int64_t outer, int64_t ld, int box_lines) {
  auto fn = encode_fn();
  if (!fn) return false;
  // The stride of a single line is never used; give it a valid value.
  if (outer == 1) ld = (inner + 7) / 8 * 8;
  cuuint64_t dims[2] = {cuuint64_t(inner), cuuint64_t(outer)};
  cuuint64_t strides[1] = {cuuint64_t(ld) * 2};
  cuuint32_t box[2] = {64, cuuint32_t(box_lines)};
  cuuint32_t estr[2] = {1, 1};
  return encode([&] {
    return fn(map,
              dtype == VECTRA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
              2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

bool make_result_map(CUtensorMap* map, const void* base, int dtype,
                     int64_t cols, int64_t rows, int64_t planes, int64_t ld) {
  auto fn = encode_fn();
  const int64_t es = dtype == VECTRA_F32 ? 4 : 2;
  if (rows == 1) ld = (cols * es + 15) / 16 * 16 / es;
  if (!fn || (reinterpret_cast<uintptr_t>(base) & 15) || ld * es % 16 != 0 ||
      (planes > 1 && ld != cols))
    return false;
  cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows),
                        cuuint64_t(planes)};
  cuuint64_t strides[2] = {cuuint64_t(ld * es), cuuint64_t(ld * es * rows)};
  cuuint32_t box[3] = {cuuint32_t(64 / es), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      dtype == VECTRA_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
      : dtype == VECTRA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return encode([&] {
    return fn(map, type, planes > 1 ? 3 : 2, const_cast<void*>(base), dims,
              strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

}  // namespace vectra
