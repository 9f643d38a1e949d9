// cross.cuh: problem description of attention to an encoder's states
// (vectra_cross_* in include/vectra_block.h) and what its kernels share.
//
//   s_ij = -g |q_i - k_j|^2,  P = softmax_j(s) over j < len,  out = P v
// and for an upstream gradient e of out, with c_i = e_i . out_i:
//   dv_j = sum_i P_ij e_i
//   z_ij = P_ij (e_i . v_j - c_i)                (the gradient of s_ij)
//   dq_i = 2 g sum_j z_ij (k_j - q_i),  dk_j = sum_i 2 g z_ij (q_i - k_j)
//   dg = -sum_ij z_ij |q_i - k_j|^2
// A row of z sums to zero, but for the rounding of c_i and of z: the sums keep
// their q_i and k_j terms, so that what that rounding leaves is weighed by
// distances and not by positions, and dg takes distances from their mean. (The
// sums' own rounding, 2^-24 of a term, is weighed by positions: float32 tensors
// 1,000 deviations from the origin have dq 2.4e-4 off, dk 1.2e-4; 16-bit ones
// show it below their own rounding.)
//
// Query heads that share a key head are rows of one problem: packed row
// i G + g is query i of the g-th of the G heads. Their keys and values are
// read once, and the gradients of shared heads are sums inside a block.
// float16 operands: a product takes P and z as 16-bit numbers, and with
// thousands of keys both lie below 2^-14, where float16 loses bits, while the
// results, sums over keys or queries, do not. They are multiplied by powers of
// two first, exactly, and the sums in float32 divided by them again.
// Whatever a kernel does not finish itself (a long axis split over blocks) it
// leaves in the workspace in float32, and the finish kernels join it in order.
#pragma once

#include "block_common.cuh"

namespace vectra {

struct CrossProblem {
  int32_t dtype = VECTRA_F32;
  int32_t scale_dtype = VECTRA_F32;
  int64_t B = 0, H = 0, Hk = 0, G = 1, Nq = 0, Nk = 0;
  int32_t D = 0, Dv = 0;
  const void* q = nullptr;
  const void* k = nullptr;
  const void* v = nullptr;
  const void* scale = nullptr;
  const void* lengths = nullptr;
  int32_t length_bytes = 8;
  int64_t length_stride = 0;
  int64_t sq[4], sk[4], sv[4], ss[2];
  void* out = nullptr;
  int64_t so[4];
  float* lse = nullptr;  // [B, H, Nq]
  void* rest = nullptr;  // [B, H, Nq, Dv]: what out's rounding left
  // Backward.
  const void* dout = nullptr;
  void* dq = nullptr;
  void* dk = nullptr;
  void* dv = nullptr;
  int64_t se[4], sdq[4], sdk[4], sdv[4];
  float* dscale = nullptr;        // [B, H]
  const float* delta = nullptr;   // [B, H, Nq]: c_i
  float* dscale_rows = nullptr;   // [splits][B, H, Nq][3]
  const float* key_squares = nullptr;  // [B, Hk, Nk]: |k_j|^2, or not formed
  // [B, Hk][2], float16 on the tensor cores: the largest 2 |g| |e_i| of a key
  // head's queries and the largest |v_j| of its seen keys.
  const float* bounds = nullptr;
  // A split axis: parts of it, and their float32 results.
  int32_t splits = 1;
  int64_t row_blocks = 1;    // blocks of one sequence's key head
  float* part = nullptr;     // out or dq or dk: [splits][rows][width]
  float* part_v = nullptr;   // dv
  float* part_ml = nullptr;  // forward: [splits][rows][2], maximum and sum
  unsigned int* err = nullptr;
};

__device__ __forceinline__ int cross_length(const CrossProblem& p, int64_t b) {
  if (p.lengths == nullptr) return int(p.Nk);
  const int64_t i = b * p.length_stride;
  const int64_t n = p.length_bytes == 8
                        ? static_cast<const int64_t*>(p.lengths)[i]
                        : int64_t(static_cast<const int32_t*>(p.lengths)[i]);
  return int(n < 0 ? 0 : (n < p.Nk ? n : p.Nk));
}

// A result and what its rounding left.
template <typename T>
__device__ __forceinline__ void store_with_rest(T* out, T* rest, float x) {
  const T r = from_f32<T>(x);
  *out = r;
  if (rest) *rest = from_f32<T>((x - to_f32(r)) * kRestLift<T>);
}

__device__ __forceinline__ float cross_scale(const CrossProblem& p, int64_t b,
                                             int64_t h) {
  return load_any(p.scale, p.scale_dtype, b * p.ss[0] + h * p.ss[1]);
}

// What weights of float16 are multiplied by before a product with them, if
// they are 1 at most (and a little more by rounding).
constexpr float kLift = 0x1p14f;

// A power of two that brings x >= 0 to [2^to, 2^(to + 1)), and 2^60 for what
// is smaller than that could; its inverse is exact too.
__device__ __forceinline__ float scale_up_to(float x, int to) {
  const int exponent = int(__float_as_uint(x) >> 23 & 0xff) - 127;
  const int k = min(to - exponent, 60);
  return __uint_as_float(uint32_t(k + 127) << 23);
}
__device__ __forceinline__ float inverse_of(float power_of_two) {
  return __uint_as_float((254u << 23) - __float_as_uint(power_of_two));
}

// Tiles [first, last) of `tiles` that part s of `splits` takes.
__device__ __forceinline__ void split_range(int tiles, int s, int splits,
                                            int* first, int* last) {
  *first = int(int64_t(tiles) * s / splits);
  *last = int(int64_t(tiles) * (s + 1) / splits);
}

// cross_simple.cu: any type, width up to 256, and strides.
cudaError_t run_cross_simple_forward(const CrossProblem& p, Workspace& ws,
                                     cudaStream_t stream);
cudaError_t run_cross_simple_backward(const CrossProblem& p, Workspace& ws,
                                      cudaStream_t stream);

// cross_tc.cu: bf16 and f16 on the tensor cores, widths up to 128.
bool cross_tc_supports(const CrossProblem& p, bool backward);
cudaError_t run_cross_tc_forward(const CrossProblem& p, Workspace& ws,
                                 cudaStream_t stream);
cudaError_t run_cross_tc_backward(const CrossProblem& p, Workspace& ws,
                                  cudaStream_t stream);

// cross_rows.cu: bf16 and f16, up to 16 packed rows, widths up to 128.
bool cross_rows_supports(const CrossProblem& p, bool backward);
cudaError_t run_cross_rows_forward(const CrossProblem& p, Workspace& ws,
                                   cudaStream_t stream);
cudaError_t run_cross_rows_backward(const CrossProblem& p, Workspace& ws,
                                    cudaStream_t stream);

// cross_finish.cu.
// c_i of every row into delta.
cudaError_t launch_cross_delta(const CrossProblem& p, float* delta,
                               cudaStream_t stream);
// |k_j|^2 of every key into `squares` [B, Hk, Nk] (16-byte pieces: what
// cross_tc_supports allows).
cudaError_t launch_cross_squares(const CrossProblem& p, float* squares,
                                 cudaStream_t stream);
// p.bounds (16-byte pieces too): zeros, then the maxima.
cudaError_t launch_cross_bounds(const CrossProblem& p, float* bounds,
                                cudaStream_t stream);
// out and lse from the parts.
cudaError_t launch_cross_join(const CrossProblem& p, cudaStream_t stream);
// `out` [B, H, N, width] from [splits][B, H, N][width].
cudaError_t launch_cross_sum(int32_t dtype, const float* part, int splits,
                             int64_t B, int64_t H, int64_t N, int width,
                             void* out, const int64_t* so,
                             cudaStream_t stream);
// dscale from dscale_rows.
cudaError_t launch_cross_dscale(const CrossProblem& p, int splits,
                                cudaStream_t stream);

constexpr int kMaxCrossWidth = 256;

}  // namespace vectra
