// block_ext.h: what the PyTorch registrations of the transformer-block
// operators share (block_ext.cpp, decoder_ext.cpp): argument checks,
// descriptions of tensors for the C ABI, workspaces and errors, and the rules
// of their autograd functions.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <vector>

#include "vectra_block.h"

namespace vectra_ext {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// ---------------------------------------------------------------------------
// Checks and descriptions.
// ---------------------------------------------------------------------------
inline bool io_dtype(at::ScalarType t) {
  return t == at::kFloat || t == at::kHalf || t == at::kBFloat16;
}

inline int32_t abi_dtype(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return VECTRA_F32;
    case at::kHalf:
      return VECTRA_F16;
    case at::kBFloat16:
      return VECTRA_BF16;
    default:
      return -1;
  }
}

inline bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

inline void check_like(const Tensor& t, const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ",
                    x.device(), ", got ", t.device());
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type(), name, " must be ",
                    x.scalar_type(), ", got ", t.scalar_type());
}

inline void check_sizes(const Tensor& t, const char* name, at::IntArrayRef sizes) {
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, " must have shape ", sizes,
                    ", got ", t.sizes());
}


// [..., C] as [rows, C]: a view where the leading dimensions allow one.
inline Tensor as_rows(const Tensor& t) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  return t.dim() == 2 ? t : t.reshape({rows, t.size(-1)});
}

inline vectra_tensor describe(const Tensor& t) {
  vectra_tensor d{};
  d.data = t.data_ptr();
  d.dtype = abi_dtype(t.scalar_type());
  d.ndim = int32_t(t.dim());
  for (int64_t i = 0; i < t.dim(); ++i) {
    d.size[i] = t.size(i);
    d.stride[i] = t.stride(i);
  }
  return d;
}

inline vectra_tensor describe(const OptTensor& t) {
  return has(t) ? describe(*t) : vectra_tensor{};
}

// The same view as the ABI's description, without making a tensor of it;
// where the leading dimensions do not allow one, `copy` keeps the copy.
inline vectra_tensor describe_rows(const Tensor& t, Tensor* copy) {
  const int64_t last = t.dim() - 1;
  int64_t rows = 1, ld = 0;
  bool regular = true;
  for (int64_t i = last - 1; i >= 0; --i) {
    if (t.size(i) != 1) {
      if (rows == 1) {
        ld = t.stride(i);
      } else if (t.stride(i) != ld * rows) {
        regular = false;
      }
    }
    rows *= t.size(i);
  }
  if (!regular && rows > 0) {
    *copy = as_rows(t);
    return describe(*copy);
  }
  vectra_tensor d{};
  d.data = t.data_ptr();
  d.dtype = abi_dtype(t.scalar_type());
  d.ndim = 2;
  d.size[0] = rows;
  d.size[1] = t.size(last);
  d.stride[0] = rows > 1 ? ld : t.size(last);
  d.stride[1] = t.stride(last);
  return d;
}

[[noreturn]] inline void raise_status(const char* op, int status) {
  const char* msg = vectra_block_strerror(status);
  switch (status) {
    case VECTRA_ERR_UNSUPPORTED:
      TORCH_CHECK_NOT_IMPLEMENTED(false, "vectra_b200::", op, ": ", msg);
    case VECTRA_ERR_CUDA:
    case VECTRA_ERR_DEVICE:
    case VECTRA_ERR_WORKSPACE:
      TORCH_CHECK(false, "vectra_b200::", op, ": ", msg);
    default:
      TORCH_CHECK_VALUE(false, "vectra_b200::", op, ": ", msg);
  }
  TORCH_CHECK(false, "unreachable");
}

// Sizes the workspace, allocates it and makes the call.
template <typename Args, typename Size, typename Call>
inline void call_with_workspace(const char* op, Args& a, const Tensor& like,
                         Size&& size, Call&& call) {
  const int64_t bytes = size(&a);
  if (bytes < 0) raise_status(op, int(bytes));
  Tensor ws;
  if (bytes > 0) {
    ws = at::empty({bytes + 256}, like.options().dtype(at::kByte));
    const uintptr_t p = reinterpret_cast<uintptr_t>(ws.data_ptr());
    a.workspace = reinterpret_cast<void*>((p + 255) & ~uintptr_t(255));
    a.workspace_bytes = size_t(bytes);
  }
  const int st = call(
      &a, at::cuda::getCurrentCUDAStream(like.device().index()).stream());
  if (st != VECTRA_OK) raise_status(op, st);
}

inline Tensor f32(const Tensor& t) { return t.to(at::kFloat); }
inline OptTensor f32(const OptTensor& t) {
  return has(t) ? OptTensor(f32(*t)) : OptTensor();
}

// Results follow their input's order of heads and tokens, by the rule of
// vectra::rbf_attention's output (torch_ext.cpp).
inline Tensor empty_like_heads(const Tensor& t) {
  const int64_t b = t.size(0), h = t.size(1), n = t.size(2), d = t.size(3);
  if (h > 1 && n > 1 && t.stride(2) > t.stride(1))
    return at::empty_strided({b, h, n, d}, {n * h * d, d, h * d, 1},
                             t.options());
  return at::empty({b, h, n, d}, t.options());
}

// ---------------------------------------------------------------------------
// Autograd.
// ---------------------------------------------------------------------------
inline bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
inline bool wants_grad(const OptTensor& t) { return has(t) && t->requires_grad(); }

inline bool has_tangent(const Tensor& t) {
  return t.defined() && t._fw_grad(/*level=*/0).defined();
}
inline bool has_tangent(const OptTensor& t) { return has(t) && has_tangent(*t); }

// The operators have no forward-mode formula; below autograd a tangent would
// be dropped, which reads as zero.
template <typename... Args>
inline void refuse_tangents(const char* op, const Args&... args) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !(has_tangent(args) || ...), "vectra_b200::", op,
      ": forward-mode differentiation is not implemented");
}

inline OptTensor optional(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}

// Backward calls go straight to the kernels unless their results are to be
// differentiated again, which the operators' own autograd entry refuses.
struct BelowUnlessRecording {
  std::optional<at::AutoDispatchBelowADInplaceOrView> below;
  BelowUnlessRecording() {
    if (!at::GradMode::is_enabled()) below.emplace();
  }
};

// What stands for an input that the backward pass reads the shape of only:
// one element, expanded. Saving the input itself would keep its memory and
// forbid writing it in place.
inline Tensor shape_of(const Tensor& t) {
  return at::empty({1}, t.options()).expand_symint(t.sym_sizes());
}

}  // namespace vectra_ext
