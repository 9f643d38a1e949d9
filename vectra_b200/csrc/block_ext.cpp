// block_ext.cpp: PyTorch registration of the transformer-block operators
// (include/vectra_block.h) in the vectra_b200 namespace:
//
//   linear, gated_linear, qk_norm_rope        differentiable entry points
//   linear_with_pre, gated_linear_with_pre    the forward that also returns
//                                             what the backward needs
//   linear_backward, gated_linear_backward,
//   qk_norm_rope_backward                     gradients
//
// CUDA tensors run the kernels of libvectra_rbf.so on the current stream,
// with results and workspace from PyTorch's allocator; CPU tensors run the
// ATen formulation below in float32. The entry points differentiate through
// C++ autograd functions; the backward operators are not differentiable
// again (they raise). Fake implementations are in vectra_b200/block.py.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "vectra_block.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// ---------------------------------------------------------------------------
// Shared checks.
// ---------------------------------------------------------------------------
int32_t activation_of(c10::string_view name) {
  if (name == "none") return VECTRA_ACT_NONE;
  if (name == "relu") return VECTRA_ACT_RELU;
  if (name == "gelu") return VECTRA_ACT_GELU;
  if (name == "gelu_tanh") return VECTRA_ACT_GELU_TANH;
  if (name == "silu") return VECTRA_ACT_SILU;
  TORCH_CHECK_VALUE(false, "activation must be 'none', 'relu', 'gelu', "
                           "'gelu_tanh' or 'silu', got '", std::string(name), "'");
}

bool io_dtype(at::ScalarType t) {
  return t == at::kFloat || t == at::kHalf || t == at::kBFloat16;
}

int32_t abi_dtype(at::ScalarType t) {
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

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_like(const Tensor& t, const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ",
                    x.device(), ", got ", t.device());
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type(), name, " must be ",
                    x.scalar_type(), ", got ", t.scalar_type());
}

void check_sizes(const Tensor& t, const char* name, at::IntArrayRef sizes) {
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, " must have shape ", sizes,
                    ", got ", t.sizes());
}

void check_layer(const Tensor& x, const Tensor& w, const char* w_name) {
  TORCH_CHECK_VALUE(io_dtype(x.scalar_type()),
                    "x must be float32, float16 or bfloat16, got ",
                    x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must be [..., K]");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(-1), w_name,
                    " must be [N, K] with K = x.shape[-1] = ", x.size(-1),
                    ", got ", w.sizes());
  check_like(w, w_name, x);
}

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s = sizes.vec();
  s.back() = last;
  return s;
}

// [..., C] as [rows, C]: a view where the leading dimensions allow one.
Tensor as_rows(const Tensor& t) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  return t.dim() == 2 ? t : t.reshape({rows, t.size(-1)});
}

vectra_tensor describe(const Tensor& t) {
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

vectra_tensor describe(const OptTensor& t) {
  return has(t) ? describe(*t) : vectra_tensor{};
}

// The same view as the ABI's description, without making a tensor of it;
// where the leading dimensions do not allow one, `copy` keeps the copy.
vectra_tensor describe_rows(const Tensor& t, Tensor* copy) {
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

[[noreturn]] void raise_status(const char* op, int status) {
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
void call_with_workspace(const char* op, Args& a, const Tensor& like,
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

// ---------------------------------------------------------------------------
// Float32 formulation on CPU tensors.
// ---------------------------------------------------------------------------
// The kernels' forms (block_common.cuh): ATen's GELU and its gradient lose
// the negative tail, and some infinite or very large arguments, in float32.
constexpr double kGeluTanhC = 0.7978845608028654;  // sqrt(2 / pi)
constexpr double kGeluTanhA = 0.044715;

// Phi(z).
Tensor cpu_cdf(const Tensor& z) {
  return at::special_erfc(z * -0.7071067811865476) * 0.5;
}
// The argument of tanh GELU's sigmoid.
Tensor cpu_tanh_argument(const Tensor& z) {
  return (z + z * z * z * kGeluTanhA) * (2 * kGeluTanhC);
}

Tensor cpu_act(const Tensor& z, int32_t act) {
  switch (act) {
    case VECTRA_ACT_RELU:
      return at::relu(z);
    case VECTRA_ACT_GELU:
      return z * cpu_cdf(z);
    case VECTRA_ACT_GELU_TANH:
      return z * at::sigmoid(cpu_tanh_argument(z));
    case VECTRA_ACT_SILU:
      return at::silu(z);
    default:
      return z;
  }
}

// dy act'(z).
Tensor cpu_act_grad(const Tensor& dy, const Tensor& z, int32_t act) {
  switch (act) {
    case VECTRA_ACT_RELU:
      return dy * (z > 0);
    case VECTRA_ACT_GELU:
      return dy * (cpu_cdf(z) +
                   z * at::exp(z * z * -0.5) * 0.3989422804014327);
    case VECTRA_ACT_GELU_TANH: {
      const Tensor x = cpu_tanh_argument(z), s = at::sigmoid(x);
      // 0 * z^2 far out has to stay 0.
      const Tensor t = at::clamp_max(z * z, 1e4);
      return dy * (s + z * s * at::sigmoid(-x) *
                           ((t * (3 * kGeluTanhA) + 1) * (2 * kGeluTanhC)));
    }
    case VECTRA_ACT_SILU: {
      const Tensor s = at::sigmoid(z);
      return dy * (s * (z * at::sigmoid(-z) + 1));
    }
    default:
      return dy;
  }
}

Tensor f32(const Tensor& t) { return t.to(at::kFloat); }
OptTensor f32(const OptTensor& t) {
  return has(t) ? OptTensor(f32(*t)) : OptTensor();
}

// ---------------------------------------------------------------------------
// linear
// ---------------------------------------------------------------------------
void check_linear(const Tensor& x, const Tensor& w, const OptTensor& bias,
                  const OptTensor& residual) {
  check_layer(x, w, "weight");
  if (has(bias)) {
    check_like(*bias, "bias", x);
    check_sizes(*bias, "bias", {w.size(0)});
  }
  if (has(residual)) {
    check_like(*residual, "residual", x);
    check_sizes(*residual, "residual", with_last(x.sizes(), w.size(0)));
  }
}

Tensor linear_run(const Tensor& x, const Tensor& w, const OptTensor& bias,
                  const OptTensor& residual, c10::string_view activation,
                  Tensor* pre) {
  check_linear(x, w, bias, residual);
  c10::cuda::CUDAGuard guard(x.device());
  const auto shape = with_last(x.sizes(), w.size(0));
  Tensor y = at::empty(shape, x.options());
  Tensor x_copy, res_copy;
  vectra_linear_args a{};
  a.activation = activation_of(activation);
  a.x = describe_rows(x, &x_copy);
  a.weight = describe(w);
  a.bias = describe(bias);
  if (has(residual)) a.residual = describe_rows(*residual, &res_copy);
  a.y = describe_rows(y, nullptr);
  if (pre != nullptr) {
    *pre = at::empty(shape, x.options());
    a.pre = describe_rows(*pre, nullptr);
  }
  call_with_workspace("linear", a, x, vectra_linear_forward_workspace_bytes,
                      vectra_linear_forward);
  return y;
}

std::tuple<Tensor, Tensor> linear_cuda(const Tensor& x, const Tensor& w,
                                       const OptTensor& bias,
                                       const OptTensor& residual,
                                       const std::string& activation,
                                       bool want_pre) {
  Tensor pre;
  Tensor y = linear_run(x, w, bias, residual, activation,
                        want_pre ? &pre : nullptr);
  if (!want_pre) pre = at::empty({0}, x.options());
  return {y, pre};
}

Tensor linear_only_cuda(const Tensor& x, const Tensor& w,
                        const OptTensor& bias, const OptTensor& residual,
                        c10::string_view activation) {
  return linear_run(x, w, bias, residual, activation, nullptr);
}

std::tuple<Tensor, Tensor> linear_cpu(const Tensor& x, const Tensor& w,
                                      const OptTensor& bias,
                                      const OptTensor& residual,
                                      const std::string& activation,
                                      bool want_pre) {
  check_linear(x, w, bias, residual);
  const int32_t act = activation_of(activation);
  Tensor z = at::matmul(f32(x), f32(w).t());
  if (has(bias)) z = z + f32(*bias);
  Tensor y = cpu_act(z, act);
  if (has(residual)) y = y + f32(*residual);
  // Results of their own, also where no cast makes a copy.
  Tensor out = at::empty(y.sizes(), x.options()).copy_(y);
  Tensor pre = want_pre ? at::empty(z.sizes(), x.options()).copy_(z)
                        : at::empty({0}, x.options());
  return {out, pre};
}

void check_linear_grad(const Tensor& dy, const Tensor& x, const Tensor& w,
                       const Tensor& pre, int32_t act) {
  check_layer(x, w, "weight");
  check_like(dy, "dy", x);
  const auto shape = with_last(x.sizes(), w.size(0));
  check_sizes(dy, "dy", shape);
  if (act != VECTRA_ACT_NONE) {
    check_like(pre, "pre", x);
    check_sizes(pre, "pre", shape);
  }
}

using Grads3 = std::tuple<Tensor, Tensor, Tensor>;

Grads3 linear_backward_cuda(const Tensor& dy, const Tensor& x,
                            const Tensor& w, const Tensor& pre,
                            const std::string& activation, bool need_dx,
                            bool need_dw, bool need_db) {
  const int32_t act = activation_of(activation);
  check_linear_grad(dy, x, w, pre, act);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor x_copy, dy_copy, pre_copy;
  Tensor dx = at::empty(need_dx ? x.sizes().vec() : std::vector<int64_t>{0},
                        x.options());
  Tensor dw = need_dw ? at::empty(w.sizes(), x.options())
                      : at::empty({0}, x.options());
  Tensor db = at::empty({need_db ? w.size(0) : 0}, x.options());
  vectra_linear_grad_args a{};
  a.activation = act;
  a.dy = describe_rows(dy, &dy_copy);
  a.x = describe_rows(x, &x_copy);
  a.weight = describe(w);
  if (act != VECTRA_ACT_NONE) {
    pre_copy = pre.contiguous();
    a.pre = describe_rows(pre_copy, nullptr);
  }
  if (need_dx) a.dx = describe_rows(dx, nullptr);
  if (need_dw) a.dweight = describe(dw);
  if (need_db) a.dbias = describe(db);
  call_with_workspace("linear_backward", a, x,
                      vectra_linear_backward_workspace_bytes,
                      vectra_linear_backward);
  return {dx, dw, db};
}

Grads3 linear_backward_cpu(const Tensor& dy, const Tensor& x, const Tensor& w,
                           const Tensor& pre, const std::string& activation,
                           bool need_dx, bool need_dw, bool need_db) {
  const int32_t act = activation_of(activation);
  check_linear_grad(dy, x, w, pre, act);
  Tensor dz = f32(as_rows(dy));
  if (act != VECTRA_ACT_NONE)
    dz = cpu_act_grad(dz, f32(as_rows(pre)), act);
  const auto none = [&] { return at::empty({0}, x.options()); };
  Tensor dx = need_dx ? at::matmul(dz, f32(w)).to(x.scalar_type())
                            .reshape(x.sizes())
                      : none();
  Tensor dw = need_dw ? at::matmul(dz.t(), f32(as_rows(x)))
                            .to(x.scalar_type())
                      : none();
  Tensor db = need_db ? dz.sum(0).to(x.scalar_type()) : none();
  return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// gated_linear
// ---------------------------------------------------------------------------
void check_gated(const Tensor& x, const Tensor& wg, const Tensor& wu,
                 const OptTensor& bg, const OptTensor& bu) {
  check_layer(x, wg, "w_gate");
  check_like(wu, "w_up", x);
  check_sizes(wu, "w_up", wg.sizes());
  if (has(bg)) {
    check_like(*bg, "b_gate", x);
    check_sizes(*bg, "b_gate", {wg.size(0)});
  }
  if (has(bu)) {
    check_like(*bu, "b_up", x);
    check_sizes(*bu, "b_up", {wg.size(0)});
  }
}

Tensor gated_run(const Tensor& x, const Tensor& wg, const Tensor& wu,
                 const OptTensor& bg, const OptTensor& bu,
                 c10::string_view activation, Tensor* gate, Tensor* up) {
  check_gated(x, wg, wu, bg, bu);
  c10::cuda::CUDAGuard guard(x.device());
  const auto shape = with_last(x.sizes(), wg.size(0));
  Tensor h = at::empty(shape, x.options());
  Tensor x_copy;
  vectra_gated_args a{};
  a.activation = activation_of(activation);
  a.x = describe_rows(x, &x_copy);
  a.w_gate = describe(wg);
  a.w_up = describe(wu);
  a.b_gate = describe(bg);
  a.b_up = describe(bu);
  a.h = describe_rows(h, nullptr);
  if (gate != nullptr) {
    const auto f32_options = x.options().dtype(at::kFloat);
    *gate = at::empty(shape, f32_options);
    *up = at::empty(shape, f32_options);
    a.gate = describe_rows(*gate, nullptr);
    a.up = describe_rows(*up, nullptr);
  }
  call_with_workspace("gated_linear", a, x,
                      vectra_gated_linear_forward_workspace_bytes,
                      vectra_gated_linear_forward);
  return h;
}

Grads3 gated_cuda(const Tensor& x, const Tensor& wg, const Tensor& wu,
                  const OptTensor& bg, const OptTensor& bu,
                  const std::string& activation, bool want_pre) {
  Tensor gate, up;
  Tensor h = gated_run(x, wg, wu, bg, bu, activation,
                       want_pre ? &gate : nullptr, &up);
  if (!want_pre)
    for (Tensor* t : {&gate, &up})
      *t = at::empty({0}, x.options().dtype(at::kFloat));
  return {h, gate, up};
}

Tensor gated_only_cuda(const Tensor& x, const Tensor& wg, const Tensor& wu,
                       const OptTensor& bg, const OptTensor& bu,
                       c10::string_view activation) {
  return gated_run(x, wg, wu, bg, bu, activation, nullptr, nullptr);
}

Grads3 gated_cpu(const Tensor& x, const Tensor& wg, const Tensor& wu,
                 const OptTensor& bg, const OptTensor& bu,
                 const std::string& activation, bool want_pre) {
  check_gated(x, wg, wu, bg, bu);
  const int32_t act = activation_of(activation);
  Tensor g = at::matmul(f32(x), f32(wg).t());
  Tensor u = at::matmul(f32(x), f32(wu).t());
  if (has(bg)) g = g + f32(*bg);
  if (has(bu)) u = u + f32(*bu);
  Tensor h = (cpu_act(g, act) * u).to(x.scalar_type());
  const auto none = [&] {
    return at::empty({0}, x.options().dtype(at::kFloat));
  };
  if (!want_pre) return {h, none(), none()};
  return {h, g, u};
}

// Gradients of x, of both weights [2, F, K] and of both biases [2, F].
// gate and up may both be empty: they are formed again.
void check_gated_grad(const Tensor& dh, const Tensor& x, const Tensor& wg,
                      const Tensor& wu, const OptTensor& bg,
                      const OptTensor& bu, const Tensor& gate,
                      const Tensor& up) {
  check_gated(x, wg, wu, bg, bu);
  check_like(dh, "dh", x);
  const auto shape = with_last(x.sizes(), wg.size(0));
  check_sizes(dh, "dh", shape);
  if (gate.numel() == 0 && up.numel() == 0) return;
  for (const Tensor* t : {&gate, &up}) {
    check_sizes(*t, "gate and up", shape);
    TORCH_CHECK_VALUE(t->device() == x.device() &&
                          t->scalar_type() == at::kFloat,
                      "gate and up must be float32 on ", x.device());
  }
}

Grads3 gated_backward_cuda(const Tensor& dh, const Tensor& x,
                           const Tensor& wg, const Tensor& wu,
                           const OptTensor& bg, const OptTensor& bu,
                           const Tensor& gate, const Tensor& up,
                           const std::string& activation, bool need_dx,
                           bool need_dw, bool need_db) {
  check_gated_grad(dh, x, wg, wu, bg, bu, gate, up);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor x_copy, dh_copy;
  const Tensor g = gate.contiguous(), u = up.contiguous();
  Tensor dx = at::empty(need_dx ? x.sizes().vec() : std::vector<int64_t>{0},
                        x.options());
  const int64_t f = wg.size(0);
  Tensor dw = need_dw ? at::empty({2, f, wg.size(1)}, x.options())
                      : at::empty({0}, x.options());
  Tensor db = need_db ? at::empty({2, f}, x.options())
                      : at::empty({0}, x.options());
  vectra_gated_grad_args a{};
  a.activation = activation_of(activation);
  a.dh = describe_rows(dh, &dh_copy);
  a.x = describe_rows(x, &x_copy);
  a.w_gate = describe(wg);
  a.w_up = describe(wu);
  a.b_gate = describe(bg);
  a.b_up = describe(bu);
  if (g.numel()) {
    a.gate = describe_rows(g, nullptr);
    a.up = describe_rows(u, nullptr);
  }
  if (need_dx) a.dx = describe_rows(dx, nullptr);
  if (need_dw) {
    a.dw_gate = describe(dw.select(0, 0));
    a.dw_up = describe(dw.select(0, 1));
  }
  if (need_db) {
    a.db_gate = describe(db.select(0, 0));
    a.db_up = describe(db.select(0, 1));
  }
  call_with_workspace("gated_linear_backward", a, x,
                      vectra_gated_linear_backward_workspace_bytes,
                      vectra_gated_linear_backward);
  return {dx, dw, db};
}

Grads3 gated_backward_cpu(const Tensor& dh, const Tensor& x,
                          const Tensor& wg, const Tensor& wu,
                          const OptTensor& bg, const OptTensor& bu,
                          const Tensor& gate, const Tensor& up,
                          const std::string& activation, bool need_dx,
                          bool need_dw, bool need_db) {
  check_gated_grad(dh, x, wg, wu, bg, bu, gate, up);
  const int32_t act = activation_of(activation);
  const auto dt = x.scalar_type();
  const Tensor d = f32(as_rows(dh));
  Tensor g, u;
  if (gate.numel() || d.numel() == 0) {
    g = as_rows(gate).reshape(d.sizes());
    u = as_rows(up).reshape(d.sizes());
  } else {
    g = at::matmul(f32(as_rows(x)), f32(wg).t());
    u = at::matmul(f32(as_rows(x)), f32(wu).t());
    if (has(bg)) g = g + f32(*bg);
    if (has(bu)) u = u + f32(*bu);
  }
  const Tensor dg = cpu_act_grad(d * u, g, act), du = d * cpu_act(g, act);
  const auto none = [&] { return at::empty({0}, x.options()); };
  Tensor dx = need_dx ? (at::matmul(dg, f32(wg)) + at::matmul(du, f32(wu)))
                            .to(dt)
                            .reshape(x.sizes())
                      : none();
  const Tensor x2 = f32(as_rows(x));
  Tensor dw = need_dw ? at::stack({at::matmul(dg.t(), x2),
                                   at::matmul(du.t(), x2)}).to(dt)
                      : none();
  Tensor db = need_db ? at::stack({dg.sum(0), du.sum(0)}).to(dt) : none();
  return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// qk_norm_rope
// ---------------------------------------------------------------------------
void check_qk(const Tensor& q, const Tensor& k, const Tensor& cos,
              const Tensor& sin, const OptTensor& qw, const OptTensor& kw,
              const OptTensor& positions) {
  TORCH_CHECK_VALUE(io_dtype(q.scalar_type()),
                    "q must be float32, float16 or bfloat16, got ",
                    q.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4,
                    "q and k must be rank 4 ([B, H, N, D])");
  check_like(k, "k", q);
  TORCH_CHECK_VALUE(k.size(0) == q.size(0) && k.size(2) == q.size(2) &&
                        k.size(3) == q.size(3),
                    "q ", q.sizes(), " and k ", k.sizes(),
                    " may differ in heads only");
  const int64_t d = q.size(3);
  for (const Tensor* t : {&cos, &sin}) {
    TORCH_CHECK_VALUE(t->dim() == 2 && t->sizes() == cos.sizes() &&
                          t->scalar_type() == at::kFloat &&
                          t->device() == q.device(),
                      "cos and sin must be float32 [P, R / 2] tables on ",
                      q.device());
    TORCH_CHECK_VALUE(t->size(1) <= 1 || t->stride(1) == 1,
                      "cos and sin need a unit inner stride");
  }
  TORCH_CHECK_VALUE(2 * cos.size(1) <= d, "the tables rotate ",
                    2 * cos.size(1), " components of vectors of ", d);
  const OptTensor* weights[2] = {&qw, &kw};
  for (const OptTensor* w : weights) {
    if (!has(*w)) continue;
    TORCH_CHECK_VALUE((*w)->device() == q.device() &&
                          ((*w)->scalar_type() == q.scalar_type() ||
                           (*w)->scalar_type() == at::kFloat),
                      "norm weights must be ", q.scalar_type(),
                      " or float32 on ", q.device());
    check_sizes(**w, "norm weights", {d});
  }
  if (has(positions)) {
    TORCH_CHECK_VALUE(positions->device() == q.device() &&
                          (positions->scalar_type() == at::kLong ||
                           positions->scalar_type() == at::kInt),
                      "positions must be int64 or int32 on ", q.device());
    TORCH_CHECK_VALUE(
        positions->dim() <= 2 &&
            (positions->dim() < 1 || positions->size(-1) == 1 ||
             positions->size(-1) == q.size(2)) &&
            (positions->dim() < 2 || positions->size(0) == 1 ||
             positions->size(0) == q.size(0)),
        "positions must broadcast to [B, N] = [", q.size(0), ", ", q.size(2),
        "], got ", positions->sizes());
  }
}

// Results follow their input's order of heads and tokens, by the rule of
// vectra::rbf_attention's output (torch_ext.cpp).
Tensor empty_like_heads(const Tensor& t) {
  const int64_t b = t.size(0), h = t.size(1), n = t.size(2), d = t.size(3);
  if (h > 1 && n > 1 && t.stride(2) > t.stride(1))
    return at::empty_strided({b, h, n, d}, {n * h * d, d, h * d, 1},
                             t.options());
  return at::empty({b, h, n, d}, t.options());
}

vectra_qk_args describe_qk(const Tensor& q, const Tensor& k,
                           const Tensor& cos, const Tensor& sin,
                           const OptTensor& qw, const OptTensor& kw,
                           const OptTensor& positions, double eps,
                           bool interleaved) {
  vectra_qk_args a{};
  a.q = describe(q);
  a.k = describe(k);
  a.cos = describe(cos);
  a.sin = describe(sin);
  a.q_weight = describe(qw);
  a.k_weight = describe(kw);
  a.eps = eps;
  a.interleaved = interleaved;
  if (has(positions) && positions->numel() > 0) {
    const Tensor& p = *positions;
    a.positions = p.data_ptr();
    a.position_bytes = int32_t(p.element_size());
    if (p.dim() == 2 && p.size(0) > 1) a.position_stride[0] = p.stride(0);
    if (p.dim() >= 1 && p.size(-1) > 1) a.position_stride[1] = p.stride(-1);
  }
  return a;
}

std::tuple<Tensor, Tensor> qk_cuda(const Tensor& q, const Tensor& k,
                                   const Tensor& cos, const Tensor& sin,
                                   const OptTensor& qw, const OptTensor& kw,
                                   const OptTensor& positions, double eps,
                                   bool interleaved) {
  check_qk(q, k, cos, sin, qw, kw, positions);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor qo = empty_like_heads(q), ko = empty_like_heads(k);
  vectra_qk_args a =
      describe_qk(q, k, cos, sin, qw, kw, positions, eps, interleaved);
  a.q_out = describe(qo);
  a.k_out = describe(ko);
  const int st = vectra_qk_norm_rope_forward(
      &a, at::cuda::getCurrentCUDAStream(q.device().index()).stream());
  if (st != VECTRA_OK) raise_status("qk_norm_rope", st);
  return {qo, ko};
}

using Grads4 = std::tuple<Tensor, Tensor, Tensor, Tensor>;

void check_qk_grad(const Tensor& dq, const Tensor& dk, const Tensor& q,
                   const Tensor& k) {
  check_like(dq, "dq", q);
  check_like(dk, "dk", q);
  check_sizes(dq, "dq", q.sizes());
  check_sizes(dk, "dk", k.sizes());
}

Grads4 qk_backward_cuda(const Tensor& dq_out, const Tensor& dk_out,
                        const Tensor& q, const Tensor& k, const Tensor& cos,
                        const Tensor& sin, const OptTensor& qw,
                        const OptTensor& kw, const OptTensor& positions,
                        double eps, bool interleaved, bool need_dw) {
  check_qk(q, k, cos, sin, qw, kw, positions);
  check_qk_grad(dq_out, dk_out, q, k);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor dq = empty_like_heads(q), dk = empty_like_heads(k);
  const auto weight = [&](const OptTensor& w) {
    return has(w) && need_dw ? at::empty_like(*w, at::MemoryFormat::Contiguous)
                             : at::empty({0}, q.options());
  };
  Tensor dqw = weight(qw), dkw = weight(kw);
  vectra_qk_grad_args a{};
  a.fwd = describe_qk(q, k, cos, sin, qw, kw, positions, eps, interleaved);
  a.dq_out = describe(dq_out);
  a.dk_out = describe(dk_out);
  a.dq = describe(dq);
  a.dk = describe(dk);
  if (dqw.numel()) a.dq_weight = describe(dqw);
  if (dkw.numel()) a.dk_weight = describe(dkw);
  call_with_workspace("qk_norm_rope_backward", a, q,
                      vectra_qk_norm_rope_backward_workspace_bytes,
                      vectra_qk_norm_rope_backward);
  return {dq, dk, dqw, dkw};
}

// [B, 1, N, R / 2] rows of a table; rows outside it are NaN.
Tensor cpu_rows(const Tensor& table, const Tensor& pos) {
  const int64_t rows = table.size(0);
  const Tensor inside = (pos >= 0).logical_and(pos < rows);
  Tensor got =
      rows > 0
          ? table.index({pos.clamp(0, rows - 1)})
          : at::zeros({pos.size(0), pos.size(1), table.size(1)},
                      table.options());
  return at::where(inside.unsqueeze(-1), got,
                   at::full({}, std::nan(""), table.options()))
      .unsqueeze(1);
}

Tensor cpu_turn(const Tensor& x, const Tensor& c, const Tensor& s,
                const Tensor& pos, int64_t table, bool interleaved) {
  const int64_t r2 = c.size(-1), d = x.size(-1);
  const Tensor head = x.narrow(-1, 0, 2 * r2);
  Tensor tail = x.narrow(-1, 2 * r2, d - 2 * r2);
  const Tensor inside = (pos >= 0).logical_and(pos < table)
                            .unsqueeze(1)
                            .unsqueeze(-1);
  tail = at::where(inside, tail, at::full({}, std::nan(""), x.options()));
  if (interleaved) {
    const Tensor p = head.unflatten(-1, {r2, 2});
    const Tensor a = p.select(-1, 0), b = p.select(-1, 1);
    return at::cat({at::stack({a * c - b * s, b * c + a * s}, -1).flatten(-2),
                    tail}, -1);
  }
  const Tensor a = head.narrow(-1, 0, r2), b = head.narrow(-1, r2, r2);
  return at::cat({a * c - b * s, b * c + a * s, tail}, -1);
}

Tensor cpu_positions(const OptTensor& positions, const Tensor& q) {
  const Tensor p = has(positions)
                       ? positions->to(at::kLong)
                       : at::arange(q.size(2), q.options().dtype(at::kLong));
  return p.expand({q.size(0), q.size(2)});
}

std::tuple<Tensor, Tensor> qk_cpu(const Tensor& q, const Tensor& k,
                                  const Tensor& cos, const Tensor& sin,
                                  const OptTensor& qw, const OptTensor& kw,
                                  const OptTensor& positions, double eps,
                                  bool interleaved) {
  check_qk(q, k, cos, sin, qw, kw, positions);
  TORCH_CHECK_NOT_IMPLEMENTED(q.size(3) <= 512,
                              "vectra_b200::qk_norm_rope: a head width above "
                              "512");
  const Tensor pos = cpu_positions(positions, q);
  const Tensor c = cpu_rows(cos, pos), s = cpu_rows(sin, pos);
  const auto side = [&](const Tensor& x, const OptTensor& w) {
    const Tensor v = f32(x);
    Tensor y = v * at::rsqrt(v.square().mean({-1}, true) + eps);
    if (has(w)) y = y * f32(*w);
    return empty_like_heads(x).copy_(
        cpu_turn(y, c, s, pos, cos.size(0), interleaved));
  };
  return {side(q, qw), side(k, kw)};
}

Grads4 qk_backward_cpu(const Tensor& dq_out, const Tensor& dk_out,
                       const Tensor& q, const Tensor& k, const Tensor& cos,
                       const Tensor& sin, const OptTensor& qw,
                       const OptTensor& kw, const OptTensor& positions,
                       double eps, bool interleaved, bool need_dw) {
  check_qk(q, k, cos, sin, qw, kw, positions);
  check_qk_grad(dq_out, dk_out, q, k);
  const Tensor pos = cpu_positions(positions, q);
  const Tensor c = cpu_rows(cos, pos), s = cpu_rows(sin, pos);
  const auto side = [&](const Tensor& dy, const Tensor& x,
                        const OptTensor& w) {
    const Tensor v = f32(x);
    const Tensor r = at::rsqrt(v.square().mean({-1}, true) + eps);
    const Tensor n = v * r;
    Tensor g = cpu_turn(f32(dy), c, -s, pos, cos.size(0), interleaved);
    Tensor dw = has(w) && need_dw
                    ? (g * n).sum(at::IntArrayRef{0, 1, 2})
                          .to(w->scalar_type())
                    : at::empty({0}, q.options());
    if (has(w)) g = g * f32(*w);
    const Tensor dx = r * (g - n * (g * n).mean({-1}, true));
    return std::make_pair(empty_like_heads(x).copy_(dx), dw);
  };
  const auto [dq, dqw] = side(dq_out, q, qw);
  const auto [dk, dkw] = side(dk_out, k, kw);
  return {dq, dk, dqw, dkw};
}

// ---------------------------------------------------------------------------
// Dispatcher calls and autograd.
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor> call_linear(const Tensor& x, const Tensor& w,
                                       const OptTensor& bias,
                                       const OptTensor& residual,
                                       const std::string& activation,
                                       bool want_pre) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::linear_with_pre", "")
          .typed<std::tuple<Tensor, Tensor>(
              const Tensor&, const Tensor&, const OptTensor&,
              const OptTensor&, c10::string_view, bool)>();
  return op.call(x, w, bias, residual, activation, want_pre);
}

Grads3 call_linear_backward(const Tensor& dy, const Tensor& x,
                            const Tensor& w, const Tensor& pre,
                            const std::string& activation, bool need_dx,
                            bool need_dw, bool need_db) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::linear_backward", "")
          .typed<Grads3(const Tensor&, const Tensor&, const Tensor&,
                        const Tensor&, c10::string_view, bool, bool,
                        bool)>();
  return op.call(dy, x, w, pre, activation, need_dx, need_dw, need_db);
}

Grads3 call_gated(const Tensor& x, const Tensor& wg, const Tensor& wu,
                  const OptTensor& bg, const OptTensor& bu,
                  const std::string& activation, bool want_pre) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::gated_linear_with_pre", "")
          .typed<Grads3(const Tensor&, const Tensor&, const Tensor&,
                        const OptTensor&, const OptTensor&, c10::string_view,
                        bool)>();
  return op.call(x, wg, wu, bg, bu, activation, want_pre);
}

Grads3 call_gated_backward(const Tensor& dh, const Tensor& x,
                           const Tensor& wg, const Tensor& wu,
                           const OptTensor& bg, const OptTensor& bu,
                           const Tensor& gate, const Tensor& up,
                           const std::string& activation, bool need_dx,
                           bool need_dw, bool need_db) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::gated_linear_backward", "")
          .typed<Grads3(const Tensor&, const Tensor&, const Tensor&,
                        const Tensor&, const OptTensor&, const OptTensor&,
                        const Tensor&, const Tensor&, c10::string_view, bool,
                        bool, bool)>();
  return op.call(dh, x, wg, wu, bg, bu, gate, up, activation, need_dx,
                 need_dw, need_db);
}

std::tuple<Tensor, Tensor> call_qk(const Tensor& q, const Tensor& k,
                                   const Tensor& cos, const Tensor& sin,
                                   const OptTensor& qw, const OptTensor& kw,
                                   const OptTensor& positions, double eps,
                                   bool interleaved) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::qk_norm_rope", "")
          .typed<std::tuple<Tensor, Tensor>(
              const Tensor&, const Tensor&, const Tensor&, const Tensor&,
              const OptTensor&, const OptTensor&, const OptTensor&, double,
              bool)>();
  return op.call(q, k, cos, sin, qw, kw, positions, eps, interleaved);
}

Grads4 call_qk_backward(const Tensor& dq, const Tensor& dk, const Tensor& q,
                        const Tensor& k, const Tensor& cos,
                        const Tensor& sin, const OptTensor& qw,
                        const OptTensor& kw, const OptTensor& positions,
                        double eps, bool interleaved, bool need_dw) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::qk_norm_rope_backward", "")
          .typed<Grads4(const Tensor&, const Tensor&, const Tensor&,
                        const Tensor&, const Tensor&, const Tensor&,
                        const OptTensor&, const OptTensor&, const OptTensor&,
                        double, bool, bool)>();
  return op.call(dq, dk, q, k, cos, sin, qw, kw, positions, eps, interleaved,
                 need_dw);
}

// On CPU the plain entry points are the with_pre operators without the extra
// results.
Tensor linear_only_cpu(const Tensor& x, const Tensor& w, const OptTensor& bias,
                    const OptTensor& residual, c10::string_view activation) {
  return std::get<0>(linear_cpu(x, w, bias, residual,
                                std::string(activation), false));
}
Tensor gated_only_cpu(const Tensor& x, const Tensor& wg, const Tensor& wu,
                   const OptTensor& bg, const OptTensor& bu,
                   c10::string_view activation) {
  return std::get<0>(
      gated_cpu(x, wg, wu, bg, bu, std::string(activation), false));
}

// The entry points below autograd.
Tensor linear_below(const Tensor& x, const Tensor& w, const OptTensor& bias,
                    const OptTensor& residual, c10::string_view activation) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::linear", "")
          .typed<Tensor(const Tensor&, const Tensor&, const OptTensor&,
                        const OptTensor&, c10::string_view)>();
  return op.call(x, w, bias, residual, activation);
}
Tensor gated_below(const Tensor& x, const Tensor& wg, const Tensor& wu,
                   const OptTensor& bg, const OptTensor& bu,
                   c10::string_view activation) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra_b200::gated_linear", "")
          .typed<Tensor(const Tensor&, const Tensor&, const Tensor&,
                        const OptTensor&, const OptTensor&,
                        c10::string_view)>();
  return op.call(x, wg, wu, bg, bu, activation);
}

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return has(t) && t->requires_grad(); }

bool has_tangent(const Tensor& t) {
  return t.defined() && t._fw_grad(/*level=*/0).defined();
}
bool has_tangent(const OptTensor& t) { return has(t) && has_tangent(*t); }

// The operators have no forward-mode formula; below autograd a tangent would
// be dropped, which reads as zero.
template <typename... Args>
void refuse_tangents(const char* op, const Args&... args) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !(has_tangent(args) || ...), "vectra_b200::", op,
      ": forward-mode differentiation is not implemented");
}

OptTensor optional(const Tensor& t) {
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

// What a backward pass has to know, in one number: which inputs want a
// gradient, and the activation.
int64_t pack_call(const std::string& activation,
                  std::initializer_list<bool> wants) {
  int64_t packed = int64_t(activation_of(activation)) << 8;
  int i = 0;
  for (const bool w : wants) packed |= int64_t(w) << i++;
  return packed;
}
const char* activation_name(int64_t activation) {
  static const char* const names[] = {"none", "relu", "gelu", "gelu_tanh",
                                      "silu"};
  return names[activation];
}

// What stands for an input that the backward pass reads the shape of only:
// one element, expanded. Saving the input itself would keep its memory and
// forbid writing it in place.
Tensor shape_of(const Tensor& t) {
  return at::empty({1}, t.options()).expand_symint(t.sym_sizes());
}

struct LinearFunction : public Function<LinearFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Tensor& w, const OptTensor& bias,
                        const OptTensor& residual,
                        const std::string& activation) {
    at::AutoDispatchBelowADInplaceOrView below;
    const bool layer =
        wants_grad(x) || wants_grad(w) || wants_grad(bias);
    auto [y, pre] = call_linear(x, w, bias, residual, activation,
                                layer && activation != "none");
    // dx reads the weight, dw reads x.
    ctx->save_for_backward({wants_grad(w) ? x : shape_of(x),
                            wants_grad(x) ? w : shape_of(w), pre});
    ctx->saved_data["call"] = pack_call(
        activation, {wants_grad(x), wants_grad(w), wants_grad(bias),
                     wants_grad(residual)});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t packed = ctx->saved_data["call"].toInt();
    const bool dx = packed & 1, dw = packed & 2, db = packed & 4,
               dr = packed & 8;
    variable_list out(5);
    if (!grads[0].defined()) return out;
    if (dx || dw || db) {
      BelowUnlessRecording below;
      auto [gx, gw, gb] = call_linear_backward(
          grads[0], saved[0], saved[1], saved[2], activation_name(packed >> 8),
          dx, dw, db);
      if (dx) out[0] = gx;
      if (dw) out[1] = gw;
      if (db) out[2] = gb;
    }
    if (dr) out[3] = grads[0];
    return out;
  }
};

struct GatedFunction : public Function<GatedFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Tensor& wg, const Tensor& wu,
                        const OptTensor& bg, const OptTensor& bu,
                        const std::string& activation) {
    at::AutoDispatchBelowADInplaceOrView below;
    // Short reductions: the backward forms gate and up again.
    const bool sums = wants_grad(bg) || wants_grad(bu);
    const bool save = x.scalar_type() == at::kFloat ||
                      wg.size(1) > (sums ? VECTRA_GATED_RECOMPUTE_K_SUMS
                                         : VECTRA_GATED_RECOMPUTE_K);
    auto [h, gate, up] = call_gated(x, wg, wu, bg, bu, activation, save);
    if (save) {
      // dx reads the weights, dw reads x; the biases are in gate and up.
      const bool dw = wants_grad(wg) || wants_grad(wu), dx = wants_grad(x);
      ctx->save_for_backward({dw ? x : shape_of(x), dx ? wg : shape_of(wg),
                              dx ? wu : shape_of(wu), gate, up, Tensor(),
                              Tensor()});
    } else {
      ctx->save_for_backward({x, wg, wu, gate, up, bg.value_or(Tensor()),
                              bu.value_or(Tensor())});
    }
    ctx->saved_data["call"] = pack_call(
        activation, {wants_grad(x), wants_grad(wg), wants_grad(wu),
                     wants_grad(bg), wants_grad(bu)});
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const int64_t mask = ctx->saved_data["call"].toInt();
    variable_list out(6);
    if (!grads[0].defined()) return out;
    BelowUnlessRecording below;
    auto [dx, dw, db] = call_gated_backward(
        grads[0], s[0], s[1], s[2], optional(s[5]), optional(s[6]), s[3],
        s[4], activation_name(mask >> 8), (mask & 1) != 0, (mask & 6) != 0,
        (mask & 24) != 0);
    if (mask & 1) out[0] = dx;
    for (int i = 0; i < 2; ++i) {
      if (mask >> (1 + i) & 1) out[1 + i] = dw.select(0, i);
      if (mask >> (3 + i) & 1) out[3 + i] = db.select(0, i);
    }
    return out;
  }
};

struct QkFunction : public Function<QkFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q,
                               const Tensor& k, const Tensor& cos,
                               const Tensor& sin, const OptTensor& qw,
                               const OptTensor& kw,
                               const OptTensor& positions, double eps,
                               bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [qo, ko] =
        call_qk(q, k, cos, sin, qw, kw, positions, eps, interleaved);
    ctx->save_for_backward({q, k, cos, sin, qw.value_or(Tensor()),
                            kw.value_or(Tensor()),
                            positions.value_or(Tensor())});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["call"] =
        pack_call("none", {wants_grad(q), wants_grad(k), wants_grad(qw),
                           wants_grad(kw), interleaved});
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const int64_t packed = ctx->saved_data["call"].toInt();
    const bool dqw = packed & 4, dkw = packed & 8;
    variable_list out(9);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    BelowUnlessRecording below;
    // A result that nothing used has no gradient: its share is zero.
    const Tensor gq =
        grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
    const Tensor gk =
        grads[1].defined() ? grads[1] : at::zeros_like(s[1]);
    auto [dq, dk, gqw, gkw] = call_qk_backward(
        gq, gk, s[0], s[1], s[2], s[3], optional(s[4]), optional(s[5]),
        optional(s[6]), ctx->saved_data["eps"].toDouble(),
        (packed & 16) != 0, dqw || dkw);
    if (packed & 1) out[0] = dq;
    if (packed & 2) out[1] = dk;
    if (dqw) out[4] = gqw;
    if (dkw) out[5] = gkw;
    return out;
  }
};

Tensor linear_autograd(const Tensor& x, const Tensor& w,
                       const OptTensor& bias, const OptTensor& residual,
                       c10::string_view activation) {
  refuse_tangents("linear", x, w, bias, residual);
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(w) || wants_grad(bias) ||
       wants_grad(residual)))
    return LinearFunction::apply(x, w, bias, residual,
                                 std::string(activation));
  at::AutoDispatchBelowADInplaceOrView below;
  return linear_below(x, w, bias, residual, activation);
}

Tensor gated_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu,
                      const OptTensor& bg, const OptTensor& bu,
                      c10::string_view activation) {
  refuse_tangents("gated_linear", x, wg, wu, bg, bu);
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(wg) || wants_grad(wu) || wants_grad(bg) ||
       wants_grad(bu)))
    return GatedFunction::apply(x, wg, wu, bg, bu, std::string(activation));
  at::AutoDispatchBelowADInplaceOrView below;
  return gated_below(x, wg, wu, bg, bu, activation);
}

std::tuple<Tensor, Tensor> qk_autograd(
    const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin,
    const OptTensor& qw, const OptTensor& kw, const OptTensor& positions,
    double eps, bool interleaved) {
  refuse_tangents("qk_norm_rope", q, k, cos, sin, qw, kw);
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) ||
                                     wants_grad(qw) || wants_grad(kw))) {
    auto out = QkFunction::apply(q, k, cos, sin, qw, kw, positions, eps,
                                 interleaved);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_qk(q, k, cos, sin, qw, kw, positions, eps, interleaved);
}

// The implementations with the schema's string type.
template <auto F>
std::tuple<Tensor, Tensor> linear_impl(const Tensor& x, const Tensor& w,
                                       const OptTensor& bias,
                                       const OptTensor& residual,
                                       c10::string_view activation,
                                       bool want_pre) {
  return F(x, w, bias, residual, std::string(activation), want_pre);
}
template <auto F>
Grads3 linear_backward_impl(const Tensor& dy, const Tensor& x,
                            const Tensor& w, const Tensor& pre,
                            c10::string_view activation, bool need_dx,
                            bool need_dw, bool need_db) {
  return F(dy, x, w, pre, std::string(activation), need_dx, need_dw,
           need_db);
}
template <auto F>
Grads3 gated_impl(const Tensor& x, const Tensor& wg, const Tensor& wu,
                  const OptTensor& bg, const OptTensor& bu,
                  c10::string_view activation, bool want_pre) {
  return F(x, wg, wu, bg, bu, std::string(activation), want_pre);
}
template <auto F>
Grads3 gated_backward_impl(const Tensor& dh, const Tensor& x,
                           const Tensor& wg, const Tensor& wu,
                           const OptTensor& bg, const OptTensor& bu,
                           const Tensor& gate, const Tensor& up,
                           c10::string_view activation, bool need_dx,
                           bool need_dw, bool need_db) {
  return F(dh, x, wg, wu, bg, bu, gate, up, std::string(activation),
           need_dx, need_dw, need_db);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(vectra_b200, m) {
  m.def(
      "linear(Tensor x, Tensor weight, Tensor? bias=None, "
      "Tensor? residual=None, str activation='none') -> Tensor");
  m.def(
      "linear_with_pre(Tensor x, Tensor weight, Tensor? bias, "
      "Tensor? residual, str activation, bool want_pre) -> (Tensor, Tensor)");
  m.def(
      "linear_backward(Tensor dy, Tensor x, Tensor weight, Tensor pre, "
      "str activation, bool need_dx, bool need_dw, bool need_db) "
      "-> (Tensor, Tensor, Tensor)");
  m.def(
      "gated_linear(Tensor x, Tensor w_gate, Tensor w_up, "
      "Tensor? b_gate=None, Tensor? b_up=None, str activation='silu') "
      "-> Tensor");
  m.def(
      "gated_linear_with_pre(Tensor x, Tensor w_gate, Tensor w_up, "
      "Tensor? b_gate, Tensor? b_up, str activation, bool want_pre) "
      "-> (Tensor, Tensor, Tensor)");
  m.def(
      "gated_linear_backward(Tensor dh, Tensor x, Tensor w_gate, "
      "Tensor w_up, Tensor? b_gate, Tensor? b_up, Tensor gate, Tensor up, "
      "str activation, bool need_dx, bool need_dw, bool need_db) "
      "-> (Tensor, Tensor, Tensor)");
  m.def(
      "qk_norm_rope(Tensor q, Tensor k, Tensor cos, Tensor sin, "
      "Tensor? q_weight=None, Tensor? k_weight=None, "
      "Tensor? positions=None, float eps=1e-6, bool interleaved=False) "
      "-> (Tensor, Tensor)");
  m.def(
      "qk_norm_rope_backward(Tensor dq_out, Tensor dk_out, Tensor q, "
      "Tensor k, Tensor cos, Tensor sin, Tensor? q_weight, "
      "Tensor? k_weight, Tensor? positions, float eps, bool interleaved, "
      "bool need_dw) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(vectra_b200, CUDA, m) {
  m.impl("linear", &linear_only_cuda);
  m.impl("linear_with_pre", &linear_impl<linear_cuda>);
  m.impl("linear_backward", &linear_backward_impl<linear_backward_cuda>);
  m.impl("gated_linear", &gated_only_cuda);
  m.impl("gated_linear_with_pre", &gated_impl<gated_cuda>);
  m.impl("gated_linear_backward", &gated_backward_impl<gated_backward_cuda>);
  m.impl("qk_norm_rope", &qk_cuda);
  m.impl("qk_norm_rope_backward", &qk_backward_cuda);
}

TORCH_LIBRARY_IMPL(vectra_b200, CPU, m) {
  m.impl("linear", &linear_only_cpu);
  m.impl("linear_with_pre", &linear_impl<linear_cpu>);
  m.impl("linear_backward", &linear_backward_impl<linear_backward_cpu>);
  m.impl("gated_linear", &gated_only_cpu);
  m.impl("gated_linear_with_pre", &gated_impl<gated_cpu>);
  m.impl("gated_linear_backward", &gated_backward_impl<gated_backward_cpu>);
  m.impl("qk_norm_rope", &qk_cpu);
  m.impl("qk_norm_rope_backward", &qk_backward_cpu);
}

TORCH_LIBRARY_IMPL(vectra_b200, Autograd, m) {
  m.impl("linear", &linear_autograd);
  m.impl("gated_linear", &gated_autograd);
  m.impl("qk_norm_rope", &qk_autograd);
  for (const char* op :
       {"linear_with_pre", "linear_backward", "gated_linear_with_pre",
        "gated_linear_backward", "qk_norm_rope_backward"})
    m.impl(op, torch::autograd::autogradNotImplementedFallback());
}
