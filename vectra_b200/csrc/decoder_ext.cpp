// decoder_ext.cpp: PyTorch registration of the operators that complete a
// decoder block (include/vectra_block.h) in the vectra_b200 namespace:
//
//   dropout, residual_norm, cross_attention   differentiable entry points
//   residual_norm_with_stats,
//   cross_attention_with_lse                  the forward that also returns
//                                             what the backward needs
//   residual_norm_backward,
//   cross_attention_backward                  gradients
//
// by the rules of block_ext.cpp: CUDA tensors run the kernels on the current
// stream, CPU tensors an ATen formulation in float32, and the backward
// operators are not differentiable again. Fake implementations are in
// vectra_b200/block.py.
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>

#include <cmath>
#include <limits>
#include <tuple>
#include <vector>

#include "block_ext.h"
#include "philox.cuh"

namespace {

using namespace vectra_ext;

// ---------------------------------------------------------------------------
// Dropout.
// ---------------------------------------------------------------------------
void check_drop(const Tensor& x, double p, const OptTensor& rng) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must be from 0 to 1, got ", p);
  TORCH_CHECK_VALUE(p == 0.0 || has(rng), "dropout needs rng");
  if (has(rng))
    TORCH_CHECK_VALUE(rng->device() == x.device() &&
                          rng->scalar_type() == at::kLong &&
                          rng->dim() == 1 && rng->size(0) == 2 &&
                          rng->stride(0) == 1,
                      "rng must be a contiguous int64 tensor (seed, step) on ",
                      x.device());
}

vectra_drop describe_drop(double p, const OptTensor& rng, int64_t stream) {
  vectra_drop d{};
  d.p = p;
  d.rng = p > 0.0 ? rng->const_data_ptr<int64_t>() : nullptr;
  d.stream = uint32_t(stream);
  return d;
}

void check_io(const Tensor& x) {
  TORCH_CHECK_VALUE(io_dtype(x.scalar_type()),
                    "x must be float32, float16 or bfloat16, got ",
                    x.scalar_type());
}

Tensor dropout_cuda(const Tensor& x, double p, const OptTensor& rng,
                    int64_t stream) {
  check_io(x);
  check_drop(x, p, rng);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return y;
  Tensor copy;
  vectra_dropout_args a{};
  a.x = describe_rows(x.dim() ? x : x.view({1}), &copy);
  a.y = a.x;
  a.y.data = y.data_ptr();
  a.y.stride[0] = a.y.size[1];
  a.y.stride[1] = 1;
  a.drop = describe_drop(p, rng, stream);
  const int st = vectra_dropout(
      &a, at::cuda::getCurrentCUDAStream(x.device().index()).stream());
  if (st != VECTRA_OK) raise_status("dropout", st);
  return y;
}

// Which elements of a tensor of these sizes are kept.
Tensor cpu_keep(at::IntArrayRef sizes, const vectra::Drop& d) {
  Tensor keep = at::empty(sizes, at::kBool);
  bool* out = keep.data_ptr<bool>();
  const int64_t n = keep.numel();
  const uint64_t seed = uint64_t(d.rng[0]);
  const vectra::PhiloxKey key{uint32_t(seed), uint32_t(seed >> 32),
                              uint32_t(uint64_t(d.rng[1])), d.stream};
  for (int64_t g = 0; 8 * g < n; ++g) {
    const uint32_t bits = vectra::keep_bits(key, uint64_t(g), d.cut);
    for (int i = 0; i < 8 && 8 * g + i < n; ++i)
      out[8 * g + i] = bits >> i & 1;
  }
  return keep;
}

// dropout(x) in float32.
Tensor cpu_drop(const Tensor& x, const vectra_drop& drop) {
  if (drop.p == 0.0) return x;
  const vectra::Drop d = vectra::make_drop(drop);
  return at::where(cpu_keep(x.sizes(), d), x * d.scale,
                   at::zeros({}, x.options()));
}

Tensor dropout_cpu(const Tensor& x, double p, const OptTensor& rng,
                   int64_t stream) {
  check_io(x);
  check_drop(x, p, rng);
  return at::empty(x.sizes(), x.options())
      .copy_(cpu_drop(f32(x), describe_drop(p, rng, stream)));
}

// ---------------------------------------------------------------------------
// residual_norm
// ---------------------------------------------------------------------------
int32_t kind_of(c10::string_view kind) {
  if (kind == "rms") return VECTRA_NORM_RMS;
  if (kind == "layer") return VECTRA_NORM_LAYER;
  TORCH_CHECK_VALUE(false, "kind must be 'rms' or 'layer', got '",
                    std::string(kind), "'");
}

// The operator's scalar arguments.
struct NormCall {
  double residual_scale, p;
  OptTensor rng;
  int64_t stream;
  double eps;
  int32_t kind;
};

// Rows of x that share a gate row: gate's leading sizes are x's up to some
// dimension and 1 from there on.
int64_t gate_rows(const Tensor& gate, at::IntArrayRef x) {
  const int64_t lead = int64_t(x.size()) - 1, own = gate.dim() - 1;
  const auto bad = [&] {
    TORCH_CHECK_VALUE(false, "gate must have x's last size, and before it "
                             "x's sizes up to some dimension and 1 behind "
                             "that; got ", gate.sizes(), " for ", x);
  };
  if (own < 0 || own > lead || gate.size(own) != x[size_t(lead)]) bad();
  int64_t rows = 1;
  bool shared = true;  // every size so far, from the last, was 1
  for (int64_t i = lead - 1; i >= 0; --i) {
    const int64_t at = i - (lead - own);
    const int64_t g = at >= 0 ? gate.size(at) : 1, n = x[size_t(i)];
    if (shared && g == 1) {
      rows *= n;
    } else if (g == n) {
      shared = false;
    } else {
      bad();
    }
  }
  return rows;
}

void check_norm(const Tensor& x, const OptTensor& branch,
                const OptTensor& weight, const OptTensor& bias,
                const OptTensor& branch_weight, const OptTensor& gate,
                const NormCall& call, bool norm) {
  check_io(x);
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must be [..., C]");
  TORCH_CHECK_NOT_IMPLEMENTED(x.size(-1) <= 16384,
                              "vectra_b200::residual_norm: rows above 16384");
  check_drop(x, call.p, call.rng);
  if (has(branch)) {
    check_like(*branch, "branch", x);
    check_sizes(*branch, "branch", x.sizes());
  } else {
    TORCH_CHECK_VALUE(norm, "without a branch there is only the norm");
    TORCH_CHECK_VALUE(!has(branch_weight) && !has(gate) && call.p == 0.0 &&
                          call.residual_scale == 1.0,
                      "branch_weight, gate, p and residual_scale need a "
                      "branch");
  }
  TORCH_CHECK_VALUE(norm || (!has(weight) && !has(bias)),
                    "weight and bias need the norm");
  const std::pair<const OptTensor*, const char*> vectors[3] = {
      {&weight, "weight"}, {&bias, "bias"}, {&branch_weight, "branch_weight"}};
  for (const auto& [t, name] : vectors) {
    if (!has(*t)) continue;
    check_like(**t, name, x);
    check_sizes(**t, name, {x.size(-1)});
  }
  if (has(gate)) {
    check_like(*gate, "gate", x);
    gate_rows(*gate, x.sizes());
  }
}

// gate as [G, C].
Tensor gate_matrix(const Tensor& gate) {
  return gate.dim() == 1 ? gate.unsqueeze(0) : as_rows(gate);
}

vectra_residual_norm_args describe_norm(const NormCall& call) {
  vectra_residual_norm_args a{};
  a.drop = describe_drop(call.p, call.rng, call.stream);
  a.residual_scale = call.residual_scale;
  a.eps = call.eps;
  a.kind = call.kind;
  return a;
}

using Three = std::tuple<Tensor, Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;
using Six = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

// What a 16-bit value's rounding left is kept times this (block_common.cuh).
double rest_lift(const Tensor& t) {
  return t.scalar_type() == at::kHalf ? 2048.0 : 1.0;
}

// What x_out's rounding leaves, for the backward pass of the norm behind.
Tensor rest_of_sum(const Tensor& x, bool branched, bool norm, bool want) {
  const bool kept =
      want && branched && norm && x.scalar_type() != at::kFloat;
  return kept ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options());
}

// `only`: x_out and y alone; the others stay undefined.
Four norm_cuda(const Tensor& x, const OptTensor& branch,
               const OptTensor& weight, const OptTensor& bias,
               const OptTensor& branch_weight, const OptTensor& gate,
               const NormCall& call, bool norm, bool want_stats, bool only) {
  check_norm(x, branch, weight, bias, branch_weight, gate, call, norm);
  c10::cuda::CUDAGuard guard(x.device());
  const auto none = [&] { return at::empty({0}, x.options()); };
  const int64_t c = x.size(-1), rows = c > 0 ? x.numel() / c : 0;
  Tensor x_out = has(branch) ? at::empty(x.sizes(), x.options()) : none();
  Tensor y = norm ? at::empty(x.sizes(), x.options()) : none();
  Tensor stats, rest;
  if (!only) {
    stats = at::empty({want_stats ? rows : 0, 4},
                      x.options().dtype(at::kFloat));
    rest = rest_of_sum(x, has(branch), norm, want_stats);
  }
  if (x.numel() == 0) return {x_out, y, stats, rest};
  vectra_residual_norm_train_args train{};
  train.fwd = describe_norm(call);
  if (!only && rest.numel()) train.rest = describe_rows(rest, nullptr);
  vectra_residual_norm_args& a = train.fwd;
  Tensor x_copy, branch_copy, gate_copy;
  a.x = describe_rows(x, &x_copy);
  if (has(branch)) {
    a.branch = describe_rows(*branch, &branch_copy);
    a.x_out = describe_rows(x_out, nullptr);
  }
  a.weight = describe(weight);
  a.bias = describe(bias);
  a.branch_weight = describe(branch_weight);
  if (has(gate)) {
    gate_copy = gate_matrix(*gate);
    a.gate = describe(gate_copy);
  }
  if (norm) a.y = describe_rows(y, nullptr);
  if (want_stats) a.stats = describe(stats);
  const int st = vectra_residual_norm_forward_train(
      &train, at::cuda::getCurrentCUDAStream(x.device().index()).stream());
  if (st != VECTRA_OK) raise_status("residual_norm", st);
  return {x_out, y, stats, rest};
}

// The gradients that a backward pass is to form, as bits.
enum Need { kDx = 1, kDbranch = 2, kDweight = 4, kDbias = 8,
            kDbranchWeight = 16, kDgate = 32 };

// What the gradients are shaped like, and the pass has checked: one of the
// upstream gradients is there.
const Tensor& upstream(const OptTensor& dx_out, const OptTensor& dy) {
  TORCH_CHECK_VALUE(has(dx_out) || has(dy), "dx_out or dy must be given");
  return has(dy) ? *dy : *dx_out;
}

void check_norm_grad(const OptTensor& dx_out, const OptTensor& dy,
                     const Tensor& x_out, const Tensor& rest,
                     const Tensor& stats,
                     const OptTensor& branch, const OptTensor& weight,
                     const OptTensor& branch_weight, const OptTensor& gate,
                     const NormCall& call, int64_t need) {
  const Tensor& g = upstream(dx_out, dy);
  check_norm(g, g, has(dy) ? weight : OptTensor(), {}, branch_weight, gate,
             call, has(dy));
  if (has(dx_out)) {
    check_like(*dx_out, "dx_out", g);
    check_sizes(*dx_out, "dx_out", g.sizes());
  }
  if (has(dy)) {
    check_like(x_out, "x_out", g);
    check_sizes(x_out, "x_out", g.sizes());
    if (rest.numel()) {
      check_like(rest, "rest", g);
      check_sizes(rest, "rest", g.sizes());
      TORCH_CHECK_VALUE(rest.is_contiguous() && g.scalar_type() != at::kFloat,
                        "rest must be the forward's");
    }
  }
  if (has(dy) || has(branch_weight)) {
    const int64_t c = g.size(-1);
    TORCH_CHECK_VALUE(stats.device() == g.device() &&
                          stats.scalar_type() == at::kFloat &&
                          stats.is_contiguous(),
                      "stats must be the forward's");
    check_sizes(stats, "stats", {c > 0 ? g.numel() / c : 0, 4});
  }
  TORCH_CHECK_VALUE(has(dy) || !(need & (kDweight | kDbias)),
                    "weight and bias have no gradient without dy");
  TORCH_CHECK_VALUE(!(need & kDbranchWeight) || has(branch_weight),
                    "dbranch_weight needs branch_weight");
  TORCH_CHECK_VALUE(!(need & kDgate) || has(gate), "dgate needs gate");
  if (has(branch_weight) || (need & kDgate)) {
    TORCH_CHECK_VALUE(has(branch), "branch must be given");
    check_like(*branch, "branch", g);
    check_sizes(*branch, "branch", g.sizes());
  }
}

Six norm_backward_cuda(const OptTensor& dx_out, const OptTensor& dy,
                       const Tensor& x_out, const Tensor& rest,
                       const Tensor& stats,
                       const OptTensor& branch, const OptTensor& weight,
                       const OptTensor& branch_weight, const OptTensor& gate,
                       const NormCall& call, int64_t need) {
  check_norm_grad(dx_out, dy, x_out, rest, stats, branch, weight,
                  branch_weight, gate, call, need);
  const Tensor& g = upstream(dx_out, dy);
  c10::cuda::CUDAGuard guard(g.device());
  const int64_t c = g.size(-1);
  const auto result = [&](int64_t bit, at::IntArrayRef sizes) {
    return need & bit ? at::empty(sizes, g.options())
                      : at::empty({0}, g.options());
  };
  Tensor dx = result(kDx, g.sizes()), dbranch = result(kDbranch, g.sizes());
  Tensor dweight = result(kDweight, {c}), dbias = result(kDbias, {c});
  Tensor dbw = result(kDbranchWeight, {c});
  Tensor dgate = need & kDgate ? at::empty(gate->sizes(), g.options())
                               : at::empty({0}, g.options());
  if (g.numel() == 0) {
    for (Tensor* t : {&dweight, &dbias, &dbw, &dgate}) t->zero_();
    return {dx, dbranch, dweight, dbias, dbw, dgate};
  }
  // The workspace is the grad part's.
  struct Args : vectra_residual_norm_train_grad_args {
    void*& workspace = grad.workspace;
    size_t& workspace_bytes = grad.workspace_bytes;
  } train{};
  vectra_residual_norm_grad_args& a = train.grad;
  a.fwd = describe_norm(call);
  Tensor copies[5], gate_copy;
  if (has(dx_out)) a.dx_out = describe_rows(*dx_out, &copies[0]);
  if (has(dy)) {
    a.dy = describe_rows(*dy, &copies[1]);
    a.fwd.x_out = describe_rows(x_out, &copies[2]);
    if (rest.numel()) train.rest = describe_rows(rest, nullptr);
    a.fwd.weight = describe(weight);
  }
  if (has(branch)) a.fwd.branch = describe_rows(*branch, &copies[3]);
  if (has(dy) || has(branch_weight)) a.fwd.stats = describe(stats);
  a.fwd.branch_weight = describe(branch_weight);
  if (has(gate)) {
    gate_copy = gate_matrix(*gate);
    a.fwd.gate = describe(gate_copy);
  }
  if (need & kDx) a.dx = describe_rows(dx, nullptr);
  if (need & kDbranch) a.dbranch = describe_rows(dbranch, nullptr);
  if (need & kDweight) a.dweight = describe(dweight);
  if (need & kDbias) a.dbias = describe(dbias);
  if (need & kDbranchWeight) a.dbranch_weight = describe(dbw);
  if (need & kDgate) {
    a.dgate = a.fwd.gate;
    a.dgate.data = dgate.data_ptr();
    a.dgate.stride[0] = c;
    a.dgate.stride[1] = 1;
  }
  call_with_workspace("residual_norm_backward", train, g,
                      vectra_residual_norm_backward_train_workspace_bytes,
                      vectra_residual_norm_backward_train);
  return {dx, dbranch, dweight, dbias, dbw, dgate};
}

// (mean, factor) of every row, [..., 1] each; the mean is 0 for 'rms'.
std::pair<Tensor, Tensor> cpu_row_norm(const Tensor& v, const NormCall& call) {
  Tensor mean = call.kind == VECTRA_NORM_LAYER
                    ? v.mean({-1}, true)
                    : at::zeros({1}, v.options());
  Tensor r = at::rsqrt((v - mean).square().mean({-1}, true) + call.eps);
  return {mean.expand(r.sizes()), r};
}

Four norm_cpu(const Tensor& x, const OptTensor& branch,
              const OptTensor& weight, const OptTensor& bias,
              const OptTensor& branch_weight, const OptTensor& gate,
              const NormCall& call, bool norm, bool want_stats, bool /*only*/) {
  check_norm(x, branch, weight, bias, branch_weight, gate, call, norm);
  const int64_t c = x.size(-1), rows = c > 0 ? x.numel() / c : 0;
  const auto none = [&] { return at::empty({0}, x.options()); };
  Tensor stats = at::zeros({want_stats ? rows : 0, 4}, at::kFloat);
  Tensor v = f32(x), x_out = none(), y = none();
  Tensor rest = rest_of_sum(x, has(branch), norm, want_stats);
  const auto keep = [&](int64_t at, const std::pair<Tensor, Tensor>& n) {
    if (!want_stats) return;
    stats.select(1, at).copy_(n.first.reshape({rows}));
    stats.select(1, at + 1).copy_(n.second.reshape({rows}));
  };
  if (has(branch)) {
    Tensor u = f32(*branch);
    if (has(branch_weight)) {
      const auto n = cpu_row_norm(u, call);
      keep(2, n);
      u = (u - n.first) * n.second * f32(*branch_weight);
    }
    u = cpu_drop(u, describe_drop(call.p, call.rng, call.stream));
    if (has(gate)) u = u * f32(*gate);
    v = v * call.residual_scale + u;
    x_out = at::empty(x.sizes(), x.options()).copy_(v);
    if (rest.numel()) rest.copy_((v - f32(x_out)) * rest_lift(x));
  }
  if (norm) {
    const auto n = cpu_row_norm(v, call);
    keep(0, n);
    v = (v - n.first) * n.second;
    if (has(weight)) v = v * f32(*weight);
    if (has(bias)) v = v + f32(*bias);
    y = at::empty(x.sizes(), x.options()).copy_(v);
  }
  return {x_out, y, stats, rest};
}

Six norm_backward_cpu(const OptTensor& dx_out, const OptTensor& dy,
                      const Tensor& x_out, const Tensor& rest,
                      const Tensor& stats,
                      const OptTensor& branch, const OptTensor& weight,
                      const OptTensor& branch_weight, const OptTensor& gate,
                      const NormCall& call, int64_t need) {
  check_norm_grad(dx_out, dy, x_out, rest, stats, branch, weight,
                  branch_weight, gate, call, need);
  const Tensor& like = upstream(dx_out, dy);
  const int64_t c = like.size(-1), rows = c > 0 ? like.numel() / c : 0;
  const at::ScalarType dt = like.scalar_type();
  const auto none = [&] { return at::empty({0}, like.options()); };
  const auto flat = [&](const Tensor& t) {
    return f32(t).reshape({rows, c});
  };
  // The gradient of normalised rows' argument.
  const auto back = [&](const Tensor& g, const Tensor& n, const Tensor& r) {
    Tensor d = g - n * (g * n).mean({-1}, true);
    if (call.kind == VECTRA_NORM_LAYER) d = d - g.mean({-1}, true);
    return d * r;
  };
  const auto column = [&](int64_t at) {
    return stats.select(1, at).unsqueeze(1);
  };
  Tensor g = has(dx_out) ? flat(*dx_out) : at::zeros({rows, c}, at::kFloat);
  Tensor dweight = none(), dbias = none(), dbw = none(), dgate = none();
  if (has(dy)) {
    const Tensor f = flat(*dy), r = column(1);
    Tensor v = flat(x_out);
    if (rest.numel()) v = v + flat(rest) / rest_lift(rest);
    const Tensor n = (v - column(0)) * r;
    if (need & kDweight) dweight = (f * n).sum(0).to(dt);
    if (need & kDbias) dbias = f.sum(0).to(dt);
    g = g + back(has(weight) ? f * f32(*weight) : f, n, r);
  }
  Tensor dx = need & kDx
                  ? (g * call.residual_scale).to(dt).reshape(like.sizes())
                  : none();
  Tensor n0, r0, u;
  if (has(branch_weight) || (need & kDgate)) {
    u = flat(*branch);
    if (has(branch_weight)) {
      r0 = column(3);
      n0 = (u - column(2)) * r0;
      u = n0 * f32(*branch_weight);
    }
  }
  const vectra_drop drop = describe_drop(call.p, call.rng, call.stream);
  if (has(gate)) {
    const int64_t shared = gate_rows(*gate, like.sizes());
    const Tensor gm = f32(gate_matrix(*gate));
    if (need & kDgate)
      dgate = (g * cpu_drop(u, drop)).reshape({gm.size(0), shared, c}).sum(1)
                  .to(dt).reshape(gate->sizes());
    g = (g.reshape({gm.size(0), shared, c}) * gm.unsqueeze(1))
            .reshape({rows, c});
  }
  g = cpu_drop(g, drop);
  if (has(branch_weight)) {
    if (need & kDbranchWeight) dbw = (g * n0).sum(0).to(dt);
    g = back(g * f32(*branch_weight), n0, r0);
  }
  Tensor dbranch =
      need & kDbranch ? g.to(dt, false, true).reshape(like.sizes()) : none();
  return {dx, dbranch, dweight, dbias, dbw, dgate};
}

// ---------------------------------------------------------------------------
// cross_attention
// ---------------------------------------------------------------------------
void check_cross(const Tensor& q, const Tensor& k, const Tensor& v,
                 const Tensor& scale, const OptTensor& lengths) {
  TORCH_CHECK_VALUE(io_dtype(q.scalar_type()),
                    "q must be float32, float16 or bfloat16, got ",
                    q.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                    "q, k and v must be rank 4 ([B, H, N, D])");
  check_like(k, "k", q);
  check_like(v, "v", q);
  TORCH_CHECK_VALUE(k.size(0) == q.size(0) && k.size(3) == q.size(3),
                    "k ", k.sizes(), " must have q's batch and width, q ",
                    q.sizes());
  TORCH_CHECK_VALUE(v.size(0) == k.size(0) && v.size(1) == k.size(1) &&
                        v.size(2) == k.size(2),
                    "v ", v.sizes(), " must have k's batch, heads and length, "
                    "k ", k.sizes());
  TORCH_CHECK_VALUE(q.size(3) >= 1 && v.size(3) >= 1,
                    "head vectors must not be empty");
  TORCH_CHECK_NOT_IMPLEMENTED(q.size(3) <= 256 && v.size(3) <= 256,
                              "vectra_b200::cross_attention: a head width "
                              "above 256");
  TORCH_CHECK_VALUE(k.size(1) > 0 ? q.size(1) % k.size(1) == 0
                                  : q.size(1) == 0,
                    "q's ", q.size(1), " heads must be a multiple of k's ",
                    k.size(1));
  TORCH_CHECK_VALUE(scale.device() == q.device() &&
                        (io_dtype(scale.scalar_type()) ||
                         scale.scalar_type() == at::kDouble),
                    "scale must be a float tensor on ", q.device());
  const int64_t full[4] = {q.size(0), q.size(1), 1, 1};
  bool fits = scale.dim() <= 4;
  for (int64_t i = 0; fits && i < scale.dim(); ++i) {
    const int64_t n = scale.size(scale.dim() - 1 - i);
    fits = n == 1 || n == full[3 - i];
  }
  TORCH_CHECK_VALUE(fits, "scale must broadcast to [B, H, 1, 1] = [", full[0],
                    ", ", full[1], ", 1, 1], got ", scale.sizes());
  if (has(lengths))
    TORCH_CHECK_VALUE(lengths->device() == q.device() &&
                          (lengths->scalar_type() == at::kLong ||
                           lengths->scalar_type() == at::kInt) &&
                          lengths->dim() == 1 && lengths->size(0) == q.size(0),
                      "key_lengths must be int64 or int32 [B] = [", q.size(0),
                      "] on ", q.device());
}

Tensor rank4(const Tensor& t) {
  std::vector<int64_t> sizes(size_t(4 - t.dim()), 1);
  sizes.insert(sizes.end(), t.sizes().begin(), t.sizes().end());
  return t.reshape(sizes);
}

// [B, H, N, width], laid out as q's heads and tokens are.
Tensor heads_like(const Tensor& q, int64_t width) {
  const int64_t b = q.size(0), h = q.size(1), n = q.size(2);
  if (h > 1 && n > 1 && q.stride(2) > q.stride(1))
    return at::empty_strided({b, h, n, width}, {n * h * width, width,
                                                h * width, 1}, q.options());
  return at::empty({b, h, n, width}, q.options());
}

vectra_cross_args describe_cross(const Tensor& q, const Tensor& k,
                                 const Tensor& v, const Tensor& scale4,
                                 const OptTensor& lengths) {
  vectra_cross_args a{};
  a.q = describe(q);
  a.k = describe(k);
  a.v = describe(v);
  a.scale = describe(scale4);
  if (scale4.scalar_type() == at::kDouble) a.scale.dtype = VECTRA_F64;
  if (has(lengths) && lengths->numel() > 0) {
    a.key_lengths = lengths->data_ptr();
    a.length_bytes = int32_t(lengths->element_size());
    a.length_stride = lengths->size(0) > 1 ? lengths->stride(0) : 0;
  }
  return a;
}

// What out's rounding left, for the backward pass of 16-bit tensors.
Tensor rest_like(const Tensor& q, int64_t width, bool want) {
  if (!want || q.scalar_type() == at::kFloat) return at::empty({0}, q.options());
  return at::empty({q.size(0), q.size(1), q.size(2), width}, q.options());
}

Three cross_cuda(const Tensor& q, const Tensor& k, const Tensor& v,
                 const Tensor& scale, const OptTensor& lengths,
                 bool want_lse) {
  check_cross(q, k, v, scale, lengths);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = heads_like(q, v.size(3));
  Tensor rest = rest_like(q, v.size(3), want_lse);
  Tensor lse = want_lse ? at::empty({q.size(0), q.size(1), q.size(2)},
                                    q.options().dtype(at::kFloat))
                        : at::empty({0, q.size(1), q.size(2)},
                                    q.options().dtype(at::kFloat));
  if (out.numel() == 0) return {out, lse, rest};
  const Tensor s4 = rank4(scale);
  vectra_cross_args a = describe_cross(q, k, v, s4, lengths);
  a.out = describe(out);
  if (want_lse) a.lse = describe(lse);
  if (rest.numel()) a.rest = describe(rest);
  call_with_workspace("cross_attention", a, q,
                      vectra_cross_attention_forward_workspace_bytes,
                      vectra_cross_attention_forward);
  return {out, lse, rest};
}

void check_cross_grad(const Tensor& dout, const Tensor& q, const Tensor& v,
                      const Tensor& out, const Tensor& lse,
                      const Tensor& rest) {
  const std::vector<int64_t> sizes = {q.size(0), q.size(1), q.size(2),
                                      v.size(3)};
  check_like(dout, "dout", q);
  check_sizes(dout, "dout", sizes);
  check_like(out, "out", q);
  check_sizes(out, "out", sizes);
  TORCH_CHECK_VALUE(out.size(3) <= 1 || out.stride(3) == 1,
                    "out must be the forward's");
  TORCH_CHECK_VALUE(lse.device() == q.device() &&
                        lse.scalar_type() == at::kFloat &&
                        lse.is_contiguous(),
                    "lse must be the forward's");
  check_sizes(lse, "lse", {q.size(0), q.size(1), q.size(2)});
  if (q.scalar_type() != at::kFloat) {
    check_like(rest, "rest", q);
    check_sizes(rest, "rest", sizes);
    TORCH_CHECK_VALUE(rest.is_contiguous(), "rest must be the forward's");
  }
}

Four cross_backward_cuda(const Tensor& dout, const Tensor& q, const Tensor& k,
                         const Tensor& v, const Tensor& scale,
                         const OptTensor& lengths, const Tensor& out,
                         const Tensor& lse, const Tensor& rest, bool need_dq,
                         bool need_dkv, bool need_dscale) {
  check_cross(q, k, v, scale, lengths);
  check_cross_grad(dout, q, v, out, lse, rest);
  c10::cuda::CUDAGuard guard(q.device());
  const auto none = [&] { return at::empty({0}, q.options()); };
  Tensor dq = need_dq ? heads_like(q, q.size(3)) : none();
  Tensor dk = need_dkv ? heads_like(k, k.size(3)) : none();
  Tensor dv = need_dkv ? heads_like(v, v.size(3)) : none();
  Tensor dscale = at::empty({need_dscale ? q.size(0) : 0, q.size(1)},
                            q.options().dtype(at::kFloat));
  // Without queries or keys there is nothing to sum.
  if (q.numel() == 0 || k.numel() == 0) {
    for (Tensor* t : {&dq, &dk, &dv, &dscale}) t->zero_();
    return {dq, dk, dv, dscale};
  }
  const Tensor s4 = rank4(scale);
  // The 16-bit kernels read rows in 16-byte pieces: an upstream gradient that
  // has none (an expanded one) is packed.
  Tensor e = dout;
  if (q.scalar_type() != at::kFloat && dout.numel() > 0) {
    bool pieces = dout.stride(3) == 1 &&
                  reinterpret_cast<uintptr_t>(dout.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i)
      pieces = pieces && (dout.size(i) == 1 || dout.stride(i) % 8 == 0);
    if (!pieces) e = heads_like(q, v.size(3)).copy_(dout);
  }
  vectra_cross_grad_args a{};
  a.fwd = describe_cross(q, k, v, s4, lengths);
  a.fwd.out = describe(out);
  a.fwd.lse = describe(lse);
  if (rest.numel() && q.scalar_type() != at::kFloat) a.fwd.rest = describe(rest);
  a.dout = describe(e);
  if (need_dq) a.dq = describe(dq);
  if (need_dkv) {
    a.dk = describe(dk);
    a.dv = describe(dv);
  }
  if (need_dscale) a.dscale = describe(dscale);
  call_with_workspace("cross_attention_backward", a, q,
                      vectra_cross_attention_backward_workspace_bytes,
                      vectra_cross_attention_backward);
  return {dq, dk, dv, dscale};
}

// The operands in float32, [B, Hk, G, N, width] with G 1 for keys; unseen keys
// and values are zeros, and `seen` [B, 1, 1, 1, Nk] says which are not.
struct CpuCross {
  Tensor q, k, v, scale, seen, dist;
};
CpuCross cpu_cross(const Tensor& q, const Tensor& k, const Tensor& v,
                   const Tensor& scale, const OptTensor& lengths) {
  const int64_t b = q.size(0), h = q.size(1), hk = k.size(1), nk = k.size(2);
  const int64_t g = hk > 0 ? h / hk : 1;
  CpuCross t;
  t.seen = at::ones({b, 1, 1, 1, nk}, at::kBool);
  if (has(lengths))
    t.seen = at::arange(nk, at::kLong).lt(lengths->to(at::kLong).unsqueeze(1))
                 .reshape({b, 1, 1, 1, nk});
  const Tensor zero = at::zeros({}, at::kFloat);
  const Tensor rows = t.seen.reshape({b, 1, 1, nk, 1});
  t.q = f32(q).reshape({b, hk, g, q.size(2), q.size(3)});
  t.k = at::where(rows, f32(k).unsqueeze(2), zero);
  t.v = at::where(rows, f32(v).unsqueeze(2), zero);
  t.scale = f32(rank4(scale)).expand({b, h, 1, 1}).reshape({b, hk, g, 1, 1});
  // Distances from differences (mode 2), as the float32 kernels form them.
  t.dist = at::cdist(t.q, t.k.expand({b, hk, g, nk, k.size(3)}), 2.0, 2)
               .square();
  return t;
}

// What lse leaves out (include/vectra_block.h).
Tensor cpu_left_out(const CpuCross& t, const Tensor& q) {
  return q.scalar_type() == at::kFloat
             ? at::zeros({}, at::kFloat)
             : t.scale * t.q.square().sum({-1}, true) * 1.4426950408889634;
}

Three cross_cpu(const Tensor& q, const Tensor& k, const Tensor& v,
                const Tensor& scale, const OptTensor& lengths,
                bool want_lse) {
  check_cross(q, k, v, scale, lengths);
  const CpuCross t = cpu_cross(q, k, v, scale, lengths);
  Tensor out = heads_like(q, v.size(3));
  Tensor lse = at::full({want_lse ? q.size(0) : 0, q.size(1), q.size(2)},
                        std::numeric_limits<float>::infinity(), at::kFloat);
  Tensor rest = rest_like(q, v.size(3), want_lse);
  if (out.numel() == 0 || k.size(2) == 0) {
    out.zero_();
    rest.zero_();
    return {out, lse, rest};
  }
  const Tensor inf =
      at::full({}, -std::numeric_limits<float>::infinity(), at::kFloat);
  const Tensor s = at::where(t.seen, -t.scale * t.dist, inf);
  const Tensor any = t.seen.any(-1, true);
  const Tensor zero = at::zeros({}, at::kFloat);
  const Tensor o =
      at::where(any, at::matmul(at::softmax(s, -1), t.v), zero)
          .reshape(out.sizes());
  out.copy_(o);
  if (rest.numel()) rest.copy_((o - f32(out)) * rest_lift(q));
  if (want_lse)
    lse.copy_(at::where(any,
                        at::logsumexp(s, {-1}, true) * 1.4426950408889634 +
                            cpu_left_out(t, q),
                        -inf)
                  .reshape(lse.sizes()));
  return {out, lse, rest};
}

Four cross_backward_cpu(const Tensor& dout, const Tensor& q, const Tensor& k,
                        const Tensor& v, const Tensor& scale,
                        const OptTensor& lengths, const Tensor& out,
                        const Tensor& lse, const Tensor& rest, bool need_dq,
                        bool need_dkv, bool need_dscale) {
  check_cross(q, k, v, scale, lengths);
  check_cross_grad(dout, q, v, out, lse, rest);
  const auto none = [&] { return at::empty({0}, q.options()); };
  Tensor dq = need_dq ? heads_like(q, q.size(3)) : none();
  Tensor dk = need_dkv ? heads_like(k, k.size(3)) : none();
  Tensor dv = need_dkv ? heads_like(v, v.size(3)) : none();
  Tensor dscale = at::zeros({need_dscale ? q.size(0) : 0, q.size(1)},
                            at::kFloat);
  if (q.numel() == 0 || k.numel() == 0) {
    for (Tensor* t : {&dq, &dk, &dv}) t->zero_();
    return {dq, dk, dv, dscale};
  }
  const CpuCross t = cpu_cross(q, k, v, scale, lengths);
  const int64_t b = t.q.size(0), hk = t.q.size(1), g = t.q.size(2),
                nq = t.q.size(3);
  const Tensor e = f32(dout).reshape({b, hk, g, nq, v.size(3)});
  Tensor o = f32(out);
  if (q.scalar_type() != at::kFloat) o = o + f32(rest) / rest_lift(q);
  o = o.reshape(e.sizes());
  const Tensor zero = at::zeros({}, at::kFloat);
  const Tensor from =
      lse.reshape({b, hk, g, nq, 1}) - cpu_left_out(t, q);
  const Tensor w = at::where(
      t.seen,
      at::exp2(-t.scale * t.dist * 1.4426950408889634 - from), zero);
  Tensor z = at::where(
      t.seen,
      w * (at::matmul(e, t.v.transpose(-1, -2)) - (e * o).sum({-1}, true)),
      zero);
  if (need_dscale) {
    const Tensor near = t.dist - (w * t.dist).sum({-1}, true);
    dscale = -at::where(t.seen, z * near, zero)
                  .sum(at::IntArrayRef{3, 4})
                  .reshape({b, hk * g});
  }
  z = z * t.scale * 2;
  if (need_dq)
    dq.copy_((at::matmul(z, t.k) - t.q * z.sum({-1}, true))
                 .reshape(dq.sizes()));
  if (need_dkv) {
    const Tensor zt = z.transpose(-1, -2);
    dk.copy_((at::matmul(zt, t.q) - t.k * zt.sum({-1}, true)).sum(2));
    dv.copy_(at::matmul(w.transpose(-1, -2), e).sum(2));
  }
  return {dq, dk, dv, dscale};
}

// ---------------------------------------------------------------------------
// Dispatcher calls and autograd.
// ---------------------------------------------------------------------------
template <typename F>
auto find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

Tensor call_dropout(const Tensor& x, double p, const OptTensor& rng,
                    int64_t stream) {
  static const auto op =
      find_op<Tensor(const Tensor&, double, const OptTensor&, int64_t)>(
          "vectra_b200::dropout");
  return op.call(x, p, rng, stream);
}

// Saved inputs that may be missing.
Tensor or_undefined(const OptTensor& t) { return t.value_or(Tensor()); }
OptTensor optional(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}

struct DropoutFunction : public Function<DropoutFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p,
                        const OptTensor& rng, int64_t stream) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({or_undefined(rng)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["stream"] = stream;
    return call_dropout(x, p, rng, stream);
  }
  // Its own gradient: the same mask on the upstream one, and differentiable
  // again like it.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    out[0] = call_dropout(grads[0], ctx->saved_data["p"].toDouble(),
                          optional(s[0]),
                          ctx->saved_data["stream"].toInt());
    return out;
  }
};

Tensor dropout_autograd(const Tensor& x, double p, const OptTensor& rng,
                        int64_t stream) {
  refuse_tangents("dropout", x);
  if (at::GradMode::is_enabled() && wants_grad(x))
    return DropoutFunction::apply(x, p, rng, stream);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_dropout(x, p, rng, stream);
}

using NormOnlyOp = std::tuple<Tensor, Tensor>(
    const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
    const OptTensor&, const OptTensor&, double, double, const OptTensor&,
    int64_t, double, c10::string_view, bool);
using NormOp = Four(const Tensor&, const OptTensor&, const OptTensor&,
                     const OptTensor&, const OptTensor&, const OptTensor&,
                     double, double, const OptTensor&, int64_t, double,
                     c10::string_view, bool, bool);
using NormBackwardOp = Six(const OptTensor&, const OptTensor&, const Tensor&,
                           const Tensor&, const Tensor&, const OptTensor&,
                           const OptTensor&, const OptTensor&,
                           const OptTensor&, double, double, const OptTensor&,
                           int64_t, double, c10::string_view, int64_t);

struct NormFunction : public Function<NormFunction> {
  static variable_list forward(
      AutogradContext* ctx, const Tensor& x, const OptTensor& branch,
      const OptTensor& weight, const OptTensor& bias,
      const OptTensor& branch_weight, const OptTensor& gate,
      double residual_scale, double p, const OptTensor& rng, int64_t stream,
      double eps, const std::string& kind, bool norm) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op =
        find_op<NormOp>("vectra_b200::residual_norm_with_stats");
    auto [x_out, y, stats, rest] =
        op.call(x, branch, weight, bias, branch_weight, gate, residual_scale,
                p, rng, stream, eps, kind, norm, true);
    const bool branched = has(branch);
    // The branch is read again for its norm and for the gate's gradient.
    const bool keep = has(branch_weight) || wants_grad(gate);
    ctx->save_for_backward(
        {norm ? (branched ? x_out : x) : shape_of(x), rest, stats,
         branched && keep ? *branch : Tensor(), or_undefined(weight),
         or_undefined(branch_weight), or_undefined(gate), or_undefined(rng)});
    ctx->saved_data["residual_scale"] = residual_scale;
    ctx->saved_data["p"] = p;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["kind"] = kind;
    int64_t need = 0;
    const bool wants[6] = {wants_grad(x),    wants_grad(branch),
                           wants_grad(weight), wants_grad(bias),
                           wants_grad(branch_weight), wants_grad(gate)};
    for (int i = 0; i < 6; ++i) need |= int64_t(wants[i]) << i;
    ctx->saved_data["need"] = need;
    ctx->saved_data["outputs"] = int64_t(branched) | int64_t(norm) << 1;
    variable_list out;
    if (branched) out.push_back(x_out);
    if (norm) out.push_back(y);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const int64_t outputs = ctx->saved_data["outputs"].toInt();
    int64_t need = ctx->saved_data["need"].toInt();
    variable_list out(13);
    const Tensor dx_out = outputs & 1 ? grads[0] : Tensor();
    const Tensor dy = outputs & 2 ? grads[outputs & 1] : Tensor();
    if (!dx_out.defined() && !dy.defined()) return out;
    // A result that nothing used has no gradient, and its norm's parameters
    // have none.
    if (!dy.defined()) need &= ~int64_t(kDweight | kDbias);
    std::optional<at::AutoDispatchBelowADInplaceOrView> below;
    if (!at::GradMode::is_enabled()) below.emplace();
    static const auto op =
        find_op<NormBackwardOp>("vectra_b200::residual_norm_backward");
    auto [dx, dbranch, dweight, dbias, dbw, dgate] = op.call(
        optional(dx_out), optional(dy), s[0], s[1], s[2], optional(s[3]),
        optional(s[4]), optional(s[5]), optional(s[6]),
        ctx->saved_data["residual_scale"].toDouble(),
        ctx->saved_data["p"].toDouble(), optional(s[7]),
        ctx->saved_data["stream"].toInt(), ctx->saved_data["eps"].toDouble(),
        ctx->saved_data["kind"].toStringRef(), need);
    const Tensor results[6] = {dx, dbranch, dweight, dbias, dbw, dgate};
    for (int i = 0; i < 6; ++i)
      if (need >> i & 1) out[size_t(i)] = results[i];
    return out;
  }
};

std::tuple<Tensor, Tensor> norm_autograd(
    const Tensor& x, const OptTensor& branch, const OptTensor& weight,
    const OptTensor& bias, const OptTensor& branch_weight,
    const OptTensor& gate, double residual_scale, double p,
    const OptTensor& rng, int64_t stream, double eps, c10::string_view kind,
    bool norm) {
  refuse_tangents("residual_norm", x, branch, weight, bias, branch_weight,
                  gate);
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(branch) || wants_grad(weight) ||
       wants_grad(bias) || wants_grad(branch_weight) || wants_grad(gate))) {
    auto out = NormFunction::apply(x, branch, weight, bias, branch_weight,
                                   gate, residual_scale, p, rng, stream, eps,
                                   std::string(kind), norm);
    const auto none = [&] { return at::empty({0}, x.options()); };
    const bool branched = has(branch);
    return {branched ? out[0] : none(),
            norm ? out[branched ? 1 : 0] : none()};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = find_op<NormOnlyOp>("vectra_b200::residual_norm");
  return op.call(x, branch, weight, bias, branch_weight, gate, residual_scale,
                 p, rng, stream, eps, kind, norm);
}

using CrossOp = Three(const Tensor&, const Tensor&, const Tensor&,
                      const Tensor&, const OptTensor&, bool);
using CrossBackwardOp = Four(const Tensor&, const Tensor&, const Tensor&,
                             const Tensor&, const Tensor&, const OptTensor&,
                             const Tensor&, const Tensor&, const Tensor&, bool,
                             bool, bool);

struct CrossFunction : public Function<CrossFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q,
                        const Tensor& k, const Tensor& v, const Tensor& scale,
                        const OptTensor& lengths) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op =
        find_op<CrossOp>("vectra_b200::cross_attention_with_lse");
    auto [out, lse, rest] = op.call(q, k, v, scale, lengths, true);
    ctx->save_for_backward(
        {q, k, v, scale, or_undefined(lengths), out, lse, rest});
    ctx->saved_data["need"] = int64_t(wants_grad(q)) |
                              int64_t(wants_grad(k)) << 1 |
                              int64_t(wants_grad(v)) << 2 |
                              int64_t(wants_grad(scale)) << 3;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    std::optional<at::AutoDispatchBelowADInplaceOrView> below;
    if (!at::GradMode::is_enabled()) below.emplace();
    static const auto op =
        find_op<CrossBackwardOp>("vectra_b200::cross_attention_backward");
    auto [dq, dk, dv, dscale] =
        op.call(grads[0], s[0], s[1], s[2], s[3], optional(s[4]), s[5], s[6],
                s[7], (need & 1) != 0, (need & 6) != 0, (need & 8) != 0);
    if (need & 1) out[0] = dq;
    if (need & 2) out[1] = dk;
    if (need & 4) out[2] = dv;
    if (need & 8)
      out[3] = at::sum_to(dscale.unsqueeze(-1).unsqueeze(-1), s[3].sizes())
                   .to(s[3].scalar_type());
    return out;
  }
};

Tensor cross_autograd(const Tensor& q, const Tensor& k, const Tensor& v,
                      const Tensor& scale, const OptTensor& lengths) {
  refuse_tangents("cross_attention", q, k, v, scale);
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) ||
                                     wants_grad(v) || wants_grad(scale)))
    return CrossFunction::apply(q, k, v, scale, lengths);
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op =
      find_op<CrossOp>("vectra_b200::cross_attention_with_lse");
  return std::get<0>(op.call(q, k, v, scale, lengths, false));
}

// The implementations with the schemas' types.
template <auto F>
Four norm_impl(const Tensor& x, const OptTensor& branch,
                const OptTensor& weight, const OptTensor& bias,
                const OptTensor& branch_weight, const OptTensor& gate,
                double residual_scale, double p, const OptTensor& rng,
                int64_t stream, double eps, c10::string_view kind, bool norm,
                bool want_stats) {
  return F(x, branch, weight, bias, branch_weight, gate,
           NormCall{residual_scale, p, rng, stream, eps, kind_of(kind)}, norm,
           want_stats, false);
}
template <auto F>
std::tuple<Tensor, Tensor> norm_only_impl(
    const Tensor& x, const OptTensor& branch, const OptTensor& weight,
    const OptTensor& bias, const OptTensor& branch_weight,
    const OptTensor& gate, double residual_scale, double p,
    const OptTensor& rng, int64_t stream, double eps, c10::string_view kind,
    bool norm) {
  auto out = F(x, branch, weight, bias, branch_weight, gate,
               NormCall{residual_scale, p, rng, stream, eps, kind_of(kind)},
               norm, false, true);
  return {std::get<0>(out), std::get<1>(out)};
}
template <auto F>
Six norm_backward_impl(const OptTensor& dx_out, const OptTensor& dy,
                       const Tensor& x_out, const Tensor& rest,
                       const Tensor& stats,
                       const OptTensor& branch, const OptTensor& weight,
                       const OptTensor& branch_weight, const OptTensor& gate,
                       double residual_scale, double p, const OptTensor& rng,
                       int64_t stream, double eps, c10::string_view kind,
                       int64_t need) {
  return F(dx_out, dy, x_out, rest, stats, branch, weight, branch_weight, gate,
           NormCall{residual_scale, p, rng, stream, eps, kind_of(kind)},
           need);
}
template <auto F>
Tensor cross_only_impl(const Tensor& q, const Tensor& k, const Tensor& v,
                       const Tensor& scale, const OptTensor& lengths) {
  return std::get<0>(F(q, k, v, scale, lengths, false));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(vectra_b200, m) {
  m.def(
      "dropout(Tensor x, float p, Tensor? rng=None, int stream=0) -> Tensor");
  m.def(
      "residual_norm(Tensor x, Tensor? branch=None, Tensor? weight=None, "
      "Tensor? bias=None, Tensor? branch_weight=None, Tensor? gate=None, "
      "float residual_scale=1.0, float p=0.0, Tensor? rng=None, "
      "int stream=0, float eps=1e-6, str kind='rms', bool norm=True) "
      "-> (Tensor, Tensor)");
  m.def(
      "residual_norm_with_stats(Tensor x, Tensor? branch, Tensor? weight, "
      "Tensor? bias, Tensor? branch_weight, Tensor? gate, "
      "float residual_scale, float p, Tensor? rng, int stream, float eps, "
      "str kind, bool norm, bool want_stats) "
      "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "residual_norm_backward(Tensor? dx_out, Tensor? dy, Tensor x_out, "
      "Tensor rest, Tensor stats, Tensor? branch, Tensor? weight, Tensor? branch_weight, "
      "Tensor? gate, float residual_scale, float p, Tensor? rng, int stream, "
      "float eps, str kind, int need) "
      "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "cross_attention(Tensor q, Tensor k, Tensor v, Tensor scale, "
      "Tensor? key_lengths=None) -> Tensor");
  m.def(
      "cross_attention_with_lse(Tensor q, Tensor k, Tensor v, Tensor scale, "
      "Tensor? key_lengths, bool want_lse) -> (Tensor, Tensor, Tensor)");
  m.def(
      "cross_attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, "
      "Tensor scale, Tensor? key_lengths, Tensor out, Tensor lse, "
      "Tensor rest, bool need_dq, bool need_dkv, bool need_dscale) "
      "-> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(vectra_b200, CUDA, m) {
  m.impl("dropout", &dropout_cuda);
  m.impl("residual_norm", &norm_only_impl<norm_cuda>);
  m.impl("residual_norm_with_stats", &norm_impl<norm_cuda>);
  m.impl("residual_norm_backward", &norm_backward_impl<norm_backward_cuda>);
  m.impl("cross_attention", &cross_only_impl<cross_cuda>);
  m.impl("cross_attention_with_lse", &cross_cuda);
  m.impl("cross_attention_backward", &cross_backward_cuda);
}

TORCH_LIBRARY_IMPL(vectra_b200, CPU, m) {
  m.impl("dropout", &dropout_cpu);
  m.impl("residual_norm", &norm_only_impl<norm_cpu>);
  m.impl("residual_norm_with_stats", &norm_impl<norm_cpu>);
  m.impl("residual_norm_backward", &norm_backward_impl<norm_backward_cpu>);
  m.impl("cross_attention", &cross_only_impl<cross_cpu>);
  m.impl("cross_attention_with_lse", &cross_cpu);
  m.impl("cross_attention_backward", &cross_backward_cpu);
}

TORCH_LIBRARY_IMPL(vectra_b200, Autograd, m) {
  m.impl("dropout", &dropout_autograd);
  m.impl("residual_norm", &norm_autograd);
  m.impl("cross_attention", &cross_autograd);
  for (const char* op :
       {"residual_norm_with_stats", "residual_norm_backward",
        "cross_attention_with_lse", "cross_attention_backward"})
    m.impl(op, torch::autograd::autogradNotImplementedFallback());
}
