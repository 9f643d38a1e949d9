// decoder_capi.cu: the C ABI of dropout, the norms between two sublayers and
// attention to an encoder's states (include/vectra_block.h): argument checks,
// and each pass as a short sequence of kernels on the caller's stream.
#include "block_checks.cuh"
#include "cross.cuh"
#include "residual_norm.cuh"

namespace vectra {
namespace {

int check_drop(const vectra_drop& d) {
  if (!(d.p >= 0.0 && d.p <= 1.0)) return VECTRA_ERR_UNSUPPORTED;
  return d.rng == nullptr && d.p > 0.0 ? VECTRA_ERR_NULL : VECTRA_OK;
}

int check_contiguous(const vectra_tensor& t, int32_t dtype, int64_t rows,
                     int64_t cols) {
  VECTRA_TRY(check(t, dtype, {rows, cols}));
  if ((cols > 1 && t.stride[1] != 1) || (rows > 1 && t.stride[0] != cols))
    return VECTRA_ERR_LAYOUT;
  return VECTRA_OK;
}
int check_contiguous(const vectra_tensor& t, int32_t dtype, int64_t n) {
  VECTRA_TRY(check(t, dtype, {n}));
  if (n > 1 && t.stride[0] != 1) return VECTRA_ERR_LAYOUT;
  return VECTRA_OK;
}

// [rows, 4] float32, which the kernels move a row at a time.
int check_stats(const vectra_tensor& t, int64_t rows) {
  VECTRA_TRY(check_contiguous(t, VECTRA_F32, rows, 4));
  return reinterpret_cast<uintptr_t>(t.data) & 15 ? VECTRA_ERR_LAYOUT
                                                  : VECTRA_OK;
}

RowView view(const vectra_tensor& t) {  // [rows, columns]
  return {t.data, t.stride[0], t.size[1] > 1 ? t.stride[1] : 1};
}
RowView vector_view(const vectra_tensor& t) {  // [columns]
  return {t.data, 0, t.size[0] > 1 ? t.stride[0] : 1};
}

int dropout(const vectra_dropout_args& a, cudaStream_t stream) {
  if (a.x.ndim != 2) return VECTRA_ERR_RANK;
  if (!io_dtype_ok(a.x.dtype)) return VECTRA_ERR_DTYPE;
  const int64_t m = a.x.size[0], c = a.x.size[1];
  if (m < 0 || c < 0) return VECTRA_ERR_SHAPE;
  VECTRA_TRY(check(a.x, a.x.dtype, {m, c}));
  VECTRA_TRY(check_contiguous(a.y, a.x.dtype, m, c));
  VECTRA_TRY(check_drop(a.drop));
  return launch_dropout(a.x.dtype, view(a.x), m, c,
                        const_cast<void*>(a.y.data), make_drop(a.drop),
                        stream) == cudaSuccess
             ? VECTRA_OK
             : VECTRA_ERR_CUDA;
}

// What both passes check and describe; the rows are those of `rows`.
int build_norm(const vectra_residual_norm_args& a, const vectra_tensor& rows,
               bool norm1, bool backward, NormProblem* p) {
  if (rows.ndim != 2) return VECTRA_ERR_RANK;
  const int32_t dtype = rows.dtype;
  if (!io_dtype_ok(dtype)) return VECTRA_ERR_DTYPE;
  const int64_t m = rows.size[0], c = rows.size[1];
  if (m < 0 || c < 0) return VECTRA_ERR_SHAPE;
  if (c > kMaxNormCols || m > kMaxSize) return VECTRA_ERR_UNSUPPORTED;
  if (a.kind != VECTRA_NORM_RMS && a.kind != VECTRA_NORM_LAYER)
    return VECTRA_ERR_UNSUPPORTED;
  VECTRA_TRY(check_drop(a.drop));
  const bool branch = present(a.branch);
  if (branch) VECTRA_TRY(check(a.branch, dtype, {m, c}));
  // No branch: nothing that would change x, and something to do. (Rows of
  // no elements may have no address.)
  if (!branch && !backward && m * c > 0 &&
      (!norm1 || present(a.gate) || present(a.branch_weight) ||
       a.drop.p != 0.0 || a.residual_scale != 1.0))
    return VECTRA_ERR_NULL;
  if (!norm1 && !backward && (present(a.weight) || present(a.bias)))
    return VECTRA_ERR_NULL;
  if (present(a.weight)) VECTRA_TRY(check(a.weight, dtype, {c}));
  if (present(a.bias)) VECTRA_TRY(check(a.bias, dtype, {c}));
  if (present(a.branch_weight)) VECTRA_TRY(check(a.branch_weight, dtype, {c}));
  *p = NormProblem{};
  if (present(a.gate)) {
    if (a.gate.ndim != 2) return VECTRA_ERR_RANK;
    const int64_t g = a.gate.size[0];
    VECTRA_TRY(check(a.gate, dtype, {g, c}));
    if (g < 1 || m % g != 0) return VECTRA_ERR_SHAPE;
    p->gate = view(a.gate);
    p->gate_count = g;
    p->gate_rows = m > 0 ? m / g : 1;
  }
  p->dtype = dtype;
  p->M = m;
  p->C = int32_t(c);
  p->layer = a.kind == VECTRA_NORM_LAYER;
  p->eps = float(a.eps);
  p->residual_scale = float(a.residual_scale);
  p->drop = make_drop(a.drop);
  if (branch) p->branch = view(a.branch);
  if (present(a.weight)) p->weight = vector_view(a.weight);
  if (present(a.bias)) p->bias = vector_view(a.bias);
  if (present(a.branch_weight))
    p->branch_weight = vector_view(a.branch_weight);
  return VECTRA_OK;
}

// What x_out's rounding left; 16-bit tensors with a branch and a norm.
int check_rest(const vectra_tensor& rest, const NormProblem& p,
               bool rounded) {
  if (p.dtype == VECTRA_F32) return VECTRA_ERR_DTYPE;
  if (!rounded) return VECTRA_ERR_NULL;
  return check_contiguous(rest, p.dtype, p.M, p.C);
}

int norm_forward(const vectra_residual_norm_args& a, const vectra_tensor& rest,
                 cudaStream_t stream) {
  NormProblem p;
  VECTRA_TRY(build_norm(a, a.x, present(a.y), false, &p));
  VECTRA_TRY(check(a.x, p.dtype, {p.M, p.C}));
  p.x = view(a.x);
  if (present(a.branch))
    VECTRA_TRY(check_contiguous(a.x_out, p.dtype, p.M, p.C));
  p.x_out = const_cast<void*>(a.x_out.data);
  if (present(a.y)) VECTRA_TRY(check_contiguous(a.y, p.dtype, p.M, p.C));
  p.y = const_cast<void*>(a.y.data);
  if (present(a.stats)) {
    VECTRA_TRY(check_stats(a.stats, p.M));
    p.stats = static_cast<float*>(const_cast<void*>(a.stats.data));
  }
  if (present(rest)) {
    VECTRA_TRY(check_rest(rest, p, present(a.branch) && present(a.y)));
    p.rest = const_cast<void*>(rest.data);
  }
  return launch_norm_forward(p, stream) == cudaSuccess ? VECTRA_OK
                                                       : VECTRA_ERR_CUDA;
}

int norm_backward_with(const vectra_residual_norm_grad_args& a,
                       const vectra_tensor& rest, Workspace& ws,
                       cudaStream_t stream) {
  NormProblem p;
  const bool norm1 = present(a.dy);
  const vectra_tensor& rows = norm1 ? a.dy : a.dx_out;
  VECTRA_TRY(build_norm(a.fwd, rows, norm1, true, &p));
  const int64_t m = p.M, c = p.C;
  VECTRA_TRY(check(rows, p.dtype, {m, c}));
  if (present(a.dx_out)) {
    VECTRA_TRY(check(a.dx_out, p.dtype, {m, c}));
    p.e = view(a.dx_out);
  }
  if (norm1) {
    VECTRA_TRY(check(a.fwd.x_out, p.dtype, {m, c}));
    p.x = view(a.fwd.x_out);
    p.f = view(a.dy);
  }
  if (present(rest)) {
    VECTRA_TRY(check_rest(rest, p, norm1));
    p.rest = const_cast<void*>(rest.data);
  }
  if (norm1 || present(a.fwd.branch_weight)) {
    VECTRA_TRY(check_stats(a.fwd.stats, m));
    p.stats = static_cast<float*>(const_cast<void*>(a.fwd.stats.data));
  }
  // The branch itself is read for its norm and for the gate's gradient only.
  if ((present(a.fwd.branch_weight) || present(a.dgate)) &&
      !present(a.fwd.branch) && m * c > 0)
    return VECTRA_ERR_NULL;
  const vectra_tensor* matrices[2] = {&a.dx, &a.dbranch};
  void** results[2] = {&p.dx, &p.dbranch};
  for (int i = 0; i < 2; ++i) {
    if (!present(*matrices[i])) continue;
    VECTRA_TRY(check_contiguous(*matrices[i], p.dtype, m, c));
    *results[i] = const_cast<void*>(matrices[i]->data);
  }
  const vectra_tensor* vectors[3] = {&a.dweight, &a.dbias, &a.dbranch_weight};
  const bool allowed[3] = {norm1, norm1, present(a.fwd.branch_weight)};
  void** sums[3] = {&p.dweight, &p.dbias, &p.dbranch_weight};
  for (int i = 0; i < 3; ++i) {
    if (!present(*vectors[i])) continue;
    if (!allowed[i]) return VECTRA_ERR_NULL;
    VECTRA_TRY(check_contiguous(*vectors[i], p.dtype, c));
    *sums[i] = const_cast<void*>(vectors[i]->data);
  }
  if (present(a.dgate)) {
    if (!present(a.fwd.gate)) return VECTRA_ERR_NULL;
    VECTRA_TRY(check_contiguous(a.dgate, p.dtype, p.gate_count, c));
    p.dgate = const_cast<void*>(a.dgate.data);
  }
  return to_status(run_norm_backward(p, ws, stream), ws);
}
int norm_backward(const vectra_residual_norm_grad_args& a, Workspace& ws,
                  cudaStream_t stream) {
  return norm_backward_with(a, vectra_tensor{}, ws, stream);
}
// The workspace of the call with `rest` is its other part's.
auto norm_backward_train(const vectra_tensor& rest) {
  return [&rest](const vectra_residual_norm_grad_args& a, Workspace& ws,
                 cudaStream_t stream) {
    return norm_backward_with(a, rest, ws, stream);
  };
}

void strides_of(const vectra_tensor& t, int64_t* s) {
  for (int i = 0; i < 4; ++i) s[i] = t.stride[i];
}

// A [B, H, N, width] result.
int set_heads(const vectra_tensor& t, int32_t dtype, int64_t b, int64_t h,
              int64_t n, int64_t width, void** data, int64_t* s) {
  VECTRA_TRY(check(t, dtype, {b, h, n, width}));
  if (width > 1 && t.stride[3] != 1) return VECTRA_ERR_LAYOUT;
  *data = const_cast<void*>(t.data);
  strides_of(t, s);
  s[3] = 1;
  return VECTRA_OK;
}

int build_cross(const vectra_cross_args& a, CrossProblem* p) {
  if (a.q.ndim != 4 || a.k.ndim != 4 || a.v.ndim != 4 || a.scale.ndim != 4)
    return VECTRA_ERR_RANK;
  const int32_t dtype = a.q.dtype;
  if (!io_dtype_ok(dtype)) return VECTRA_ERR_DTYPE;
  const int64_t b = a.q.size[0], h = a.q.size[1], nq = a.q.size[2],
                d = a.q.size[3];
  const int64_t hk = a.k.size[1], nk = a.k.size[2], dv = a.v.size[3];
  for (const int64_t s : {b, h, nq, d, hk, nk, dv})
    if (s < 0) return VECTRA_ERR_SHAPE;
    else if (s > kMaxSize) return VECTRA_ERR_UNSUPPORTED;
  VECTRA_TRY(check(a.q, dtype, {b, h, nq, d}));
  VECTRA_TRY(check(a.k, dtype, {b, hk, nk, d}));
  VECTRA_TRY(check(a.v, dtype, {b, hk, nk, dv}));
  if (h > 0 && (hk < 1 || h % hk != 0)) return VECTRA_ERR_SHAPE;
  if (h == 0 && hk != 0) return VECTRA_ERR_SHAPE;
  if (d < 1 || dv < 1) return VECTRA_ERR_SHAPE;
  if (d > kMaxCrossWidth || dv > kMaxCrossWidth) return VECTRA_ERR_UNSUPPORTED;
  // Packed rows and planes are counted in 32 bits.
  if (hk > 0 && (nq * (h / hk) > kMaxSize || b * h > 0x7fffffff))
    return VECTRA_ERR_UNSUPPORTED;
  if (a.scale.dtype < VECTRA_F32 || a.scale.dtype > VECTRA_F64)
    return VECTRA_ERR_DTYPE;
  if (b * h > 0 && a.scale.data == nullptr) return VECTRA_ERR_NULL;
  const int64_t full[2] = {b, h};
  for (int i = 0; i < 2; ++i)
    if ((a.scale.size[i] != 1 && a.scale.size[i] != full[i]) ||
        a.scale.size[i + 2] != 1)
      return VECTRA_ERR_SCALE_SHAPE;
  if (a.key_lengths && a.length_bytes != 4 && a.length_bytes != 8)
    return VECTRA_ERR_DTYPE;
  *p = CrossProblem{};
  p->dtype = dtype;
  p->scale_dtype = a.scale.dtype;
  p->B = b;
  p->H = h;
  p->Hk = hk;
  p->G = hk > 0 ? h / hk : 1;
  p->Nq = nq;
  p->Nk = nk;
  p->D = int32_t(d);
  p->Dv = int32_t(dv);
  p->q = a.q.data;
  p->k = a.k.data;
  p->v = a.v.data;
  p->scale = a.scale.data;
  p->lengths = a.key_lengths;
  p->length_bytes = a.length_bytes;
  p->length_stride = a.length_stride;
  strides_of(a.q, p->sq);
  strides_of(a.k, p->sk);
  strides_of(a.v, p->sv);
  for (int i = 0; i < 2; ++i)
    p->ss[i] = a.scale.size[i] == 1 ? 0 : a.scale.stride[i];
  VECTRA_TRY(set_heads(a.out, dtype, b, h, nq, dv, &p->out, p->so));
  if (present(a.lse)) {
    VECTRA_TRY(check(a.lse, VECTRA_F32, {b, h, nq}));
    if ((nq > 1 && a.lse.stride[2] != 1) || (h > 1 && a.lse.stride[1] != nq) ||
        (b > 1 && a.lse.stride[0] != nq * h))
      return VECTRA_ERR_LAYOUT;
    p->lse = static_cast<float*>(const_cast<void*>(a.lse.data));
  }
  if (present(a.rest)) {
    if (dtype == VECTRA_F32) return VECTRA_ERR_DTYPE;
    VECTRA_TRY(check(a.rest, dtype, {b, h, nq, dv}));
    int64_t step = 1;
    for (int i = 3; i >= 0; --i) {
      if (a.rest.size[i] > 1 && a.rest.stride[i] != step)
        return VECTRA_ERR_LAYOUT;
      step *= a.rest.size[i];
    }
    p->rest = const_cast<void*>(a.rest.data);
  }
  return VECTRA_OK;
}

int cross_forward(const vectra_cross_args& a, Workspace& ws,
                  cudaStream_t stream) {
  CrossProblem p;
  VECTRA_TRY(build_cross(a, &p));
  p.err = ws.dry ? nullptr : device_error_ptr();
  return to_status(cross_rows_supports(p, false)
                       ? run_cross_rows_forward(p, ws, stream)
                   : cross_tc_supports(p, false)
                       ? run_cross_tc_forward(p, ws, stream)
                       : run_cross_simple_forward(p, ws, stream),
                   ws);
}

int cross_backward(const vectra_cross_grad_args& a, Workspace& ws,
                   cudaStream_t stream) {
  CrossProblem p;
  VECTRA_TRY(build_cross(a.fwd, &p));
  if (p.B * p.H * p.Nq > 0 &&
      (p.lse == nullptr || (p.dtype != VECTRA_F32 && p.rest == nullptr)))
    return VECTRA_ERR_NULL;
  VECTRA_TRY(check(a.dout, p.dtype, {p.B, p.H, p.Nq, int64_t(p.Dv)}));
  p.dout = a.dout.data;
  strides_of(a.dout, p.se);
  if (present(a.dq))
    VECTRA_TRY(set_heads(a.dq, p.dtype, p.B, p.H, p.Nq, p.D, &p.dq, p.sdq));
  if (present(a.dk) != present(a.dv)) return VECTRA_ERR_NULL;
  if (present(a.dk)) {
    VECTRA_TRY(set_heads(a.dk, p.dtype, p.B, p.Hk, p.Nk, p.D, &p.dk, p.sdk));
    VECTRA_TRY(set_heads(a.dv, p.dtype, p.B, p.Hk, p.Nk, p.Dv, &p.dv, p.sdv));
  }
  if (present(a.dscale)) {
    VECTRA_TRY(check_contiguous(a.dscale, VECTRA_F32, p.B, p.H));
    p.dscale = static_cast<float*>(const_cast<void*>(a.dscale.data));
  }
  p.err = ws.dry ? nullptr : device_error_ptr();
  return to_status(cross_rows_supports(p, true)
                       ? run_cross_rows_backward(p, ws, stream)
                   : cross_tc_supports(p, true)
                       ? run_cross_tc_backward(p, ws, stream)
                       : run_cross_simple_backward(p, ws, stream),
                   ws);
}

}  // namespace
}  // namespace vectra

using namespace vectra;

extern "C" {

int vectra_dropout(const vectra_dropout_args* a, void* stream) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return dropout(*a, static_cast<cudaStream_t>(stream));
}
int vectra_residual_norm_forward(const vectra_residual_norm_args* a,
                                 void* stream) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return norm_forward(*a, vectra_tensor{}, static_cast<cudaStream_t>(stream));
}
int vectra_residual_norm_forward_train(const vectra_residual_norm_train_args* a,
                                       void* stream) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return norm_forward(a->fwd, a->rest, static_cast<cudaStream_t>(stream));
}
int vectra_residual_norm_backward(const vectra_residual_norm_grad_args* a,
                                  void* stream) {
  return run_with_workspace(a, stream, norm_backward);
}
int vectra_residual_norm_backward_train(
    const vectra_residual_norm_train_grad_args* a, void* stream) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return run_with_workspace(&a->grad, stream, norm_backward_train(a->rest));
}
int64_t vectra_residual_norm_backward_train_workspace_bytes(
    const vectra_residual_norm_train_grad_args* a) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return workspace_of(&a->grad, norm_backward_train(a->rest));
}
int vectra_cross_attention_forward(const vectra_cross_args* a, void* stream) {
  return run_with_workspace(a, stream, cross_forward);
}
int vectra_cross_attention_backward(const vectra_cross_grad_args* a,
                                    void* stream) {
  return run_with_workspace(a, stream, cross_backward);
}

int64_t vectra_residual_norm_backward_workspace_bytes(
    const vectra_residual_norm_grad_args* a) {
  return workspace_of(a, norm_backward);
}
int64_t vectra_cross_attention_forward_workspace_bytes(
    const vectra_cross_args* a) {
  return workspace_of(a, cross_forward);
}
int64_t vectra_cross_attention_backward_workspace_bytes(
    const vectra_cross_grad_args* a) {
  return workspace_of(a, cross_backward);
}

}  // extern "C"
