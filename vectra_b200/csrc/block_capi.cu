// block_capi.cu: the C ABI of the transformer-block operators
// (include/vectra_block.h): argument checks, and each operator's forward and
// backward pass as a short sequence of matrix products and elementwise
// kernels on the caller's stream.
#include "block_checks.cuh"

namespace vectra {
namespace {

MatView rows_of(const vectra_tensor& t) {  // reduced over the columns
  return {t.data, t.stride[0], t.stride[1]};
}
MatView cols_of(const vectra_tensor& t) {  // reduced over the rows
  return {t.data, t.stride[1], t.stride[0]};
}

int check_common(const vectra_tensor& x, const vectra_tensor& w,
                 int32_t activation) {
  if (x.ndim != 2 || w.ndim != 2) return VECTRA_ERR_RANK;
  if (!io_dtype_ok(x.dtype)) return VECTRA_ERR_DTYPE;
  if (activation < VECTRA_ACT_NONE || activation > VECTRA_ACT_SILU)
    return VECTRA_ERR_UNSUPPORTED;
  for (int i = 0; i < 2; ++i) {
    if (x.size[i] < 0 || w.size[i] < 0) return VECTRA_ERR_SHAPE;
    // Sizes count blocks and tensor-map lines, which are 32-bit.
    if (x.size[i] > kMaxSize || w.size[i] > kMaxSize)
      return VECTRA_ERR_UNSUPPORTED;
  }
  return VECTRA_OK;
}

// Above the few-row kernel's sizes, float32 gradients are split once.
constexpr int64_t kSplitOnceRows = 64;

// Rows of the gradients in the workspace start on 16-byte boundaries, which
// the tensor-core products need.
int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

// The operators' passes. Each runs twice: dry, to size the workspace, and
// for real.
int linear_forward(const vectra_linear_args& a, Workspace& ws,
                   cudaStream_t stream) {
  VECTRA_TRY(check_common(a.x, a.weight, a.activation));
  const int64_t M = a.x.size[0], K = a.x.size[1], N = a.weight.size[0];
  const int32_t dt = a.x.dtype;
  VECTRA_TRY(check(a.x, dt, {M, K}));
  VECTRA_TRY(check(a.weight, dt, {N, K}));
  if (present(a.bias)) VECTRA_TRY(check(a.bias, dt, {N}));
  if (present(a.residual)) VECTRA_TRY(check(a.residual, dt, {M, N}));
  VECTRA_TRY(check_result(a.y, dt, {M, N}));
  if (present(a.pre)) VECTRA_TRY(check_result(a.pre, dt, {M, N}));
  if (M == 0 || N == 0) return VECTRA_OK;
  GemmProblem p;
  p.dtype = dt;
  // A bare product needs no more than a store.
  p.epilogue = present(a.bias) || present(a.residual) || present(a.pre) ||
                       a.activation != VECTRA_ACT_NONE
                   ? kEpiLinear
                   : kEpiStore;
  p.act = a.activation;
  p.M = M;
  p.N = N;
  p.K = K;
  p.a[0] = rows_of(a.x);
  p.b[0] = rows_of(a.weight);
  p.bias[0] = a.bias.data;
  p.bias_stride[0] = a.bias.stride[0];
  p.res = a.residual.data;
  p.res_sm = a.residual.stride[0];
  p.res_sn = a.residual.stride[1];
  p.out = const_cast<void*>(a.y.data);
  p.out_ld = a.y.stride[0];
  p.pre = const_cast<void*>(a.pre.data);
  p.pre_ld = a.pre.stride[0];
  return to_status(run_gemm(p, ws, stream), ws);
}

int linear_backward(const vectra_linear_grad_args& a, Workspace& ws,
                    cudaStream_t stream) {
  VECTRA_TRY(check_common(a.x, a.weight, a.activation));
  const int64_t M = a.x.size[0], K = a.x.size[1], N = a.weight.size[0];
  const int32_t dt = a.x.dtype;
  VECTRA_TRY(check(a.x, dt, {M, K}));
  VECTRA_TRY(check(a.weight, dt, {N, K}));
  VECTRA_TRY(check(a.dy, dt, {M, N}));
  const bool act = a.activation != VECTRA_ACT_NONE;
  if (act) VECTRA_TRY(check_result(a.pre, dt, {M, N}));
  if (present(a.dx)) VECTRA_TRY(check_result(a.dx, dt, {M, K}));
  if (present(a.dweight)) VECTRA_TRY(check_result(a.dweight, dt, {N, K}));
  if (present(a.dbias)) VECTRA_TRY(check_result(a.dbias, dt, {N}));
  const size_t es = dt == VECTRA_F32 ? 4 : 2;
  const bool products = (present(a.dx) || present(a.dweight)) && M > 0;

  MatView dz_rows = rows_of(a.dy), dz_cols = cols_of(a.dy);
  if ((act && products) || present(a.dbias)) {
    GradProblem g;
    g.dtype = dt;
    g.act = a.activation;
    g.M = M;
    g.N = N;
    g.dy = a.dy.data;
    g.dy_sm = a.dy.stride[0];
    g.dy_sn = a.dy.stride[1];
    g.pre = act ? a.pre.data : nullptr;
    g.pre_ld = a.pre.stride[0];
    if (act && products) {
      g.dz_ld = pad8(N);
      g.dz = ws.take(size_t(M) * g.dz_ld * es);
      dz_rows = {g.dz, g.dz_ld, 1};
      dz_cols = {g.dz, 1, g.dz_ld};
    }
    g.db = const_cast<void*>(a.dbias.data);
    VECTRA_TRY(to_status(run_grad(g, ws, stream), ws));
  }
  // float32: dz is split once for both products.
  if (dt == VECTRA_F32 && present(a.dx) && present(a.dweight) &&
      M > kSplitOnceRows && N > 0 && K > 0)
    VECTRA_TRY(to_status(
        split_for_products(dz_rows.p, M, N, dz_rows.sr, dz_rows.sk, ws,
                           &dz_rows, &dz_cols, stream), ws));
  GemmProblem p;
  p.dtype = dt;
  p.epilogue = kEpiStore;
  if (present(a.dx) && M > 0 && K > 0) {
    p.M = M;
    p.N = K;
    p.K = N;
    p.a[0] = dz_rows;
    p.b[0] = cols_of(a.weight);
    p.out = const_cast<void*>(a.dx.data);
    p.out_ld = a.dx.stride[0];
    VECTRA_TRY(to_status(run_gemm(p, ws, stream), ws));
  }
  if (present(a.dweight) && N > 0 && K > 0) {
    p.M = N;
    p.N = K;
    p.K = M;
    p.a[0] = dz_cols;
    p.b[0] = cols_of(a.x);
    p.out = const_cast<void*>(a.dweight.data);
    p.out_ld = a.dweight.stride[0];
    VECTRA_TRY(to_status(run_gemm(p, ws, stream), ws));
  }
  return VECTRA_OK;
}

int gated_forward(const vectra_gated_args& a, Workspace& ws,
                  cudaStream_t stream) {
  VECTRA_TRY(check_common(a.x, a.w_gate, a.activation));
  const int64_t M = a.x.size[0], K = a.x.size[1], F = a.w_gate.size[0];
  const int32_t dt = a.x.dtype;
  VECTRA_TRY(check(a.x, dt, {M, K}));
  VECTRA_TRY(check(a.w_gate, dt, {F, K}));
  VECTRA_TRY(check(a.w_up, dt, {F, K}));
  if (present(a.b_gate)) VECTRA_TRY(check(a.b_gate, dt, {F}));
  if (present(a.b_up)) VECTRA_TRY(check(a.b_up, dt, {F}));
  VECTRA_TRY(check_result(a.h, dt, {M, F}));
  if (present(a.gate) != present(a.up)) return VECTRA_ERR_NULL;
  if (present(a.gate)) {
    VECTRA_TRY(check_result(a.gate, VECTRA_F32, {M, F}));
    VECTRA_TRY(check_result(a.up, VECTRA_F32, {M, F}));
  }
  if (M == 0 || F == 0) return VECTRA_OK;
  GemmProblem p;
  p.dtype = dt;
  p.epilogue = kEpiGated;
  p.act = a.activation;
  p.M = M;
  p.N = F;
  p.K = K;
  p.a[0] = rows_of(a.x);
  p.b[0] = rows_of(a.w_gate);
  p.b[1] = rows_of(a.w_up);
  p.bias[0] = a.b_gate.data;
  p.bias_stride[0] = a.b_gate.stride[0];
  p.bias[1] = a.b_up.data;
  p.bias_stride[1] = a.b_up.stride[0];
  p.out = const_cast<void*>(a.h.data);
  p.out_ld = a.h.stride[0];
  p.gate = static_cast<float*>(const_cast<void*>(a.gate.data));
  p.gate_ld = a.gate.stride[0];
  p.up = static_cast<float*>(const_cast<void*>(a.up.data));
  p.up_ld = a.up.stride[0];
  return to_status(run_gemm(p, ws, stream), ws);
}

int gated_backward(const vectra_gated_grad_args& a, Workspace& ws,
                   cudaStream_t stream) {
  VECTRA_TRY(check_common(a.x, a.w_gate, a.activation));
  const int64_t M = a.x.size[0], K = a.x.size[1], F = a.w_gate.size[0];
  const int32_t dt = a.x.dtype;
  VECTRA_TRY(check(a.x, dt, {M, K}));
  VECTRA_TRY(check(a.w_gate, dt, {F, K}));
  VECTRA_TRY(check(a.w_up, dt, {F, K}));
  VECTRA_TRY(check(a.dh, dt, {M, F}));
  if (present(a.gate) != present(a.up)) return VECTRA_ERR_NULL;
  if (present(a.gate)) {
    VECTRA_TRY(check_result(a.gate, VECTRA_F32, {M, F}));
    VECTRA_TRY(check_result(a.up, VECTRA_F32, {M, F}));
  }
  if (present(a.b_gate)) VECTRA_TRY(check(a.b_gate, dt, {F}));
  if (present(a.b_up)) VECTRA_TRY(check(a.b_up, dt, {F}));
  if (present(a.dx)) VECTRA_TRY(check_result(a.dx, dt, {M, K}));
  if (present(a.dw_gate) != present(a.dw_up) ||
      present(a.db_gate) != present(a.db_up))
    return VECTRA_ERR_NULL;
  if (present(a.dw_gate)) {
    VECTRA_TRY(check_result(a.dw_gate, dt, {F, K}));
    VECTRA_TRY(check_result(a.dw_up, dt, {F, K}));
  }
  if (present(a.db_gate)) {
    VECTRA_TRY(check_result(a.db_gate, dt, {F}));
    VECTRA_TRY(check_result(a.db_up, dt, {F}));
  }
  const size_t es = dt == VECTRA_F32 ? 4 : 2;
  // dg and du side by side, [M][2 pad8(F)].
  const int64_t ld = 2 * pad8(F);
  char* d = static_cast<char*>(ws.take(size_t(M) * ld * es));
  char* d2 = d ? d + ld / 2 * es : nullptr;
  void* db = const_cast<void*>(a.db_gate.data);
  void* db2 = const_cast<void*>(a.db_up.data);
  // The layer's own product, for values that were not saved.
  GemmProblem layer;
  layer.dtype = dt;
  layer.act = a.activation;
  layer.M = M;
  layer.N = F;
  layer.K = K;
  layer.a[0] = rows_of(a.x);
  layer.b[0] = rows_of(a.w_gate);
  layer.b[1] = rows_of(a.w_up);
  layer.bias[0] = a.b_gate.data;
  layer.bias_stride[0] = a.b_gate.stride[0];
  layer.bias[1] = a.b_up.data;
  layer.bias_stride[1] = a.b_up.stride[0];
  const bool saved = present(a.gate) || M == 0 || F == 0;
  if (!saved && dt != VECTRA_F32 && K > 0) {
    const int64_t blocks = (M + 31) / 32;
    layer.epilogue = kEpiGatedGrad;
    layer.res = a.dh.data;
    layer.res_sm = a.dh.stride[0];
    layer.res_sn = a.dh.stride[1];
    layer.out = d;
    layer.pre = d2;
    layer.out_ld = layer.pre_ld = ld;
    if (db) {
      layer.gate = static_cast<float*>(ws.take(size_t(blocks) * F * 4));
      layer.up = static_cast<float*>(ws.take(size_t(blocks) * F * 4));
    }
    VECTRA_TRY(to_status(run_gemm(layer, ws, stream), ws));
    if (db && !ws.dry)
      VECTRA_TRY(to_status(
          launch_column_finish(dt, layer.gate, layer.up, int(blocks), F, db,
                               db2, stream), ws));
  } else {
    GradProblem g;
    g.dtype = dt;
    g.act = a.activation;
    g.gated = true;
    g.M = M;
    g.N = F;
    g.dy = a.dh.data;
    g.dy_sm = a.dh.stride[0];
    g.dy_sn = a.dh.stride[1];
    g.gate = static_cast<const float*>(a.gate.data);
    g.gate_ld = a.gate.stride[0];
    g.up = static_cast<const float*>(a.up.data);
    g.up_ld = a.up.stride[0];
    if (!saved) {
      layer.epilogue = kEpiGated;
      layer.out = ws.take(size_t(M) * F * es);
      layer.gate = static_cast<float*>(ws.take(size_t(M) * F * 4));
      layer.up = static_cast<float*>(ws.take(size_t(M) * F * 4));
      layer.out_ld = layer.gate_ld = layer.up_ld = F;
      VECTRA_TRY(to_status(run_gemm(layer, ws, stream), ws));
      g.gate = layer.gate;
      g.up = layer.up;
      g.gate_ld = g.up_ld = F;
    }
    g.dz = d;
    g.dz2 = d2;
    g.dz_ld = ld;
    g.db = db;
    g.db2 = db2;
    VECTRA_TRY(to_status(run_grad(g, ws, stream), ws));
  }
  MatView dg_rows{d, ld, 1}, du_rows{d2, ld, 1};
  MatView dg_cols{d, 1, ld}, du_cols{d2, 1, ld};
  if (dt == VECTRA_F32 && present(a.dx) && present(a.dw_gate) &&
      M > kSplitOnceRows && F > 0 && K > 0) {
    // dg and du are split once for both products, as one matrix.
    VECTRA_TRY(to_status(
        split_for_products(d, M, ld, ld, 1, ws, &dg_rows, &dg_cols, stream),
        ws));
    const int64_t half = ld / 2 * 2;  // bytes of a bf16 row's half
    du_rows = dg_rows;
    du_cols = dg_cols;
    du_rows.p = dg_rows.p ? static_cast<const char*>(dg_rows.p) + half
                          : nullptr;
    du_cols.p = du_rows.p;
  }
  GemmProblem p;
  p.dtype = dt;
  p.epilogue = kEpiStore;
  if (present(a.dx) && M > 0 && K > 0) {
    p.M = M;
    p.N = K;
    p.K = F;
    p.segments = 2;
    p.a[0] = dg_rows;
    p.a[1] = du_rows;
    p.b[0] = cols_of(a.w_gate);
    p.b[1] = cols_of(a.w_up);
    p.out = const_cast<void*>(a.dx.data);
    p.out_ld = a.dx.stride[0];
    VECTRA_TRY(to_status(run_gemm(p, ws, stream), ws));
    p.segments = 1;
  }
  if (present(a.dw_gate) && F > 0 && K > 0) {
    const vectra_tensor* out[2] = {&a.dw_gate, &a.dw_up};
    // Results that lie one behind the other, like dg and du, are one product
    // of twice the rows: x is read once for both.
    const bool joined =
        F % 8 == 0 && a.dw_gate.stride[0] == a.dw_up.stride[0] &&
        static_cast<const char*>(a.dw_gate.data) +
                size_t(F) * a.dw_gate.stride[0] * es ==
            static_cast<const char*>(a.dw_up.data);
    for (int i = 0; i < (joined ? 1 : 2); ++i) {
      p.M = joined ? 2 * F : F;
      p.N = K;
      p.K = M;
      p.a[0] = i ? du_cols : dg_cols;
      p.b[0] = cols_of(a.x);
      p.out = const_cast<void*>(out[i]->data);
      p.out_ld = out[i]->stride[0];
      VECTRA_TRY(to_status(run_gemm(p, ws, stream), ws));
    }
  }
  return VECTRA_OK;
}

int build_qk(const vectra_qk_args& a, const vectra_qk_axes* axes,
             QkProblem* p) {
  if (a.q.ndim != 4 || a.k.ndim != 4 || a.cos.ndim != 2 || a.sin.ndim != 2)
    return VECTRA_ERR_RANK;
  if (!io_dtype_ok(a.q.dtype)) return VECTRA_ERR_DTYPE;
  const int64_t B = a.q.size[0], N = a.q.size[2], D = a.q.size[3];
  VECTRA_TRY(check(a.q, a.q.dtype, {B, a.q.size[1], N, D}));
  VECTRA_TRY(check(a.k, a.q.dtype, {B, a.k.size[1], N, D}));
  if (D > 512) return VECTRA_ERR_UNSUPPORTED;
  for (const int64_t s : {B, N, a.q.size[1], a.k.size[1]})
    if (s < 0) return VECTRA_ERR_SHAPE;
    else if (s > kMaxSize) return VECTRA_ERR_UNSUPPORTED;
  const int64_t P = a.cos.size[0], R2 = a.cos.size[1];
  VECTRA_TRY(check(a.cos, VECTRA_F32, {P, R2}));
  VECTRA_TRY(check(a.sin, VECTRA_F32, {P, R2}));
  if (R2 < 0 || 2 * R2 > D) return VECTRA_ERR_SHAPE;
  if (R2 > 1 && (a.cos.stride[1] != 1 || a.sin.stride[1] != 1))
    return VECTRA_ERR_LAYOUT;
  if (a.positions && a.position_bytes != 4 && a.position_bytes != 8)
    return VECTRA_ERR_DTYPE;
  *p = QkProblem{};
  if (axes != nullptr) {
    if (axes->count < 1 || axes->count > VECTRA_MAX_AXES)
      return VECTRA_ERR_UNSUPPORTED;
    if (a.positions == nullptr && B * N > 0) return VECTRA_ERR_NULL;
    int64_t sum = 0;
    for (int i = 0; i < axes->count; ++i) {
      if (axes->section[i] < 0) return VECTRA_ERR_SHAPE;
      p->first_pair[i] = int32_t(sum);
      if (sum % 4) p->whole_quads = false;
      sum += axes->section[i];
      if (sum > R2) return VECTRA_ERR_SHAPE;
    }
    if (sum != R2) return VECTRA_ERR_SHAPE;
    p->axes = axes->count;
    p->pos_sa = axes->stride;
  }
  const vectra_tensor* x[2] = {&a.q, &a.k};
  const vectra_tensor* w[2] = {&a.q_weight, &a.k_weight};
  for (int i = 0; i < 2; ++i) {
    QkSide& s = p->side[i];
    s.x = x[i]->data;
    s.H = int32_t(x[i]->size[1]);
    for (int j = 0; j < 4; ++j) s.sx[j] = x[i]->stride[j];
    if (present(*w[i])) {
      if (w[i]->dtype != a.q.dtype && w[i]->dtype != VECTRA_F32)
        return VECTRA_ERR_DTYPE;
      VECTRA_TRY(check(*w[i], w[i]->dtype, {D}));
      s.w = w[i]->data;
      s.sw = w[i]->stride[0];
      s.w_dtype = w[i]->dtype;
    }
  }
  p->dtype = a.q.dtype;
  p->interleaved = a.interleaved != 0;
  p->B = B;
  p->N = N;
  p->D = int32_t(D);
  p->R2 = int32_t(R2);
  p->P = P;
  p->cos = static_cast<const float*>(a.cos.data);
  p->sin = static_cast<const float*>(a.sin.data);
  p->cos_ld = a.cos.stride[0];
  p->sin_ld = a.sin.stride[0];
  p->pos = a.positions;
  p->pos_bytes = a.position_bytes;
  p->pos_sb = a.position_stride[0];
  p->pos_sn = a.position_stride[1];
  p->eps = float(a.eps);
  return VECTRA_OK;
}

int set_result(const vectra_tensor& t, const vectra_tensor& like,
               QkSide* s) {
  VECTRA_TRY(check(t, like.dtype, {like.size[0], like.size[1], like.size[2],
                                   like.size[3]}));
  if (t.size[3] > 1 && t.stride[3] != 1) return VECTRA_ERR_LAYOUT;
  s->out = const_cast<void*>(t.data);
  for (int j = 0; j < 4; ++j) s->so[j] = t.stride[j];
  return VECTRA_OK;
}

int qk_forward(const vectra_qk_args& a, const vectra_qk_axes* axes,
               cudaStream_t stream) {
  QkProblem p;
  VECTRA_TRY(build_qk(a, axes, &p));
  VECTRA_TRY(set_result(a.q_out, a.q, &p.side[0]));
  VECTRA_TRY(set_result(a.k_out, a.k, &p.side[1]));
  return launch_qk_forward(p, stream) == cudaSuccess ? VECTRA_OK
                                                     : VECTRA_ERR_CUDA;
}

int qk_backward_with(const vectra_qk_grad_args& a, const vectra_qk_axes* axes,
                     Workspace& ws, cudaStream_t stream) {
  QkProblem p;
  VECTRA_TRY(build_qk(a.fwd, axes, &p));
  const vectra_tensor* x[2] = {&a.fwd.q, &a.fwd.k};
  const vectra_tensor* dy[2] = {&a.dq_out, &a.dk_out};
  const vectra_tensor* dx[2] = {&a.dq, &a.dk};
  const vectra_tensor* dw[2] = {&a.dq_weight, &a.dk_weight};
  for (int i = 0; i < 2; ++i) {
    QkSide& s = p.side[i];
    VECTRA_TRY(check(*dy[i], p.dtype, {x[i]->size[0], x[i]->size[1],
                                       x[i]->size[2], x[i]->size[3]}));
    s.dy = dy[i]->data;
    for (int j = 0; j < 4; ++j) s.sy[j] = dy[i]->stride[j];
    VECTRA_TRY(set_result(*dx[i], *x[i], &s));
    if (present(*dw[i])) {
      if (s.w == nullptr) return VECTRA_ERR_NULL;
      VECTRA_TRY(check(*dw[i], s.w_dtype, {int64_t(p.D)}));
      s.dw = const_cast<void*>(dw[i]->data);
      s.sdw = dw[i]->stride[0];
    }
  }
  return to_status(run_qk_backward(p, ws, stream), ws);
}
int qk_backward(const vectra_qk_grad_args& a, Workspace& ws,
                cudaStream_t stream) {
  return qk_backward_with(a, nullptr, ws, stream);
}
// The workspace of the axes' call is its qk part's.
auto qk_axes_backward(const vectra_qk_axes& axes) {
  return [&axes](const vectra_qk_grad_args& a, Workspace& ws,
                 cudaStream_t stream) {
    return qk_backward_with(a, &axes, ws, stream);
  };
}

}  // namespace
}  // namespace vectra

using namespace vectra;

extern "C" {

int vectra_linear_forward(const vectra_linear_args* a, void* stream) {
  return run_with_workspace(a, stream, linear_forward);
}
int vectra_linear_backward(const vectra_linear_grad_args* a, void* stream) {
  return run_with_workspace(a, stream, linear_backward);
}
int vectra_gated_linear_forward(const vectra_gated_args* a, void* stream) {
  return run_with_workspace(a, stream, gated_forward);
}
int vectra_gated_linear_backward(const vectra_gated_grad_args* a,
                                 void* stream) {
  return run_with_workspace(a, stream, gated_backward);
}
int vectra_qk_norm_rope_forward(const vectra_qk_args* a, void* stream) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return qk_forward(*a, nullptr, static_cast<cudaStream_t>(stream));
}
int vectra_qk_norm_rope_backward(const vectra_qk_grad_args* a,
                                 void* stream) {
  return run_with_workspace(a, stream, qk_backward);
}
int vectra_qk_norm_rope_axes_forward(const vectra_qk_axes_args* a,
                                     void* stream) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return qk_forward(a->qk, &a->axes, static_cast<cudaStream_t>(stream));
}
int vectra_qk_norm_rope_axes_backward(const vectra_qk_axes_grad_args* a,
                                      void* stream) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return run_with_workspace(&a->qk, stream, qk_axes_backward(a->axes));
}
int64_t vectra_qk_norm_rope_axes_backward_workspace_bytes(
    const vectra_qk_axes_grad_args* a) {
  if (a == nullptr) return VECTRA_ERR_NULL;
  return workspace_of(&a->qk, qk_axes_backward(a->axes));
}

int64_t vectra_linear_forward_workspace_bytes(const vectra_linear_args* a) {
  return workspace_of(a, linear_forward);
}
int64_t vectra_linear_backward_workspace_bytes(
    const vectra_linear_grad_args* a) {
  return workspace_of(a, linear_backward);
}
int64_t vectra_gated_linear_forward_workspace_bytes(
    const vectra_gated_args* a) {
  return workspace_of(a, gated_forward);
}
int64_t vectra_gated_linear_backward_workspace_bytes(
    const vectra_gated_grad_args* a) {
  return workspace_of(a, gated_backward);
}
int64_t vectra_qk_norm_rope_backward_workspace_bytes(
    const vectra_qk_grad_args* a) {
  return workspace_of(a, qk_backward);
}

const char* vectra_block_strerror(int status) {
  switch (status) {
    case VECTRA_ERR_NULL:
      return "a required pointer is NULL";
    case VECTRA_ERR_RANK:
      return "a tensor has the wrong rank";
    case VECTRA_ERR_SHAPE:
      return "tensor sizes disagree";
    case VECTRA_ERR_DTYPE:
      return "tensors must share one of float32, float16, bfloat16 (rotation "
             "tables float32, norm weights that type or float32, positions "
             "int32 or int64)";
    case VECTRA_ERR_UNSUPPORTED:
      return "unsupported activation, a head width above 512 (in cross "
             "attention 256), a normalised row above 16384, more than 4 axes, "
             "or a size above 2^29 - 256";
    case VECTRA_ERR_LAYOUT:
      return "results and rotation tables need a unit inner stride and rows "
             "that do not overlap, a norm's statistics 16-byte alignment";
    case VECTRA_ERR_WORKSPACE:
      return "the workspace is too small or not 256-byte aligned";
    default:
      return vectra_rbf_strerror(status);
  }
}

}  // extern "C"
