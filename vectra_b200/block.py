"""The operators of a transformer block around RBF attention, on B200.

    y = linear(x, weight, bias, residual, activation)
        act(x W^T + b) + r in one kernel: a projection with its bias,
        activation and residual.
    h = gated_linear(x, w_gate, w_up, b_gate, b_up, activation)
        act(x Wg^T + bg) * (x Wu^T + bu): both projections of a gated
        feed-forward layer, the activation and the product in one kernel.
    q, k = qk_norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps,
                        interleaved)
        the RMS norm of every query and key head vector and the rotation of
        its position in one pass, ready for torch.ops.vectra.rbf_attention.
    q, k = qk_norm_rope_axes(q, k, cos, sin, positions, sections, ...)
        the same with positions on several axes (time, height, width).
    x, y = residual_norm(x, branch, weight, bias, gate, branch_weight,
                         residual_scale, p, rng, ...)
        a sublayer's result normalised, dropped out, gated and added to the
        scaled residual, and the next sublayer's norm, in one pass.
    y = dropout(x, p, rng, stream)
        dropout whose mask is a function of an element's index.
    o = cross_attention(q, k, v, scale, key_lengths)
        RBF attention to an encoder's states of another length, with shared
        key heads; with gradients, unlike torch.ops.vectra.rbf_attention.

Tensors are float32, float16 or bfloat16 with any strides, one type per
call. CUDA tensors run this library's sm_100a kernels on the current stream
(include/vectra_block.h is their C ABI); CPU tensors run an ATen formulation
in float32. Sums, norms and activations are in float32 and each result is
rounded once; with 16-bit tensors a gradient is also rounded before its
products with the weight and the input, and `linear` keeps act's argument for
the backward pass in its type. `cross_attention` takes weights and their
gradients into its products as two 16-bit numbers each, with 16-bit tensors: its
results are off by their own rounding. Like `residual_norm` it keeps what a
result's rounding left beside it for the backward pass.
All differentiate (once, in reverse, `dropout` again and again;
forward mode raises NotImplementedError); under torch.no_grad(), or when no
argument needs a gradient, nothing is kept for a backward pass.
torch.autocast does not reach them: cast the inputs, mixed types raise.
A kernel whose wait runs out leaves its result unfinished, which
`_lib.check_device_errors` reports.

`RbfBlock` is a pre-norm transformer block built from them, `RbfCrossBlock`
one that reads an encoder's states.
"""

import math

import torch
from torch import nn

from vectra_b200 import _lib
from vectra_b200 import custom_ops

ACTIVATIONS = ('none', 'relu', 'gelu', 'gelu_tanh', 'silu')

# Every symbol include/vectra_block.h declares.
EXPORTED = (
    'vectra_linear_forward',
    'vectra_linear_backward',
    'vectra_gated_linear_forward',
    'vectra_gated_linear_backward',
    'vectra_qk_norm_rope_forward',
    'vectra_qk_norm_rope_backward',
    'vectra_linear_forward_workspace_bytes',
    'vectra_linear_backward_workspace_bytes',
    'vectra_gated_linear_forward_workspace_bytes',
    'vectra_gated_linear_backward_workspace_bytes',
    'vectra_qk_norm_rope_backward_workspace_bytes',
    'vectra_qk_norm_rope_axes_forward',
    'vectra_qk_norm_rope_axes_backward',
    'vectra_dropout',
    'vectra_residual_norm_forward',
    'vectra_residual_norm_forward_train',
    'vectra_residual_norm_backward_train',
    'vectra_residual_norm_backward_train_workspace_bytes',
    'vectra_residual_norm_backward',
    'vectra_cross_attention_forward',
    'vectra_cross_attention_backward',
    'vectra_qk_norm_rope_axes_backward_workspace_bytes',
    'vectra_residual_norm_backward_workspace_bytes',
    'vectra_cross_attention_forward_workspace_bytes',
    'vectra_cross_attention_backward_workspace_bytes',
    'vectra_block_strerror',
)

_OPS = torch.ops.vectra_b200
_LINEAR = _OPS.linear.default
_GATED = _OPS.gated_linear.default
_QK = _OPS.qk_norm_rope.default
_AXES = _OPS.qk_norm_rope_axes.default
_DROPOUT = _OPS.dropout.default
_NORM = _OPS.residual_norm.default
_CROSS = _OPS.cross_attention.default


def linear(x, weight, bias=None, residual=None,
           activation: str = 'none') -> torch.Tensor:
    """act(x @ weight.T + bias) + residual.

    Args:
      x: [..., K].
      weight: [N, K].
      bias: Optional [N].
      residual: Optional [..., N] (expand a broadcast one; stride 0 is
        read in place).
      activation: 'none', 'relu', 'gelu' (erf), 'gelu_tanh' or 'silu'.

    Returns:
      [..., N], contiguous, in x's dtype.

    Raises:
      ValueError: shapes, dtypes or devices that do not agree, or an unknown
        activation.
    """
    return _LINEAR(x, weight, bias, residual, activation)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None,
                 activation: str = 'silu') -> torch.Tensor:
    """act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up).

    Args:
      x: [..., K].
      w_gate, w_up: [F, K].
      b_gate, b_up: Optional [F].
      activation: As in `linear`.

    Returns:
      [..., F], contiguous, in x's dtype.

    Raises:
      ValueError: as `linear`.
    """
    return _GATED(x, w_gate, w_up, b_gate, b_up, activation)


def qk_norm_rope(q, k, cos, sin, q_weight=None, k_weight=None,
                 positions=None, eps: float = 1e-6,
                 interleaved: bool = False):
    """RMS-normalises and rotates every query and key head vector.

    Each vector v becomes n = v / sqrt(mean(v^2) + eps), y = n * weight, and
    the first R = 2 * cos.shape[1] components of y turn in pairs (a, b) ->
    (a cos - b sin, b cos + a sin) by the table rows of the vector's
    position.

    Args:
      q: [B, Hq, N, D], D at most 512.
      k: [B, Hk, N, D].
      cos, sin: float32 [P, R / 2] tables (see `rotation_tables`), R <= D.
      q_weight, k_weight: Optional [D], in q's dtype or float32.
      positions: Optional int32 or int64, broadcastable to [B, N]; by default
        a token's index. A position outside [0, P) makes its vectors NaN.
      eps: Added to the mean square.
      interleaved: Pairs are (2i, 2i + 1) instead of (i, i + R / 2).

    Returns:
      (q, k) of the same shapes, laid out as
      `custom_ops.output_strides` says for each.

    Raises:
      ValueError: shapes, dtypes or devices that do not agree.
      NotImplementedError: D above 512.
    """
    return _QK(q, k, cos, sin, q_weight, k_weight, positions, eps,
               interleaved)


def qk_norm_rope_axes(q, k, cos, sin, positions, sections, q_weight=None,
                      k_weight=None, eps: float = 1e-6,
                      interleaved: bool = False):
    """`qk_norm_rope` with positions on one to four axes.

    The tables' pairs belong to the axes in order, sections[a] of them to axis
    a: pair i turns by entry i of the row that its axis' position names, so
    the tables' columns decide every pair's frequency.

    Args:
      q, k, cos, sin, q_weight, k_weight, eps, interleaved: As in
        `qk_norm_rope`.
      positions: int32 or int64, broadcastable to [A, B, N] (its first size is
        A). A position outside the tables makes its token's vectors NaN.
      sections: A pair counts, not negative, that add up to cos.shape[1].

    Returns, raises:
      As `qk_norm_rope`.
    """
    return _AXES(q, k, cos, sin, positions, sections, q_weight, k_weight, eps,
                 interleaved)


def dropout(x, p: float, rng=None, stream: int = 0) -> torch.Tensor:
    """Zeros a share p of x and scales the rest by the inverse of what is kept.

    The mask is a function of rng, stream and an element's index in row-major
    order (whatever the strides) and is never stored: the backward pass makes
    it again, and a captured graph takes a new one when rng is written between
    replays. Masks of different steps or streams are independent. An element
    that is not kept is 0, whatever it holds. p is taken to the nearest
    multiple of 2^-16 (the numbers: include/vectra_block.h, vectra_drop).

    Args:
      x: Any shape and strides.
      p: From 0 to 1.
      rng: int64 [2] on x's device, contiguous: (seed, step). All 64 bits of
        the seed and the low 32 of the step count. Not needed for p = 0. It
        must not change between a forward pass and its backward pass.
      stream: Keeps the masks of one step apart: a number for each place of
        a model that drops; its low 32 bits count.

    Returns:
      A tensor like x, contiguous.

    Raises:
      ValueError: p outside [0, 1], a type that is not supported, or an rng
        that is missing or not as above.
    """
    return _DROPOUT(x, p, rng, stream)


def residual_norm(x, branch=None, weight=None, bias=None, gate=None,
                  branch_weight=None, residual_scale: float = 1.0,
                  p: float = 0.0, rng=None, stream: int = 0,
                  eps: float = 1e-6, kind: str = 'rms', norm: bool = True):
    """What stands between two sublayers:

        u = norm(branch) * branch_weight    (u = branch without one)
        x_out = residual_scale * x + gate * dropout(u, p, rng, stream)
        y = norm(x_out) * weight + bias

    with norm(v) = v / sqrt(mean(v^2) + eps), of v - mean(v) for 'layer'.

    Args:
      x: [..., C], the residual stream, C at most 16384.
      branch: Like x, a sublayer's result; None: x_out is x.
      weight, bias: Optional [C], of the norm behind.
      gate: Optional, C last and before it x's sizes up to some dimension and
        ones from there on: [C], [B, 1, C] or [B, N, C] for x [B, N, C].
      branch_weight: Optional [C]: the branch is normalised first.
      residual_scale: Multiplies x.
      p, rng, stream: As in `dropout`, of the branch.
      kind: 'rms' or 'layer', of both norms.
      norm: False: no norm behind; y is None.

    Returns:
      (x_out, y), contiguous. y is formed from x_out before its rounding, and
      so are the gradients of its norm. Without a branch x_out is x itself.

    Raises:
      ValueError: shapes, dtypes or devices that do not agree, arguments of a
        branch or norm that is not there.
      NotImplementedError: C above 16384.
    """
    x_out, y = _NORM(x, branch, weight, bias, branch_weight, gate,
                     residual_scale, p, rng, stream, eps, kind, norm)
    return x if branch is None else x_out, y if norm else None


def cross_attention(q, k, v, scale, key_lengths=None) -> torch.Tensor:
    """RBF attention to states of another length: for query i of head h

        sum over j < key_lengths[b] of softmax_j(-scale |q_i - k_j|^2) v_j

    with the keys of head h // (H / Hk).

    Args:
      q: [B, H, Nq, D], D at most 256.
      k: [B, Hk, Nk, D], H a multiple of Hk.
      v: [B, Hk, Nk, Dv], Dv at most 256.
      scale: Broadcastable to [B, H, 1, 1], any float type. Zero and negative
        values are legal.
      key_lengths: Optional int32 or int64 [B]; values outside [0, Nk] count
        as the nearer end. Keys and values at or past a length are never used
        and have zero gradients, whatever they hold; a sequence of length 0
        has zero results.

    Returns:
      [B, H, Nq, Dv], laid out as `custom_ops.output_strides` says; the same
      bits with and without gradients. A NaN in a seen key or value reaches
      every query of its heads.

    Raises:
      ValueError: shapes, dtypes or devices that do not agree.
      NotImplementedError: D or Dv above 256.
    """
    return _CROSS(q, k, v, scale, key_lengths)


def rotation_tables(length: int, dim: int, base: float = 10000.0,
                    device=None):
    """(cos, sin), float32 [length, dim / 2]: the angles position *
    base^(-2i / dim), formed in float64."""
    half = dim // 2
    inv = base ** (-torch.arange(half, dtype=torch.float64) / half)
    angle = torch.arange(length, dtype=torch.float64)[:, None] * inv
    return (angle.cos().float().to(device), angle.sin().float().to(device))


# ---------------------------------------------------------------------------
# Fake implementations (shapes and layouts).
# ---------------------------------------------------------------------------
def _heads_like(t):
    return t.new_empty_strided(t.shape,
                               custom_ops.output_strides(t, t.shape[-1]))


@torch.library.register_fake('vectra_b200::linear')
def _linear_fake(x, weight, bias=None, residual=None, activation='none'):
    del bias, residual, activation
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.register_fake('vectra_b200::linear_with_pre')
def _linear_with_pre_fake(x, weight, bias, residual, activation, want_pre):
    del bias, residual, activation
    shape = (*x.shape[:-1], weight.shape[0])
    return x.new_empty(shape), x.new_empty(shape if want_pre else (0,))


@torch.library.register_fake('vectra_b200::linear_backward')
def _linear_backward_fake(dy, x, weight, pre, activation, need_dx, need_dw,
                          need_db):
    del dy, pre, activation
    return (x.new_empty(x.shape if need_dx else (0,)),
            x.new_empty(weight.shape if need_dw else (0,)),
            x.new_empty((weight.shape[0] if need_db else 0,)))


@torch.library.register_fake('vectra_b200::gated_linear')
def _gated_fake(x, w_gate, w_up, b_gate=None, b_up=None, activation='silu'):
    del w_up, b_gate, b_up, activation
    return x.new_empty((*x.shape[:-1], w_gate.shape[0]))


@torch.library.register_fake('vectra_b200::gated_linear_with_pre')
def _gated_with_pre_fake(x, w_gate, w_up, b_gate, b_up, activation,
                         want_pre):
    del w_up, b_gate, b_up, activation
    shape = (*x.shape[:-1], w_gate.shape[0])
    pre = shape if want_pre else (0,)
    return (x.new_empty(shape), x.new_empty(pre, dtype=torch.float32),
            x.new_empty(pre, dtype=torch.float32))


@torch.library.register_fake('vectra_b200::gated_linear_backward')
def _gated_backward_fake(dh, x, w_gate, w_up, b_gate, b_up, gate, up,
                         activation, need_dx, need_dw, need_db):
    del dh, w_up, b_gate, b_up, gate, up, activation
    return (x.new_empty(x.shape if need_dx else (0,)),
            x.new_empty((2, *w_gate.shape) if need_dw else (0,)),
            x.new_empty((2, w_gate.shape[0]) if need_db else (0,)))


@torch.library.register_fake('vectra_b200::qk_norm_rope')
def _qk_fake(q, k, cos, sin, q_weight=None, k_weight=None, positions=None,
             eps=1e-6, interleaved=False):
    del cos, sin, q_weight, k_weight, positions, eps, interleaved
    return _heads_like(q), _heads_like(k)


@torch.library.register_fake('vectra_b200::qk_norm_rope_backward')
def _qk_backward_fake(dq_out, dk_out, q, k, cos, sin, q_weight, k_weight,
                      positions, eps, interleaved, need_dw):
    del dq_out, dk_out, cos, sin, positions, eps, interleaved

    def weight(w):
        if w is None or not need_dw:
            return q.new_empty((0,))
        return w.new_empty(w.shape)

    return (_heads_like(q), _heads_like(k), weight(q_weight),
            weight(k_weight))


@torch.library.register_fake('vectra_b200::qk_norm_rope_axes')
def _axes_fake(q, k, cos, sin, positions, sections, q_weight=None,
               k_weight=None, eps=1e-6, interleaved=False):
    del cos, sin, positions, sections, q_weight, k_weight, eps, interleaved
    return _heads_like(q), _heads_like(k)


@torch.library.register_fake('vectra_b200::qk_norm_rope_axes_backward')
def _axes_backward_fake(dq_out, dk_out, q, k, cos, sin, positions, sections,
                        q_weight, k_weight, eps, interleaved, need_dw):
    del sections
    return _qk_backward_fake(dq_out, dk_out, q, k, cos, sin, q_weight,
                             k_weight, positions, eps, interleaved, need_dw)


@torch.library.register_fake('vectra_b200::dropout')
def _dropout_fake(x, p, rng=None, stream=0):
    del p, rng, stream
    return x.new_empty(x.shape)


@torch.library.register_fake('vectra_b200::residual_norm')
def _norm_fake(x, branch=None, weight=None, bias=None, branch_weight=None,
               gate=None, residual_scale=1.0, p=0.0, rng=None, stream=0,
               eps=1e-6, kind='rms', norm=True):
    return _norm_with_stats_fake(x, branch, weight, bias, branch_weight, gate,
                                 residual_scale, p, rng, stream, eps, kind,
                                 norm, False)[:2]


@torch.library.register_fake('vectra_b200::residual_norm_with_stats')
def _norm_with_stats_fake(x, branch, weight, bias, branch_weight, gate,
                          residual_scale, p, rng, stream, eps, kind, norm,
                          want_stats):
    del weight, bias, branch_weight, gate, residual_scale, p, rng, stream
    del eps, kind
    rows = math.prod(x.shape[:-1]) if want_stats and x.shape[-1] else 0
    return (x.new_empty(x.shape if branch is not None else (0,)),
            x.new_empty(x.shape if norm else (0,)),
            x.new_empty((rows, 4), dtype=torch.float32),
            x.new_empty(x.shape if want_stats and norm and
                        branch is not None and x.dtype != torch.float32
                        else (0,)))


@torch.library.register_fake('vectra_b200::residual_norm_backward')
def _norm_backward_fake(dx_out, dy, x_out, rest, stats, branch, weight,
                        branch_weight, gate, residual_scale, p, rng, stream,
                        eps, kind, need):
    del x_out, rest, stats, branch, weight, branch_weight, residual_scale, p, rng
    del stream, eps, kind
    g = dx_out if dy is None else dy
    c = g.shape[-1:]
    shapes = (g.shape, g.shape, c, c, c, () if gate is None else gate.shape)
    return tuple(g.new_empty(shape if need >> i & 1 else (0,))
                 for i, shape in enumerate(shapes))


def _rows_like(t, width):
    return t.new_empty_strided((*t.shape[:-1], width),
                               custom_ops.output_strides(t, width))


@torch.library.register_fake('vectra_b200::cross_attention')
def _cross_fake(q, k, v, scale, key_lengths=None):
    del k, scale, key_lengths
    return _rows_like(q, v.shape[-1])


@torch.library.register_fake('vectra_b200::cross_attention_with_lse')
def _cross_with_lse_fake(q, k, v, scale, key_lengths, want_lse):
    del k, scale, key_lengths
    rest = want_lse and q.dtype != torch.float32
    return (_rows_like(q, v.shape[-1]),
            q.new_empty(q.shape[:-1] if want_lse else (0, *q.shape[1:3]),
                        dtype=torch.float32),
            q.new_empty((*q.shape[:-1], v.shape[-1]) if rest else (0,)))


@torch.library.register_fake('vectra_b200::cross_attention_backward')
def _cross_backward_fake(dout, q, k, v, scale, key_lengths, out, lse, rest,
                         need_dq, need_dkv, need_dscale):
    del dout, scale, key_lengths, out, lse, rest

    def grad(t, need):
        return _rows_like(t, t.shape[-1]) if need else t.new_empty((0,))

    return (grad(q, need_dq), grad(k, need_dkv), grad(v, need_dkv),
            q.new_empty((q.shape[0] if need_dscale else 0, q.shape[1]),
                        dtype=torch.float32))


# ---------------------------------------------------------------------------
# Blocks that run them together.
# ---------------------------------------------------------------------------
class RbfBlock(nn.Module):
    """A pre-norm transformer block: RBF attention over normalised, rotated
    heads and a gated feed-forward layer, each with its residual.

    Serving (no gradient needed) runs attention on
    torch.ops.vectra.rbf_attention. That operator has no backward pass, so
    with gradients the same formula runs as matrix products, and the layers
    around it train through this module's operators. `.to(dtype)` and its
    like leave the rotation tables and `log_scale` in float32.

    With `sections`, positions have an axis each (`qk_norm_rope_axes`) and have
    to be given.
    """

    def __init__(self, d_model: int, heads: int, ffn: int,
                 activation: str = 'silu', max_positions: int = 4096,
                 device=None, dtype=None, sections=None):
        super().__init__()
        if d_model % heads or (d_model // heads) % 2:
            raise ValueError('d_model must be an even multiple of heads')
        if sections is not None and \
                sum(sections) != d_model // heads // 2:
            raise ValueError('sections must add up to half the head width')
        kw = {'device': device, 'dtype': dtype}
        self.heads, self.head_dim = heads, d_model // heads
        self.activation = activation
        self.sections = None if sections is None else tuple(sections)
        self.norm1 = nn.LayerNorm(d_model, **kw)
        self.qkv = nn.Linear(d_model, 3 * d_model, **kw)
        self.q_weight = nn.Parameter(torch.ones(self.head_dim, **kw))
        self.k_weight = nn.Parameter(torch.ones(self.head_dim, **kw))
        self.out = nn.Linear(d_model, d_model, **kw)
        self.log_scale = nn.Parameter(
            torch.full((1, heads, 1, 1), -2.0, device=device,
                       dtype=torch.float32))
        self.norm2 = nn.LayerNorm(d_model, **kw)
        self.gate = nn.Linear(d_model, ffn, **kw)
        self.up = nn.Linear(d_model, ffn, **kw)
        self.down = nn.Linear(ffn, d_model, **kw)
        cos, sin = rotation_tables(max_positions, self.head_dim,
                                   device=device)
        self.register_buffer('cos', cos, persistent=False)
        self.register_buffer('sin', sin, persistent=False)

    def _apply(self, fn, recurse=True):
        # What .to(), .half() and the like do to every tensor. The operators
        # take float32 tables only, and a scale rounded to 16 bits would move
        # every logit: these keep their type and values.
        tables, scale = (self.cos, self.sin), self.log_scale.detach()
        grad = self.log_scale.grad
        if grad is not None:
            grad = grad.detach()
        super()._apply(fn, recurse)
        if self.cos.is_meta < tables[0].is_meta:
            tables = rotation_tables(tables[0].shape[0], self.head_dim)
        elif self.cos.dtype == torch.float32:
            tables = (self.cos, self.sin)
        self.cos, self.sin = (t.to(self.cos.device) for t in tables)
        if self.log_scale.dtype != torch.float32:
            self.log_scale.grad = None
            self.log_scale.data = scale.to(self.log_scale.device)
            if grad is not None:
                self.log_scale.grad = grad.to(self.log_scale.device)
        return self

    def _attend(self, q, k, v, bias):
        scale = self.log_scale.exp()
        if not (torch.is_grad_enabled() and
                any(t.requires_grad for t in (q, k, v, scale))):
            return custom_ops.rbf_attention(q, k, v, scale, bias)
        q, k, v32 = q.float(), k.float(), v.float()
        d2 = (q.square().sum(-1, keepdim=True) +
              k.square().sum(-1).unsqueeze(-2) - 2 * q @ k.transpose(-1, -2))
        logits = -scale * d2.clamp(min=0)
        if bias is not None:
            logits = logits + bias
        return (logits.softmax(-1) @ v32).to(v.dtype)

    def forward(self, x, key_bias=None, positions=None):
        """x [B, N, d_model]; key_bias broadcastable to [B, 1|H, 1, N] (0 or
        -inf); positions as in `qk_norm_rope` (one outside the tables of
        max_positions rows makes its token NaN), with sections as in
        `qk_norm_rope_axes`. Without positions, sections or N above
        max_positions raise ValueError."""
        b, n, _ = x.shape
        if positions is None and self.sections is not None:
            raise ValueError('a block with sections needs positions')
        if positions is None and n > self.cos.shape[0]:
            raise ValueError(f'{n} tokens, but max_positions is '
                             f'{self.cos.shape[0]}')
        qkv = linear(self.norm1(x), self.qkv.weight, self.qkv.bias)
        q, k, v = qkv.view(b, n, 3, self.heads,
                           self.head_dim).permute(2, 0, 3, 1, 4)
        if self.sections is not None:
            q, k = qk_norm_rope_axes(q, k, self.cos, self.sin, positions,
                                     self.sections, self.q_weight,
                                     self.k_weight)
        else:
            q, k = qk_norm_rope(q, k, self.cos, self.sin, self.q_weight,
                                self.k_weight, positions)
        a = self._attend(q, k, v, key_bias)
        a = a.transpose(1, 2).reshape(b, n, -1)
        x = linear(a, self.out.weight, self.out.bias, residual=x)
        h = gated_linear(self.norm2(x), self.gate.weight, self.up.weight,
                         self.gate.bias, self.up.bias, self.activation)
        return linear(h, self.down.weight, self.down.bias, residual=x)


class RbfCrossBlock(nn.Module):
    """A transformer block whose attention reads an encoder's states: RBF
    cross attention and a gated feed-forward layer, each between two RMS
    norms, with a learned gate and dropout on its way into the residual
    stream.

    It runs the same operators with and without gradients. `.to(dtype)` and
    its like leave `log_scale` in float32.
    """

    # Dropout's streams of one block: attention, feed-forward, hidden layer.
    STREAMS = 3

    def __init__(self, d_model: int, d_states: int, heads: int,
                 kv_heads: int, ffn: int, activation: str = 'silu',
                 dropout: float = 0.0, residual_scale: float = 1.0,
                 device=None, dtype=None):
        super().__init__()
        if d_model % heads or heads % kv_heads:
            raise ValueError('d_model must be a multiple of heads, and heads '
                             'of kv_heads')
        kw = {'device': device, 'dtype': dtype}
        self.heads, self.kv_heads = heads, kv_heads
        self.head_dim = d_model // heads
        self.activation, self.p = activation, dropout
        self.residual_scale = residual_scale
        for name in ('norm1', 'norm2', 'attn_norm', 'ffn_norm', 'attn_gate',
                     'ffn_gate'):
            setattr(self, name, nn.Parameter(torch.ones(d_model, **kw)))
        self.q = nn.Linear(d_model, d_model, bias=False, **kw)
        self.kv = nn.Linear(d_states, 2 * kv_heads * self.head_dim,
                            bias=False, **kw)
        self.out = nn.Linear(d_model, d_model, bias=False, **kw)
        self.log_scale = nn.Parameter(
            torch.full((1, heads, 1, 1), -2.0, device=device,
                       dtype=torch.float32))
        self.gate = nn.Linear(d_model, ffn, bias=False, **kw)
        self.up = nn.Linear(d_model, ffn, bias=False, **kw)
        self.down = nn.Linear(ffn, d_model, bias=False, **kw)

    def _apply(self, fn, recurse=True):
        # As RbfBlock's.
        scale, grad = self.log_scale.detach(), self.log_scale.grad
        super()._apply(fn, recurse)
        if self.log_scale.dtype != torch.float32:
            self.log_scale.grad = None
            self.log_scale.data = scale.to(self.log_scale.device)
            if grad is not None:
                self.log_scale.grad = grad.detach().to(self.log_scale.device)
        return self

    def forward(self, x, states, state_lengths=None, rng=None,
                stream: int = 0):
        """x [B, N, d_model]; states [B, M, d_states], of which a sequence has
        state_lengths[b] (int32 or int64 [B]; all M by default). In training
        mode with dropout, rng is as in `dropout` and the block's streams are
        stream .. stream + STREAMS - 1."""
        b, n, _ = x.shape
        p = self.p if self.training else 0.0
        drop = {'p': p, 'rng': rng, 'residual_scale': self.residual_scale}
        _, y = residual_norm(x, weight=self.norm1)
        q = linear(y, self.q.weight).view(b, n, self.heads, self.head_dim)
        k, v = linear(states, self.kv.weight).view(
            b, states.shape[1], 2, self.kv_heads,
            self.head_dim).permute(2, 0, 3, 1, 4)
        a = cross_attention(q.transpose(1, 2), k, v, self.log_scale.exp(),
                            state_lengths)
        a = linear(a.transpose(1, 2).reshape(b, n, -1), self.out.weight)
        x, y = residual_norm(x, a, self.norm2, gate=self.attn_gate,
                             branch_weight=self.attn_norm, stream=stream,
                             **drop)
        h = gated_linear(y, self.gate.weight, self.up.weight,
                         activation=self.activation)
        if p > 0:
            h = dropout(h, p, rng, stream + 2)
        h = linear(h, self.down.weight)
        x, _ = residual_norm(x, h, gate=self.ffn_gate,
                             branch_weight=self.ffn_norm, stream=stream + 1,
                             norm=False, **drop)
        return x


def strerror(status: int) -> str:
    """Text of a status of include/vectra_block.h's functions."""
    return _lib.LIB.vectra_block_strerror(status).decode()
