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

Tensors are float32, float16 or bfloat16 with any strides, one type per
call. CUDA tensors run this library's sm_100a kernels on the current stream
(include/vectra_block.h is their C ABI); CPU tensors run an ATen formulation
in float32. Sums, norms and activations are in float32 and each result is
rounded once; with 16-bit tensors a gradient is also rounded before its
products with the weight and the input, and `linear` keeps act's argument for
the backward pass in its type. All three differentiate (once, in reverse;
forward mode raises NotImplementedError); under torch.no_grad(), or when no
argument needs a gradient, nothing is kept for a backward pass.
torch.autocast does not reach them: cast the inputs, mixed types raise.
A kernel whose wait runs out leaves its result unfinished, which
`_lib.check_device_errors` reports.

`RbfBlock` is a pre-norm transformer block built from them.
"""

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
    'vectra_block_strerror',
)

_OPS = torch.ops.vectra_b200
_LINEAR = _OPS.linear.default
_GATED = _OPS.gated_linear.default
_QK = _OPS.qk_norm_rope.default


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


# ---------------------------------------------------------------------------
# A block that runs them together.
# ---------------------------------------------------------------------------
class RbfBlock(nn.Module):
    """A pre-norm transformer block: RBF attention over normalised, rotated
    heads and a gated feed-forward layer, each with its residual.

    Serving (no gradient needed) runs attention on
    torch.ops.vectra.rbf_attention. That operator has no backward pass, so
    with gradients the same formula runs as matrix products, and the layers
    around it train through this module's operators. `.to(dtype)` and its
    like leave the rotation tables and `log_scale` in float32.
    """

    def __init__(self, d_model: int, heads: int, ffn: int,
                 activation: str = 'silu', max_positions: int = 4096,
                 device=None, dtype=None):
        super().__init__()
        if d_model % heads or (d_model // heads) % 2:
            raise ValueError('d_model must be an even multiple of heads')
        kw = {'device': device, 'dtype': dtype}
        self.heads, self.head_dim = heads, d_model // heads
        self.activation = activation
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
        max_positions rows makes its token NaN). Without positions, N above
        max_positions raises ValueError."""
        b, n, _ = x.shape
        if positions is None and n > self.cos.shape[0]:
            raise ValueError(f'{n} tokens, but max_positions is '
                             f'{self.cos.shape[0]}')
        qkv = linear(self.norm1(x), self.qkv.weight, self.qkv.bias)
        q, k, v = qkv.view(b, n, 3, self.heads,
                           self.head_dim).permute(2, 0, 3, 1, 4)
        q, k = qk_norm_rope(q, k, self.cos, self.sin, self.q_weight,
                            self.k_weight, positions)
        a = self._attend(q, k, v, key_bias)
        a = a.transpose(1, 2).reshape(b, n, -1)
        x = linear(a, self.out.weight, self.out.bias, residual=x)
        h = gated_linear(self.norm2(x), self.gate.weight, self.up.weight,
                         self.gate.bias, self.up.bias, self.activation)
        return linear(h, self.down.weight, self.down.bias, residual=x)


def strerror(status: int) -> str:
    """Text of a status of include/vectra_block.h's functions."""
    return _lib.LIB.vectra_block_strerror(status).decode()
