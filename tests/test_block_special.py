"""The transformer-block operators (vectra_b200.block) beside the ordinary:
values that are not finite or far out, and uses that a call has to refuse.

Tolerances are those of test_block.py unless a test derives its own.
"""

import math
import threading

import pytest
import torch

import vectra_b200
from tests.test_block import ACTS
from tests.test_block import DEVICES
from tests.test_block import Rand
from tests.test_block import TINY
from tests.test_block import TYPES
from tests.test_block import U
from tests.test_block import act64
from tests.test_block import close
from tests.test_block import d
from tests.test_block import slope64
from tests.test_block import sums
from tests.test_block import turn64
from vectra_b200 import block


# ---------------------------------------------------------------------------
# Forward mode
# ---------------------------------------------------------------------------
def _calls(device):
    """Each entry point with the tensors that can carry a tangent."""
    rand = Rand(3, device, torch.float32)
    cos, sin = block.rotation_tables(5, 8, device=device)
    return {
        'linear': (block.linear, [rand(3, 8), rand(4, 8), rand(4),
                                  rand(3, 4)]),
        'gated': (block.gated_linear, [rand(3, 8), rand(4, 8), rand(4, 8),
                                       rand(4), rand(4)]),
        'qk': (block.qk_norm_rope, [rand(2, 3, 5, 8), rand(2, 1, 5, 8), cos,
                                    sin, rand(8), rand(8)]),
    }


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('op', ['linear', 'gated', 'qk'])
@pytest.mark.parametrize('grad', [False, True])
def test_forward_mode_is_refused(device, op, grad):
    """A tangent in any argument raises (dropped, it would read as zero)."""
    fun, args = _calls(device)[op]
    ad = torch.autograd.forward_ad
    for i, t in enumerate(args):
        with ad.dual_level():
            tensors = [a.clone().requires_grad_(grad) for a in args]
            tensors[i] = ad.make_dual(tensors[i], torch.ones_like(t))
            with pytest.raises(NotImplementedError):
                fun(*tensors)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                fun(*tensors)
        if i == 0 and not grad:
            one = lambda a: fun(a, *args[1:])  # noqa: E731
            with pytest.raises(NotImplementedError):
                torch.func.jvp(one, (t,), (torch.ones_like(t),))
            with pytest.raises(NotImplementedError):
                torch.func.jacfwd(one)(t)
        # Outside the level the same tensors run.
        fun(*args)


# ---------------------------------------------------------------------------
# Values that are not finite
# ---------------------------------------------------------------------------
# (rows, K, N) of a few rows, one CTA's tiles, a reduction in parts, and CTA
# pairs (16-bit types); odd columns among them.
KERNELS = [(4, 64, 72), (150, 64, 520), (130, 4096, 96), (2570, 192, 1032),
           (70, 72, 33)]


def _others_equal(got, clean, columns, dim, what):
    """All of `dim` but `columns` as without the special values."""
    keep = [i for i in range(clean.shape[dim]) if i not in columns]
    index = torch.tensor(keep, device=got.device)
    assert torch.equal(got.index_select(dim, index),
                       clean.index_select(dim, index)), what


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('size', KERNELS)
def test_nan_stays_in_its_column(device, dtype, act, size):
    """NaN in one weight row and in one bias entry: those columns only, in
    the result and in the gradients of the parameters."""
    m, k, n = size
    rand = Rand(m + k + n, device, dtype)
    x, dy = rand(m, k), rand(m, n)
    w, b = rand(n, k, scale=k**-0.5), rand(n)
    wu, bu = rand(n, k, scale=k**-0.5), rand(n)
    bad = (3, 6)

    def linear(*leaves):
        leaves = [t.clone().requires_grad_() for t in leaves]
        y = block.linear(x, *leaves, activation=act)
        return (y, *torch.autograd.grad(y, leaves, dy))

    def gated(*leaves):
        leaves = [t.clone().requires_grad_() for t in leaves]
        h = block.gated_linear(x, leaves[0], leaves[2], leaves[1], leaves[3],
                               act)
        return (h, *torch.autograd.grad(h, leaves, dy))

    clean, clean_h = linear(w, b), gated(w, b, wu, bu)
    w[bad[0], k // 2] = float('nan')
    b[bad[1]] = float('nan')
    for got, want, what in ((linear(w, b), clean, 'linear'),
                            (gated(w, b, wu, bu), clean_h, 'gated')):
        assert got[0][:, list(bad)].isnan().all(), what
        _others_equal(got[0], want[0], bad, 1, what)
        for i in range(1, len(got)):
            _others_equal(got[i], want[i], bad, 0, f'{what} gradient {i}')


def _close_or_past(got, want, bound, what):
    """`close`; what lies past the type's range is infinite (within its bound
    of the edge it may be either)."""
    most = torch.finfo(got.dtype).max
    sure = want.abs() - bound > most
    near = want.abs() + bound < most
    assert torch.equal(d(got)[sure], want[sure].sign() * float('inf')), what
    close(got[near], want[near], bound[near], what)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('rows', [40, 300])
@pytest.mark.parametrize('saved', [False, True])
def test_slopes_far_out(device, dtype, act, rows, saved):
    """Gates of up to 1e4 either side of zero, beside ordinary ones. The
    weights are zero, so the gates are the biases, exactly, and the slope is
    off by the 4e-6 (its float32 form), act by 2e-6 of the gate."""
    u = U[dtype]
    rand = Rand(rows, device, dtype)
    far = [50., 100., 1e3, 1e4, 25., 12., 7., -7., -12., -50., -1e3, -1e4]
    gates = torch.tensor([v for f in far for v in (f, -0.7, f, 2.5, f, 6.)])
    bg = gates.to(device, dtype)
    n, k = bg.numel(), 64
    x, dh = rand(rows, k), rand(rows, n)
    zero = x.new_zeros(n, k)
    bu = torch.full_like(bg, 0.75)
    ops = torch.ops.vectra_b200
    h, gate, up = ops.gated_linear_with_pre(x, zero, zero, bg, bu, act, True)
    if not saved:
        gate, up = gate.new_empty(0), up.new_empty(0)
    _, dw, db = ops.gated_linear_backward(dh, x, zero, zero, bg, bu, gate, up,
                                          act, True, True, True)
    g, dy = d(bg).expand(rows, n), d(dh)
    a, slope = act64(g, act), slope64(g, act)
    ab = 2e-6 * g.abs().clamp(min=1)
    tiny = TINY[dtype]
    close(h, 0.75 * a, 0.75 * ab * (1 + u) + u * 0.75 * a.abs() + tiny, 'h')
    for i, (want, off) in enumerate(((dy * 0.75 * slope,
                                      dy.abs() * 0.75 * 4e-6),
                                     (dy * a, dy.abs() * ab))):
        spread = off.sum(0) + sums(rows) * want.abs().sum(0)
        total = want.sum(0)
        _close_or_past(db[i], total,
                       spread * (1 + u) + u * total.abs() + tiny, 'db')
        # As rounded for the product.
        off = off * (1 + u) + u * want.abs() + tiny
        total = want.t() @ d(x)
        spread = off.t() @ d(x).abs() + sums(rows) * (
            want.abs().t() @ d(x).abs())
        _close_or_past(dw[i], total,
                       spread * (1 + u) + u * total.abs() + tiny, 'dw')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('size', KERNELS)
def test_infinite_preactivations(device, dtype, act, size):
    """Biases that are infinite, NaN or very large: every kernel gives what
    the definition gives in floating point (act(-inf) is -inf * 0, NaN, for
    the smooth ones), and so do the slopes (ReLU's is z > 0)."""
    m, k, n = size
    rand = Rand(m * 3 + n, device, dtype)
    big = 6e4 if dtype == torch.float16 else 1e30
    x, dy = rand(m, k), rand(m, n)
    w, b = rand(n, k, scale=k**-0.5), rand(n)
    far = [float('inf'), float('-inf'), float('nan'), big, -big]
    b[2:12:2] = torch.tensor(far, device=device)
    columns = torch.arange(2, 12, 2)
    z = torch.tensor(far, dtype=torch.float64)
    want, slope = act64(z, act), slope64(z, act)
    if act == 'relu':
        slope = (z > 0).double()
    leaf = b.clone().requires_grad_()
    y = block.linear(x, w, leaf, activation=act)
    db, = torch.autograd.grad(y, leaf, dy)
    checks = [('linear', y, want, db, slope)]
    wu, bu = rand(n, k, scale=0.01 / k), torch.ones_like(b)
    ops = torch.ops.vectra_b200
    h, gate, up = ops.gated_linear_with_pre(x, w, wu, b, bu, act, True)
    for saved in (True, False):
        if not saved:
            gate, up = gate.new_empty(0), up.new_empty(0)
        _, _, both = ops.gated_linear_backward(
            dy, x, w, wu, b, bu, gate, up, act, False, False, True)
        checks += [('dg', h, want, both[0], slope),
                   ('du', h, want, both[1], want)]
    for what, result, value, grad, factor in checks:
        got = d(result)[:, columns]
        value = value.expand(m, 5)
        assert torch.equal(got.isnan(), value.isnan()), what
        inf = value.isinf()
        assert torch.equal(got[inf], value[inf]), what
        fin = value.isfinite()
        # Beside the bias the product is nothing, or within the rounding of
        # the type; the up factor is 1 to within 0.01 x sqrt(k) / k.
        err = (got - value)[fin].abs()
        assert (err <= 0.03 * value[fin].abs()).all(), what
        total = (d(dy)[:, columns] * factor).sum(0)
        got = d(grad)[columns]
        assert torch.equal(got.isnan(), total.isnan()), what
        if what != 'du':
            fin = total.isfinite()
            spread = (d(dy).abs().sum(0)[columns][fin] * 0.03)
            assert ((got - total)[fin].abs() <= spread).all(), what


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('act', ['gelu', 'gelu_tanh', 'silu'])
@pytest.mark.parametrize('size', KERNELS)
def test_float32_tails(device, act, size):
    """float32 activations of -8 to -4 to a relative accuracy, by every
    kernel. The weights are zero, so z is the bias, exactly. An exponent of
    size e takes at most four roundings (its polynomial included) and so puts
    4 e 2^-24 on its exponential; the rest of the form is within 16 of
    them."""
    m, k, n = size
    rand = Rand(m, device, torch.float32)
    x, zero = rand(m, k), torch.zeros(n, k, device=device)
    b = torch.linspace(-8, -4, n, device=device)
    z = d(b)
    e = {'gelu': z * z / 2, 'silu': -z,
         'gelu_tanh': -math.sqrt(8 / math.pi) * (z + 0.044715 * z**3)}[act]
    # (act64's 1 + tanh is 0 from z = -6 on, in float64 too.)
    want = (z * torch.sigmoid(-e) if act == 'gelu_tanh' else
            act64(z, act)).expand(m, n)
    bound = (4 * e + 16) * 2.0**-24 * want.abs()
    close(block.linear(x, zero, b, activation=act), want, bound, 'linear')
    one = torch.ones_like(b)
    h = block.gated_linear(x, zero, zero, b, one, activation=act)
    close(h, want, bound, 'gated')
    # The slope, act(z) / z + z phi(z) or its like: terms of one size.
    leaf = b.clone().requires_grad_()
    db, = torch.autograd.grad(block.linear(x, zero, leaf, activation=act),
                              leaf, torch.ones(m, n, device=device))
    slope = slope64(z, act)
    if act == 'gelu_tanh':
        s = torch.sigmoid(-e)
        slope = s + z * s * (1 - s) * math.sqrt(8 / math.pi) * (
            1 + 3 * 0.044715 * z * z)
    size = (want[0] / z).abs() * (1 + z * z * (3 if act == 'gelu_tanh' else
                                               1))
    close(db, m * slope, m * (4 * e + 16 + m) * 2.0**-24 * size, 'db')


def _same_kinds(got, want, what):
    """NaN and infinities where `want` (float64) has them."""
    got = d(got)
    assert torch.equal(got.isnan(), want.isnan()), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    assert got[want.isfinite()].isfinite().all(), what


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', KERNELS)
def test_infinite_operands(device, dtype, size):
    """Infinities in x, the weight and the gradient: against finite numbers
    of either sign, zeros, other infinities and NaN, as in any product."""
    m, k, n = size
    rand = Rand(k + n, device, dtype)
    x, w, dy = rand(m, k), rand(n, k, scale=k**-0.5), rand(m, n)
    inf, nan = float('inf'), float('nan')
    w[2, 3] = 0
    clean = block.linear(x, w)
    x[0, 3], x[1, 5], x[2, 1], x[2, 9], x[3, 7] = inf, -inf, inf, -inf, -inf
    w[4, 5], w[6, 7], w[8, 3], w[10, 7] = inf, -inf, nan, inf
    dy[1, 4], dy[3, 12], dy[0, 6] = inf, -inf, 0
    xs, ws, g = d(x), d(w), d(dy)
    x.requires_grad_(), w.requires_grad_()
    y = block.linear(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    _same_kinds(y, xs @ ws.t(), 'y')
    _same_kinds(dx, g @ ws, 'dx')
    _same_kinds(dw, g.t() @ xs, 'dw')
    rows = list(range(4, m))
    cols = [i for i in range(n) if i not in (4, 6, 8, 10)]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    r = block.linear(x, w, activation='relu')
    _same_kinds(r, (xs @ ws.t()).clamp(min=0), 'relu')
    h = block.gated_linear(x, w, torch.ones_like(w), activation='none')
    _same_kinds(h, (xs @ ws.t()) * xs.sum(1, keepdim=True), 'gated')


# ---------------------------------------------------------------------------
# RbfBlock
# ---------------------------------------------------------------------------
CASTS = {
    'half': lambda m, device: m.half(),
    'bfloat16': lambda m, device: m.bfloat16(),
    'to': lambda m, device: m.to(torch.float16),
    'both': lambda m, device: m.to(device, torch.bfloat16),
    'back': lambda m, device: m.half().float(),
    'parent': lambda m, device: torch.nn.Sequential(m).to(torch.bfloat16)[0],
}


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('cast', CASTS)
def test_block_can_be_cast(device, cast):
    """The rotation tables and the attention's scale stay float32, bit for
    bit; everything else takes the type, and the block runs and trains."""
    torch.manual_seed(0)
    blk = block.RbfBlock(64, 4, 96, max_positions=32).to(device)
    blk.log_scale.data.uniform_(-2.5, -1.5)
    x = Rand(47, device, torch.float32)(3, 17, 64)
    blk(x).square().mean().backward()
    scale, grad = blk.log_scale.detach().clone(), blk.log_scale.grad.clone()
    blk = CASTS[cast](blk, device)
    dtype = blk.out.weight.dtype
    tables = block.rotation_tables(32, 16, device=device)
    for got, want in ((blk.cos, tables[0]), (blk.sin, tables[1]),
                      (blk.log_scale, scale), (blk.log_scale.grad, grad)):
        assert got.dtype == torch.float32 and torch.equal(got, want)
    assert {p.dtype for n, p in blk.named_parameters()
            if n != 'log_scale'} == {dtype}
    x = x.to(dtype)
    with torch.no_grad():
        served = blk(x)
    blk.zero_grad()
    trained = blk(x)
    assert served.dtype == trained.dtype == dtype
    assert torch.isfinite(served).all()
    trained.float().square().mean().backward()
    for name, p in blk.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert p.grad.dtype == p.dtype, name


def test_block_from_meta():
    """Tables that never had values are made on the first real device."""
    blk = block.RbfBlock(64, 4, 96, max_positions=32, device='meta')
    assert blk.cos.is_meta and blk.half().cos.dtype == torch.float32
    blk = blk.to_empty(device='cpu')
    cos, sin = block.rotation_tables(32, 16)
    assert torch.equal(blk.cos, cos) and torch.equal(blk.sin, sin)


@pytest.mark.parametrize('device', DEVICES)
def test_block_refuses_longer_sequences(device):
    """More tokens than rotations, without positions, raise instead of
    giving NaN; positions inside the tables serve them."""
    blk = block.RbfBlock(32, 2, 48, max_positions=8).to(device)
    x = Rand(5, device, torch.float32)(2, 9, 32)
    with torch.no_grad():
        assert torch.isfinite(blk(x[:, :8])).all()
        with pytest.raises(ValueError, match='max_positions'):
            blk(x)
        at = torch.arange(9, device=device) % 8
        assert torch.isfinite(blk(x, positions=at)).all()


# ---------------------------------------------------------------------------
# Saved values
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['none', 'gelu', 'silu'])
@pytest.mark.parametrize('size', [(2570, 192, 2056), (5001, 72, 1032),
                                  (257, 1100, 5000), (150, 64, 520)])
def test_saved_values(dtype, act, size):
    """The pre-activation beside the result, with and without a residual:
    within their bounds, the same with and without the other, and the same
    every time."""
    m, k, n = size
    u, tiny = U[dtype], TINY[dtype]
    rand = Rand(m, 'cuda', dtype)
    x, w, b, r = rand(m, k), rand(n, k, scale=k**-0.5), rand(n), rand(m, n)
    z = d(x) @ d(w).t() + d(b)
    off = sums(k) * (d(x).abs() @ d(w).abs().t() + d(b).abs())
    run = torch.ops.vectra_b200.linear_with_pre
    plain, pre = run(x, w, b, None, act, True)
    close(pre, z, off * (1 + u) + u * z.abs() + tiny, 'pre')
    want = act64(z, act)
    bound = 1.13 * off + 2e-6 * z.abs().clamp(min=1) + tiny
    close(plain, want, bound * (1 + u) + u * want.abs(), 'y')
    first = None
    for _ in range(20):
        y, again = run(x, w, b, r, act, True)
        assert torch.equal(again, pre)
        if first is None:
            first = y
            want = want + d(r)
            bound = bound + 2.0**-23 * want.abs()
            close(y, want, bound * (1 + u) + u * want.abs(), 'y + r')
            assert torch.equal(y, run(x, w, b, r, act, False)[0])
        assert torch.equal(y, first)


# ---------------------------------------------------------------------------
# What a backward pass keeps
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('k', [64, 1024])
@pytest.mark.parametrize('want', [(0,), (1,), (2,), (3,), (0, 2), (1, 2)])
def test_unneeded_inputs_may_change(device, dtype, k, want):
    """A backward pass holds only the inputs that its gradients read: the
    others may be written in place between forward and backward, and the
    gradients are those of the values before."""
    rand = Rand(k, device, dtype)
    m, n = 33, 48
    args = [rand(m, k), rand(n, k, scale=k**-0.5), rand(n), rand(m, n)]
    dy = rand(m, n)

    def grads(change):
        leaves = [t.clone().requires_grad_(i in want)
                  for i, t in enumerate(args)]
        # x, weight, bias and residual as intermediate results.
        use = [t * 1 for t in leaves]
        y = block.linear(*use, activation='gelu')
        held = {0: (1,), 1: (0,)}
        needed = {j for i in want for j in held.get(i, ())}
        if change:
            for j, t in enumerate(use):
                if j not in needed:
                    t.add_(1)
        return torch.autograd.grad(y, [leaves[i] for i in want], dy)

    for got, expected in zip(grads(True), grads(False)):
        assert torch.equal(got, expected)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('want', [(0,), (1,), (2,), (3,), (4,), (0, 3)])
def test_unneeded_inputs_may_change_gated(device, want):
    """The same where a gated layer's projections were saved (float32)."""
    rand = Rand(7, device, torch.float32)
    m, k, n = 33, 64, 48
    args = [rand(m, k), rand(n, k, scale=0.1), rand(n, k, scale=0.1), rand(n),
            rand(n)]
    dy = rand(m, n)

    def grads(change):
        leaves = [t.clone().requires_grad_(i in want)
                  for i, t in enumerate(args)]
        use = [t * 1 for t in leaves]
        y = block.gated_linear(*use)
        needed = {j for i in want for j in {0: (1, 2), 1: (0,),
                                            2: (0,)}.get(i, ())}
        if change:
            for j, t in enumerate(use):
                if j not in needed:
                    t.add_(1)
        return torch.autograd.grad(y, [leaves[i] for i in want], dy)

    for got, expected in zip(grads(True), grads(False)):
        assert torch.equal(got, expected)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('op', ['linear', 'gated_linear'])
def test_partial_gradients_trace(device, op):
    """Calls with frozen inputs go through AOT dispatch with static and
    dynamic shapes."""
    rand = Rand(5, device, torch.float32)
    args = [rand(6, 8), rand(4, 8), rand(4, 8)][:2 if op == 'linear' else 3]
    for i in range(len(args)):
        call = [t.clone().requires_grad_(i == j) for j, t in enumerate(args)]
        torch.library.opcheck(
            getattr(torch.ops.vectra_b200, op).default, tuple(call),
            test_utils=('test_schema', 'test_faketensor',
                        'test_aot_dispatch_static',
                        'test_aot_dispatch_dynamic'))


# ---------------------------------------------------------------------------
# qk_norm_rope
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dims', [(64, 16), (64, 32), (64, 64), (48, 0),
                                  (40, 16), (7, 6)])
@pytest.mark.parametrize('aligned', [True, False])
def test_infinite_components(device, dtype, interleaved, dims, aligned):
    """An infinite component of a vector, or of its gradient, reaches what
    the formula says, and its partner only where the two are rotated: the
    same for the 16-byte and the general kernel."""
    dim, r = dims
    rand = Rand(dim + r, device, dtype)
    b, h, n = 2, 3, 7
    cos, sin = block.rotation_tables(20, r, device=device)
    pos = torch.randint(1, 20, (b, n), generator=rand.gen)
    q, dq = rand(b, h, n, dim), rand(b, h, n, dim)
    inf = float('inf')
    for t in (q, dq):
        for e in range(dim):  # one vector each, as far as there are any
            i, j = divmod(e * 5 % dim, n)
            if i < h:
                t[0 if t is q else 1, i, j, e] = inf if e % 2 else -inf
    w = 1 + rand(dim, scale=0.1)
    if not aligned:
        wide = rand(b, h, n, dim + 1)
        wide[..., 1:] = q
        q = wide[..., 1:]
    q = q.detach().requires_grad_()
    w.requires_grad_()
    out, _ = block.qk_norm_rope(q, q.detach(), cos, sin, w, None,
                                pos.to(device), 1e-6, interleaved)
    dx, dw = torch.autograd.grad(out, [q, w], dq)
    c, s = d(cos)[pos][:, None], d(sin)[pos][:, None]
    v, g = d(q), d(dq)
    scale = (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    nrm = v * scale
    _same_kinds(out, turn64(nrm * d(w), c, s, interleaved), 'y')
    g = turn64(g, c, -s, interleaved)
    gw = g * d(w)
    _same_kinds(dx, scale * (gw - nrm * (gw * nrm).mean(-1, keepdim=True)),
                'dx')
    _same_kinds(dw, (g * nrm).sum((0, 1, 2)), 'dw')


# ---------------------------------------------------------------------------
# Products with tensor maps, in threads and graphs
# ---------------------------------------------------------------------------
# More than 64 rows, which the few-row kernel never takes: one CTA's tiles, a
# reduction in parts (two launches), CTA pairs.
TENSOR_MAPS = {'tile': (150, 64, 520), 'parts': (130, 4096, 96),
               'pair': (2570, 192, 2056)}


def _launches(call):
    before = vectra_b200.launch_count()
    out = call()
    return out, vectra_b200.launch_count() - before


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('size', TENSOR_MAPS)
def test_products_from_a_fresh_thread(dtype, size):
    """A thread without a current CUDA context encodes tensor maps, of
    operands and of results."""
    m, k, n = TENSOR_MAPS[size]
    rand = Rand(m, 'cuda', dtype)
    x, w, b, wu = rand(m, k), rand(n, k), rand(n), rand(n, k)
    for call in (lambda: block.linear(x, w, b, None, 'gelu'),
                 lambda: block.gated_linear(x, w, wu)):
        want, launches = _launches(call)
        planes = dtype == torch.float32  # split first, in a launch
        if size == 'parts':
            assert launches == 2 + planes
        torch.cuda.synchronize()
        got = []
        thread = threading.Thread(target=lambda c=call: got.append(c()))
        thread.start()
        thread.join()
        assert len(got) == 1 and torch.equal(got[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('size', TENSOR_MAPS)
def test_products_in_a_cuda_graph(dtype, size):
    """Forward and backward passes, captured and replayed on new inputs:
    tensor maps, clusters and workspaces of parts."""
    m, k, n = TENSOR_MAPS[size]
    rand = Rand(n, 'cuda', dtype)
    x, w, wu, b, dy = rand(m, k), rand(n, k), rand(n, k), rand(n), rand(m, n)
    ops = torch.ops.vectra_b200
    none = torch.empty(0, device='cuda')

    def step():
        y, pre = ops.linear_with_pre(x, w, b, dy, 'gelu', True)
        h = block.gated_linear(x, w, wu, b, b)
        return (y, h, *ops.linear_backward(dy, x, w, pre, 'gelu', True, True,
                                           True),
                *ops.gated_linear_backward(dy, x, w, wu, b, b, none, none,
                                           'silu', True, True, True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, launches = _launches(step)
    torch.cuda.current_stream().wait_stream(side)
    assert launches >= 8 + (size == 'parts')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in (x, w, dy):
        t.copy_(rand(*t.shape))
    for _ in range(2):
        graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
