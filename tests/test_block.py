"""linear, gated_linear and qk_norm_rope (vectra_b200.block) against plain
float64 formulations, on CPU tensors and, marked gpu, on the kernels.

Bounds. With u the unit roundoff of the tensors' type (2^-24, 2^-11, 2^-8
for float32, float16, bfloat16), a float32 sum of K products is off by at
most (K + 16) 2^-23 times the sum S of the products' magnitudes (2^-23, not
2^-24: the tensor cores may truncate), the activations' slopes are below
1.13 and their float32 forms off by 2e-6 of max(1, |z|), and the result is
rounded once: u |y|. A gradient dz enters its products rounded to the type,
and for `linear` it is formed from z in that type, where |z act''(z)| < 0.5:
dz is off by u (|dz| + |dy| / 2), which a product turns into at most that
summed against the other factor's magnitudes. float16's subnormal spacing
adds 2^-24 per rounding.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

import vectra_b200
from vectra_b200 import _lib
from vectra_b200 import block
from vectra_b200 import custom_ops

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11,
     torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 1e-38, torch.float16: 2.0**-24,
        torch.bfloat16: 1e-38}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ['none', 'relu', 'gelu', 'gelu_tanh', 'silu']


def act64(z, kind):
    if kind == 'none':
        return z
    if kind == 'relu':
        return z.clamp(min=0)
    if kind == 'silu':
        return z * torch.sigmoid(z)
    if kind == 'gelu':
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) *
                                     (z + 0.044715 * z**3)))


def slope64(z, kind):
    z = z.clone().requires_grad_()
    return torch.autograd.grad(act64(z, kind).sum(), z)[0]


class Rand:

    def __init__(self, seed, device, dtype):
        self.gen = torch.Generator().manual_seed(seed)
        self.device, self.dtype = device, dtype

    def __call__(self, *shape, scale=1.0):
        t = torch.randn(*shape, generator=self.gen) * scale
        return t.to(self.device, self.dtype)


def d(t):
    return t.detach().double().cpu()


def close(got, want, bound, what=''):
    assert got.shape == want.shape, what
    err = (d(got) - want).abs()
    assert torch.isfinite(d(got)).all(), what
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f'{what}: error is {worst:.2f} of its bound'


def sums(n):
    return (n + 16) * 2.0**-23


def check_linear(x, w, b, r, act, dy=None):
    """Result (and gradients for dy) of block.linear within bounds."""
    u, tiny = U[x.dtype], TINY[x.dtype]
    leaves = [t for t in (x, w, b, r) if t is not None]
    if dy is not None:
        for t in leaves:
            t.requires_grad_()
    y = block.linear(x, w, b, r, act)
    k, n = w.shape[1], w.shape[0]
    xs, ws = d(x).reshape(-1, k) if k else d(x).reshape(
        math.prod(x.shape[:-1]), 0), d(w)
    m = xs.shape[0]
    z, s = xs @ ws.t(), xs.abs() @ ws.abs().t()
    if b is not None:
        z, s = z + d(b), s + d(b).abs()
    want = act64(z, act)
    zerr = sums(k) * s
    bound = 1.13 * zerr + 2e-6 * z.abs().clamp(min=1) + tiny
    if r is not None:
        want = want + d(r).reshape(m, n)
        bound = bound + 2.0**-23 * want.abs()
    assert y.dtype == x.dtype and y.is_contiguous()
    assert y.shape == (*x.shape[:-1], n)
    close(y.reshape(m, n), want, bound * (1 + u) + u * want.abs(), 'y')
    if dy is None:
        return y
    grads = torch.autograd.grad(y, leaves, dy)
    got = dict(zip([i for i, t in enumerate((x, w, b, r)) if t is not None],
                   grads))
    g = d(dy).reshape(m, n)
    dz = g * slope64(z, act)
    # Rounding of z and of dz, the float32 error of z (|act''| < 1.2), and
    # the slope's own error.
    dzb = u * (dz.abs() + 0.5 * g.abs()) + g.abs() * (
        1.2 * zerr * (1 + u) + 4e-6) + 2 * tiny
    if act == 'none':
        dzb = torch.zeros_like(dzb)
    for i, want, spread, count in (
            (0, dz @ ws, dzb @ ws.abs() + sums(n) * (dz.abs() @ ws.abs()),
             n),
            (1, dz.t() @ xs,
             dzb.t() @ xs.abs() + sums(m) * (dz.abs().t() @ xs.abs()), m)):
        del count
        shape = (x if i == 0 else w).shape
        close(got[i], want.reshape(shape),
              (spread * (1 + u) + u * want.abs() + tiny).reshape(shape),
              ('dx', 'dw')[i])
    if b is not None:
        spread = dzb.sum(0) + sums(m) * dz.abs().sum(0)
        close(got[2], dz.sum(0),
              spread * (1 + u) + u * dz.sum(0).abs() + tiny, 'db')
    if r is not None:
        assert torch.equal(got[3], dy)
    return y


def check_gated(x, wg, wu, bg, bu, act, dy=None):
    u, tiny = U[x.dtype], TINY[x.dtype]
    leaves = [t for t in (x, wg, wu, bg, bu) if t is not None]
    if dy is not None:
        for t in leaves:
            t.requires_grad_()
    h = block.gated_linear(x, wg, wu, bg, bu, act)
    k, f = wg.shape[1], wg.shape[0]
    m = math.prod(x.shape[:-1])
    xs, wgs, wus = d(x).reshape(m, k), d(wg), d(wu)
    g, sg = xs @ wgs.t(), xs.abs() @ wgs.abs().t()
    p, sp = xs @ wus.t(), xs.abs() @ wus.abs().t()
    if bg is not None:
        g, sg = g + d(bg), sg + d(bg).abs()
    if bu is not None:
        p, sp = p + d(bu), sp + d(bu).abs()
    a = act64(g, act)
    ge, pe = sums(k) * sg, sums(k) * sp
    ab = 1.13 * ge + 2e-6 * g.abs().clamp(min=1)
    want = a * p
    bound = ab * (p.abs() + pe) + a.abs() * pe + 2.0**-23 * want.abs() + tiny
    assert h.dtype == x.dtype and h.is_contiguous()
    close(h.reshape(m, f), want, bound * (1 + u) + u * want.abs(), 'h')
    if dy is None:
        return h
    grads = torch.autograd.grad(h, leaves, dy)
    got = dict(zip([i for i, t in enumerate((x, wg, wu, bg, bu))
                    if t is not None], grads))
    up = d(dy).reshape(m, f)
    slope = slope64(g, act)
    dg, du = up * p * slope, up * a
    sb = 1.2 * ge + 4e-6
    dgb = up.abs() * (sb * (p.abs() + pe) + 1.13 * pe)
    dub = up.abs() * ab
    dgs = dgb * (1 + u) + u * dg.abs() + tiny  # as rounded for the products
    dus = dub * (1 + u) + u * du.abs() + tiny
    want = dg @ wgs + du @ wus
    spread = (dgs @ wgs.abs() + dus @ wus.abs() + sums(2 * f) *
              (dg.abs() @ wgs.abs() + du.abs() @ wus.abs()))
    close(got[0], want.reshape(x.shape),
          (spread * (1 + u) + u * want.abs() + tiny).reshape(x.shape), 'dx')
    for i, t, ts in ((1, dg, dgs), (2, du, dus)):
        want = t.t() @ xs
        spread = ts.t() @ xs.abs() + sums(m) * (t.abs().t() @ xs.abs())
        close(got[i], want, spread * (1 + u) + u * want.abs() + tiny,
              ('', 'dwg', 'dwu')[i])
    for i, t, tb in ((3, dg, dgb), (4, du, dub)):
        if i not in got:
            continue
        want = t.sum(0)
        spread = tb.sum(0) + sums(m) * t.abs().sum(0)
        close(got[i], want, spread * (1 + u) + u * want.abs() + tiny, 'db')
    return h


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------
# (rows, K, N): single tokens, few tokens, tile edges, odd and tiny sizes,
# a long reduction over few outputs.
SIZES = [(1, 64, 64), (1, 4096, 200), (2, 1, 1), (3, 7, 5), (8, 512, 136),
         (9, 520, 72), (16, 100, 96), (17, 256, 264), (33, 1000, 31),
         (64, 128, 128), (65, 72, 300), (127, 96, 257), (128, 192, 256),
         (130, 64, 520), (257, 136, 129), (300, 2048, 8), (515, 64, 64)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_linear_sizes(device, dtype, size):
    m, k, n = size
    rand = Rand(m * 1000003 + k * 1009 + n, device, dtype)
    act = ACTS[(m + k + n) % 5]
    check_linear(rand(m, k), rand(n, k, scale=k**-0.5),
                 rand(n) if m % 2 else None,
                 rand(m, n) if n % 2 == 0 else None, act, rand(m, n))


# Enough tiles for every launch shape: wide results, long and short
# reductions, ragged edges, weight gradients over many rows.
LARGE = [(2570, 192, 2056), (5001, 72, 1032), (1030, 2304, 600),
         (257, 1100, 5000), (20000, 64, 72), (700, 520, 1304)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', LARGE)
def test_large_products(dtype, size):
    m, k, n = size
    rand = Rand(m + k + n, 'cuda', dtype)
    check_linear(rand(m, k), rand(n, k, scale=k**-0.5), rand(n), rand(m, n),
                 'gelu', rand(m, n))
    check_gated(rand(m, k), rand(n, k, scale=k**-0.5),
                rand(n, k, scale=k**-0.5), rand(n), rand(n), 'silu',
                rand(m, n))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('rows', [5, 150])
def test_linear_activations(device, dtype, act, rows):
    rand = Rand(7, device, dtype)
    check_linear(rand(rows, 64, scale=3), rand(80, 64, scale=0.125),
                 rand(80), rand(rows, 80), act, rand(rows, 80))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows', [1, 6, 200])
def test_linear_layouts(device, dtype, rows):
    """Strided, offset and broadcast operands give what contiguous ones do."""
    rand = Rand(11, device, dtype)
    k, n = 72, 88
    wide = rand(rows, 3 * k + 1)
    x = wide[:, k + 1:2 * k + 1]                  # rows not 16-byte aligned
    w = rand(k, n).t()                            # [N, K], stride 1 along N
    bias = rand(2 * n)[::2]
    row = rand(n)
    y = check_linear(x.detach(), w.detach(), bias, row.expand(rows, n), 'gelu',
                     rand(rows, n))
    again = block.linear(x.contiguous(), w.contiguous(), bias.contiguous(),
                         row.expand(rows, n).contiguous(), 'gelu')
    np.testing.assert_allclose(d(y).numpy(), d(again).numpy(),
                               rtol=2 * U[dtype], atol=1e-5)
    xt = rand(k, rows).t()
    check_linear(xt.detach(), rand(n, 2 * k)[:, ::2].detach(), None, None,
                 'none', rand(1, 1).expand(rows, n))
    check_linear(rand(2, 3, rows, k).transpose(0, 2).detach(),
                 rand(n, k).detach(), None, None, 'silu',
                 rand(rows, 3, 2, n))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(0, 8, 16), (4, 0, 16), (4, 8, 0),
                                  (0, 0, 0)])
def test_linear_empty(device, dtype, size):
    """No rows, no outputs, or an empty sum (act(bias) + residual)."""
    m, k, n = size
    rand = Rand(3, device, dtype)
    check_linear(rand(m, k), rand(n, k), rand(n), rand(m, n), 'silu',
                 rand(m, n))


@pytest.mark.parametrize('device', DEVICES)
def test_linear_only_wanted_gradients(device):
    rand = Rand(5, device, torch.bfloat16)
    x, w, b, r = rand(20, 64), rand(48, 64), rand(48), rand(20, 48)
    dy = rand(20, 48)
    full = [t.clone().requires_grad_() for t in (x, w, b, r)]
    every = torch.autograd.grad(block.linear(*full, 'gelu'), full, dy)
    for i in range(4):
        one = [t.clone() for t in (x, w, b, r)]
        one[i].requires_grad_()
        got, = torch.autograd.grad(block.linear(*one, 'gelu'), one[i], dy)
        assert torch.equal(got, every[i])
    with torch.no_grad():
        assert not block.linear(*full, 'gelu').requires_grad


# ---------------------------------------------------------------------------
# gated_linear
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_gated_sizes(device, dtype, size):
    m, k, f = size
    rand = Rand(m * 1000003 + k * 1009 + f, device, dtype)
    act = ACTS[1 + (m + k + f) % 4]
    check_gated(rand(m, k), rand(f, k, scale=k**-0.5),
                rand(f, k, scale=k**-0.5), rand(f) if m % 2 else None,
                rand(f) if k % 2 == 0 else None, act, rand(m, f))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('rows', [5, 150])
def test_gated_activations(device, dtype, act, rows):
    rand = Rand(17, device, dtype)
    check_gated(rand(rows, 64, scale=3), rand(80, 64, scale=0.125),
                rand(80, 64, scale=0.125), rand(80), rand(80), act,
                rand(rows, 80))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows', [1, 6, 200])
def test_gated_layouts(device, dtype, rows):
    rand = Rand(13, device, dtype)
    k, f = 72, 88
    both = rand(2 * f, k)
    x = rand(rows, k + 3)[:, 3:]
    check_gated(x.detach(), both[:f].detach(), both[f:].detach(), None,
                rand(2 * f)[::2], 'silu', rand(rows, f))
    check_gated(rand(k, rows).t().detach(), rand(k, f).t().detach(),
                both[1::2].detach(), None, None, 'gelu_tanh',
                rand(1, 1).expand(rows, f))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(0, 8, 16), (4, 0, 16), (4, 8, 0)])
def test_gated_empty(device, dtype, size):
    m, k, f = size
    rand = Rand(3, device, dtype)
    check_gated(rand(m, k), rand(f, k), rand(f, k), rand(f), rand(f), 'silu',
                rand(m, f))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(1, 64, 64), (7, 40, 33), (70, 96, 200),
                                  (300, 264, 136), (40, 1100, 72)])
def test_gated_backward_without_saved_values(device, dtype, size):
    """The backward operator with gate and up saved, and formed again: the
    same gradients but for the order of float32 sums (each is within half an
    output rounding and the accumulation's error, so they differ by at most
    two roundings of dz or of the result)."""
    m, k, f = size
    rand = Rand(19, device, dtype)
    x, dh = rand(m, k), rand(m, f)
    wg, wu = rand(f, k, scale=k**-0.5), rand(f, k, scale=k**-0.5)
    bg, bu = rand(f), rand(f)
    ops = torch.ops.vectra_b200
    for act in ('silu', 'gelu', 'gelu_tanh', 'relu', 'none'):
        _, gate, up = ops.gated_linear_with_pre(x, wg, wu, bg, bu, act, True)
        none = gate.new_empty(0)
        for sums in (True, False):
            want = ops.gated_linear_backward(dh, x, wg, wu, bg, bu, gate, up,
                                             act, True, True, sums)
            got = ops.gated_linear_backward(dh, x, wg, wu, bg, bu, none,
                                            none, act, True, True, sums)
            # dz differs by one rounding where it lies between two values;
            # a product sums those against factors of order 1.
            for a, b, n in zip(got, want, (2 * f, m, m)):
                assert a.shape == b.shape
                scale = 16 * U[dtype] * math.sqrt(n) + 16 * U[dtype] * d(
                    b).abs() + 1e-4
                assert ((d(a) - d(b)).abs() <= scale).all()


@pytest.mark.parametrize('device', DEVICES)
def test_gated_only_wanted_gradients(device):
    rand = Rand(5, device, torch.float16)
    args = [rand(20, 64), rand(48, 64), rand(48, 64), rand(48), rand(48)]
    dy = rand(20, 48)
    full = [t.clone().requires_grad_() for t in args]
    every = torch.autograd.grad(block.gated_linear(*full), full, dy)
    for i in range(5):
        one = [t.clone() for t in args]
        one[i].requires_grad_()
        got, = torch.autograd.grad(block.gated_linear(*one), one[i], dy)
        assert torch.equal(got, every[i])


# ---------------------------------------------------------------------------
# qk_norm_rope
# ---------------------------------------------------------------------------
def turn64(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    head, tail = x[..., :r], x[..., r:]
    a, b = ((head[..., 0::2], head[..., 1::2]) if interleaved else
            (head[..., :r // 2], head[..., r // 2:]))
    a, b = a * cos - b * sin, b * cos + a * sin
    head = (torch.stack([a, b], -1).flatten(-2) if interleaved else
            torch.cat([a, b], -1))
    return torch.cat([head, tail], -1)


def check_qk(q, k, cos, sin, qw, kw, positions, eps, interleaved, dq=None,
             dk=None):
    u, tiny = U[q.dtype], TINY[q.dtype]
    args = [q, k, qw, kw]
    if dq is not None:
        for t in args:
            if t is not None:
                t.requires_grad_()
    got = block.qk_norm_rope(q, k, cos, sin, qw, kw, positions, eps,
                             interleaved)
    b, _, n, dim = q.shape
    pos = (torch.arange(n) if positions is None else
           positions.cpu().long()).expand(b, n)
    c, s = d(cos)[pos][:, None], d(sin)[pos][:, None]
    grads = {}
    if dq is not None:
        leaves = [t for t in args if t is not None]
        grads = dict(zip([i for i, t in enumerate(args) if t is not None],
                         torch.autograd.grad(got, leaves, [dq, dk])))
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        assert got[i].stride() == custom_ops.output_strides(x, dim)
        v = d(x)
        r = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
        nrm = v * r
        y = nrm if w is None else nrm * d(w)
        want = turn64(y, c, s, interleaved)
        # float32 mean of D squares, rsqrt (2 ulp), products and rotation.
        f = (dim + 32) * 2.0**-24
        size = turn64(y.abs(), c.abs(), -s.abs(), interleaved).abs() + \
            turn64(y.abs(), c.abs(), s.abs(), interleaved).abs()
        close(got[i], want, u * want.abs() * (1 + f) + f * size + tiny,
              'qk'[i])
        if dy is None:
            continue
        g = turn64(d(dy), c, -s, interleaved)
        gm = turn64(d(dy).abs(), c.abs(), -s.abs(), interleaved).abs() + \
            turn64(d(dy).abs(), c.abs(), s.abs(), interleaved).abs()
        gw, gwm = (g, gm) if w is None else (g * d(w), gm * d(w).abs())
        dx = r * (gw - nrm * (gw * nrm).mean(-1, keepdim=True))
        spread = r * (gwm + nrm.abs() *
                      (gwm * nrm.abs()).mean(-1, keepdim=True))
        close(grads[i], dx, u * dx.abs() * (1 + f) + 3 * f * spread + tiny,
              'd' + 'qk'[i])
        assert grads[i].stride() == custom_ops.output_strides(x, dim)
        if w is not None:
            dw = (g * nrm).sum((0, 1, 2))
            rows = v.numel() // max(dim, 1)
            spread = (gm * nrm.abs()).sum((0, 1, 2))
            close(grads[2 + i], dw, U[w.dtype] * dw.abs() * (1 + f) +
                  (3 * f + sums(rows)) * spread + tiny,
                  'd' + 'qk'[i] + 'w')
    return got


# (B, Hq, Hk, N, D, R): single tokens, odd widths, partial rotation, grouped
# keys, no rotation at all.
QK_SIZES = [(1, 1, 1, 1, 64, 64), (5, 8, 2, 1, 128, 128),
            (2, 4, 4, 33, 32, 32), (2, 6, 3, 17, 80, 40),
            (1, 3, 1, 65, 96, 96), (2, 2, 2, 9, 256, 256),
            (1, 2, 1, 5, 7, 6), (3, 2, 2, 4, 1, 0), (2, 1, 1, 3, 512, 512),
            (1, 5, 5, 130, 64, 16), (2, 2, 1, 7, 40, 0),
            (1, 1, 1, 3, 511, 2), (2, 3, 3, 21, 128, 64)]


def qk_inputs(rand, b, hq, hk, n, dim, fused):
    if not fused:
        return rand(b, hq, n, dim), rand(b, hk, n, dim)
    qkv = rand(b, n, (hq + 2 * hk) * dim)
    q = qkv[..., :hq * dim].view(b, n, hq, dim).transpose(1, 2)
    k = qkv[..., hq * dim:(hq + hk) * dim].view(b, n, hk, dim).transpose(1, 2)
    return q.detach(), k.detach()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', QK_SIZES)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('fused', [False, True])
def test_qk_sizes(device, dtype, size, interleaved, fused):
    b, hq, hk, n, dim, r = size
    rand = Rand(dim * 31 + n, device, dtype)
    q, k = qk_inputs(rand, b, hq, hk, n, dim, fused)
    cos, sin = block.rotation_tables(n + 50, r, device=device)
    positions = torch.randint(0, n + 50, (b, n), generator=rand.gen).to(
        device)
    check_qk(q, k, cos, sin, 1 + rand(dim, scale=0.2),
             1 + rand(dim, scale=0.2), positions, 1e-5, interleaved,
             rand(b, hq, n, dim), rand(b, hk, n, dim))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_qk_options(device, dtype):
    """No weights, float32 weights, int32, row and default positions, odd
    strides, broadcast gradients."""
    rand = Rand(23, device, dtype)
    cos, sin = block.rotation_tables(40, 64, device=device)
    q, k = qk_inputs(rand, 2, 4, 2, 19, 64, True)
    check_qk(q.clone(), k.clone(), cos, sin, None, None, None, 1e-6, False,
             rand(2, 4, 19, 64), rand(2, 2, 19, 64))
    f32w = 1 + 0.2 * torch.randn(2, 64, generator=rand.gen).to(device)
    row = torch.randint(0, 40, (19,), generator=rand.gen).to(device)
    check_qk(q.clone(), k.clone(), cos, sin, f32w[0].clone(), None,
             row.int(), 1e-6, True, rand(2, 4, 19, 64),
             rand(1, 1, 1, 1).expand(2, 2, 19, 64))
    each = torch.randint(0, 40, (2, 1), generator=rand.gen).to(device)
    odd = rand(2, 4, 19, 129)[..., ::2][..., :64]
    shifted = rand(2, 2, 19, 65)[..., 1:]
    check_qk(odd.detach(), shifted.detach(), cos, sin,
             (1 + rand(128, scale=0.1))[::2].detach(), f32w[1].clone(), each,
             1e-6, False, rand(2, 19, 4, 64).transpose(1, 2),
             rand(2, 2, 64, 19).transpose(2, 3))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_qk_zero_vectors(device, dtype):
    """A zero vector stays zero and its gradient is finite (eps)."""
    rand = Rand(29, device, dtype)
    cos, sin = block.rotation_tables(8, 64, device=device)
    q, k = rand(1, 2, 8, 64), rand(1, 2, 8, 64)
    q[0, 1, 3] = 0
    # r = 1000 there: keep its gradient inside float16.
    got = check_qk(q, k, cos, sin, None, None, None, 1e-6, False,
                   rand(1, 2, 8, 64, scale=0.1), rand(1, 2, 8, 64))
    assert (got[0][0, 1, 3] == 0).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dim', [64, 48])
def test_qk_positions_outside_the_tables(device, dim):
    """They make their vectors NaN, and no others."""
    rand = Rand(31, device, torch.bfloat16)
    cos, sin = block.rotation_tables(16, 32, device=device)
    q, k = rand(2, 3, 5, dim), rand(2, 1, 5, dim)
    positions = torch.tensor([[0, 15, 16, 3, 2], [-1, 1, 2, 2**40, 4]],
                             device=device)
    bad = torch.tensor([[0, 0, 1, 0, 0], [1, 0, 0, 1, 0]], dtype=torch.bool)
    q.requires_grad_()
    qo, ko = block.qk_norm_rope(q, k, cos, sin, None, None, positions)
    dq, = torch.autograd.grad(qo, q, torch.ones_like(qo))
    for t in (qo, ko, dq):
        nan = d(t).isnan()
        assert torch.equal(nan.any(-1).any(1), bad)
        assert torch.equal(nan.all(-1).all(1), bad)


@pytest.mark.parametrize('device', DEVICES)
def test_qk_empty(device):
    cos, sin = block.rotation_tables(4, 8, device=device)
    for shape, heads in (((0, 2, 3, 8), 1), ((2, 2, 0, 8), 1),
                         ((2, 0, 3, 8), 1), ((2, 2, 3, 8), 0)):
        q = torch.ones(shape, device=device, requires_grad=True)
        k = torch.ones((shape[0], heads, *shape[2:]), device=device)
        w = torch.ones(8, device=device, requires_grad=True)
        qo, ko = block.qk_norm_rope(q, k, cos, sin, w, w)
        assert qo.shape == q.shape and ko.shape == k.shape
        dq, dw = torch.autograd.grad(qo.sum() + ko.sum(), [q, w])
        assert dq.shape == q.shape and torch.isfinite(dw).all()
        if q.numel() == 0 and k.numel() == 0:
            assert (dw == 0).all()


@pytest.mark.parametrize('device', DEVICES)
def test_qk_only_one_result_used(device):
    rand = Rand(37, device, torch.float32)
    cos, sin = block.rotation_tables(8, 32, device=device)
    q, k, w = (rand(1, 2, 8, 32).requires_grad_(),
               rand(1, 2, 8, 32).requires_grad_(), rand(32).requires_grad_())
    qo, _ = block.qk_norm_rope(q, k, cos, sin, w, w)
    dy = rand(1, 2, 8, 32)
    dq, dk, dw = torch.autograd.grad(qo, [q, k, w], dy)
    assert (dk == 0).all()
    w2 = w.detach().clone().requires_grad_()
    qo2, _ = block.qk_norm_rope(q, k.detach(), cos, sin, w2, None)
    want_q, want_w = torch.autograd.grad(qo2, [q, w2], dy)
    assert torch.equal(dq, want_q) and torch.equal(dw, want_w)


# ---------------------------------------------------------------------------
# Gradients against differences.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('act', ['gelu', 'gelu_tanh', 'silu'])
@pytest.mark.parametrize('op', ['linear', 'gated', 'qk'])
def test_gradients_against_differences(device, act, op):
    """Central differences along random directions, float32.

    With step h the difference of F = <y, dy> is off by h^2 / 6 |F'''| and by
    2^-22 sum|y dy| / h; the inputs are of order 1 and the directions of unit
    length, so |F'''| stays below 30 |dy| and h = 2^-6 leaves less than
    2e-3 |dy|.
    """
    if op == 'qk' and act != 'silu':
        pytest.skip('no activation')
    rand = Rand(41, device, torch.float32)
    if op == 'linear':
        args = [rand(6, 12), rand(9, 12, scale=0.3), rand(9), rand(6, 9)]
        fun = lambda *a: [block.linear(*a, act)]  # noqa: E731
        dys = [rand(6, 9)]
    elif op == 'gated':
        args = [rand(6, 12), rand(9, 12, scale=0.3), rand(9, 12, scale=0.3),
                rand(9), rand(9)]
        fun = lambda *a: [block.gated_linear(*a, act)]  # noqa: E731
        dys = [rand(6, 9)]
    else:
        cos, sin = block.rotation_tables(5, 12, device=device)
        args = [rand(1, 2, 5, 16), rand(1, 1, 5, 16), rand(16), rand(16)]
        fun = lambda q, k, w, v: block.qk_norm_rope(  # noqa: E731
            q, k, cos, sin, w, v)
        dys = [rand(1, 2, 5, 16), rand(1, 1, 5, 16)]
    size = math.sqrt(sum(float(t.double().square().sum()) for t in dys))
    leaves = [t.clone().requires_grad_() for t in args]
    grads = torch.autograd.grad(fun(*leaves), leaves, dys)
    value = lambda a: sum(float((y.double() * t.double()).sum())  # noqa: E731
                          for y, t in zip(fun(*a), dys))
    h = 2.0**-6
    for i, t in enumerate(args):
        for _ in range(3):
            v = rand(*t.shape)
            v = v / v.norm()
            hi = [a + h * v if j == i else a for j, a in enumerate(args)]
            lo = [a - h * v if j == i else a for j, a in enumerate(args)]
            want = (value(hi) - value(lo)) / (2 * h)
            got = float((grads[i].double() * v.double()).sum())
            assert abs(got - want) <= 2e-3 * size, (i, got, want)


# ---------------------------------------------------------------------------
# Refusals and dispatch.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    def t(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device=device)

    x, w = t(3, 8), t(4, 8)
    for bad in (lambda: block.linear(x, w, activation='tanh'),
                lambda: block.linear(x, t(4, 7)),
                lambda: block.linear(x, t(8)),
                lambda: block.linear(x, w.half()),
                lambda: block.linear(x.double(), w.double()),
                lambda: block.linear(x, w, t(5)),
                lambda: block.linear(x, w, t(1, 4)),
                lambda: block.linear(x, w, t(4, dtype=torch.float16)),
                lambda: block.linear(x, w, None, t(4)),
                lambda: block.linear(x, w, None, t(3, 5)),
                lambda: block.linear(t(), w),
                lambda: block.gated_linear(x, w, t(5, 8)),
                lambda: block.gated_linear(x, w, w.half()),
                lambda: block.gated_linear(x, w, w, t(5)),
                lambda: block.gated_linear(x, w, w, None, t(4, 1)),
                lambda: block.gated_linear(x, w, w, activation='swish')):
        with pytest.raises(ValueError):
            bad()
    q, k, c = t(2, 3, 5, 8), t(2, 1, 5, 8), t(6, 4)
    long = lambda *s: t(*s, dtype=torch.int64)  # noqa: E731
    rope = block.qk_norm_rope
    for bad in (lambda: rope(q[0], k, c, c), lambda: rope(q, k[:1], c, c),
                lambda: rope(q, t(2, 1, 5, 6), c, c),
                lambda: rope(q, k.half(), c, c),
                lambda: rope(q.double(), k.double(), c, c),
                lambda: rope(q, k, c.half(), c.half()),
                lambda: rope(q, k, c, t(6, 3)),
                lambda: rope(q, k, t(6, 5), t(6, 5)),
                lambda: rope(q, k, t(6, 8)[:, ::2], c),
                lambda: rope(q, k, c, c, t(7)),
                lambda: rope(q, k, c, c, None, t(8).half()),
                lambda: rope(q, k, c, c, None, None, t(5)),
                lambda: rope(q, k, c, c, None, None, long(4)),
                lambda: rope(q, k, c, c, None, None, long(3, 5)),
                lambda: rope(q, k, c, c, None, None, long(1, 2, 5))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        rope(t(1, 1, 1, 520), t(1, 1, 1, 520), c, c)


@pytest.mark.parametrize('device', DEVICES)
def test_no_second_derivative(device):
    x = torch.randn(3, 8, device=device, requires_grad=True)
    w = torch.randn(4, 8, device=device, requires_grad=True)
    dx, = torch.autograd.grad(block.linear(x, w, activation='gelu').sum(), x,
                              create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def _op_calls(device):
    rand = Rand(43, device, torch.float32)
    leaf = lambda *s: rand(*s).requires_grad_()  # noqa: E731
    cos, sin = block.rotation_tables(5, 8, device=device)
    ops = torch.ops.vectra_b200
    return [
        (ops.linear.default, (leaf(3, 8), leaf(4, 8), leaf(4), leaf(3, 4),
                              'gelu')),
        (ops.linear.default, (leaf(2, 3, 8), leaf(4, 8))),
        (ops.gated_linear.default, (leaf(3, 8), leaf(4, 8), leaf(4, 8),
                                    leaf(4), leaf(4))),
        (ops.qk_norm_rope.default, (leaf(2, 3, 5, 8), leaf(2, 1, 5, 8), cos,
                                    sin, leaf(8), leaf(8))),
    ]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('case', range(4))
def test_opcheck(device, case):
    op, args = _op_calls(device)[case]
    torch.library.opcheck(op, args, test_utils=(
        'test_schema', 'test_faketensor', 'test_aot_dispatch_static',
        'test_aot_dispatch_dynamic'))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_block_runs_them_together(device, dtype):
    """RbfBlock serves what it trains: the attention operator and the
    differentiable formula agree, and every parameter gets a gradient."""
    torch.manual_seed(0)
    blk = block.RbfBlock(64, 4, 96, max_positions=32).to(device, dtype)
    blk.log_scale.data = blk.log_scale.data.float()
    blk.cos, blk.sin = (t.to(device) for t in block.rotation_tables(32, 16))
    x = Rand(47, device, dtype)(3, 17, 64)
    bias = torch.zeros(3, 1, 1, 17, device=device)
    bias[1, ..., 12:] = float('-inf')
    trained = blk(x, bias)
    with torch.no_grad():
        served = blk(x, bias)
    # The two attentions round their weights differently (once, to the
    # type, in the kernels); the residual stream is of order 4.
    np.testing.assert_allclose(d(trained).numpy(), d(served).numpy(),
                               rtol=0, atol=16 * U[dtype] + 1e-4)
    trained.float().square().mean().backward()
    for name, p in blk.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name


def test_exports():
    """The library exports what include/vectra_block.h declares."""
    import os
    import re
    header = os.path.join(os.path.dirname(os.path.dirname(
        os.path.abspath(__file__))), 'include', 'vectra_block.h')
    text = re.sub(r'/\*.*?\*/', '', open(header, encoding='utf-8').read(),
                  flags=re.S)
    declared = sorted(set(re.findall(r'VECTRA_API[^;]*?\b(vectra_\w+)\s*\(',
                                     text)))
    assert sorted(block.EXPORTED) == declared
    for name in declared:
        assert hasattr(_lib.LIB, name), name
    assert block.strerror(-13).startswith('the workspace')
    assert block.strerror(0) == 'ok'


class _LinearArgs(ctypes.Structure):
    """vectra_linear_args."""
    _fields_ = [(n, _lib.Tensor) for n in ('x', 'weight', 'bias', 'residual',
                                           'y', 'pre')] + [
        ('activation', ctypes.c_int32), ('workspace', ctypes.c_void_p),
        ('workspace_bytes', ctypes.c_size_t)]


def _abi_tensor(shape, dtype=_lib.BF16, strides=None, addr=0x10000):
    t = _lib.Tensor()
    t.data, t.dtype, t.ndim = addr, dtype, len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        t.size[i] = shape[i]
        t.stride[i] = step if strides is None else strides[i]
        step *= shape[i]
    return t


def test_abi_statuses():
    """The C entries answer statuses and sizes without touching a device."""
    size = _lib.LIB.vectra_linear_forward_workspace_bytes
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_void_p]
    call = _lib.LIB.vectra_linear_forward
    call.restype, call.argtypes = ctypes.c_int, [ctypes.c_void_p,
                                                 ctypes.c_void_p]

    def args(**over):
        a = _LinearArgs()
        a.x, a.weight = _abi_tensor((64, 4096)), _abi_tensor((512, 4096))
        a.y = _abi_tensor((64, 512))
        for name, value in over.items():
            setattr(a, name, value)
        return a

    def status(**over):
        return size(ctypes.byref(args(**over)))

    # 64 x 512 over 4,096: cut into parts, whose sums need the workspace.
    need = status()
    assert need > 0 and need % 256 == 0
    assert call(ctypes.byref(args()), None) == -13  # no workspace given
    assert call(ctypes.byref(args(workspace=0x10001,
                                  workspace_bytes=need)), None) == -13
    assert call(ctypes.byref(args(workspace=0x10000,
                                  workspace_bytes=need - 1)), None) == -13
    assert status(x=_abi_tensor((64, 4096), strides=(4100, 1))) > need
    assert size(None) == _lib.ERR_NULL
    assert status(x=_abi_tensor((64,))) == _lib.ERR_RANK
    assert status(weight=_abi_tensor((512, 4095))) == _lib.ERR_SHAPE
    assert status(y=_abi_tensor((64, 511))) == _lib.ERR_SHAPE
    assert status(x=_abi_tensor((64, 4096), _lib.F64)) == _lib.ERR_DTYPE
    assert status(weight=_abi_tensor((512, 4096), _lib.F16)) == _lib.ERR_DTYPE
    assert status(bias=_abi_tensor((511,))) == _lib.ERR_SHAPE
    assert status(residual=_abi_tensor((64, 512), _lib.F32)) == _lib.ERR_DTYPE
    assert status(y=_abi_tensor((64, 512), addr=None)) == _lib.ERR_NULL
    assert status(y=_abi_tensor((64, 512), strides=(512, 2))) == -12
    assert status(y=_abi_tensor((64, 512), strides=(500, 1))) == -12
    assert status(activation=5) == _lib.ERR_UNSUPPORTED
    assert status(x=_abi_tensor((2**30, 4096)),
                  y=_abi_tensor((2**30, 512))) == _lib.ERR_UNSUPPORTED
    # A handful of rows needs none; nor does an empty product.
    assert status(x=_abi_tensor((4, 4096)), y=_abi_tensor((4, 512))) == 0
    assert status(x=_abi_tensor((0, 4096)), y=_abi_tensor((0, 512))) == 0


# ---------------------------------------------------------------------------
# The kernels.
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_repeats_are_bit_identical(dtype):
    rand = Rand(53, 'cuda', dtype)
    x, w, wu = rand(515, 264), rand(200, 264), rand(200, 264)
    leaves = [t.requires_grad_() for t in (x, w, wu)]
    dy = rand(515, 200)
    before = vectra_b200.launch_count()
    first = None
    for _ in range(3):
        y = block.linear(x, w, None, None, 'gelu')
        h = block.gated_linear(x, w, wu)
        got = [y, h, *torch.autograd.grad([y, h], leaves, [dy, dy])]
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    assert vectra_b200.launch_count() > before


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_rows_do_not_depend_on_each_other(dtype):
    """NaN and infinities in one token stay in its rows."""
    rand = Rand(59, 'cuda', dtype)
    for rows in (4, 140):
        x, w, wu = rand(rows, 128), rand(96, 128), rand(96, 128)
        clean = block.linear(x, w, activation='silu')
        clean_h = block.gated_linear(x, w, wu)
        x[2, 5], x[0, 7] = float('nan'), float('inf')
        y = block.linear(x, w, activation='silu')
        h = block.gated_linear(x, w, wu)
        keep = [i for i in range(rows) if i not in (0, 2)]
        assert torch.equal(y[keep], clean[keep])
        assert torch.equal(h[keep], clean_h[keep])
        assert y[2].isnan().all() and h[2].isnan().all()


@pytest.mark.gpu
def test_other_streams():
    """Calls run on the current stream, after what it holds."""
    rand = Rand(61, 'cuda', torch.bfloat16)
    w = rand(512, 512, scale=0.05)
    base = rand(700, 512)
    want = block.linear(base * 2, w, activation='gelu')
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000)  # pylint: disable=protected-access
        x = base * 2
        got = block.linear(x, w, activation='gelu')
        back = got.clone()
    stream.synchronize()
    assert torch.equal(back, want)


@pytest.mark.gpu
def test_from_a_fresh_thread():
    """A thread without a current CUDA context: tensor maps still encode
    (products here, and the long-sequence attention)."""
    import threading
    rand = Rand(73, 'cuda', torch.bfloat16)
    x, w = rand(64, 512), rand(256, 512)
    q = rand(1, 2, 256, 64)
    scale = torch.full((1, 2, 1, 1), 0.05, device='cuda')
    calls = [lambda: block.linear(x, w),
             lambda: vectra_b200.rbf_attention(q, q, q, scale)]
    for call in calls:
        want, got = call(), []
        torch.cuda.synchronize()
        thread = threading.Thread(target=lambda c=call: got.append(c()))
        thread.start()
        thread.join()
        assert len(got) == 1 and torch.equal(got[0], want)


@pytest.mark.gpu
def test_results_past_32_bit_offsets():
    """More than 2^31 result elements."""
    rand = Rand(67, 'cuda', torch.bfloat16)
    m, k, n = 66000, 16, 32768
    x, w = rand(m, k), rand(n, k, scale=0.25)
    y = block.linear(x, w)
    for rows in (slice(0, 3), slice(65533, 66000, 100)):
        want = d(x[rows]) @ d(w).t()
        bound = U[x.dtype] * want.abs() + 2 * sums(k) * (
            d(x[rows]).abs() @ d(w).abs().t())
        close(y[rows], want, bound, 'rows')


@pytest.mark.gpu
def test_captured_in_a_cuda_graph():
    rand = Rand(71, 'cuda', torch.bfloat16)
    x, w, wu = rand(9, 256), rand(192, 256), rand(192, 256)
    q = rand(2, 4, 3, 64)
    cos, sin = block.rotation_tables(8, 64, device='cuda')

    def step():
        y = block.linear(x, w, activation='silu')
        return (y, block.gated_linear(x, w, wu),
                *block.qk_norm_rope(q, q, cos, sin))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(rand(9, 256))
    q.copy_(rand(2, 4, 3, 64))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
