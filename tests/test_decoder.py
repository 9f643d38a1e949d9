"""dropout, residual_norm, qk_norm_rope_axes and cross_attention
(vectra_b200.block) against plain float64 formulations, on CPU tensors and,
marked gpu, on the kernels.

Bounds. u is the unit roundoff of the tensors' type, E = 2^-23 one float32
rounding (two: the tensor cores may truncate). A float32 sum of n terms is off
by (n + 16) E times the sum of their magnitudes. What is said about magnitudes
below is formed from absolute values in float64 beside the value itself, and
every error is carried through the formula by its partial derivatives'
magnitudes; second-order terms are covered by the 16.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

from vectra_b200 import _lib
from vectra_b200 import block
from vectra_b200 import custom_ops

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11,
     torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 1e-38, torch.float16: 2.0**-24,
        torch.bfloat16: 1e-38}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
E = 2.0**-23


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
    return (n + 16) * E


# ---------------------------------------------------------------------------
# Dropout.
# ---------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 in Python integers."""
    c, k, m = list(counter), list(key), 0xffffffff
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def test_philox_known_answers():
    """The method's published vectors (its authors' kat_vectors)."""
    assert philox([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c,
                                        0x9b00dbd8]
    assert philox([0xffffffff] * 4, [0xffffffff] * 2) == [
        0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def keep_mask(n, seed, step, stream, p):
    m, cut = 0xffffffff, int(math.floor(p * 65536 + 0.5))
    out = []
    for g in range((n + 7) // 8):
        words = philox([g & m, g >> 32, step & m, stream & m],
                       [seed & m, (seed >> 32) & m])
        for w in words:
            out += [(w & 0xffff) >= cut, (w >> 16) >= cut]
    return torch.tensor(out[:n])


def rng_of(seed, step, device):
    return torch.tensor([seed, step], dtype=torch.int64, device=device)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1,), (7,), (8,), (3, 5), (2, 3, 40),
                                   (1, 1, 1, 17), (4, 250)])
@pytest.mark.parametrize('p', [0.1, 0.5])
def test_dropout_values(device, dtype, shape, p):
    rand = Rand(1, device, dtype)
    seed, step, stream = -(1 << 61) + 12345, (5 << 32) + 7, 3
    x, dy = rand(*shape).requires_grad_(), rand(*shape)
    y = block.dropout(x, p, rng_of(seed, step, device), stream)
    n = x.numel()
    keep = keep_mask(n, seed, step, stream, p).view(shape)
    scale = 1 / (1 - math.floor(p * 65536 + 0.5) / 65536)
    assert y.dtype == dtype and y.is_contiguous()
    for got, t in ((y, x), (torch.autograd.grad(y, x, dy)[0], dy)):
        want = d(t) * keep * scale
        # The scale and the product are rounded, then the result.
        close(got, want, (U[dtype] + 2 * E) * want.abs() + TINY[dtype])
        assert torch.equal(d(got) == 0, ~keep | (d(t) == 0))


@pytest.mark.parametrize('device', DEVICES)
def test_dropout_streams_steps_and_shares(device):
    x = torch.ones(100000, device=device)

    def kept(p, seed=1, step=2, stream=3):
        return block.dropout(x, p, rng_of(seed, step, device), stream) != 0

    base = kept(0.3)
    assert torch.equal(base, kept(0.3))
    for other in (kept(0.3, seed=2), kept(0.3, seed=1 + (1 << 32)),
                  kept(0.3, step=3), kept(0.3, stream=4)):
        # Independent masks agree on 0.58 of the elements; the deviation of
        # the share is 0.0016.
        assert abs((base == other).float().mean().item() - 0.58) < 0.012
    for p in (0.05, 0.3, 0.9):
        assert abs(kept(p).float().mean().item() - (1 - p)) < 0.01
    assert not kept(1.0).any() and kept(0.0).all()
    assert torch.equal(block.dropout(x, 0.0), x)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_dropout_layouts(device, dtype):
    rand, rng = Rand(2, device, dtype), rng_of(9, 1, device)
    x = rand(6, 40, 24)
    for view in (x[:, ::2, :], x.transpose(0, 1), x[..., 1:], x[..., ::3],
                 x[:1].expand(4, 40, 24), x[:, :, :8], x[:0], x[0, 0, 0]):
        want = block.dropout(view.contiguous(), 0.4, rng, 2)
        assert torch.equal(block.dropout(view, 0.4, rng, 2), want)
    y = x.clone().requires_grad_()
    got, = torch.autograd.grad(block.dropout(y, 0.4, rng, 2).sum(), y)
    assert torch.equal(got, block.dropout(torch.ones_like(x), 0.4, rng, 2))


@pytest.mark.parametrize('device', DEVICES)
def test_dropped_values_are_zero_whatever_they_hold(device):
    rng = rng_of(4, 4, device)
    keep = block.dropout(torch.ones(64, device=device), 0.5, rng) != 0
    x = torch.full((64,), float('nan'), device=device)
    x[::2] = float('inf')
    y = block.dropout(x, 0.5, rng)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


# ---------------------------------------------------------------------------
# residual_norm
# ---------------------------------------------------------------------------
def norm64(v, kind, eps):
    """(normalised, factor) and the magnitudes that the normalised came of."""
    mean = v.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros(
        (), dtype=torch.float64)
    t = v - mean
    r = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    size = v.abs() + (v.abs().mean(-1, keepdim=True)
                      if kind == 'layer' else 0)
    return t * r, r, size * r


def mean(t):
    return t.mean(-1, keepdim=True)


def norm_error(n, r, size, e, f, kind):
    """Error of normalised rows whose argument is off by e."""
    own = r * e + n.abs() * mean(n.abs() * r * e) + f * size
    return own + (r * mean(e) + 0 * n if kind == 'layer' else 0)


def back64(g, n, r, kind):
    out = g - n * mean(g * n)
    return r * (out - mean(g) if kind == 'layer' else out)


def back_error(g, eg, n, en, r, f, kind):
    """Error of back64 for errors eg and en of g and n; all of their orders,
    since en may be more than n where a row hardly varies."""
    cross = mean(eg * (n.abs() + en)) + mean(g.abs() * en)
    e = eg + n.abs() * cross + en * (mean(g * n).abs() + cross)
    size = g.abs() + n.abs() * mean((g * n).abs())
    if kind == 'layer':
        e, size = e + mean(eg), size + mean(g.abs())
    return r * (e + 3 * f * size)


def check_norm(x, branch, weight, bias, gate, bw, a, p, rng, stream, kind, eps,
               norm=True, dx_out=None, dy=None, keep=None):
    """Results (and gradients) of block.residual_norm within bounds."""
    dtype, c = x.dtype, x.shape[-1]
    u, tiny, f = U[dtype], TINY[dtype], sums(c)
    named = {'x': x, 'branch': branch, 'weight': weight, 'bias': bias,
             'gate': gate, 'bw': bw}
    named = {k: t for k, t in named.items() if t is not None}
    train = dx_out is not None or dy is not None
    if train:
        for t in named.values():
            t.requires_grad_()
    got_x, got_y = block.residual_norm(
        x, branch, weight, bias, gate=gate, branch_weight=bw,
        residual_scale=a, p=p, rng=rng, stream=stream, eps=eps, kind=kind,
        norm=norm)
    xv = d(x)
    n0 = r0 = None
    if branch is None:
        x_out, ex = xv, torch.zeros_like(xv)
        assert got_x is x
    else:
        uv = d(branch)
        eu = torch.zeros_like(uv)
        if bw is not None:
            n0, r0, size0 = norm64(uv, kind, eps)
            en0 = f * size0
            uv = n0 * d(bw)
            eu = en0 * d(bw).abs() + E * uv.abs()
        drop = torch.ones_like(uv) if keep is None else keep.double() / (
            1 - math.floor(p * 65536 + 0.5) / 65536)
        dv, ed = uv * drop, eu * drop + 2 * E * (uv * drop).abs()
        gv = torch.ones((), dtype=torch.float64) if gate is None else d(gate)
        x_out = a * xv + gv * dv
        ex = gv.abs() * ed + 2 * E * ((a * xv).abs() + (gv * dv).abs())
        assert got_x.is_contiguous() and got_x.dtype == dtype
        close(got_x, x_out, ex * (1 + u) + u * x_out.abs() + tiny, 'x_out')
    if norm:
        n1, r1, size1 = norm64(x_out, kind, eps)
        wv = torch.ones(c, dtype=torch.float64) if weight is None else \
            d(weight)
        y = n1 * wv + (0 if bias is None else d(bias))
        en1 = norm_error(n1, r1, size1, ex, f, kind)
        ey = en1 * wv.abs() + 2 * E * ((n1 * wv).abs() + y.abs())
        close(got_y, y, ey * (1 + u) + u * y.abs() + tiny, 'y')
    else:
        assert got_y is None
    if not train:
        return
    outs = [(got_x, dx_out), (got_y, dy)]
    outs = [o for o in outs if o[1] is not None]
    grads = dict(zip(named, torch.autograd.grad(
        [o[0] for o in outs], list(named.values()), [o[1] for o in outs],
        allow_unused=True)))
    rows = x_out.numel() // c
    g = torch.zeros_like(x_out) if dx_out is None else d(dx_out)
    eg = torch.zeros_like(g)
    if branch is None:
        # x_out is x: its gradient is added to dx, both rounded.
        direct, g = g, torch.zeros_like(g)
    if dy is not None:
        # The backward pass forms n1 from x_out as it was rounded.
        en1 = norm_error(n1, r1, size1, ex, f, kind) + r1 * (
            u * x_out.abs() + tiny)
        fv = d(dy)
        if weight is not None:
            want = (fv * n1).reshape(rows, c).sum(0)
            close(grads['weight'], want,
                  (fv.abs() * en1 + sums(rows) * (fv * n1).abs()).reshape(
                      rows, c).sum(0) * (1 + u) + u * want.abs() + tiny, 'dw')
        if bias is not None:
            want = fv.reshape(rows, c).sum(0)
            close(grads['bias'], want, sums(rows) * fv.abs().reshape(
                rows, c).sum(0) * (1 + u) + u * want.abs() + tiny, 'db')
        fw = fv * wv
        term = back64(fw, n1, r1, kind)
        eg = back_error(fw, E * fw.abs(), n1, en1, r1, f, kind) + \
            2 * E * (term.abs() + g.abs())
        g = g + term
    if branch is None:
        want = g + direct
        close(grads['x'], want, eg * (1 + u) + u * (g.abs() + want.abs()) +
              2 * tiny, 'dx')
        return
    close(grads['x'], a * g, abs(a) * eg * (1 + u) + (u + E) * (a * g).abs() +
          tiny, 'dx')
    if gate is not None:
        t, et = g * dv, eg * dv.abs() + g.abs() * ed
        shape, lead = gate.shape, x.dim() - gate.dim()
        dims = tuple(range(lead)) + tuple(
            i + lead for i in range(gate.dim() - 1) if shape[i] == 1)
        want, count = t, 1
        spread = et
        if dims:
            count = math.prod(x.shape[i] for i in dims)
            spread = (et + sums(count) * t.abs()).sum(dims).reshape(shape)
            want = t.sum(dims).reshape(shape)
        close(grads['gate'], want, spread * (1 + u) + (u + E) * want.abs() +
              tiny, 'dgate')
    h = g * gv * drop
    eh = eg * gv.abs() * drop + 3 * E * h.abs()
    if bw is None:
        close(grads['branch'], h, eh * (1 + u) + u * h.abs() + tiny,
              'dbranch')
        return
    want = (h * n0).reshape(rows, c).sum(0)
    close(grads['bw'], want,
          (eh * n0.abs() + h.abs() * en0 + sums(rows) * (h * n0).abs())
          .reshape(rows, c).sum(0) * (1 + u) + u * want.abs() + tiny, 'dbw')
    hb = h * d(bw)
    want = back64(hb, n0, r0, kind)
    close(grads['branch'], want,
          back_error(hb, eh * d(bw).abs() + E * hb.abs(), n0, en0, r0, f,
                     kind) * (1 + u) + u * want.abs() + tiny, 'dbranch')


# Rows and widths: single rows, odd widths, a warp's, a block's, its limits.
NORM_SIZES = [(1, 1), (3, 7), (5, 64), (2, 250), (9, 256), (4, 320),
              (3, 512), (2, 520), (7, 1000), (3, 2056), (2, 4096), (2, 5121),
              (1, 8192)]
FORMS = [dict(kind='rms', bias=False, bw=False, gate='none', p=0.0),
         dict(kind='layer', bias=True, bw=True, gate='channel', p=0.3),
         dict(kind='rms', bias=True, bw=True, gate='token', p=0.1),
         dict(kind='layer', bias=False, bw=False, gate='sequence', p=0.5)]


def norm_inputs(rand, b, n, c, form):
    gate = {'none': None, 'channel': (c,), 'sequence': (b, 1, c),
            'token': (b, n, c)}[form['gate']]
    return dict(x=rand(b, n, c), branch=rand(b, n, c, scale=1.5),
                weight=1 + rand(c, scale=0.2),
                bias=rand(c) if form['bias'] else None,
                gate=None if gate is None else rand(*gate),
                bw=1 + rand(c, scale=0.2) if form['bw'] else None)


def mask_of(form, shape, seed, step, stream):
    if not form['p']:
        return None
    n = math.prod(shape)
    return keep_mask(n, seed, step, stream, form['p']).view(shape)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', NORM_SIZES)
@pytest.mark.parametrize('form', range(len(FORMS)))
def test_norm_sizes(device, dtype, size, form):
    (n, c), form = size, FORMS[form]
    rand = Rand(n * 100 + c, device, dtype)
    a = norm_inputs(rand, 2, n, c, form)
    check_norm(**a, a=0.7, p=form['p'], rng=rng_of(11, 12, device), stream=1,
               kind=form['kind'], eps=1e-5, dx_out=rand(2, n, c),
               dy=rand(2, n, c), keep=mask_of(form, (2, n, c), 11, 12, 1))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_norm_many_rows(device, dtype):
    """More rows than teams, so sums over rows are joined from all places."""
    for c, b, n in ((64, 3, 2100), (768, 2, 700)):
        for form in (FORMS[1], FORMS[3]):
            rand = Rand(c, device, dtype)
            form = dict(form, p=0.0)
            a = norm_inputs(rand, b, n, c, form)
            check_norm(**a, a=1.0, p=0.0, rng=None, stream=0,
                       kind=form['kind'], eps=1e-6, dx_out=rand(b, n, c),
                       dy=rand(b, n, c))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('c', [8200, 12000, 16384])
def test_norm_widest_rows(dtype, c):
    rand = Rand(c, 'cuda', dtype)
    form = dict(FORMS[1], p=0.0)
    a = norm_inputs(rand, 2, 3, c, form)
    check_norm(**a, a=0.5, p=0.0, rng=None, stream=0, kind='layer', eps=1e-6,
               dx_out=rand(2, 3, c), dy=rand(2, 3, c))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', ['rms', 'layer'])
def test_norm_forms(device, dtype, kind):
    """The norm alone, the residual alone, either result's gradient alone."""
    rand = Rand(21, device, dtype)
    b, n, c = 2, 5, 96
    kw = dict(p=0.0, rng=None, stream=0, kind=kind, eps=1e-6)

    def fresh():
        return norm_inputs(rand, b, n, c, FORMS[1])

    one = dict(branch=None, gate=None, bw=None)
    check_norm(**{**fresh(), **one}, a=1.0, **kw)
    check_norm(**{**fresh(), **one}, a=1.0, dy=rand(b, n, c),
               dx_out=rand(b, n, c), **kw)
    check_norm(**{**fresh(), **one, 'weight': None, 'bias': None}, a=1.0,
               dy=rand(b, n, c), **kw)
    for extra in ({}, {'bw': None}, {'bw': None, 'gate': None}):
        check_norm(**{**fresh(), 'weight': None, 'bias': None, **extra},
                   a=0.3, norm=False, dx_out=rand(b, n, c), **kw)
        check_norm(**{**fresh(), **extra}, a=0.3, dy=rand(b, n, c), **kw)
        check_norm(**{**fresh(), **extra}, a=0.3, dx_out=rand(b, n, c), **kw)
    check_norm(**{**fresh(), 'bias': None}, a=0.3, dy=rand(b, n, c), **kw)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_norm_layouts(device, dtype):
    """Strided, sliced and broadcast inputs give what contiguous ones do."""
    rand = Rand(22, device, dtype)
    b, n, c = 3, 6, 40
    base = [rand(b, n, 2 * c + 1) for _ in range(4)]
    assert base[0][..., 1::2].shape == (b, n, c)
    wide = rand(4 * c)
    turned = rand(n, b, 2 * c).transpose(0, 1)
    views = [t[..., 1:2 * c + 1:2] for t in base[:2]] + \
        [turned[..., :c], base[3][..., 1:c + 1]]
    weights = [wide[:c], wide[1:2 * c:2], wide[c + 1:2 * c + 1]]
    for order in ((0, 1, 2, 3), (2, 3, 0, 1)):
        x, branch, dx_out, dy = (views[i] for i in order)
        for gate in (wide[2 * c:3 * c], base[0][:, :1, :c],
                     base[1][..., 3:3 + c]):
            results = []
            for flat in (False, True):
                ts = [x, branch, weights[0], weights[1], gate, weights[2]]
                gs = [dx_out, dy]
                if flat:
                    ts = [t.contiguous() for t in ts]
                    gs = [t.contiguous() for t in gs]
                ts = [t.detach().requires_grad_() for t in ts]
                out = block.residual_norm(ts[0], ts[1], ts[2], ts[3],
                                          gate=ts[4], branch_weight=ts[5],
                                          kind='layer')
                results.append([*out, *torch.autograd.grad(out, ts, gs)])
            for s, t in zip(*results):
                # One order of sums a thread, another a layout: a rounding.
                np.testing.assert_allclose(
                    d(s).numpy(), d(t).numpy(), rtol=2 * U[dtype],
                    atol=1e-5 + 4 * U[dtype] * float(d(t).abs().max()))


@pytest.mark.parametrize('device', DEVICES)
def test_norm_empty(device):
    x = torch.zeros(0, 5, 16, device=device, requires_grad=True)
    w = torch.ones(16, device=device, requires_grad=True)
    g = torch.ones(16, device=device, requires_grad=True)
    out = block.residual_norm(x, x, w, gate=g, branch_weight=w)
    assert out[0].shape == out[1].shape == x.shape
    grads = torch.autograd.grad([t.sum() for t in out], [x, w, g])
    assert grads[0].shape == x.shape
    assert (grads[1] == 0).all() and (grads[2] == 0).all()
    y = torch.zeros(3, 0, device=device)
    assert block.residual_norm(y, y)[1].shape == (3, 0)


@pytest.mark.parametrize('device', DEVICES)
def test_norm_only_wanted_gradients(device):
    rand = Rand(23, device, torch.float16)
    a = norm_inputs(rand, 2, 9, 128, FORMS[1])
    rng = rng_of(1, 2, device)
    order = ('x', 'branch', 'weight', 'bias', 'gate', 'bw')
    ups = [rand(2, 9, 128), rand(2, 9, 128)]

    def run(ts):
        out = block.residual_norm(ts[0], ts[1], ts[2], ts[3], gate=ts[4],
                                  branch_weight=ts[5], p=0.3, rng=rng)
        leaves = [t for t in ts if t.requires_grad]
        return torch.autograd.grad(out, leaves, ups)

    every = run([a[k].clone().requires_grad_() for k in order])
    for i in range(6):
        ts = [a[k].clone() for k in order]
        ts[i].requires_grad_()
        assert torch.equal(run(ts)[0], every[i]), order[i]


# ---------------------------------------------------------------------------
# qk_norm_rope_axes
# ---------------------------------------------------------------------------
def axis_rows(table, positions, sections):
    parts, at = [], 0
    for a, n in enumerate(sections):
        parts.append(d(table)[:, at:at + n][positions[a].cpu().long()])
        at += n
    return torch.cat(parts, -1)[:, None]


# (heads, key heads, width, sections): whole fours, ends anywhere, an axis
# without a pair, one axis, unrotated components, odd widths.
AXES = [(4, 2, 64, (8, 12, 12)), (3, 3, 32, (4, 6, 6)), (2, 1, 128, (16, 48)),
        (1, 1, 48, (5, 0, 7, 9)), (2, 2, 16, (8,)), (8, 2, 80, (3, 17)),
        (2, 1, 14, (2, 5)), (1, 1, 256, (40, 44, 44))]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', AXES)
@pytest.mark.parametrize('interleaved', [False, True])
def test_axes(device, dtype, size, interleaved):
    hq, hk, dim, sections = size
    b, n, table = 3, 11, 70
    rand = Rand(dim, device, dtype)
    u, tiny, f = U[dtype], TINY[dtype], (dim + 32) * 2.0**-24
    q, k = rand(b, n, hq, dim).transpose(1, 2), rand(b, hk, n, dim)
    cos, sin = block.rotation_tables(table, 2 * sum(sections), device=device)
    positions = torch.randint(0, table, (len(sections), b, n),
                              generator=rand.gen).to(device)
    ws = [1 + rand(dim, scale=0.2), 1 + rand(dim, scale=0.2)]
    leaves = [t.detach().requires_grad_() for t in (q, k, *ws)]
    got = block.qk_norm_rope_axes(leaves[0], leaves[1], cos, sin, positions,
                                  sections, leaves[2], leaves[3], 1e-5,
                                  interleaved)
    ups = [rand(b, hq, n, dim), rand(b, hk, n, dim)]
    grads = torch.autograd.grad(got, leaves, ups)
    c, s = (axis_rows(t, positions, sections) for t in (cos, sin))
    rotary = 2 * sum(sections)

    def turn(x, c, s):
        head, tail = x[..., :rotary], x[..., rotary:]
        a, z = ((head[..., 0::2], head[..., 1::2]) if interleaved else
                head.chunk(2, -1))
        a, z = a * c - z * s, z * c + a * s
        head = torch.stack([a, z], -1).flatten(-2) if interleaved else \
            torch.cat([a, z], -1)
        return torch.cat([head, tail], -1)

    def size_of(x):
        return turn(x.abs(), c.abs(), -s.abs()).abs() + \
            turn(x.abs(), c.abs(), s.abs()).abs()

    for i, (x, w, dy) in enumerate(zip((q, k), ws, ups)):
        v = d(x)
        r = (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        nrm = v * r
        want = turn(nrm * d(w), c, s)
        assert got[i].stride() == custom_ops.output_strides(x, dim)
        close(got[i], want, u * want.abs() * (1 + f) +
              f * size_of(nrm * d(w)) + tiny, 'qk'[i])
        g, gm = turn(d(dy), c, -s), size_of(d(dy))
        gw, gwm = g * d(w), gm * d(w).abs()
        dx = r * (gw - nrm * mean(gw * nrm))
        spread = r * (gwm + nrm.abs() * mean(gwm * nrm.abs()))
        close(grads[i], dx, u * dx.abs() * (1 + f) + 3 * f * spread + tiny,
              'd' + 'qk'[i])
        dw = (g * nrm).sum((0, 1, 2))
        spread = (gm * nrm.abs()).sum((0, 1, 2))
        close(grads[2 + i], dw, u * dw.abs() * (1 + f) +
              (3 * f + sums(b * n * hq)) * spread + tiny, 'dw')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('interleaved', [False, True])
def test_axes_agree_with_one_position(device, interleaved):
    """The same position on all axes is qk_norm_rope, bit for bit."""
    rand = Rand(31, device, torch.bfloat16)
    q, k = rand(2, 4, 9, 64), rand(2, 2, 9, 64)
    cos, sin = block.rotation_tables(40, 64, device=device)
    pos = torch.randint(0, 40, (2, 9), generator=rand.gen).to(device)
    want = block.qk_norm_rope(q, k, cos, sin, None, None, pos, 1e-6,
                              interleaved)
    for p, sections in ((pos.expand(3, 2, 9), (8, 12, 12)),
                        (pos.int().expand(2, 2, 9), (7, 25)),
                        (pos[None], (32,))):
        got = block.qk_norm_rope_axes(q, k, cos, sin, p, sections, None, None,
                                      1e-6, interleaved)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dim', [64, 14])
def test_axes_outside_the_tables(device, dim):
    rand = Rand(32, device, torch.float32)
    q, k = rand(1, 2, 6, dim), rand(1, 1, 6, dim)
    cos, sin = block.rotation_tables(5, dim, device=device)
    pos = torch.zeros(2, 1, 6, dtype=torch.int64, device=device)
    pos[0, 0, 1], pos[1, 0, 3], pos[1, 0, 4] = -1, 5, 1 << 40
    got = block.qk_norm_rope_axes(q, k, cos, sin, pos,
                                  (dim // 2 - 2, 2))
    for t in got:
        bad = torch.isnan(t).all(-1)
        assert bad[..., [1, 3, 4]].all() and not bad[..., [0, 2, 5]].any()
        assert torch.isfinite(t[..., [0, 2, 5], :]).all()


# ---------------------------------------------------------------------------
# cross_attention
# ---------------------------------------------------------------------------
def check_cross(q, k, v, scale, lengths=None, dout=None):
    """Result (and gradients) of block.cross_attention within bounds.

    A logit comes of a distance that is off by sums(D) (2 |q|.|k| + |k|^2 +
    |q|^2) at most, however it is formed, and of at most four roundings; the
    weights are off by that of both the logit and the row's sum, relatively:
    `ew`. 16-bit products round weights (u, and float16's spacing), training
    keeps what that rounding left (u^2).
    """
    dtype, dim, dv_ = q.dtype, q.shape[3], v.shape[3]
    u, tiny = U[dtype], TINY[dtype]
    half = dtype != torch.float32
    train = dout is not None
    if train:
        for t in (q, k, v, scale):
            t.requires_grad_()
    out = block.cross_attention(q, k, v, scale, lengths)
    assert out.dtype == dtype
    assert out.stride() == custom_ops.output_strides(q, dv_)
    b, h, nq = q.shape[:3]
    hk, nk = k.shape[1:3]
    rep = h // hk
    Q, K, V = d(q), d(k), d(v)
    n = torch.full((b,), nk) if lengths is None else \
        lengths.cpu().long().clamp(0, nk)
    seen = (torch.arange(nk) < n[:, None])[:, None, None]
    K = torch.where(seen[:, :, 0, :, None], K, 0.0)
    V = torch.where(seen[:, :, 0, :, None], V, 0.0)
    K, V = K.repeat_interleave(rep, 1), V.repeat_interleave(rep, 1)
    S = d(scale).reshape((1,) * (4 - scale.dim()) + scale.shape).expand(
        b, h, 1, 1)
    diff = Q[:, :, :, None] - K[:, :, None]
    dist = diff.square().sum(-1)
    size = 2 * Q.abs() @ K.abs().mT + K.square().sum(-1)[:, :, None] + \
        Q.square().sum(-1, keepdim=True)
    logits = torch.where(seen, -S * dist, -math.inf)
    w = torch.softmax(logits, -1)
    w = torch.where(seen & (n > 0)[:, None, None, None], w, 0.0)
    el = S.abs() * (sums(dim) * size) + 4 * E * (S * size).abs()
    ew = torch.where(seen, el, 0.0)
    ew = torch.expm1(2 * ew.amax(-1, keepdim=True) + sums(nk)) if nk else ew
    spare = tiny * (nk + 1) if half else 0.0  # float16 weights far down
    o = w @ V
    per = w * ew + w * (sums(nk) + (2 * u if half and not train else
                                    3 * u * u)) + spare
    eo = per @ V.abs()
    close(out, o, eo * (1 + u) + u * o.abs() + tiny, 'out')
    if not train:
        return out
    got = dict(zip(('q', 'k', 'v', 'scale'), torch.autograd.grad(
        out, (q, k, v, scale), dout)))
    G = d(dout)
    c = (G * o).sum(-1, keepdim=True)
    # out's rounding is kept in another 16-bit number.
    ec = (G.abs() * (eo + 2 * u * u * o.abs() + tiny)).sum(
        -1, keepdim=True) + sums(dv_) * (G.abs() * o.abs()).sum(
            -1, keepdim=True)
    t = G @ V.mT
    et = sums(dv_) * (G.abs() @ V.abs().mT)
    z = w * (t - c)
    ez = w * (ew * (t - c).abs() + et + ec) + 2 * E * z.abs()
    rough = (u * z.abs() + tiny) if half else 0.0

    def shared(x):  # sums over the query heads of a key head
        return x.reshape(b, hk, rep, *x.shape[2:]).sum(2)

    reach = diff.abs()
    two = 2 * S.abs()
    want = 2 * S * ((z[..., None] * -diff).sum(3))
    bound = two * ((ez + rough)[..., None] * reach).sum(3) + \
        sums(nk) * two * (z.abs() @ K.abs() +
                          z.abs().sum(-1, keepdim=True) * Q.abs())
    close(got['q'], want, bound * (1 + u) + u * want.abs() + tiny, 'dq')
    # For dk, z is rounded with its scale.
    rough_k = (u * two * z.abs() + tiny) if half else 0.0
    want = shared(2 * S * ((z[..., None] * diff).sum(2)
                           if nq else 0 * K))
    bound = shared(((two * ez + rough_k)[..., None] * reach).sum(2) +
                   sums(nq * rep) * ((two * z.abs()).mT @ Q.abs() +
                                     (two * z.abs()).sum(2)[..., None] *
                                     K.abs()))
    close(got['k'], want, bound * (1 + u) + u * want.abs() + tiny, 'dk')
    want = shared(w.mT @ G)
    bound = shared((w * (ew + (u if half else 0.0)) + spare +
                    sums(nq * rep) * w).mT @ G.abs())
    close(got['v'], want, bound * (1 + u) + u * want.abs() + tiny, 'dv')
    near = dist - (w * dist).sum(-1, keepdim=True)
    per = -(z * near).sum((2, 3), keepdim=True)
    # A centred distance is off by its own error and the mean's: of the
    # weights, of the distances and of the sum. z may be smaller than its
    # error (over a single key it is zero), so that goes along.
    zz = z.abs() + ez
    en = sums(dim) * size + (w * size * (ew + sums(dim) + sums(nk))).sum(
        -1, keepdim=True)
    bound = (ez * near.abs() + zz * en).sum((2, 3), keepdim=True) + sums(nk) \
        * ((zz * size).sum(-1, keepdim=True) + zz.sum(-1, keepdim=True) *
           (w * size).sum(-1, keepdim=True)).sum((2, 3), keepdim=True)
    shape = (1,) * (4 - scale.dim()) + tuple(scale.shape)
    dims = [i for i in range(2) if shape[i] == 1]
    if dims:
        per, bound = per.sum(dims, keepdim=True), bound.sum(dims,
                                                            keepdim=True)
    us = 2.0**-53 if scale.dtype == torch.float64 else U[scale.dtype]
    close(got['scale'], per.reshape(scale.shape),
          (bound * (1 + us) + (us + E * b * h) * per.abs()).reshape(
              scale.shape) + TINY.get(scale.dtype, 1e-38), 'dscale')
    return out


def cross_inputs(rand, b, h, hk, nq, nk, dim, dv=None, gamma=None):
    dv = dim if dv is None else dv
    q = rand(b, nq, h, dim).transpose(1, 2)
    k, v = rand(b, hk, nk, dim), rand(b, nk, hk, dv).transpose(1, 2)
    if gamma is None:
        gamma = 2.0 / math.sqrt(8 * dim)
    scale = gamma * (0.5 + torch.rand(1, h, 1, 1, generator=rand.gen))
    return q, k, v, scale.to(rand.device)


# b, h, hk, nq, nk, D, Dv: single tokens and keys, tiles' ends, shared heads in
# numbers that divide a tile and not, widths that end inside a piece, other
# value widths, and those the tensor cores do not take.
CROSS = [(1, 1, 1, 1, 1, 64, 64), (2, 2, 2, 1, 64, 32, 32),
         (3, 4, 2, 5, 63, 64, 64), (2, 3, 1, 17, 65, 80, 80),
         (1, 5, 1, 40, 129, 128, 128), (2, 8, 8, 65, 65, 32, 32),
         (1, 7, 1, 30, 130, 64, 32), (2, 6, 3, 130, 40, 48, 96),
         (1, 16, 1, 9, 300, 16, 128), (1, 2, 1, 200, 257, 96, 64),
         (1, 1, 1, 3, 700, 128, 128), (2, 2, 1, 7, 33, 24, 40),
         (1, 2, 2, 20, 50, 33, 17), (1, 2, 1, 70, 70, 160, 136),
         (2, 1, 1, 5, 40, 256, 256), (1, 66, 1, 2, 20, 64, 64)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', CROSS)
@pytest.mark.parametrize('train', [False, True])
def test_cross_sizes(device, dtype, size, train):
    b, h, hk, nq, nk, dim, dv = size
    rand = Rand(nk + dim, device, dtype)
    a = cross_inputs(rand, *size)
    check_cross(*a, dout=rand(b, h, nq, dv) if train else None)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(6, 4, 2, 3, 70, 64), (6, 2, 2, 66, 150, 32),
                                  (6, 3, 1, 1, 40, 128), (6, 2, 1, 9, 20, 30)])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
def test_cross_lengths(device, dtype, size, index):
    """None, one, all, more than all and fewer than none of the keys; those
    past the length may hold anything."""
    b, h, hk, nq, nk, dim = size
    rand = Rand(51, device, dtype)
    q, k, v, scale = cross_inputs(rand, *size)
    lengths = torch.tensor([nk, 0, 1, nk - 3, nk + 9, -5], dtype=index,
                           device=device)
    dout = rand(b, h, nq, dim)
    want = check_cross(q, k, v, scale, lengths, dout)
    assert (want[[1, 5]] == 0).all()
    leaves = [t.detach().clone() for t in (q, k, v)]
    for i, n in enumerate(lengths.clamp(0, nk).tolist()):
        leaves[1][i, :, n:] = float('nan')
        leaves[2][i, :, n:] = float('inf')
    leaves = [t.requires_grad_() for t in (*leaves, scale.detach())]
    got = block.cross_attention(*leaves, lengths)
    assert torch.equal(got, want)
    mine = torch.autograd.grad(got, leaves, dout)
    clean = torch.autograd.grad(block.cross_attention(
        q, k, v, scale, lengths), (q, k, v, scale), dout)
    for x, y in zip(mine, clean):
        assert torch.equal(x, y)
    for i, n in enumerate(lengths.clamp(0, nk).tolist()):
        for t in mine[1:3]:
            assert (t[i, :, n:] == 0).all()
    assert (mine[0][[1, 5]] == 0).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_cross_scales(device, dtype):
    """Zero, negative and broadcast scales of every float type."""
    rand = Rand(52, device, dtype)
    b, h, hk, nq, nk, dim = 2, 4, 2, 6, 70, 64
    dout = rand(b, h, nq, dim)
    for scale in (torch.zeros(1, h, 1, 1), torch.full((1, h, 1, 1), -0.02),
                  torch.tensor(0.05), torch.rand(b, 1, 1, 1) * 0.1,
                  torch.rand(h, 1, 1, dtype=torch.float64) * 0.1,
                  (torch.rand(b, h, 1, 1) * 0.1).half(),
                  (torch.rand(1, 1, 1, 1) * 0.1).bfloat16()):
        q, k, v, _ = cross_inputs(rand, b, h, hk, nq, nk, dim)
        check_cross(q, k, v, scale.to(device), None, dout)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_cross_one_large_weight(device, dtype):
    """Keys beside their query among far ones: one weight near 1. Its value
    comes out but for its own rounding, and gradients keep their bounds."""
    rand = Rand(53, device, dtype)
    b, h, nq, nk, dim = 1, 2, 40, 200, 64
    q = rand(b, h, nq, dim, scale=3.0)
    k = rand(b, h, nk, dim, scale=3.0)
    k[:, :, 10:10 + nq] = q + rand(b, h, nq, dim, scale=0.05)
    v = rand(b, h, nk, dim)
    scale = torch.full((1, h, 1, 1), 0.02, device=device)
    check_cross(q, k, v, scale, None, rand(b, h, nq, dim))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_cross_layouts(device, dtype):
    """Views give what contiguous tensors do, within the two layouts' bounds
    (misaligned ones run on other kernels)."""
    rand = Rand(54, device, dtype)
    b, h, hk, nq, nk, dim = 2, 4, 2, 20, 70, 32
    wide = rand(b, nk, 2 * hk * dim + 1)
    odd = wide[..., 1:].unflatten(-1, (2, hk, dim)).permute(2, 0, 3, 1, 4)
    even = wide[..., :-1].unflatten(-1, (2, hk, dim)).permute(2, 0, 3, 1, 4)
    q = rand(b, h, nq, dim)
    stretched = rand(b, h, nq, 2 * dim)[..., ::2]
    scale = torch.full((1, h, 1, 1), 0.1, device=device)
    lengths = torch.tensor([[nk, 3], [20, 4]], device=device)[:, 0]
    one = rand(1, 1, 1, 1).expand(b, h, nq, dim)
    for qq in (q, q.transpose(0, 1).contiguous().transpose(0, 1), stretched,
               q[:, :, :1].expand(b, h, nq, dim)):
        for kv in (odd, even, even.flip(0)):
            for dout in (rand(b, h, nq, dim), one):
                check_cross(qq.detach(), kv[0].detach(), kv[1].detach(),
                            scale.detach(), lengths, dout)


@pytest.mark.parametrize('device', DEVICES)
def test_cross_empty(device):
    def t(*s):
        return torch.ones(s, device=device, requires_grad=True)

    scale = torch.ones(1, 2, 1, 1, device=device, requires_grad=True)
    for b, h, nq, nk in ((0, 2, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0)):
        q, k, v = t(b, h, nq, 8), t(b, 1, nk, 8), t(b, 1, nk, 8)
        out = block.cross_attention(q, k, v, scale)
        assert out.shape == q.shape and (out == 0).all()
        for g in torch.autograd.grad(out.sum(), (q, k, v, scale)):
            assert (g == 0).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('nq', [1, 200])
@pytest.mark.parametrize('dim', [64, 66])
def test_cross_without_keys(device, dtype, nq, dim):
    """Few and many queries, and widths of 16-byte pieces and not, over an
    encoder without states."""
    rand = Rand(59, device, dtype)
    q, k, v, scale = (t.requires_grad_() for t in
                      cross_inputs(rand, 2, 4, 2, nq, 0, dim))
    with torch.no_grad():
        assert (block.cross_attention(q, k, v, scale) == 0).all()
    out = block.cross_attention(q, k, v, scale)
    assert out.shape == q.shape and (out == 0).all()
    for t in torch.autograd.grad(out.sum(), (q, k, v, scale)):
        assert (t == 0).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_cross_only_wanted_gradients(device, dtype):
    rand = Rand(55, device, dtype)
    a = cross_inputs(rand, 2, 4, 2, 30, 70, 64)
    dout = rand(2, 4, 30, 64)

    def run(ts):
        return torch.autograd.grad(block.cross_attention(*ts),
                                   [t for t in ts if t.requires_grad], dout)

    every = run([t.clone().requires_grad_() for t in a])
    for i in range(4):
        ts = [t.clone() for t in a]
        ts[i].requires_grad_()
        assert torch.equal(run(ts)[0], every[i])


@pytest.mark.parametrize('device', DEVICES)
def test_cross_agrees_with_the_attention_operator(device):
    """Without lengths and shared heads it is torch.ops.vectra.rbf_attention:
    both within a weight's and a result's rounding of the formula."""
    rand = Rand(56, device, torch.bfloat16)
    q, k, v, scale = cross_inputs(rand, 2, 4, 4, 33, 129, 64)
    got = block.cross_attention(q, k, v, scale)
    want = custom_ops.rbf_attention(q, k, v, scale)
    np.testing.assert_allclose(d(got).numpy(), d(want).numpy(), rtol=0,
                               atol=4 * U[torch.bfloat16] *
                               float(d(v).abs().max()))


# ---------------------------------------------------------------------------
# All of them.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('op', ['norm', 'axes', 'cross'])
def test_gradients_against_differences(device, op):
    """Central differences along random directions, float32 (the bound of
    tests/test_block.py: |F'''| below 30 |dy| for inputs of order 1)."""
    rand = Rand(61, device, torch.float32)
    if op == 'norm':
        rng = rng_of(3, 4, device)
        args = [rand(2, 5, 24), rand(2, 5, 24), 1 + rand(24, scale=0.1),
                rand(24), rand(2, 1, 24), 1 + rand(24, scale=0.1)]
        fun = lambda x, r, w, b, g, bw: block.residual_norm(  # noqa: E731
            x, r, w, b, gate=g, branch_weight=bw, residual_scale=0.8, p=0.3,
            rng=rng, kind='layer')
        dys = [rand(2, 5, 24), rand(2, 5, 24)]
    elif op == 'axes':
        cos, sin = block.rotation_tables(9, 12, device=device)
        pos = torch.randint(0, 9, (2, 1, 5), generator=rand.gen).to(device)
        args = [rand(1, 2, 5, 16), rand(1, 1, 5, 16), rand(16), rand(16)]
        fun = lambda q, k, w, v: block.qk_norm_rope_axes(  # noqa: E731
            q, k, cos, sin, pos, (2, 4), w, v)
        dys = [rand(1, 2, 5, 16), rand(1, 1, 5, 16)]
    else:
        lengths = torch.tensor([7, 4], device=device)
        args = [rand(2, 2, 3, 8), rand(2, 1, 7, 8), rand(2, 1, 7, 8),
                rand(1, 2, 1, 1, scale=0.05) + 0.1]
        fun = lambda *a: [block.cross_attention(*a, lengths)]  # noqa: E731
        dys = [rand(2, 2, 3, 8)]
    size = math.sqrt(sum(float(t.double().square().sum()) for t in dys))
    leaves = [t.clone().requires_grad_() for t in args]
    grads = torch.autograd.grad(fun(*leaves), leaves, dys)
    value = lambda a: sum(float((y.double() * t.double()).sum())  # noqa: E731
                          for y, t in zip(fun(*a), dys))
    for i, t in enumerate(args):
        # A scale multiplies distances of order 16: a shorter step.
        h = 2.0**-10 if op == 'cross' and i == 3 else 2.0**-6
        for _ in range(3):
            v = rand(*t.shape)
            v = v / v.norm()
            hi = [a + h * v if j == i else a for j, a in enumerate(args)]
            lo = [a - h * v if j == i else a for j, a in enumerate(args)]
            want = (value(hi) - value(lo)) / (2 * h)
            got = float((grads[i].double() * v.double()).sum())
            slack = 2e-2 if op == 'cross' and i == 3 else 2e-3
            assert abs(got - want) <= slack * size, (i, got, want)


@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    def t(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device=device)

    x, w, rng = t(2, 3, 8), t(8), t(2, dtype=torch.int64)
    norm, drop = block.residual_norm, block.dropout
    cross, axes = block.cross_attention, block.qk_norm_rope_axes
    q, k, s = t(2, 4, 5, 8), t(2, 2, 7, 8), t(1, 4, 1, 1)
    qk, c = t(2, 4, 7, 8), t(6, 4)
    long = lambda *s: t(*s, dtype=torch.int64)  # noqa: E731
    for bad in (
            lambda: drop(x, -0.1, rng), lambda: drop(x, 1.1, rng),
            lambda: drop(x, float('nan'), rng), lambda: drop(x, 0.5),
            lambda: drop(x, 0.5, t(2)), lambda: drop(x, 0.5, long(3)),
            lambda: drop(x, 0.5, long(4)[::2]),
            lambda: drop(x.double(), 0.5, rng),
            lambda: drop(long(4), 0.5, rng),
            lambda: norm(x, t(2, 3, 7)), lambda: norm(x, x.half()),
            lambda: norm(x, x, t(7)), lambda: norm(x, x, w, t(1, 8)),
            lambda: norm(x, x, w.half()),
            lambda: norm(x, x, branch_weight=t(9)),
            lambda: norm(x, x, gate=t(7)), lambda: norm(x, x, gate=t(3, 8)),
            lambda: norm(x, x, gate=t(1, 3, 8)),
            lambda: norm(x, x, gate=t(2, 3, 1)),
            lambda: norm(x, x, gate=t(1, 1, 1, 8)),
            lambda: norm(x, x, kind='batch'), lambda: norm(x, x, p=0.5),
            lambda: norm(x, x, p=2.0, rng=rng),
            lambda: norm(x, norm=False), lambda: norm(x, gate=w),
            lambda: norm(x, branch_weight=w),
            lambda: norm(x, residual_scale=0.5),
            lambda: norm(x, p=0.5, rng=rng),
            lambda: norm(x, x, w, norm=False), lambda: norm(t(), t()),
            lambda: norm(x.double(), x.double()),
            lambda: cross(q[0], k, k, s), lambda: cross(q, k[:1], k, s),
            lambda: cross(q, k.half(), k, s), lambda: cross(q, k, k.half(), s),
            lambda: cross(q, t(2, 3, 7, 8), t(2, 3, 7, 8), s),
            lambda: cross(q, t(2, 2, 7, 6), k, s),
            lambda: cross(q, k, t(2, 2, 6, 8), s),
            lambda: cross(q, k, t(2, 1, 7, 8), s),
            lambda: cross(q, k, k, t(1, 3, 1, 1)),
            lambda: cross(q, k, k, t(1, 4, 5, 1)),
            lambda: cross(q, k, k, t(1, 1, 4, 1, 1)),
            lambda: cross(q, k, k, s.long()),
            lambda: cross(q, k, k, s, t(2)),
            lambda: cross(q, k, k, s, long(3)),
            lambda: cross(q, k, k, s, long(2, 1)),
            lambda: cross(t(2, 4, 5, 0), t(2, 2, 7, 0), k, s),
            lambda: cross(q.double(), k.double(), k.double(), s),
            lambda: axes(qk, qk, c, c, long(2, 2, 7), (1, 2)),
            lambda: axes(qk, qk, c, c, long(2, 2, 7), (5, -1)),
            lambda: axes(qk, qk, c, c, long(2, 2, 7), ()),
            lambda: axes(qk, qk, c, c, long(5, 2, 7), (1, 1, 1, 1, 0)),
            lambda: axes(qk, qk, c, c, long(3, 2, 7), (2, 2)),
            lambda: axes(qk, qk, c, c, long(2, 7), (2, 2)),
            lambda: axes(qk, qk, c, c, long(2, 2, 6), (2, 2)),
            lambda: axes(qk, qk, c, c, t(2, 2, 7), (2, 2)),
            lambda: block.RbfBlock(64, 4, 64, sections=(4, 5)),
            lambda: block.RbfCrossBlock(64, 32, 4, 3, 64),
            lambda: block.RbfBlock(64, 4, 64, sections=(4, 4))(t(1, 3, 64))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: norm(t(1, 16385), t(1, 16385)),
                lambda: cross(t(1, 1, 1, 257), t(1, 1, 1, 257), t(1, 1, 1, 8),
                              t(1, 1, 1, 1)),
                lambda: cross(t(1, 1, 1, 8), t(1, 1, 1, 8), t(1, 1, 1, 300),
                              t(1, 1, 1, 1))):
        with pytest.raises(NotImplementedError):
            bad()


@pytest.mark.parametrize('device', DEVICES)
def test_no_forward_mode_or_second_derivative(device):
    from torch.autograd import forward_ad
    x = torch.randn(2, 8, device=device, requires_grad=True)
    q = torch.randn(1, 1, 3, 8, device=device, requires_grad=True)
    rng = rng_of(1, 1, device)
    s = torch.ones(1, 1, 1, 1, device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        dq = forward_ad.make_dual(q.detach(), torch.ones_like(q))
        for call in (lambda: block.dropout(dual, 0.5, rng),
                     lambda: block.residual_norm(dual, dual),
                     lambda: block.cross_attention(dq, dq, dq, s)):
            with pytest.raises(NotImplementedError):
                call()
    for y, t in ((block.residual_norm(x, x)[1], x),
                 (block.cross_attention(q, q, q, s), q)):
        g, = torch.autograd.grad(y.square().sum(), t, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
    # Dropout is linear: it goes on.
    y = block.dropout(x, 0.5, rng)
    g, = torch.autograd.grad(y.pow(3).sum(), x, create_graph=True)
    assert torch.autograd.grad(g.sum(), x)[0].shape == x.shape


def _op_calls(device):
    rand = Rand(71, device, torch.float32)
    leaf = lambda *s: rand(*s).requires_grad_()  # noqa: E731
    cos, sin = block.rotation_tables(5, 8, device=device)
    ops = torch.ops.vectra_b200
    rng = rng_of(1, 2, device)
    pos = torch.zeros(2, 2, 5, dtype=torch.int64, device=device)
    lengths = torch.tensor([5, 2], device=device)
    return [
        (ops.dropout.default, (leaf(3, 8), 0.3, rng, 4)),
        (ops.residual_norm.default,
         (leaf(2, 3, 8), leaf(2, 3, 8), leaf(8), leaf(8), leaf(8),
          leaf(2, 1, 8), 0.5, 0.3, rng, 1, 1e-6, 'layer')),
        (ops.residual_norm.default, (leaf(3, 8),)),
        (ops.qk_norm_rope_axes.default,
         (leaf(2, 3, 5, 8), leaf(2, 1, 5, 8), cos, sin, pos, [1, 3], leaf(8),
          leaf(8))),
        (ops.cross_attention.default,
         (leaf(2, 2, 3, 8), leaf(2, 1, 5, 8), leaf(2, 1, 5, 8),
          leaf(1, 2, 1, 1), lengths)),
        (ops.cross_attention.default,
         (rand(2, 2, 3, 8).bfloat16().requires_grad_(),
          rand(2, 1, 5, 8).bfloat16(), rand(2, 1, 5, 8).bfloat16(),
          rand(1, 2, 1, 1))),
    ]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('case', range(6))
def test_opcheck(device, case):
    op, args = _op_calls(device)[case]
    torch.library.opcheck(op, args, test_utils=(
        'test_schema', 'test_faketensor', 'test_aot_dispatch_static',
        'test_aot_dispatch_dynamic'))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_cross_block_runs_them_together(device, dtype):
    """RbfCrossBlock: every parameter gets a gradient, states past a length
    change nothing, dropout acts in training only and by its rng."""
    torch.manual_seed(0)
    blk = block.RbfCrossBlock(64, 48, 4, 2, 96, dropout=0.2,
                              residual_scale=0.9).to(device, dtype)
    assert blk.log_scale.dtype == torch.float32
    rand = Rand(81, device, dtype)
    x, states = rand(3, 9, 64), rand(3, 21, 48)
    lengths = torch.tensor([21, 0, 6], device=device)
    rng = rng_of(5, 6, device)
    y = blk(x, states, lengths, rng)
    assert torch.equal(y, blk(x, states, lengths, rng))
    assert not torch.equal(y, blk(x, states, lengths, rng_of(5, 7, device)))
    assert not torch.equal(y, blk(x, states, lengths, rng,
                                  block.RbfCrossBlock.STREAMS))
    y.float().square().mean().backward()
    for name, p in blk.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    blk.eval()
    trained = blk(x, states, lengths)
    with torch.no_grad():
        served = blk(x, states, lengths)
        other = states.clone()
        other[1], other[2, 6:] = 9.0, -9.0
        assert torch.equal(served, blk(x, other, lengths))
    # Training keeps what the weights' rounding left, serving does not: one
    # rounding of the attention's result, on a stream of order 4.
    np.testing.assert_allclose(d(trained).numpy(), d(served).numpy(), rtol=0,
                               atol=16 * U[dtype] + 1e-4)


@pytest.mark.parametrize('device', DEVICES)
def test_block_with_sections(device):
    torch.manual_seed(0)
    blk = block.RbfBlock(64, 2, 96, max_positions=32,
                         sections=(4, 6, 6)).to(device)
    plain = block.RbfBlock(64, 2, 96, max_positions=32).to(device)
    plain.load_state_dict(blk.state_dict())
    x = Rand(82, device, torch.float32)(2, 7, 64)
    pos = torch.randint(0, 32, (2, 7)).to(device)
    assert torch.equal(blk(x, positions=pos.expand(3, 2, 7)),
                       plain(x, positions=pos))
    blk(x, positions=torch.randint(0, 32, (3, 2, 7)).to(
        device)).sum().backward()
    for name, p in blk.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name


# ---------------------------------------------------------------------------
# The C ABI, without a device.
# ---------------------------------------------------------------------------
class _Drop(ctypes.Structure):
    """vectra_drop."""
    _fields_ = [('p', ctypes.c_double), ('rng', ctypes.c_void_p),
                ('stream', ctypes.c_uint32)]


class _NormArgs(ctypes.Structure):
    """vectra_residual_norm_args."""
    _fields_ = [(n, _lib.Tensor) for n in (
        'x', 'branch', 'weight', 'bias', 'branch_weight', 'gate', 'x_out',
        'y', 'stats')] + [('drop', _Drop), ('residual_scale', ctypes.c_double),
                          ('eps', ctypes.c_double), ('kind', ctypes.c_int32)]


class _CrossArgs(ctypes.Structure):
    """vectra_cross_args."""
    _fields_ = [(n, _lib.Tensor) for n in ('q', 'k', 'v', 'scale')] + [
        ('key_lengths', ctypes.c_void_p), ('length_bytes', ctypes.c_int32),
        ('length_stride', ctypes.c_int64)] + [
            (n, _lib.Tensor) for n in ('out', 'lse', 'rest')] + [
                ('workspace', ctypes.c_void_p),
                ('workspace_bytes', ctypes.c_size_t)]


class _DropoutArgs(ctypes.Structure):
    """vectra_dropout_args."""
    _fields_ = [('x', _lib.Tensor), ('y', _lib.Tensor), ('drop', _Drop)]


def _abi(shape, dtype=_lib.BF16, strides=None, addr=0x10000):
    t = _lib.Tensor()
    t.data, t.dtype, t.ndim = addr, dtype, len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        t.size[i] = shape[i]
        t.stride[i] = step if strides is None else strides[i]
        step *= shape[i]
    return t


def test_abi_statuses():
    """The C entries answer statuses without touching a device."""
    def entry(name, result=ctypes.c_int):
        f = getattr(_lib.LIB, name)
        f.restype = result
        f.argtypes = [ctypes.c_void_p] * (1 if 'bytes' in name else 2)
        return f

    drop = entry('vectra_dropout')
    a = _DropoutArgs(_abi((4, 8)), _abi((4, 8)), _Drop(0.5, None, 0))
    assert drop(ctypes.byref(a), None) == _lib.ERR_NULL
    a.drop = _Drop(1.5, 0x10000, 0)
    assert drop(ctypes.byref(a), None) == _lib.ERR_UNSUPPORTED
    a.drop = _Drop(0.5, 0x10000, 0)
    a.y = _abi((4, 8), strides=(16, 1))
    assert drop(ctypes.byref(a), None) == -12  # VECTRA_ERR_LAYOUT
    assert drop(None, None) == _lib.ERR_NULL

    norm = entry('vectra_residual_norm_forward')

    def status(**over):
        n = _NormArgs(x=_abi((6, 8)), branch=_abi((6, 8)),
                      weight=_abi((8,)), x_out=_abi((6, 8)), y=_abi((6, 8)),
                      residual_scale=1.0, eps=1e-6)
        for name, value in over.items():
            setattr(n, name, value)
        return norm(ctypes.byref(n), None)

    assert status(x=_abi((48,))) == _lib.ERR_RANK
    assert status(x=_abi((6, 8), _lib.F64)) == _lib.ERR_DTYPE
    assert status(branch=_abi((6, 9))) == _lib.ERR_SHAPE
    assert status(gate=_abi((4, 8))) == _lib.ERR_SHAPE
    assert status(kind=2) == _lib.ERR_UNSUPPORTED
    assert status(y=_lib.Tensor()) == _lib.ERR_NULL  # weight without a norm
    assert status(branch=_lib.Tensor(), gate=_abi((1, 8))) == _lib.ERR_NULL
    assert status(y=_abi((6, 8), strides=(9, 1))) == -12
    assert status(x=_abi((6, 16392)), branch=_abi((6, 16392))) == \
        _lib.ERR_UNSUPPORTED

    size = entry('vectra_cross_attention_forward_workspace_bytes',
                 ctypes.c_int64)

    def need(**over):
        c = _CrossArgs(q=_abi((2, 4, 5, 64)), k=_abi((2, 2, 7, 64)),
                       v=_abi((2, 2, 7, 64)), scale=_abi((1, 4, 1, 1),
                                                         _lib.F32),
                       out=_abi((2, 4, 5, 64)))
        for name, value in over.items():
            setattr(c, name, value)
        return size(ctypes.byref(c))

    assert need() == 0
    assert need(q=_abi((2, 4, 64))) == _lib.ERR_RANK
    assert need(k=_abi((2, 3, 7, 64)), v=_abi((2, 3, 7, 64))) == \
        _lib.ERR_SHAPE
    assert need(scale=_abi((1, 3, 1, 1), _lib.F32)) == _lib.ERR_SCALE_SHAPE
    assert need(key_lengths=0x10000, length_bytes=2) == _lib.ERR_DTYPE
    assert need(lse=_abi((2, 4, 5))) == _lib.ERR_DTYPE
    assert need(out=_abi((2, 4, 5, 64), strides=(1280, 320, 1, 5))) == -12
    wide = [_abi((2, n, 7, 300)) for n in (4, 2)]
    assert need(q=wide[0], k=wide[1]) == _lib.ERR_UNSUPPORTED


# ---------------------------------------------------------------------------
# Streams, graphs, threads, far addresses.
# ---------------------------------------------------------------------------
def _together(rand, rng):
    """One call of each with gradients; (results, leaves)."""
    x, br = rand(2, 70, 64), rand(2, 70, 64)
    w, g = 1 + rand(64, scale=0.1), rand(2, 1, 64)
    kv = rand(2, 90, 2, 1, 32)
    s = torch.full((1, 2, 1, 1), 0.1, device=x.device)
    leaves = [t.requires_grad_() for t in (x, br, w, g, kv, s)]
    lengths = torch.tensor([90, 31], device=x.device)

    def run():
        y, n = block.residual_norm(x, br, w, gate=g, branch_weight=w, p=0.2,
                                   rng=rng)
        q = n.view(2, 70, 2, 32).transpose(1, 2)
        k, v = kv.permute(2, 0, 3, 1, 4)
        o = block.cross_attention(q, k, v, s, lengths)
        o = block.dropout(o.transpose(1, 2).reshape(2, 70, 64), 0.1, rng, 1)
        grads = torch.autograd.grad((o * y).float().sum(), leaves)
        # No graph stays alive between a run and a captured one.
        return [t.detach() for t in (y, n, o, *grads)]

    return run, leaves


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_repeats_streams_and_graphs(dtype):
    """Bit for bit: a second run, another stream, and a captured run replayed
    with new inputs and a new step."""
    rng = rng_of(1, 2, 'cuda')
    run, leaves = _together(Rand(91, 'cuda', dtype), rng)
    want = run()
    for a, b in zip(run(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    with torch.no_grad():
        for t in leaves[:5]:
            t.mul_(0.75)
        rng[1] += 1
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, run()):
        assert torch.equal(a, b)
    assert _lib.check_device_errors(
        torch.cuda.current_stream().cuda_stream) == _lib.OK


@pytest.mark.gpu
def test_two_graphs_and_threads():
    """Two captured runs in turn, and runs from threads, each on a stream of
    its own: workspaces are a call's own."""
    import threading
    rng = rng_of(1, 2, 'cuda')
    runs = [_together(Rand(s, 'cuda', torch.bfloat16), rng)[0]
            for s in (92, 93)]
    want = [[t.clone() for t in run()] for run in runs]
    graphs = []
    for run in runs:
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for _ in range(3):
        for graph, _out in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for (_graph, out), ref in zip(graphs, want):
        for a, b in zip(out, ref):
            assert torch.equal(a, b)
    results, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    results[i] = runs[i % 2]()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    torch.cuda.synchronize()
    for i, out in enumerate(results):
        for a, b in zip(out, want[i % 2]):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_offsets_past_32_bits(dtype):
    """Views whose elements lie more than 2^31 elements apart."""
    far = (1 << 31) + 64
    store = torch.zeros(far + (1 << 16), dtype=dtype, device='cuda')
    rand = Rand(95, 'cuda', dtype)
    q, k, v, scale = cross_inputs(rand, 2, 2, 1, 5, 70, 64)
    views = []
    at = 0
    for t in (q, k, v):
        t = t.contiguous()
        view = store.as_strided(t.shape, (far, *t.stride()[1:]), at)
        view.copy_(t)
        views.append(view)
        at += t[0].numel()
    out = check_cross(*views, scale, None, rand(2, 2, 5, 64))
    assert torch.equal(out, block.cross_attention(
        *(t.contiguous() for t in views), scale.detach()))
    rows = store.as_strided((2, 64), (far, 1), 40960)
    rows.copy_(rand(2, 64))
    near = rows.contiguous()
    w = 1 + rand(64, scale=0.1)
    for a, b in zip(block.residual_norm(rows, rows, w),
                    block.residual_norm(near, near, w)):
        assert torch.equal(a, b)
    rng = rng_of(1, 1, 'cuda')
    assert torch.equal(block.dropout(rows, 0.5, rng),
                       block.dropout(near, 0.5, rng))


@pytest.mark.gpu
def test_dropout_past_32_bits():
    """Elements past 2^32 of one tensor have numbers of their own."""
    n = (1 << 32) + 4096
    x = torch.ones(n, dtype=torch.bfloat16, device='cuda')
    y = block.dropout(x, 0.5, rng_of(7, 8, 'cuda'), 9)
    del x
    first = (1 << 32) // 8
    words = []
    for g in range(first, first + 64):
        for w in philox([g & 0xffffffff, g >> 32, 8, 9], [7, 0]):
            words += [(w & 0xffff) >= 32768, (w >> 16) >= 32768]
    at = first * 8
    assert torch.equal((y[at:at + 512] != 0).cpu(), torch.tensor(words))
