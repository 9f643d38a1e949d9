"""The decoder operators (vectra_b200.block) beside the ordinary: values that
are not finite, small gradients, rows far from zero, long walks and split axes,
and what a call has to refuse.

A test that compares whole tensors does so by their norms: with `u` the unit
roundoff (half a step, relative to the value), a result that is rounded once
is off by at most u of its norm. The roundings spread evenly over the steps,
so that it is off by 0.39 u where its mantissas spread evenly over a binade's
logarithm (the error of m 2^e is uniform in u 2^e: mean squares u^2 / 3 against
1.5 / ln 2 for m^2), and by no more than u / sqrt(3) = 0.58 u if all mantissas
were 1. ONCE = 0.5 lies between: two roundings of a value, or of the values
that it sums, are off by 0.39 sqrt(2) = 0.55 u.
"""

import ctypes
import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tests.test_decoder import DEVICES
from tests.test_decoder import TINY
from tests.test_decoder import TYPES
from tests.test_decoder import U
from tests.test_decoder import Rand
from tests.test_decoder import _abi
from tests.test_decoder import _Drop
from tests.test_decoder import _NormArgs
from tests.test_decoder import check_cross
from tests.test_decoder import cross_inputs
from tests.test_decoder import d
from tests.test_decoder import sums
from vectra_b200 import _lib
from vectra_b200 import block

HALVES = [torch.bfloat16, torch.float16]
ONCE = 0.5


def off(got, want, dtype):
    """The error of a tensor as a share of its norm, in units of u."""
    return float((d(got) - want).norm() / want.norm()) / U[dtype]


def gradients(leaves, lengths, dout):
    leaves = [t.detach().clone().requires_grad_() for t in leaves]
    out = block.cross_attention(*leaves, lengths)
    return out.detach(), torch.autograd.grad(out, leaves, dout)


def exact_cross(q, k, v, scale, lengths, dout):
    """out, dq, dk, dv in float64, by matrix products a sequence at a time."""
    b, h, nq = q.shape[:3]
    hk, nk = k.shape[1:3]
    rep = h // hk
    Q, K, V, G = d(q), d(k), d(v), d(dout)
    S = d(scale).expand(b, h, 1, 1)
    n = torch.full((b,), nk) if lengths is None else lengths.cpu()
    out, dq = torch.zeros_like(G), torch.zeros_like(Q)
    dk, dv = torch.zeros_like(K), torch.zeros_like(V)
    for i in range(b):
        m = int(n[i])
        for j in range(h):
            x, y, z = Q[i, j], K[i, j // rep, :m], V[i, j // rep, :m]
            g, e = S[i, j], G[i, j]
            dist = x.square().sum(-1, keepdim=True) + y.square().sum(-1) - \
                2 * x @ y.mT
            w = torch.softmax(-g * dist, -1)
            out[i, j] = w @ z
            t = w * (e @ z.mT - (e * out[i, j]).sum(-1, keepdim=True))
            dq[i, j] = 2 * g * (t @ y - t.sum(-1, keepdim=True) * x)
            dk[i, j // rep, :m] += 2 * g * (t.mT @ x -
                                            t.sum(0)[:, None] * y)
            dv[i, j // rep, :m] += w.mT @ e
    return out, dq, dk, dv


# ---------------------------------------------------------------------------
# cross_attention: values that are not finite.
# ---------------------------------------------------------------------------
# b, h, hk, nq, nk, D, and a length whose last key is alone in its part where
# the kernels split the keys (16 a step up to 16 packed queries, else tiles of
# 128, and of 64 in float32 and for odd widths): up to 8, up to 16 and more
# packed queries, split and not.
NAN_SIZES = [(2, 2, 2, 1, 700, 64, 17), (2, 2, 2, 1, 24, 64, 17),
             (2, 6, 2, 4, 700, 128, 17), (2, 6, 2, 4, 24, 32, 17),
             (2, 4, 2, 20, 1100, 64, 129), (2, 4, 2, 20, 1100, 128, 129),
             (2, 4, 2, 20, 140, 64, 129), (2, 4, 2, 20, 700, 33, 65)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', NAN_SIZES)
@pytest.mark.parametrize('where', ['key', 'value', 'far value'])
def test_cross_nan_in_a_seen_key(device, dtype, size, where):
    """It reaches every query of the key's heads (a value's: its component, of
    a key that weighs nothing too), and nothing else."""
    b, h, hk, nq, nk, dim, n = size
    rand = Rand(nk + dim, device, dtype)
    q, k, v, scale = cross_inputs(rand, b, h, hk, nq, nk, dim)
    dout = rand(b, h, nq, dim)
    lengths = torch.tensor([n, nk], device=device)
    if where == 'far value':
        k[0, 0, n - 1] = 60.0
    clean, cleans = gradients((q, k, v, scale), lengths, dout)
    (k if where == 'key' else v)[0, 0, n - 1, 3] = math.nan
    out, (dq, dk, dv, dscale) = gradients((q, k, v, scale), lengths, dout)
    own = h // hk
    if where == 'key':
        assert out[0, :own].isnan().all()
        assert dv[0, 0, :n].isnan().all()
    else:
        assert out[0, :own, :, 3].isnan().all()
        assert out[0, :own, :, :3].isfinite().all()
        assert dv[0, 0].isfinite().all()
    assert dq[0, :own].isnan().all()
    assert dk[0, 0, :n].isnan().all()
    assert dscale[0, :own].isnan().all()
    with torch.no_grad():
        served = block.cross_attention(q, k, v, scale, lengths)
    assert torch.equal(served.isnan(), out.isnan())
    for got, want in ((out, clean), (dq, cleans[0])):
        assert got[0, own:].isfinite().all() and got[1].isfinite().all()
        assert torch.equal(got[1], want[1])
    for got, want in ((dk, cleans[1]), (dv, cleans[2])):
        assert (got[0, :, n:] == 0).all()
        assert torch.equal(got[0, 1:], want[0, 1:])
        assert torch.equal(got[1], want[1])


# ---------------------------------------------------------------------------
# cross_attention: the range of 16-bit operands.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('size', [(1, 2, 2, 3, 4500, 64),
                                  (1, 6, 1, 2, 4500, 128),
                                  (1, 2, 1, 250, 4500, 128),
                                  (2, 2, 2, 130, 2000, 48)])
@pytest.mark.parametrize('up', [1.0, 1e-2, 1e-3, 1e-4])
def test_cross_small_gradients(device, dtype, size, up):
    """Many keys and a small upstream gradient: the gradients are within twice
    their own rounding (float16's spacing, 2^-24, counted once a result)."""
    b, h, hk, nq, nk, dim = size
    rand = Rand(nk + dim, device, dtype)
    a = cross_inputs(rand, *size)
    dout = rand(b, h, nq, dim, scale=up)
    lengths = torch.tensor([nk, nk - 9][:b], device=device)
    got = gradients(a, lengths, dout)
    want = exact_cross(*a, lengths, dout)
    for x, y, name in zip((got[0], *got[1][:3]), want,
                          ('out', 'dq', 'dk', 'dv')):
        bound = 2 * (U[dtype] * y.norm() + TINY[dtype] / 2 *
                     math.sqrt(y.numel()))
        assert (d(x) - y).norm() <= bound, name


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('nq', [1, 5, 24])
def test_cross_gradients_of_unequal_rows(device, nq):
    """Rows whose upstream gradients lie far apart: each row of dq is within
    twice its own rounding."""
    rand = Rand(nq, device, torch.float16)
    b, h, hk, nk, dim = 2, 4, 2, 3000, 64
    a = cross_inputs(rand, b, h, hk, nq, nk, dim)
    size = torch.tensor([4.0, 0.25, 2.0**-6, 2.0**-10], device=device)
    dout = rand(b, h, nq, dim) * size.view(1, 4, 1, 1).half()
    got = gradients(a, None, dout)[1][0]
    want = exact_cross(*a, None, dout)[1]
    err = (d(got) - want).norm(dim=-1)
    bound = 2 * (U[torch.float16] * want.norm(dim=-1) + 2.0**-25 *
                 math.sqrt(dim))
    assert (err <= bound).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('nq', [2, 10, 24])
def test_cross_large_gradients(device, nq):
    """Upstream gradients whose products with the values pass float16's
    largest number, though no gradient does: within twice their rounding."""
    rand = Rand(nq, device, torch.float16)
    b, h, hk, nk, dim = 2, 2, 2, 6, 64
    q, k, v, _ = cross_inputs(rand, b, h, hk, nq, nk, dim)
    scale = torch.full((1, h, 1, 1), 0.01, device=device)
    dout = rand(b, h, nq, dim, scale=10000.0)
    got = gradients((q, k, 2 * v, scale), None, dout)
    want = exact_cross(q, k, 2 * v, scale, None, dout)
    for x, y, name in zip((got[0], *got[1][:3]), want,
                          ('out', 'dq', 'dk', 'dv')):
        assert y.abs().max() < 65504, name
        assert off(x, y, torch.float16) <= 2, name


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('nq', [3, 10, 40])
def test_cross_float16_weights_far_below_one(device, nq):
    """120,000 keys. Each weighs 2^-17: values' gradients are within twice
    their rounding. And with one key beside the queries, the others weigh 2^-25
    of it and still 0.36 % together."""
    rand = Rand(nq, device, torch.float16)
    b, h, hk, nk, dim = 1, 1, 1, 120000, 32
    q = rand(b, h, 1, dim, scale=0.1).expand(b, h, nq, dim).contiguous()
    k = q[:, :, :1] + rand(b, hk, nk, dim, scale=0.05)
    v = 1 + rand(b, hk, nk, dim)
    scale = torch.full((1, h, 1, 1), 0.5, device=device)
    dout = rand(b, h, nq, dim, scale=32.0)
    got = gradients((q, k, v, scale), None, dout)[1][2]
    want = exact_cross(q, k, v, scale, None, dout)[3]
    assert off(got, want, torch.float16) <= 2 + 2.0**-24 * math.sqrt(
        want.numel()) / (U[torch.float16] * float(want.norm()))
    # All but the first at a distance of 4 from the queries.
    q = torch.zeros_like(q)
    k = rand(b, hk, nk, dim)
    k = (4 * k.float() / k.float().norm(dim=-1, keepdim=True)).half()
    k[:, :, 0] = 0.0
    v[:, :, 0] = 0.0
    scale = torch.full((1, h, 1, 1), 25 * math.log(2) / 16, device=device)
    out = block.cross_attention(q, k, v, scale)
    want = exact_cross(q, k, v, scale, None, dout)[0]
    # A distance is off by its products' rounding, 16 sums(32) at most.
    slack = 2 * float(scale.max()) * 32 * sums(dim)
    assert ((d(out) - want).abs() <= (2 * U[torch.float16] + slack) *
            want.abs()).all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('nq', [2, 6, 20])
@pytest.mark.parametrize('dim', [64, 33])
def test_cross_small_values(device, nq, dim):
    """Small values under large upstream gradients, and one large weight: what
    out's rounding left is in float16's range as well."""
    rand = Rand(nq, device, torch.float16)
    b, h, hk, nk = 2, 4, 2, 100
    q, k, v, _ = cross_inputs(rand, b, h, hk, nq, nk, dim)
    v = v * 1e-4
    scale = torch.full((1, h, 1, 1), 0.3, device=device)
    dout = rand(b, h, nq, dim, scale=4000.0)
    got = gradients((q, k, v, scale), None, dout)
    want = exact_cross(q, k, v, scale, None, dout)
    for x, y, name in zip(got[1][:2], want[1:3], ('dq', 'dk')):
        assert off(x, y, torch.float16) <= 1, name


# ---------------------------------------------------------------------------
# cross_attention: one rounding a result.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('size', [(4, 4, 4, 1, 300, 64),
                                  (2, 8, 2, 3, 300, 128),
                                  (1, 4, 2, 150, 500, 128),
                                  (2, 2, 2, 200, 300, 32)])
def test_cross_results_are_rounded_once(device, dtype, size):
    """Weights and their gradients enter the products with what their
    rounding left: results and gradients are off by their own rounding, and a
    call that will have no backward pass gives the same bits."""
    b, h, hk, nq, nk, dim = size
    rand = Rand(nk + dim, device, dtype)
    a = cross_inputs(rand, *size)
    dout = rand(b, h, nq, dim)
    out, grads = gradients(a, None, dout)
    assert torch.equal(out, block.cross_attention(*a))
    want = exact_cross(*a, None, dout)
    for got, y, name in zip((out, *grads[:3]), want,
                            ('out', 'dq', 'dk', 'dv')):
        assert off(got, y, dtype) <= ONCE, name


# ---------------------------------------------------------------------------
# cross_attention: long walks, split axes, few keys.
# ---------------------------------------------------------------------------
def check_long(a, lengths, dout):
    """check_cross for sizes whose differences of all queries and keys would
    not fit: |q - k| is at most |q| + |k| where it weighs an error. Training
    keeps what the rounding of weights left."""
    q, k, v, scale = a
    dtype, dim, dv_ = q.dtype, q.shape[3], v.shape[3]
    b, h, nq = q.shape[:3]
    hk, nk = k.shape[1:3]
    rep, u, tiny = h // hk, U[dtype], TINY[dtype]
    out, (dq, dk, dv, _) = gradients(a, lengths, dout)
    want = exact_cross(*a, lengths, dout)
    n = torch.full((b,), nk) if lengths is None else lengths.cpu()
    bounds = [torch.zeros_like(t) for t in want]
    for i in range(b):
        m = int(n[i])
        for j in range(h):
            x, y, z = d(q[i, j]), d(k[i, j // rep, :m]), d(v[i, j // rep, :m])
            e, g = d(dout[i, j]), float(d(scale).expand(b, h, 1, 1)[i, j])
            size = x.square().sum(-1, keepdim=True) + y.square().sum(-1) + \
                2 * x.abs() @ y.abs().mT
            dist = x.square().sum(-1, keepdim=True) + y.square().sum(-1) - \
                2 * x @ y.mT
            w = torch.softmax(-g * dist, -1)
            ew = torch.expm1(2 * (abs(g) * (sums(dim) + 2.0**-21) *
                                  size).amax(-1, keepdim=True) + sums(m))
            keep = 3 * u * u + sums(max(m, nq * rep))
            eo = (w * (ew + keep)) @ z.abs()
            bounds[0][i, j] = eo
            o = want[0][i, j]
            ec = (e.abs() * (eo + 3 * u * u * o.abs() + tiny)).sum(
                -1, keepdim=True) + sums(dv_) * (e * o).abs().sum(
                    -1, keepdim=True)
            t = (e @ z.mT - (e * o).sum(-1, keepdim=True)).abs()
            et = sums(dv_) * (e.abs() @ z.abs().mT)
            ez = 2 * abs(g) * w * ((ew + keep) * (t + et + ec) + et + ec)
            bounds[1][i, j] = ez.sum(-1, keepdim=True) * x.abs() + \
                ez @ y.abs()
            bounds[2][i, j // rep, :m] += ez.mT @ x.abs() + \
                ez.sum(0)[:, None] * y.abs()
            bounds[3][i, j // rep, :m] += (w * (ew + keep)).mT @ e.abs()
    for got, y, bound, name in zip((out, dq, dk, dv), want, bounds,
                                   ('out', 'dq', 'dk', 'dv')):
        err = (d(got) - y).abs()
        limit = bound * (1 + u) + u * y.abs() + tiny
        assert (err <= limit).all(), (name, float((err / limit).max()))


# By the 16-bit kernels' rules for more than 16 packed queries: keys that are
# split in the forward and the queries' pass (8 tiles of 128 and of 64 or
# more); queries that are split in the keys' pass; and enough blocks that
# nothing splits, with rings of up to four tiles that wrap twice, of keys and of
# queries.
LONG = [(1, 2, 1, 40, 1100, 64), (1, 2, 1, 40, 1030, 128),
        (1, 2, 1, 300, 200, 64), (1, 2, 1, 300, 190, 128),
        (3, 6, 2, 170, 1000, 64),
        (5, 16, 16, 20, 1290, 64), (5, 16, 16, 20, 1290, 128),
        (5, 16, 16, 600, 70, 64), (5, 16, 16, 600, 70, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('size', LONG)
@pytest.mark.parametrize('ragged', [False, True])
def test_cross_long_walks(dtype, size, ragged):
    b, h, hk, nq, nk, dim = size
    rand = Rand(nk + dim, 'cuda', dtype)
    a = cross_inputs(rand, *size)
    lengths = None
    if ragged:
        some = [nk - 1, nk // 2 + 1, nk, 1, 64]
        lengths = torch.tensor(some[:b], device='cuda')
    check_long(a, lengths, rand(b, h, nq, dim))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(2, 4, 2, 3, 64), (1, 6, 1, 2, 128),
                                  (2, 2, 1, 30, 64), (1, 1, 1, 150, 128),
                                  (1, 2, 2, 40, 33), (1, 2, 1, 20, 160)])
@pytest.mark.parametrize('nk', [2, 3])
def test_cross_two_and_three_keys(device, dtype, size, nk):
    b, h, hk, nq, dim = size
    rand = Rand(nk + dim, device, dtype)
    check_cross(*cross_inputs(rand, b, h, hk, nq, nk, dim),
                dout=rand(b, h, nq, dim))


# ---------------------------------------------------------------------------
# residual_norm: rows far from zero.
# ---------------------------------------------------------------------------
def exact_norm(x, branch, weight, bias, dx_out, dy, kind, eps):
    """Gradients of x, branch, weight and bias in float64."""
    leaves = [d(t).requires_grad_() for t in (x, branch, weight, bias)]
    v = leaves[0] + leaves[1]
    c = v - v.mean(-1, keepdim=True) if kind == 'layer' else v
    y = c * (c.square().mean(-1, keepdim=True) + eps).rsqrt() * leaves[2] + \
        leaves[3]
    return torch.autograd.grad((v, y), leaves, (d(dx_out), d(dy)))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('mean', [0.0, 16.0])
@pytest.mark.parametrize('size', [(2, 40, 256), (3, 30, 1000), (1, 7, 4096)])
def test_norm_gradients_of_rows_far_from_zero(device, dtype, kind, mean,
                                              size):
    """The stream's rounding does not enter the gradients of its norm, which a
    mean of many deviations would multiply: gradients are rounded once."""
    b, n, c = size
    rand = Rand(c, device, dtype)
    x, branch = rand(b, n, c) + mean, rand(b, n, c)
    weight, bias = 1 + rand(c, scale=0.2), rand(c)
    dx_out, dy = rand(b, n, c), rand(b, n, c)
    leaves = [t.requires_grad_() for t in (x, branch, weight, bias)]
    out = block.residual_norm(*leaves, kind=kind)
    got = torch.autograd.grad(out, leaves, (dx_out, dy))
    want = exact_norm(x, branch, weight, bias, dx_out, dy, kind, 1e-6)
    for a, y, name in zip(got, want, ('dx', 'dbranch', 'dweight', 'dbias')):
        # Of c roundings the share in a norm varies by sqrt(0.2 / c) of itself.
        assert off(a, y, dtype) <= ONCE * (1 + 3 * math.sqrt(
            0.2 / a.numel())), name


@pytest.mark.parametrize('device', DEVICES)
def test_norm_keeps_what_a_rounding_left_only_where_it_is_read(device):
    """Nothing is kept beside x_out for float32, without a branch, or where no
    norm follows."""
    op = torch.ops.vectra_b200.residual_norm_with_stats

    def rest(dtype, branch, norm, want=True):
        x = torch.ones(3, 16, device=device, dtype=dtype)
        return op(x, x if branch else None, None, None, None, None, 1.0, 0.0,
                  None, 0, 1e-6, 'rms', norm, want)[3]

    assert rest(torch.bfloat16, True, True).shape == (3, 16)
    for call in ((torch.float32, True, True), (torch.bfloat16, False, True),
                 (torch.float16, True, False),
                 (torch.float16, True, True, False)):
        assert rest(*call).numel() == 0


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('c', [256, 1000])
def test_norm_gradients_of_small_rows(device, kind, c):
    """What the stream's rounding left is in float16's range as well: rows of
    2e-5, whose own spacing is 6e-8."""
    rand = Rand(c, device, torch.float16)
    x, branch = rand(2, 30, c, scale=2e-5), rand(2, 30, c, scale=2e-5)
    # The sum with a scale is rounded where a plain one would be exact.
    weight, dy = 1 + rand(c, scale=0.2), rand(2, 30, c, scale=1e-4)
    x, branch, weight = leaves = [t.requires_grad_() for t in
                                  (x, branch, weight)]
    y = block.residual_norm(x, branch, weight, residual_scale=0.7, kind=kind,
                            eps=1e-12)[1]
    got = torch.autograd.grad(y, leaves, dy)
    X, R, W = (d(t).requires_grad_() for t in leaves)
    v = 0.7 * X + R
    t = v - v.mean(-1, keepdim=True) if kind == 'layer' else v
    t = t * (t.square().mean(-1, keepdim=True) + 1e-12).rsqrt() * W
    want = torch.autograd.grad(t, (X, R, W), d(dy))
    for a, b, name in zip(got, want, ('dx', 'dbranch', 'dweight')):
        # (dweight's own spacing: 30 gradients of 1e-4 have sums of 8e-4.)
        assert off(a, b, torch.float16) <= ONCE * (1 + 3 * math.sqrt(
            0.2 / a.numel())) + 2.0**-24 / 3 / (
                U[torch.float16] * float(b.square().mean().sqrt())), name


# ---------------------------------------------------------------------------
# All of them.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_checkpointed_block(device, dtype):
    """A block whose forward pass runs without gradients and again with them:
    the same bits, results and gradients, as one that keeps everything."""
    torch.manual_seed(1)
    blk = block.RbfCrossBlock(64, 48, 4, 2, 96, dropout=0.1).to(device, dtype)
    rand = Rand(101, device, dtype)
    x, states = rand(3, 40, 64).requires_grad_(), rand(3, 70, 48)
    lengths = torch.tensor([70, 0, 33], device=device)
    rng = torch.tensor([5, 6], device=device)
    dy = rand(3, 40, 64)
    leaves = [x, *blk.parameters()]
    y = blk(x, states, lengths, rng)
    want = torch.autograd.grad(y, leaves, dy)
    z = checkpoint(blk, x, states, lengths, rng, use_reentrant=False)
    got = torch.autograd.grad(z, leaves, dy)
    assert torch.equal(y, z)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(y, blk(x, states, lengths, rng))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', HALVES)
def test_opcheck_of_16_bit_norms(device, dtype):
    rand = Rand(102, device, dtype)
    leaves = [rand(*s).requires_grad_() for s in (
        (2, 3, 8), (2, 3, 8), (8,), (8,), (8,), (2, 1, 8))]
    torch.library.opcheck(
        torch.ops.vectra_b200.residual_norm.default,
        (*leaves, 0.5, 0.0, None, 0, 1e-6, 'layer'),
        test_utils=('test_schema', 'test_faketensor',
                    'test_aot_dispatch_static', 'test_aot_dispatch_dynamic'))
    torch.library.opcheck(
        torch.ops.vectra_b200.residual_norm_with_stats.default,
        (*(t.detach() for t in leaves), 0.5, 0.0, None, 0, 1e-6, 'layer',
         True, True), test_utils=('test_schema', 'test_faketensor'))


# ---------------------------------------------------------------------------
# The C ABI, without a device.
# ---------------------------------------------------------------------------
class _NormGradArgs(ctypes.Structure):
    """vectra_residual_norm_grad_args."""
    _fields_ = [('fwd', _NormArgs)] + [(n, _lib.Tensor) for n in (
        'dx_out', 'dy', 'dx', 'dbranch', 'dweight', 'dbias', 'dbranch_weight',
        'dgate')] + [('workspace', ctypes.c_void_p),
                     ('workspace_bytes', ctypes.c_size_t)]


def test_abi_statistics_start_on_16_bytes():
    """The kernels move a row's four statistics at once."""
    forward = _lib.LIB.vectra_residual_norm_forward
    size = _lib.LIB.vectra_residual_norm_backward_workspace_bytes
    size.restype = ctypes.c_int64
    layout = -12  # VECTRA_ERR_LAYOUT

    def args(addr, **over):
        n = _NormArgs(x=_abi((6, 8)), branch=_abi((6, 8)), x_out=_abi((6, 8)),
                      y=_abi((6, 8)), stats=_abi((6, 4), _lib.F32, addr=addr),
                      drop=_Drop(0.0, None, 0), residual_scale=1.0, eps=1e-6)
        for name, value in over.items():
            setattr(n, name, value)
        return n

    for addr in (0x10004, 0x10008):
        assert forward(ctypes.byref(args(addr)), None) == layout
    for addr, status in ((0x10004, layout), (0x10008, layout),
                         (0x10010, _lib.OK)):
        g = _NormGradArgs(fwd=args(addr), dy=_abi((6, 8)), dx=_abi((6, 8)))
        got = size(ctypes.byref(g))
        assert (got if status else min(got, 0)) == status




class _NormTrainArgs(ctypes.Structure):
    """vectra_residual_norm_train_args."""
    _fields_ = [('fwd', _NormArgs), ('rest', _lib.Tensor)]


class _NormTrainGradArgs(ctypes.Structure):
    """vectra_residual_norm_train_grad_args."""
    _fields_ = [('grad', _NormGradArgs), ('rest', _lib.Tensor)]


def test_abi_statuses_of_a_kept_rest():
    forward = _lib.LIB.vectra_residual_norm_forward_train
    size = _lib.LIB.vectra_residual_norm_backward_train_workspace_bytes
    size.restype = ctypes.c_int64
    backward = _lib.LIB.vectra_residual_norm_backward_train

    def norm(dtype, **over):
        n = _NormArgs(x=_abi((6, 8), dtype), branch=_abi((6, 8), dtype),
                      x_out=_abi((6, 8), dtype), y=_abi((6, 8), dtype),
                      stats=_abi((6, 4), _lib.F32),
                      drop=_Drop(0.0, None, 0), residual_scale=1.0, eps=1e-6)
        for name, value in over.items():
            setattr(n, name, value)
        return n

    def there(rest, dtype=_lib.BF16, **over):
        a = _NormTrainArgs(norm(dtype, **over), rest)
        return forward(ctypes.byref(a), None)

    def back(rest, dtype=_lib.BF16, **over):
        g = _NormGradArgs(fwd=norm(dtype), dy=_abi((6, 8), dtype),
                          dx=_abi((6, 8), dtype))
        for name, value in over.items():
            setattr(g, name, value)
        return size(ctypes.byref(_NormTrainGradArgs(g, rest)))

    for call in (there, back):
        assert call(_abi((6, 8), _lib.F32), _lib.F32) == _lib.ERR_DTYPE
        assert call(_abi((6, 8), _lib.F16)) == _lib.ERR_DTYPE
        assert call(_abi((6, 9))) == _lib.ERR_SHAPE
        assert call(_abi((6, 8), strides=(16, 1))) == -12
    assert there(_abi((6, 8)), y=_lib.Tensor()) == _lib.ERR_NULL
    assert back(_abi((6, 8)), dy=_lib.Tensor(),
                dx_out=_abi((6, 8))) == _lib.ERR_NULL
    assert back(_lib.Tensor()) >= 0 and back(_abi((6, 8))) >= 0
    assert forward(None, None) == backward(None, None) == size(None) == \
        _lib.ERR_NULL
