"""Cases, plain forms and float64 values of a decoder block's operators.

They stand around the attention of a transformer block that reads an
encoder's states, in serving and training, and are reached through
vectra_b200.block:

* dropout(x, p, rng, stream): zeros a share p of x and scales the rest; the
  mask is a function of rng = (seed, step), stream and an element's index,
  and is never stored.
* residual_norm(x, branch, ...): the norm of a sublayer's result, dropout,
  its gate, the scaled residual and the next sublayer's norm in one pass:
    u = norm(branch) * branch_weight        (branch_weight given)
    x_out = residual_scale * x + gate * dropout(u)
    y = norm(x_out) * weight + bias
* qk_norm_rope_axes(q, k, cos, sin, positions, sections, ...): the RMS norm
  of query and key head vectors and a rotation whose pairs take their
  position from one of several axes.
* cross_attention(q, k, v, scale, key_lengths): RBF attention of queries to
  the states of an encoder, of another and per sequence different length,
  with shared key heads:
    softmax_j(-scale * |q_i - k_j|^2) V over j < key_lengths.

A "train" case is the forward pass and the backward pass through autograd;
its outputs are the results and every gradient.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16,
           'f32': torch.float32}
_BYTES = {'bf16': 2, 'f16': 2, 'f32': 4}
_EPS = 1e-6
# No drawn case costs more than the largest listed one of its kind.
_MOST_ELEMENTS = {'dropout': 6.7e7, 'norm': 3.4e7}
_MOST_ROTATED = 3.2e7         # qk_norm_rope_axes
_MOST_FLOPS = 5.9e11          # cross_attention
_MOST_FLOPS_F32 = 2.0e10
_MOST_LOGITS = 5.8e8          # weights the plain form of attention holds


# ---------------------------------------------------------------------------
# Cases.
# ---------------------------------------------------------------------------
def _dropout(name, dtype, batch, tokens, width, p, train):
    return {'name': name, 'op': 'dropout', 'dtype': dtype, 'batch': batch,
            'tokens': tokens, 'width': width, 'p': p, 'train': train}


def _norm(name, dtype, batch, tokens, width, kind, bias, branch_norm, gate,
          scale, p, train):
    return {'name': name, 'op': 'norm', 'dtype': dtype, 'batch': batch,
            'tokens': tokens, 'width': width, 'kind': kind, 'bias': bias,
            'branch_norm': branch_norm, 'gate': gate, 'scale': scale, 'p': p,
            'train': train}


def _axes(name, dtype, batch, tokens, heads, kv_heads, dim, sections, table,
          interleaved, train):
    return {'name': name, 'op': 'axes', 'dtype': dtype, 'batch': batch,
            'tokens': tokens, 'heads': heads, 'kv_heads': kv_heads,
            'dim': dim, 'sections': sections, 'table': table,
            'interleaved': interleaved, 'train': train}


def _cross(name, dtype, batch, heads, kv_heads, queries, keys, dim, ragged,
           train):
    return {'name': name, 'op': 'cross', 'dtype': dtype, 'batch': batch,
            'heads': heads, 'kv_heads': kv_heads, 'queries': queries,
            'keys': keys, 'dim': dim, 'ragged': ragged, 'train': train}


def listed():
    return [
        # Dropout on a float32 encoder's small ragged batch.
        _dropout('dropout_encoder', 'f32', 7, 65, 250, 0.3, True),
        # Dropout on a wide layer's activations in training.
        _dropout('dropout_wide_train', 'bf16', 4, 4099, 4096, 0.1, True),
        # Between two sublayers of one serving step of 64 sequences.
        _norm('norm_step', 'bf16', 64, 1, 4096, 'rms', False, True, 'none',
              1.0, 0.0, False),
        # The price model's blocks in training: layer norm, a learned gate
        # per channel, dropout; 1,024 targets with 64 comparables each.
        _norm('norm_price_train', 'bf16', 1024, 65, 256, 'layer', True, False,
              'channel', 1.0, 0.1, True),
        # A wide block in training: norms on both sides, a gate for each
        # sequence, a scaled residual.
        _norm('norm_wide_train', 'bf16', 3, 2731, 5120, 'rms', False, True,
              'sequence', 0.7, 0.0, True),
        # A prompt of image patches: positions in time, height and width.
        _axes('axes_prompt', 'bf16', 4, 2305, 32, 8, 128, '16,24,24', 4096,
              False, False),
        # The price model in training: sale day, latitude and longitude as
        # the axes of its comparables, all float16.
        _axes('axes_price_train', 'f16', 1024, 65, 8, 8, 32, '4,6,6', 8192,
              True, True),
        # One new token of 32 sequences over an encoder's cached states.
        _cross('cross_step', 'bf16', 32, 32, 8, 1, 4001, 128, True, False),
        # A subject attends to its 64 comparables: the price model's heads,
        # in training.
        _cross('cross_price_train', 'bf16', 1024, 8, 8, 1, 64, 32, True,
               True),
        # A short float32 decoder over a longer encoder, in training.
        _cross('cross_f32_train', 'f32', 4, 8, 8, 257, 700, 64, True, True),
        # A long prompt over an encoder's states.
        _cross('cross_prompt', 'f16', 1, 32, 8, 4096, 5003, 128, False,
               False),
        # Training of a long decoder over padded encoders: the largest call.
        _cross('cross_train', 'bf16', 4, 16, 4, 2048, 4500, 128, True, True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A layer width: mostly multiples of 64, some of 8, a few odd ones."""
    w = _log_int(rng, low, high)
    kind = rng.random()
    if kind < 0.6:
        return max(64, (w + 32) // 64 * 64)
    if kind < 0.85:
        return max(8, (w + 4) // 8 * 8)
    return w


def draw(rng):
    op = rng.choice(['dropout', 'norm', 'norm', 'axes', 'cross', 'cross',
                     'cross'])
    dtype = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
    train = rng.random() < 0.6
    if op in ('dropout', 'norm'):
        while True:
            batch, tokens = _log_int(rng, 1, 1024), _log_int(rng, 1, 8192)
            if rng.random() < 0.2:
                tokens = 1
            width = _width(rng, 32, 8192)
            if batch * tokens * width <= _MOST_ELEMENTS[op] / (
                    2 if dtype == 'f32' else 1):
                break
        p = rng.choice([0.05, 0.1, 0.2, 0.5])
        case = {'op': op, 'dtype': dtype, 'batch': batch, 'tokens': tokens,
                'width': width, 'p': p, 'train': train}
        if op == 'norm':
            case.update(kind=rng.choice(['rms', 'layer']),
                        bias=rng.random() < 0.5,
                        branch_norm=rng.random() < 0.5,
                        gate=rng.choice(['none', 'channel', 'sequence',
                                         'token']),
                        scale=rng.choice([1.0, 1.0, 0.5, 1.7]),
                        p=rng.choice([0.0, p]) if train else 0.0)
        return case
    if op == 'axes':
        while True:
            batch, tokens = _log_int(rng, 1, 1024), _log_int(rng, 1, 8192)
            kv_heads = rng.choice([1, 2, 4, 8, 16])
            heads = kv_heads * rng.choice([1, 1, 2, 4])
            dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
            if batch * tokens * (heads + kv_heads) * dim <= _MOST_ROTATED / (
                    2 if dtype == 'f32' else 1):
                break
        pairs = rng.choice([dim, dim, dim // 2]) // 2
        axes = rng.choice([2, 3, 3, 4])
        # Section edges at multiples of 4 mostly, anywhere else.
        unit = 4 if rng.random() < 0.7 and pairs // 4 >= axes else 1
        cuts = sorted(unit * c for c in rng.sample(
            range(1, (pairs + unit - 1) // unit), axes - 1))
        edges = [0] + cuts + [pairs]
        return {'op': op, 'dtype': dtype, 'batch': batch, 'tokens': tokens,
                'heads': heads, 'kv_heads': kv_heads, 'dim': dim,
                'sections': ','.join(str(b - a)
                                     for a, b in zip(edges, edges[1:])),
                'table': rng.choice([4096, 8192, 32768]),
                'interleaved': rng.random() < 0.4, 'train': train}
    while True:
        batch = _log_int(rng, 1, 1024)
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
        # Over a single state all gradients but that of v are zero.
        queries = _log_int(rng, 1, 4096)
        keys = _log_int(rng, 4 if train else 1, 8192)
        if rng.random() < 0.25:
            queries = 1
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        logits = float(batch * heads * queries * keys)
        flops = 4.0 * logits * dim * (3.5 if train else 1)
        if flops <= (_MOST_FLOPS_F32 if dtype == 'f32' else _MOST_FLOPS) \
                and logits <= _MOST_LOGITS \
                and batch * kv_heads * keys * dim <= 1.4e8 \
                and batch * heads * queries * dim <= 1.4e8:
            break
    return {'op': op, 'dtype': dtype, 'batch': batch, 'heads': heads,
            'kv_heads': kv_heads, 'queries': queries, 'keys': keys,
            'dim': dim, 'ragged': rng.random() < 0.6, 'train': train}


def _sections(case):
    return [int(n) for n in case['sections'].split(',')]


def _lengths(case):
    """Key lengths of a batch, before their order is drawn: from all keys
    down to a quarter of them, and one empty sequence among four or more."""
    batch, keys = case['batch'], case['keys']
    if not case['ragged']:
        return [keys] * batch
    lengths = [keys - (3 * keys * b) // (4 * max(batch - 1, 1))
               for b in range(batch)]
    if batch >= 4:
        lengths[-1] = 0
    return lengths


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case['dtype']]
    train = case['train']

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) *
                scale).to(dtype)

    def leaf(t):
        return t.requires_grad_() if train else t

    state = {'case': dict(case)}
    b = case['batch']
    if case['op'] in ('dropout', 'norm'):
        t, c = case['tokens'], case['width']
        state['rng'] = torch.randint(0, 1 << 30, (2,), generator=gen,
                                     device=dev)
        state['stream'] = 5
        state['x'] = leaf(randn(b, t, c))
        if case['op'] == 'dropout':
            if train:
                state['dy'] = randn(b, t, c, scale=0.1)
            return state
        state['branch'] = leaf(randn(b, t, c, scale=1.5))
        state['weight'] = leaf(1 + randn(c, scale=0.1))
        state['bias'] = leaf(randn(c, scale=0.1)) if case['bias'] else None
        state['branch_weight'] = leaf(1 + randn(c, scale=0.1)) \
            if case['branch_norm'] else None
        shape = {'none': None, 'channel': (c,), 'sequence': (b, 1, c),
                 'token': (b, t, c)}[case['gate']]
        state['gate'] = None if shape is None else leaf(
            randn(*shape, scale=0.5))
        if train:
            state['dx_out'] = randn(b, t, c, scale=0.1)
            state['dy'] = randn(b, t, c, scale=0.1)
        return state
    if case['op'] == 'axes':
        t, h, hk, d = (case['tokens'], case['heads'], case['kv_heads'],
                       case['dim'])
        # Views of one projection of queries, keys and values.
        qkv = randn(b, t, (h + 2 * hk) * d, scale=1.5)
        q = qkv[..., :h * d].view(b, t, h, d).transpose(1, 2)
        k = qkv[..., h * d:(h + hk) * d].view(b, t, hk, d).transpose(1, 2)
        state['q'], state['k'] = leaf(q.detach()), leaf(k.detach())
        for name in ('q_weight', 'k_weight'):
            state[name] = leaf(1 + randn(d, scale=0.1))
        pairs = sum(_sections(case))
        inv = 10000.0 ** (-torch.arange(pairs, device=dev).double() / pairs)
        angle = torch.arange(case['table'], device=dev).double()[:, None] * inv
        state['cos'], state['sin'] = angle.cos().float(), angle.sin().float()
        state['positions'] = torch.randint(
            0, case['table'], (len(_sections(case)), b, t), generator=gen,
            device=dev)
        if train:
            state['dq'] = randn(b, h, t, d, scale=0.1)
            state['dk'] = randn(b, hk, t, d, scale=0.1)
        return state

    h, hk, d = case['heads'], case['kv_heads'], case['dim']
    nq, nk = case['queries'], case['keys']
    # Queries are a view of their projection, keys and values of theirs.
    q = randn(b, nq, h, d).transpose(1, 2)
    kv = randn(b, nk, 2, hk, d).permute(2, 0, 3, 1, 4)
    state['q'] = leaf(q.detach())
    state['k'], state['v'] = leaf(kv[0].detach()), leaf(kv[1].detach())
    # |q - k|^2 varies by sqrt(8 d): weights neither flat nor on one key.
    scale = (0.5 + torch.rand(1, h, 1, 1, generator=gen, device=dev)) * (
        2.0 / math.sqrt(8 * d))
    state['scale'] = leaf(scale.to(dtype))
    order = torch.randperm(b, generator=gen, device=dev)
    state['key_lengths'] = torch.tensor(_lengths(case), device=dev)[order] \
        if case['ragged'] else None
    if train:
        state['dout'] = randn(b, nq, h, d, scale=0.1 if case['dtype'] != 'f16'
                              else 1.0).transpose(1, 2)
    return state


# ---------------------------------------------------------------------------
# Plain forms: elementary operations in 32 bits, rounded once at the end.
# ---------------------------------------------------------------------------
def _f32(t):
    return None if t is None else t.detach().float()


def _bits(rng, stream, count):
    """`count` 16-bit random numbers: Philox4x32-10 (Salmon et al., "Parallel
    random numbers: as easy as 1, 2, 3", 2011) with key = seed and counter =
    (group, step, stream), eight numbers to a group of consecutive
    elements."""
    low = 0xffffffff
    group = torch.arange((count + 7) // 8, device=rng.device)
    key = [rng[0] & low, (rng[0] >> 32) & low]
    c = [group & low, group >> 32, (rng[1] & low).expand_as(group),
         torch.full_like(group, stream & low)]
    for _ in range(10):
        # int64 products wrap; their bits are those of the unsigned product.
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & low) ^ c[1] ^ key[0], p1 & low,
             ((p0 >> 32) & low) ^ c[3] ^ key[1], p0 & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    halves = [w for x in c for w in (x & 0xffff, x >> 16)]
    return torch.stack(halves, 1).reshape(-1)[:count]


def _mask(s, shape, p):
    """What dropout multiplies by: 0 or the inverse of the share kept."""
    cut = int(math.floor(p * 65536 + 0.5))
    keep = _bits(s['rng'], s['stream'], math.prod(shape)) >= cut
    return keep.view(shape).float() * (65536.0 / (65536 - cut))


def _plain_dropout(s, c, dtype):
    m = _mask(s, s['x'].shape, c['p'])
    out = {'y': (_f32(s['x']) * m).to(dtype)}
    if c['train']:
        out['dx'] = (_f32(s['dy']) * m).to(dtype)
    return out


def _normed(x, kind):
    """(the normalised rows, the factor that normalised them)."""
    if kind == 'layer':
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    return x * r, r


def _norm_back(g, n, r, kind):
    """The gradient of the rows from that of the normalised ones."""
    d = g - n * (g * n).mean(-1, keepdim=True)
    if kind == 'layer':
        d = d - g.mean(-1, keepdim=True)
    return d * r


def _plain_norm(s, c, dtype):
    x, branch, w = _f32(s['x']), _f32(s['branch']), _f32(s['weight'])
    bias, bw, gate = _f32(s['bias']), _f32(s['branch_weight']), _f32(s['gate'])
    u = branch
    if bw is not None:
        n0, r0 = _normed(branch, c['kind'])
        u = n0 * bw
    m = _mask(s, u.shape, c['p']) if c['p'] else None
    d = u if m is None else u * m
    x_out = c['scale'] * x + (d if gate is None else gate * d)
    n1, r1 = _normed(x_out, c['kind'])
    y = n1 * w
    if bias is not None:
        y = y + bias
    out = {'x_out': x_out.to(dtype), 'y': y.to(dtype)}
    if not c['train']:
        return out
    dy = _f32(s['dy'])
    rows = (0, 1)
    out['dweight'] = (dy * n1).sum(rows).to(dtype)
    if bias is not None:
        out['dbias'] = dy.sum(rows).to(dtype)
    g = _f32(s['dx_out']) + _norm_back(dy * w, n1, r1, c['kind'])
    out['dx'] = (c['scale'] * g).to(dtype)
    if gate is not None:
        dgate = g * d
        if c['gate'] == 'channel':
            dgate = dgate.sum(rows)
        elif c['gate'] == 'sequence':
            dgate = dgate.sum(1, keepdim=True)
        out['dgate'] = dgate.to(dtype)
        g = g * gate
    if m is not None:
        g = g * m
    if bw is not None:
        out['dbranch_weight'] = (g * n0).sum(rows).to(dtype)
        g = _norm_back(g * bw, n0, r0, c['kind'])
    out['dbranch'] = g.to(dtype)
    return out


def _pairs(x, interleaved):
    """The two members of each rotated pair of the last dimension."""
    if interleaved:
        return x[..., 0::2], x[..., 1::2]
    half = x.shape[-1] // 2
    return x[..., :half], x[..., half:]


def _join(a, b, interleaved):
    if interleaved:
        return torch.stack([a, b], dim=-1).flatten(-2)
    return torch.cat([a, b], dim=-1)


def _rotate(x, cos, sin, interleaved):
    rotary = 2 * cos.shape[-1]
    a, b = _pairs(x[..., :rotary], interleaved)
    turned = _join(a * cos - b * sin, b * cos + a * sin, interleaved)
    return torch.cat([turned, x[..., rotary:]], dim=-1)


def _axis_rows(table, positions, sections):
    """[B, 1, N, pairs]: every pair's entry at its axis' position."""
    parts, start = [], 0
    for axis, n in enumerate(sections):
        parts.append(table[:, start:start + n][positions[axis]])
        start += n
    return torch.cat(parts, -1)[:, None]


def _plain_axes(s, c, dtype):
    cos = _axis_rows(s['cos'], s['positions'], _sections(c))
    sin = _axis_rows(s['sin'], s['positions'], _sections(c))
    out = {}
    for name in ('q', 'k'):
        x, w = _f32(s[name]), _f32(s[name + '_weight'])
        n, r = _normed(x, 'rms')
        out[name] = _rotate(n * w, cos, sin, c['interleaved']).to(dtype)
        if c['train']:
            dy = _rotate(_f32(s['d' + name]), cos, -sin, c['interleaved'])
            out['d%s_weight' % name] = (dy * n).sum((0, 1, 2)).to(dtype)
            out['d' + name] = _norm_back(dy * w, n, r, 'rms').to(dtype)
    return out


def _plain_cross(s, c, dtype):
    b, h, hk = c['batch'], c['heads'], c['kv_heads']
    nq, nk, d = c['queries'], c['keys'], c['dim']
    group = h // hk
    # Heads that share their keys stand together.
    q = _f32(s['q']).reshape(b, hk, group, nq, d)
    k = _f32(s['k']).reshape(b, hk, 1, nk, d)
    v = _f32(s['v']).reshape(b, hk, 1, nk, d)
    scale = _f32(s['scale']).reshape(1, hk, group, 1, 1)
    dist = q @ k.transpose(-1, -2)
    dist = (q.square().sum(-1, keepdim=True) +
            k.square().sum(-1).unsqueeze(-2) - 2 * dist).clamp(min=0)
    w = -scale * dist
    if s['key_lengths'] is not None:
        seen = torch.arange(nk, device=q.device) < s['key_lengths'][:, None]
        w = w.masked_fill(~seen[:, None, None, None], -math.inf)
    top = w.amax(-1, keepdim=True).clamp(min=torch.finfo(w.dtype).min)
    w = torch.exp(w - top)
    w = w / w.sum(-1, keepdim=True).clamp(min=torch.finfo(w.dtype).tiny)
    o = w @ v
    out = {'out': o.reshape(b, h, nq, d).to(dtype)}
    if c['train']:
        do = _f32(s['dout']).reshape(b, hk, group, nq, d)
        out['dv'] = (w.transpose(-1, -2) @ do).sum(2).to(dtype)
        ds = w * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
        # A row of ds sums to zero, so a row of distances may be centred: its
        # mean would bring the rounding of ds into the sum.
        near = dist - (w * dist).sum(-1, keepdim=True)
        out['dscale'] = -(ds * near).sum((0, 3, 4)).reshape(1, h, 1, 1).to(
            dtype)
        ds = 2 * scale * ds
        out['dq'] = (ds @ k - q * ds.sum(-1, keepdim=True)).reshape(
            b, h, nq, d).to(dtype)
        dk = ds.transpose(-1, -2) @ q - k * ds.sum(-2).unsqueeze(-1)
        out['dk'] = dk.sum(2).to(dtype)
    return out


# ---------------------------------------------------------------------------
# The framework's operators.
# ---------------------------------------------------------------------------
def _own(s, c):
    from vectra_b200 import block
    if c['op'] == 'dropout':
        out = {'y': block.dropout(s['x'], c['p'], s['rng'], s['stream'])}
        names, seeds = ('x',), ('dy',)
    elif c['op'] == 'norm':
        x_out, y = block.residual_norm(
            s['x'], s['branch'], s['weight'], s['bias'], gate=s['gate'],
            branch_weight=s['branch_weight'], residual_scale=c['scale'],
            p=c['p'], rng=s['rng'] if c['p'] else None, stream=s['stream'],
            eps=_EPS, kind=c['kind'])
        out = {'x_out': x_out, 'y': y}
        names = ('x', 'branch', 'weight', 'bias', 'branch_weight', 'gate')
        seeds = ('dx_out', 'dy')
    elif c['op'] == 'axes':
        q, k = block.qk_norm_rope_axes(
            s['q'], s['k'], s['cos'], s['sin'], s['positions'], _sections(c),
            s['q_weight'], s['k_weight'], _EPS, c['interleaved'])
        out = {'q': q, 'k': k}
        names, seeds = ('q', 'k', 'q_weight', 'k_weight'), ('dq', 'dk')
    else:
        out = {'out': block.cross_attention(s['q'], s['k'], s['v'],
                                            s['scale'], s['key_lengths'])}
        names, seeds = ('q', 'k', 'v', 'scale'), ('dout',)
    if c['train']:
        names = [n for n in names if s[n] is not None]
        grads = torch.autograd.grad(list(out.values()), [s[n] for n in names],
                                    [s[n] for n in seeds])
        out.update(('d' + n, g) for n, g in zip(names, grads))
    return out


def run(state):
    c = state['case']
    if own:
        return _own(state, c)
    plain = {'dropout': _plain_dropout, 'norm': _plain_norm,
             'axes': _plain_axes, 'cross': _plain_cross}[c['op']]
    with torch.no_grad():
        return plain(state, c, _DTYPES[c['dtype']])


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(case):
    es = _BYTES[case['dtype']]
    train = case['train']
    if case['op'] == 'dropout':
        n = case['batch'] * case['tokens'] * case['width']
        passes = 2 if train else 1
        return {'bytes': 2 * passes * n * es, 'flops': passes * n}
    if case['op'] == 'norm':
        c = case['width']
        n = case['batch'] * case['tokens'] * c
        gate = {'none': 0, 'channel': c, 'sequence': case['batch'] * c,
                'token': n}[case['gate']]
        params = gate + c * (1 + case['bias'] + case['branch_norm'])
        n_bytes = (4 * n + params) * es
        flops = 12 * n
        if train:
            # dx_out and dy are read, dx, dbranch and the parameters'
            # gradients written.
            n_bytes += (4 * n + params) * es
            flops += 24 * n
        return {'bytes': n_bytes, 'flops': flops}
    if case['op'] == 'axes':
        rows = case['batch'] * case['tokens']
        n = rows * (case['heads'] + case['kv_heads']) * case['dim']
        # A token's positions and its entries of both tables.
        side = rows * (8 * len(_sections(case)) + 8 * sum(_sections(case)))
        weights = 2 * case['dim'] * es
        n_bytes, flops = 2 * n * es + side + weights, 8 * n
        if train:
            n_bytes += 2 * n * es + weights
            flops += 16 * n
        return {'bytes': n_bytes, 'flops': flops}
    b, h, hk = case['batch'], case['heads'], case['kv_heads']
    nq, d = case['queries'], case['dim']
    seen = sum(_lengths(case))
    n_bytes = (2 * b * h * nq * d + 2 * hk * seen * d + h) * es
    flops = 4.0 * h * nq * seen * d
    if train:
        # The result's gradient is read; dq, dk and dv are written.
        n_bytes += (2 * b * h * nq * d + 2 * b * hk * case['keys'] * d +
                    h) * es
        flops *= 3.5
    return {'bytes': n_bytes, 'flops': flops}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, gradients by differentiation.
# ---------------------------------------------------------------------------
def _exact_keep(rng, stream, count):
    """The numbers of `_bits`, in NumPy's unsigned integers."""
    seed, step = (int(v) for v in rng.cpu())
    u32 = np.uint64(0xffffffff)
    n = (count + 7) // 8
    ctr = np.zeros((n, 4), dtype=np.uint64)
    index = np.arange(n, dtype=np.uint64)
    ctr[:, 0], ctr[:, 1] = index & u32, index >> np.uint64(32)
    ctr[:, 2], ctr[:, 3] = step & 0xffffffff, stream & 0xffffffff
    k0, k1 = seed & 0xffffffff, (seed >> 32) & 0xffffffff
    for _ in range(10):
        a = ctr[:, 0] * np.uint64(0xD2511F53)
        b = ctr[:, 2] * np.uint64(0xCD9E8D57)
        ctr = np.stack([(b >> np.uint64(32)) ^ ctr[:, 1] ^ np.uint64(k0),
                        b & u32,
                        (a >> np.uint64(32)) ^ ctr[:, 3] ^ np.uint64(k1),
                        a & u32], axis=1)
        k0, k1 = (k0 + 0x9E3779B9) % 2**32, (k1 + 0xBB67AE85) % 2**32
    return ctr.astype('<u4').view('<u2').reshape(-1)[:count]


def _exact_drop(t, s, p):
    if not p:
        return t
    cut = int(math.floor(p * 65536 + 0.5))
    bits = _exact_keep(s['rng'], s['stream'], t.numel())
    keep = torch.from_numpy(bits >= cut).to(t.device).view(t.shape)
    return torch.where(keep, t / (1 - cut / 65536),
                       torch.zeros((), dtype=t.dtype, device=t.device))


def _exact_row_norm(t, w, bias, kind):
    f = torch.nn.functional
    if kind == 'layer':
        return f.layer_norm(t, t.shape[-1:], w, bias, _EPS)
    y = f.rms_norm(t, t.shape[-1:], w, _EPS)
    return y if bias is None else y + bias


def _exact_turn(x, cos, sin, interleaved):
    """The rotation as a product of complex numbers."""
    rotary = 2 * cos.shape[-1]
    head, tail = x[..., :rotary], x[..., rotary:]
    if interleaved:
        z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous())
    else:
        z = torch.complex(*head.unflatten(-1, (2, -1)).unbind(-2))
    z = z * torch.complex(cos, sin)
    if interleaved:
        head = torch.view_as_real(z).flatten(-2)
    else:
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, tail], -1)


def _exact_cross(case, s):
    """One sequence and key head at a time, over the keys it sees."""
    b, h, hk = case['batch'], case['heads'], case['kv_heads']
    group = h // hk
    train = case['train']
    t = {n: s[n].detach().double() for n in ('q', 'k', 'v', 'scale')}
    lengths = [case['keys']] * b if s['key_lengths'] is None else \
        s['key_lengths'].tolist()
    out = {'out': torch.zeros_like(t['q'])}
    if train:
        out.update(('d' + n, torch.zeros_like(t[n])) for n in t)
        do = s['dout'].double()
    # Sequences of one length go through together, at most 2^27 weights at
    # a time.
    by_length = {}
    for i, n in enumerate(lengths):
        by_length.setdefault(n, []).append(i)
    for n, rows in by_length.items():
        if n == 0:
            continue
        weights = hk * group * case['queries'] * n
        step = max(1, (1 << 27) // weights)
        for at in range(0, len(rows), step):
            i = torch.tensor(rows[at:at + step], device=t['q'].device)
            heads = [(j, j + 1) for j in range(hk)] if weights > 1 << 27 \
                else [(0, hk)]
            for lo, hi in heads:
                own_q = slice(lo * group, hi * group)
                q = t['q'][i, own_q].requires_grad_(train)
                k = t['k'][i, lo:hi, :n].requires_grad_(train)
                v = t['v'][i, lo:hi, :n].requires_grad_(train)
                sc = t['scale'][:, own_q].clone().requires_grad_(train)
                kk = k.repeat_interleave(group, 1)
                vv = v.repeat_interleave(group, 1)
                sq = (q * q).sum(-1)[..., None] - 2 * q @ kk.mT + \
                    (kk * kk).sum(-1)[..., None, :]
                o = torch.softmax(-sc * sq, -1) @ vv
                out['out'][i, own_q] = o.detach()
                if train:
                    g = torch.autograd.grad(o, (q, k, v, sc), do[i, own_q])
                    out['dq'][i, own_q] = g[0]
                    out['dk'][i, lo:hi, :n] = g[1]
                    out['dv'][i, lo:hi, :n] = g[2]
                    out['dscale'][:, own_q] += g[3]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'cross':
        # A thousand sequences of different lengths take too long one by one.
        if case['ragged'] and case['batch'] > 64:
            return _exact_cross_padded(case, s)
        return _exact_cross(case, s)
    train = case['train']
    names = {'dropout': ('x',),
             'norm': ('x', 'branch', 'weight', 'bias', 'branch_weight',
                      'gate'),
             'axes': ('q', 'k', 'q_weight', 'k_weight')}[case['op']]
    seeds = {'dropout': ('dy',), 'norm': ('dx_out', 'dy'),
             'axes': ('dq', 'dk')}[case['op']]
    v = {n: None if s[n] is None else s[n].detach().double().requires_grad_(
        train) for n in names}
    if case['op'] == 'dropout':
        out = {'y': _exact_drop(v['x'], s, case['p'])}
    elif case['op'] == 'norm':
        u = v['branch']
        if v['branch_weight'] is not None:
            u = _exact_row_norm(u, v['branch_weight'], None, case['kind'])
        u = _exact_drop(u, s, case['p'])
        if v['gate'] is not None:
            u = u * v['gate']
        x_out = torch.add(u, v['x'], alpha=case['scale'])
        out = {'x_out': x_out, 'y': _exact_row_norm(
            x_out, v['weight'], v['bias'], case['kind'])}
    else:
        # Axis of each pair, then its table entry by that axis' position.
        axis = torch.repeat_interleave(
            torch.arange(len(_sections(case))),
            torch.tensor(_sections(case))).to(s['cos'].device)
        at = s['positions'].permute(1, 2, 0)[..., axis]
        pair = torch.arange(axis.numel(), device=axis.device)
        cos = s['cos'].double()[at, pair].unsqueeze(1)
        sin = s['sin'].double()[at, pair].unsqueeze(1)
        f = torch.nn.functional
        out = {n: _exact_turn(
            f.rms_norm(v[n], (case['dim'],), v[n + '_weight'], _EPS), cos,
            sin, case['interleaved']) for n in ('q', 'k')}
    if train:
        have = [n for n in names if v[n] is not None]
        grads = torch.autograd.grad(list(out.values()), [v[n] for n in have],
                                    [s[n].double() for n in seeds])
        out.update(('d' + n, g) for n, g in zip(have, grads))
    return {n: t.detach() for n, t in out.items()}


def _exact_cross_padded(case, s):
    """All sequences of a large batch at once, unseen keys' weights zero."""
    train = case['train']
    if case['batch'] * case['heads'] * case['queries'] * case['keys'] > 1 << 29:
        return None
    group = case['heads'] // case['kv_heads']
    t = {n: s[n].detach().double().requires_grad_(train)
         for n in ('q', 'k', 'v', 'scale')}
    kk = t['k'].repeat_interleave(group, 1)
    vv = t['v'].repeat_interleave(group, 1)
    sq = (t['q'] ** 2).sum(-1)[..., None] - 2 * t['q'] @ kk.mT + \
        (kk ** 2).sum(-1)[..., None, :]
    at = torch.arange(case['keys'], device=sq.device)
    hidden = at >= s['key_lengths'][:, None, None, None]
    logits = (-t['scale'] * sq).masked_fill(hidden, -1e300)
    w = torch.softmax(logits, -1).masked_fill(hidden, 0.0)
    out = {'out': w @ vv}
    if train:
        g = torch.autograd.grad(out['out'], tuple(t.values()),
                                s['dout'].double())
        out.update(('d' + n, x) for n, x in zip(t, g))
    return {n: x.detach() for n, x in out.items()}
