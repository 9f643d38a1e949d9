"""Cases, plain forms and float64 values of the transformer-block operators.

The operators stand around torch.ops.vectra.rbf_attention in a transformer
block and are reached through vectra_b200.block:

* linear(x, weight, bias, residual, activation):
    y = act(x W^T + b) + r
* gated_linear(x, w_gate, w_up, b_gate, b_up, activation):
    h = act(x Wg^T + bg) * (x Wu^T + bu)
* qk_norm_rope(q, k, cos, sin, q_weight, k_weight, positions, eps,
  interleaved): the RMS norm of every query and key head vector and the
  rotation of its position, in one pass.

A "train" case is the forward pass and the backward pass through autograd;
its outputs are the results and every gradient.
"""

import math

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16,
           'f32': torch.float32}
_BYTES = {'bf16': 2, 'f16': 2, 'f32': 4}
_EPS = 1e-6
# No drawn case needs more operations than the largest listed one.
_MOST_FLOPS = 4.1e12
_MOST_FLOPS_F32 = 1.2e11


# ---------------------------------------------------------------------------
# Cases.
# ---------------------------------------------------------------------------
def _linear(name, dtype, batch, tokens, k, n, activation, bias, residual,
            train):
    return {'name': name, 'op': 'linear', 'dtype': dtype, 'batch': batch,
            'tokens': tokens, 'k': k, 'n': n, 'activation': activation,
            'bias': bias, 'residual': residual, 'train': train}


def _gated(name, dtype, batch, tokens, k, f, activation, bias, train):
    return {'name': name, 'op': 'gated', 'dtype': dtype, 'batch': batch,
            'tokens': tokens, 'k': k, 'f': f, 'activation': activation,
            'bias': bias, 'train': train}


def _qk(name, dtype, batch, tokens, heads, kv_heads, dim, rotary, table,
        interleaved, weights, fused, train):
    return {'name': name, 'op': 'qk', 'dtype': dtype, 'batch': batch,
            'tokens': tokens, 'heads': heads, 'kv_heads': kv_heads,
            'dim': dim, 'rotary': rotary, 'table': table,
            'interleaved': interleaved, 'weights': weights, 'fused': fused,
            'train': train}


def listed():
    return [
        # Output projection of one serving step of 8 sequences: the weights
        # are read for a handful of rows.
        _linear('linear_step_8', 'bf16', 8, 1, 4096, 4096, 'none', False,
                True, False),
        # The price model's first feed-forward layer over a served batch:
        # 1,024 targets with 64 comparables each.
        _linear('linear_price_ffn_up', 'bf16', 1024, 65, 256, 1024, 'gelu',
                True, False, False),
        # Its second feed-forward layer in training, with the residual.
        _linear('linear_price_ffn_down_train', 'bf16', 1024, 65, 1024, 256,
                'none', True, True, True),
        # A long ragged prompt through a wide layer.
        _linear('linear_prompt', 'f16', 1, 8191, 4096, 4096, 'gelu_tanh',
                True, True, False),
        # The price model's encoders stay in float32: comparables'
        # embeddings of 128 to the model width.
        _linear('linear_encoder_f32', 'f32', 1024, 64, 128, 256, 'gelu',
                True, False, False),
        # The gated layer of one sequence's next token.
        _gated('gated_step_1', 'bf16', 1, 1, 4096, 10240, 'silu', False,
               False),
        # A short ragged prompt.
        _gated('gated_prompt', 'f16', 1, 1237, 2048, 5632, 'gelu_tanh', True,
               False),
        # Training of the price model's width with a gated layer.
        _gated('gated_price_train', 'bf16', 1024, 65, 256, 704, 'silu', True,
               True),
        # Training of a wide layer: the largest call.
        _gated('gated_train', 'bf16', 4, 2048, 4096, 10240, 'silu', False,
               True),
        # Queries and keys of one serving step, views of the projection.
        _qk('qk_step', 'bf16', 64, 1, 32, 8, 128, 128, 32768, False, True,
            True, False),
        # Queries and keys of long prompts.
        _qk('qk_prompt', 'bf16', 4, 4096, 32, 8, 128, 128, 32768, False,
            True, True, False),
        # Training, half of the head width rotated in neighbouring pairs.
        _qk('qk_train', 'f16', 3, 2049, 16, 16, 64, 32, 4096, True, True,
            True, True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A layer width: mostly multiples of 64, some of 8, a few odd ones."""
    while True:
        w = _log_int(rng, low, high)
        kind = rng.random()
        if kind < 0.65:
            w = max(64, (w + 32) // 64 * 64)
        elif kind < 0.88:
            w = max(8, (w + 4) // 8 * 8)
        if w != 3072 and low <= w <= high:
            return w


def _tokens(rng, low, high):
    while True:
        t = _log_int(rng, low, high)
        if t != 3072:
            return t


def draw(rng):
    op = rng.choice(['linear', 'gated', 'qk'])
    train = rng.random() < 0.4
    if op == 'qk':
        while True:
            batch = _log_int(rng, 1, 128)
            tokens = _tokens(rng, 1, 4096)
            if rng.random() < 0.3:
                tokens = 1
            kv_heads = rng.choice([1, 2, 4, 8, 16])
            heads = kv_heads * rng.choice([1, 1, 2, 4])
            dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
            rotary = rng.choice([dim, dim, dim // 2])
            width = (heads + 2 * kv_heads) * dim
            sizes = (width, heads * dim, kv_heads * dim, batch * tokens)
            if batch * tokens * width > 2.0e8 or 3072 in sizes:
                continue
            break
        return {'op': 'qk', 'dtype': rng.choice(['bf16', 'bf16', 'f16',
                                                 'f32']),
                'batch': batch, 'tokens': tokens, 'heads': heads,
                'kv_heads': kv_heads, 'dim': dim, 'rotary': rotary,
                'table': rng.choice([4096, 8192, 32768]),
                'interleaved': rng.random() < 0.4,
                'weights': rng.random() < 0.8, 'fused': rng.random() < 0.7,
                'train': train}
    while True:
        dtype = rng.choice(['bf16', 'bf16', 'f16', 'f16', 'f32'])
        batch = _log_int(rng, 1, 64)
        tokens = _tokens(rng, 1, 4096) if train or rng.random() < 0.6 else 1
        if train and batch * tokens < 32:
            continue
        k = _width(rng, 48, 4096)
        out = _width(rng, 48, 10240 if op == 'gated' else 8192)
        rows = batch * tokens
        flops = 2.0 * rows * k * out * (3 if train else 1) * (
            2 if op == 'gated' else 1)
        most = _MOST_FLOPS_F32 if dtype == 'f32' else _MOST_FLOPS
        if flops > most or rows > 70000 or rows == 3072 or rows * out > 6e8:
            continue
        break
    case = {'op': op, 'dtype': dtype, 'batch': batch, 'tokens': tokens,
            'k': k, 'train': train, 'bias': rng.random() < 0.5}
    if op == 'linear':
        case.update(n=out, residual=rng.random() < 0.5,
                    activation=rng.choice(['none', 'none', 'relu', 'gelu',
                                           'gelu_tanh', 'silu']))
    else:
        case.update(f=out, activation=rng.choice(['silu', 'silu', 'gelu',
                                                  'gelu_tanh']))
    return case


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

    b, t = case['batch'], case['tokens']
    state = {'case': dict(case)}
    if case['op'] == 'qk':
        h, hk, d = case['heads'], case['kv_heads'], case['dim']
        half = case['rotary'] // 2
        if case['fused']:
            qkv = randn(b, t, (h + 2 * hk) * d, scale=1.5)
            q = qkv[..., :h * d].view(b, t, h, d).transpose(1, 2)
            k = qkv[..., h * d:(h + hk) * d].view(b, t, hk, d).transpose(1, 2)
            q, k = q.detach(), k.detach()
        else:
            q, k = randn(b, h, t, d, scale=1.5), randn(b, hk, t, d, scale=1.5)
        inv = 10000.0 ** (-torch.arange(half, device=dev).double() / half)
        angle = torch.arange(case['table'], device=dev).double()[:, None] * inv
        state['cos'], state['sin'] = angle.cos().float(), angle.sin().float()
        start = torch.randint(0, case['table'] - t + 1, (b, 1), generator=gen,
                              device=dev)
        state['positions'] = start + torch.arange(t, device=dev)
        state['q'], state['k'] = leaf(q), leaf(k)
        for name in ('q_weight', 'k_weight'):
            state[name] = leaf(1 + randn(d, scale=0.1)) if case['weights'] \
                else None
        if train:
            state['dq'] = randn(b, h, t, d, scale=0.1)
            state['dk'] = randn(b, hk, t, d, scale=0.1)
        return state

    k = case['k']
    state['x'] = leaf(randn(b, t, k))
    if case['op'] == 'linear':
        n = case['n']
        state['weight'] = leaf(randn(n, k, scale=k ** -0.5))
        state['bias'] = leaf(randn(n, scale=0.1)) if case['bias'] else None
        state['residual'] = leaf(randn(b, t, n)) if case['residual'] else None
    else:
        n = case['f']
        state['w_gate'] = leaf(randn(n, k, scale=k ** -0.5))
        state['w_up'] = leaf(randn(n, k, scale=k ** -0.5))
        for name in ('b_gate', 'b_up'):
            state[name] = leaf(randn(n, scale=0.1)) if case['bias'] else None
    if train:
        state['dy'] = randn(b, t, n, scale=0.1)
    return state


# ---------------------------------------------------------------------------
# Plain forms: elementary operations in 32 bits, rounded once at the end.
# ---------------------------------------------------------------------------
def _f32(t):
    return None if t is None else t.detach().float()


_TANH_C = math.sqrt(2.0 / math.pi)


def _act(z, kind):
    """act(z)."""
    if kind == 'none':
        return z
    if kind == 'relu':
        return torch.clamp(z, min=0)
    if kind == 'silu':
        return z / (1 + torch.exp(-z))
    if kind == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1 + torch.tanh(_TANH_C * (z + 0.044715 * z * z * z)))


def _act_grad(z, kind):
    """d act(z) / dz."""
    if kind == 'relu':
        return (z > 0).to(z.dtype)
    if kind == 'silu':
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if kind == 'gelu':
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(
            -0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    t = torch.tanh(_TANH_C * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _TANH_C * (
        1 + 3 * 0.044715 * z * z)


def _plain_linear(s, c, dtype):
    shape = s['x'].shape
    x, w = _f32(s['x']).reshape(-1, c['k']), _f32(s['weight'])
    z = x @ w.t()
    if c['bias']:
        z = z + _f32(s['bias'])
    y = _act(z, c['activation'])
    if c['residual']:
        y = y + _f32(s['residual']).reshape(-1, c['n'])
    out = {'y': y.to(dtype).reshape(*shape[:-1], c['n'])}
    if c['train']:
        dz = _f32(s['dy']).reshape(-1, c['n'])
        if c['activation'] != 'none':
            dz = dz * _act_grad(z, c['activation'])
        out['dx'] = (dz @ w).to(dtype).reshape(shape)
        out['dweight'] = (dz.t() @ x).to(dtype)
        if c['bias']:
            out['dbias'] = dz.sum(0).to(dtype)
        if c['residual']:
            out['dresidual'] = s['dy']
    return out


def _plain_gated(s, c, dtype):
    shape = s['x'].shape
    x = _f32(s['x']).reshape(-1, c['k'])
    wg, wu = _f32(s['w_gate']), _f32(s['w_up'])
    g, u = x @ wg.t(), x @ wu.t()
    if c['bias']:
        g, u = g + _f32(s['b_gate']), u + _f32(s['b_up'])
    a = _act(g, c['activation'])
    out = {'y': (a * u).to(dtype).reshape(*shape[:-1], c['f'])}
    if c['train']:
        dy = _f32(s['dy']).reshape(-1, c['f'])
        dg, du = dy * u * _act_grad(g, c['activation']), dy * a
        out['dx'] = (dg @ wg + du @ wu).to(dtype).reshape(shape)
        out['dw_gate'] = (dg.t() @ x).to(dtype)
        out['dw_up'] = (du.t() @ x).to(dtype)
        if c['bias']:
            out['db_gate'] = dg.sum(0).to(dtype)
            out['db_up'] = du.sum(0).to(dtype)
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


def _rotate(x, cos, sin, rotary, interleaved):
    a, b = _pairs(x[..., :rotary], interleaved)
    turned = _join(a * cos - b * sin, b * cos + a * sin, interleaved)
    return torch.cat([turned, x[..., rotary:]], dim=-1)


def _plain_qk(s, c, dtype):
    cos = s['cos'][s['positions']][:, None]
    sin = s['sin'][s['positions']][:, None]
    out = {}
    for name in ('q', 'k'):
        x, w = _f32(s[name]), _f32(s[name + '_weight'])
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        n = x * r
        y = n if w is None else n * w
        out[name] = _rotate(y, cos, sin, c['rotary'],
                            c['interleaved']).to(dtype)
        if c['train']:
            dy = _rotate(_f32(s['d' + name]), cos, -sin, c['rotary'],
                         c['interleaved'])
            if w is not None:
                out['d%s_weight' % name] = (dy * n).sum((0, 1, 2)).to(dtype)
                dy = dy * w
            dx = r * (dy - n * (dy * n).mean(-1, keepdim=True))
            out['d' + name] = dx.to(dtype)
    return out


# ---------------------------------------------------------------------------
# The framework's operators.
# ---------------------------------------------------------------------------
def _own(s, c):
    from vectra_b200 import block
    if c['op'] == 'linear':
        y = block.linear(s['x'], s['weight'], s['bias'], s['residual'],
                         c['activation'])
        names = ('x', 'weight', 'bias', 'residual')
    elif c['op'] == 'gated':
        y = block.gated_linear(s['x'], s['w_gate'], s['w_up'], s['b_gate'],
                               s['b_up'], c['activation'])
        names = ('x', 'w_gate', 'w_up', 'b_gate', 'b_up')
    else:
        q, k = block.qk_norm_rope(s['q'], s['k'], s['cos'], s['sin'],
                                  s['q_weight'], s['k_weight'],
                                  s['positions'], _EPS, c['interleaved'])
        names = ('q', 'k', 'q_weight', 'k_weight')
        out = {'q': q, 'k': k}
    if c['op'] != 'qk':
        out = {'y': y}
    if c['train']:
        names = [n for n in names if s[n] is not None]
        if c['op'] == 'qk':
            grads = torch.autograd.grad([q, k], [s[n] for n in names],
                                        [s['dq'], s['dk']])
        else:
            grads = torch.autograd.grad(y, [s[n] for n in names], s['dy'])
        out.update(('d' + n, g) for n, g in zip(names, grads))
    return out


def run(state):
    c = state['case']
    if own:
        return _own(state, c)
    plain = {'linear': _plain_linear, 'gated': _plain_gated,
             'qk': _plain_qk}[c['op']]
    with torch.no_grad():
        return plain(state, c, _DTYPES[c['dtype']])


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(case):
    es = _BYTES[case['dtype']]
    rows = case['batch'] * case['tokens']
    if case['op'] == 'qk':
        elements = rows * (case['heads'] + case['kv_heads']) * case['dim']
        # The rotation's rows of both tables once per token, and the token's
        # position.
        side = rows * (case['rotary'] * 4 + 8)
        weights = 2 * case['dim'] * es if case['weights'] else 0
        n_bytes = 2 * elements * es + side + weights
        flops = 8 * elements
        if case['train']:
            n_bytes += 2 * elements * es + weights
            flops += 16 * elements
        return {'bytes': n_bytes, 'flops': flops}
    k = case['k']
    if case['op'] == 'linear':
        out, products = case['n'], 1
        params = out * k + (out if case['bias'] else 0)
        n_bytes = (rows * k + params + rows * out *
                   (2 if case['residual'] else 1)) * es
    else:
        out, products = case['f'], 2
        params = 2 * (out * k + (out if case['bias'] else 0))
        n_bytes = (rows * k + params + rows * out) * es
    flops = 2 * products * rows * k * out
    if case['train']:
        # dy is read; the gradients of x and of the parameters are written.
        n_bytes += (rows * out + rows * k + params) * es
        flops *= 3
    return {'bytes': n_bytes, 'flops': flops}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, gradients by differentiation.
# ---------------------------------------------------------------------------
def _exact_act(z, kind):
    f = torch.nn.functional
    return {'none': lambda: z, 'relu': lambda: f.relu(z),
            'silu': lambda: f.silu(z), 'gelu': lambda: f.gelu(z),
            'gelu_tanh': lambda: f.gelu(z, approximate='tanh')}[kind]()


def _exact_turn(x, angle_cos, angle_sin, rotary, interleaved):
    """The rotation as a product of complex numbers."""
    head, tail = x[..., :rotary], x[..., rotary:]
    if interleaved:
        z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous())
    else:
        z = torch.complex(*head.unflatten(-1, (2, -1)).unbind(-2))
    z = z * torch.complex(angle_cos, angle_sin)
    if interleaved:
        head = torch.view_as_real(z).flatten(-2)
    else:
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, tail], -1)


def exact(case, seed):
    s = prepare(case, seed)
    train = case['train']
    names = {'linear': ('x', 'weight', 'bias', 'residual'),
             'gated': ('x', 'w_gate', 'w_up', 'b_gate', 'b_up'),
             'qk': ('q', 'k', 'q_weight', 'k_weight')}[case['op']]
    v = {n: None if s[n] is None else s[n].detach().double().requires_grad_(
        train) for n in names}
    f = torch.nn.functional
    if case['op'] == 'linear':
        y = _exact_act(f.linear(v['x'], v['weight'], v['bias']),
                       case['activation'])
        if v['residual'] is not None:
            y = y + v['residual']
        out = {'y': y}
    elif case['op'] == 'gated':
        out = {'y': _exact_act(f.linear(v['x'], v['w_gate'], v['b_gate']),
                               case['activation']) *
                    f.linear(v['x'], v['w_up'], v['b_up'])}
    else:
        at = s['positions'].unsqueeze(1)
        cos, sin = s['cos'].double()[at], s['sin'].double()[at]
        out = {n: _exact_turn(
            f.rms_norm(v[n], (case['dim'],), v[n + '_weight'], _EPS), cos,
            sin, case['rotary'], case['interleaved']) for n in ('q', 'k')}
    if train:
        heads = list(out)
        seeds = [s['d' + n].double() for n in heads]
        have = [n for n in names if v[n] is not None]
        grads = torch.autograd.grad([out[n] for n in heads],
                                    [v[n] for n in have], seeds)
        out.update(('d' + n, g) for n, g in zip(have, grads))
    return {n: t.detach() for n, t in out.items()}
