"""Measured cases of the transformer-block operators: query/key norm with rotation, differential attention, gated feed-forward.

Token counts and widths are those of the attention levels of the presets (32x32, 16x16 and 28x28 maps, heads of 32 to 256
channels, batches of 16 to 64), single tokens against a long cache, and generic block widths for training.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def listed():
    return [
        # one new token of each of four sequences, far into them: launch latency
        dict(name='qk_token', op='qk', dtype='bf16', B=4, T=1, Hq=12, Hk=12, D=64, R=64, start=131071, grid=0, interleaved=False,
             packed=False, train=False),
        # the 32x32 attention level of the 64x64 preset at batch 64, in its packed qkv rows
        dict(name='qk_grid', op='qk', dtype='bf16', B=64, T=1024, Hq=6, Hk=6, D=64, R=64, start=0, grid=32, interleaved=False,
             packed=True, train=False),
        # fp32, an odd number of tokens, pairs side by side, half the channels rotated; forward and backward
        dict(name='qk_odd_train_f32', op='qk', dtype='f32', B=5, T=785, Hq=4, Hk=2, D=96, R=48, start=3, grid=0, interleaved=True,
             packed=True, train=True),
        # a training step's norms over long rows with shared key heads
        dict(name='qk_train', op='qk', dtype='bf16', B=16, T=4096, Hq=12, Hk=4, D=128, R=128, start=0, grid=64, interleaved=False,
             packed=False, train=True),
        # one query against a ragged cache of 8192 keys, four query heads to a key head
        dict(name='diff_token', op='diff', dtype='bf16', B=16, Tq=1, Tk=8192, H=16, Hk=4, D=64, Dv=128, ragged=True, causal=False,
             packed=False, train=False),
        # the 32x32 level of the 64x64 preset: heads of 64 as two halves of 32
        dict(name='diff_grid', op='diff', dtype='bf16', B=64, Tq=1024, Tk=1024, H=6, Hk=6, D=32, Dv=64, ragged=False, causal=False,
             packed=True, train=False),
        # fp32 with odd, ragged lengths (one sequence empty), forward and backward
        dict(name='diff_odd_train_f32', op='diff', dtype='f32', B=3, Tq=785, Tk=785, H=4, Hk=2, D=48, Dv=96, ragged=True, causal=False,
             packed=True, train=True),
        # a training step over 2048 causal tokens
        dict(name='diff_train', op='diff', dtype='bf16', B=8, Tq=2048, Tk=2048, H=8, Hk=8, D=64, Dv=128, ragged=False, causal=True,
             packed=False, train=True),
        # one token through the block: the weights are what is read
        dict(name='ffn_token', op='ffn', dtype='bf16', B=1, T=1, C=1024, F=4096, act='silu', bias=False, residual=True, train=False),
        # the 32x32 level at batch 64
        dict(name='ffn_grid', op='ffn', dtype='bf16', B=64, T=1024, C=384, F=1024, act='gelu', bias=True, residual=True, train=False),
        # fp32 with odd rows and widths off the tiles
        dict(name='ffn_odd_train_f32', op='ffn', dtype='f32', B=3, T=785, C=264, F=680, act='gelu', bias=True, residual=True, train=True),
        # a training step of a wide block
        dict(name='ffn_train', op='ffn', dtype='bf16', B=16, T=1024, C=1024, F=4096, act='silu', bias=False, residual=True, train=True),
    ]


def _log(rng, lo, hi):
    """A whole number of lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(['qk', 'diff', 'ffn'])
    dtype = rng.choice(['bf16', 'bf16', 'f32'])
    train = rng.random() < 0.5
    if op == 'qk':
        B, Hk, D = _log(rng, 1, 64), rng.randint(1, 8), 2 * _log(rng, 8, 128)
        Hq = Hk * rng.randint(1, 4)
        T = _log(rng, 1, max(1, min(4096, (1 << 26) // (B * (Hq + Hk) * D))))
        return dict(op=op, dtype=dtype, B=B, T=T, Hq=Hq, Hk=Hk, D=D, R=rng.choice([D, D // 4 * 2]), start=_log(rng, 1, 200000), grid=0,
                    interleaved=rng.random() < 0.5, packed=rng.random() < 0.5, train=train)
    if op == 'diff':
        D, Hk = 8 * rng.randint(1, 16), rng.randint(1, 4)
        Dv, H, B = rng.choice([2 * D, D, 2 * D]), Hk * rng.randint(1, 4), _log(rng, 1, 16)
        if rng.random() < 0.3:
            Tq, Tk, train = rng.randint(1, 4), _log(rng, 16, 8192), False
        else:
            Tk = _log(rng, 1, 2048)
            Tq = Tk if rng.random() < 0.6 else _log(rng, 1, 2048)
        B = max(1, min(B, (1 << 32) // (H * Tq * Tk * D)))
        return dict(op=op, dtype=dtype, B=B, Tq=Tq, Tk=Tk, H=H, Hk=Hk, D=D, Dv=Dv, ragged=rng.random() < 0.4, causal=rng.random() < 0.4,
                    packed=Tq == Tk and rng.random() < 0.5, train=train)
    C, F = 8 * _log(rng, 8, 128), 8 * _log(rng, 8, 512)
    rows = _log(rng, 1, max(1, min(16384, (1 << 35) // (C * F) // (8 if dtype == 'f32' else 1))))
    B = rng.randint(1, min(4, rows))
    return dict(op=op, dtype=dtype, B=B, T=max(1, rows // B), C=C, F=F, act=rng.choice(['silu', 'gelu', 'gelu_tanh']),
                bias=rng.random() < 0.5, residual=rng.random() < 0.5, train=train)


_DTYPES = {'bf16': torch.bfloat16, 'f32': torch.float32}


def _lengths(c):
    """Keys of each sequence: from all of them down, the last sequence of three or more empty."""
    if not c['ragged']:
        return [c['Tk']] * c['B']
    return [0 if b and b == c['B'] - 1 and c['B'] >= 3 else max(1, c['Tk'] - b * c['Tk'] // (2 * c['B'])) for b in range(c['B'])]


def _pairs(c):
    """Unmasked (query, key) pairs of one head, over the batch."""
    if not c['causal']:
        return sum(c['Tq'] * n for n in _lengths(c))
    n = 0
    for k in _lengths(c):
        first = k - c['Tq'] + 1                       # keys that query 0 sees; one more for each next query
        lo = max(first, 0)
        n += (lo + k) * (k - lo + 1) // 2 if k else 0
    return n


def work(c):
    es = 2 if c['dtype'] == 'bf16' else 4
    if c['op'] == 'qk':
        x = c['B'] * c['T'] * (c['Hq'] + c['Hk']) * c['D']
        return {'bytes': x * es * (5 if c['train'] else 2) + 4 * c['T'] * c['R'] + 4 * c['D'] * es, 'flops': x * (25 if c['train'] else 8)}
    if c['op'] == 'diff':
        B, Tq, H, Hk, D, Dv = (c[k] for k in ('B', 'Tq', 'H', 'Hk', 'D', 'Dv'))
        rows, keys = B * Tq * H, sum(_lengths(c)) * Hk
        q, o, kv = rows * 2 * D, rows * Dv, keys * (2 * D + Dv)
        fwd = 4 * D + 2 * Dv
        if not c['train']:
            return {'bytes': es * (q + o + kv), 'flops': fwd * H * max(1, _pairs(c))}
        return {'bytes': es * (2 * (q + kv) + 2 * o + q + B * c['Tk'] * Hk * (2 * D + Dv)), 'flops': (fwd + 12 * D + 4 * Dv) * H * max(1, _pairs(c))}
    M, C, F = c['B'] * c['T'], c['C'], c['F']
    w, x = 3 * C * F, M * C
    if not c['train']:
        return {'bytes': es * (w + (3 if c['residual'] else 2) * x), 'flops': 6 * M * C * F}
    return {'bytes': es * (3 * w + 5 * x), 'flops': 18 * M * C * F}


# ------------------------------------------------------------------------------------------------------------ inputs
def _normal(c, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device='cuda') * scale + mean).to(_DTYPES[c['dtype']])
    return normal


def _tables(c):
    """cos and sin of every token's angles [T, R/2], from 64-bit angles: rows and columns of a map share the pairs, or one long axis."""
    pairs = c['R'] // 2
    t = torch.arange(c['T'], device='cuda')
    if c['grid']:
        half = pairs // 2
        f = 10000.0 ** (-torch.arange(half, device='cuda', dtype=torch.float64) / half)
        a = torch.cat([(t // c['grid']).double()[:, None] * f, (t % c['grid']).double()[:, None] * f], 1)
    else:
        f = 10000.0 ** (-torch.arange(pairs, device='cuda', dtype=torch.float64) / max(1, pairs))
        a = (t + c['start']).double()[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def prepare(case, seed):
    c, normal = case, _normal(case, seed)
    if c['op'] == 'qk':
        B, T, Hq, Hk, D = (c[k] for k in ('B', 'T', 'Hq', 'Hk', 'D'))
        if c['packed']:                               # q, k, v side by side in one row, as the qkv projection leaves them
            row = normal(B, T, (Hq + 2 * Hk) * D)
            q, k = row[..., :Hq * D].view(B, T, Hq, D), row[..., Hq * D:(Hq + Hk) * D].view(B, T, Hk, D)
        else:
            q, k = normal(B, T, Hq, D), normal(B, T, Hk, D)
        s = dict(q=q, k=k, qw=normal(D, scale=0.1, mean=1.0), kw=normal(D, scale=0.1, mean=1.0))
        names = ('q', 'k', 'qw', 'kw')
        douts = [(B, T, Hq, D), (B, T, Hk, D)]
        s['cos'], s['sin'] = _tables(c)
    elif c['op'] == 'diff':
        B, Tq, Tk, H, Hk, D, Dv = (c[k] for k in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D', 'Dv'))
        if c['packed']:
            row = normal(B, Tq, 2 * H * D + 2 * Hk * D + Hk * Dv)
            q, k, v = row.split([2 * H * D, 2 * Hk * D, Hk * Dv], -1)
            q, k, v = q.view(B, Tq, H, 2 * D), k.view(B, Tk, Hk, 2 * D), v.view(B, Tk, Hk, Dv)
        else:
            q, k, v = normal(B, Tq, H, 2 * D), normal(B, Tk, Hk, 2 * D), normal(B, Tk, Hk, Dv)
        s = dict(q=q, k=k, v=v, **{n: normal(D, scale=0.1) for n in ('lq1', 'lk1', 'lq2', 'lk2')})
        names = ('q', 'k', 'v', 'lq1', 'lk1', 'lq2', 'lk2')
        douts = [(B, Tq, H, Dv)]
        s['lengths'] = torch.tensor(_lengths(c), dtype=torch.int32, device='cuda') if c['ragged'] else None
    else:
        B, T, C, F = (c[k] for k in ('B', 'T', 'C', 'F'))
        s = dict(x=normal(B, T, C), w_in=normal(2 * F, C, scale=C ** -0.5), w_out=normal(C, F, scale=F ** -0.5))
        s['b_in'] = normal(2 * F, scale=0.1) if c['bias'] else None
        s['b_out'] = normal(C, scale=0.1) if c['bias'] else None
        s['residual'] = normal(B, T, C) if c['residual'] else None
        names = tuple(n for n in ('x', 'w_in', 'w_out', 'b_in', 'b_out', 'residual') if s[n] is not None)
        douts = [(B, T, C)]
    if c['train']:
        s['douts'] = [normal(*d) for d in douts]
        for n in names:
            s[n] = s[n].detach().requires_grad_()
    s['case'], s['names'] = c, names
    return s


# ------------------------------------------------------------------------------------------------- the plain forms
def _plain_qk(s, q, k, qw, kw):
    c = s['case']

    def one(x, w):
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        R, cos, sin = c['R'], s['cos'][:, None, :], s['sin'][:, None, :]
        y, rest = y[..., :R], y[..., R:]
        if c['interleaved']:
            a, b = y[..., 0::2], y[..., 1::2]
            return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
        a, b = y[..., :R // 2], y[..., R // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    return one(q, qw), one(k, kw)


def _plain_diff(s, q, k, v, lq1, lk1, lq2, lk2):
    c = s['case']
    B, Tq, Tk, H, Hk, D = (c[n] for n in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D'))
    lam = torch.exp((lq1 * lk1).sum()) - torch.exp((lq2 * lk2).sum()) + 0.8
    key = torch.arange(Tk, device='cuda')
    n = s['lengths'][:, None, None] if c['ragged'] else torch.full((1, 1, 1), Tk, device='cuda')
    seen = key < n
    if c['causal']:
        seen = seen & (key <= torch.arange(Tq, device='cuda')[:, None] + n - Tq)
    seen = seen[:, None]                                             # [B or 1, 1, Tq or 1, Tk]

    def softmax(a, b):                                               # [B, T, heads, D] each; a row that sees nothing is zero
        x = torch.matmul(a.transpose(1, 2), b.transpose(1, 2).transpose(-1, -2)) * D ** -0.5
        x = torch.where(seen, x, -math.inf)
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(m == -math.inf, 0.0, m).detach())
        t = e.sum(-1, keepdim=True)
        return e / torch.where(t == 0, 1.0, t)
    k, v = k.repeat_interleave(H // Hk, 2), v.repeat_interleave(H // Hk, 2)
    p = softmax(q[..., :D], k[..., :D]) - lam * softmax(q[..., D:], k[..., D:])
    return (torch.matmul(p, v.transpose(1, 2)).transpose(1, 2),)


def _plain_ffn(s, x, w_in, w_out, b_in=None, b_out=None, residual=None):
    c = s['case']
    a = torch.matmul(x, w_in.t())
    if b_in is not None:
        a = a + b_in
    a, u = a[..., :c['F']], a[..., c['F']:]
    if c['act'] == 'silu':
        h = a / (1 + torch.exp(-a)) * u
    elif c['act'] == 'gelu':
        h = 0.5 * a * (1 + torch.erf(a * 2 ** -0.5)) * u
    else:
        h = 0.5 * a * (1 + torch.tanh((2 / math.pi) ** 0.5 * (a + 0.044715 * a * a * a))) * u
    y = torch.matmul(h, w_out.t())
    if b_out is not None:
        y = y + b_out
    return (y if residual is None else y + residual,)


def _call(s, block):
    c, t = s['case'], s
    if c['op'] == 'qk':
        return block.qk_norm_rope(t['q'], t['k'], t['qw'], t['kw'], t['cos'], t['sin'], eps=1e-6, interleaved=c['interleaved'])
    if c['op'] == 'diff':
        return (block.differential_attention(t['q'], t['k'], t['v'], t['lq1'], t['lk1'], t['lq2'], t['lk2'], lambda_init=0.8,
                                             key_lengths=t['lengths'], causal=c['causal']),)
    return (block.gated_feed_forward(t['x'], t['w_in'], t['w_out'], b_in=t['b_in'], b_out=t['b_out'], residual=t['residual'],
                                     activation=c['act']),)


def run(state):
    s, c = state, state['case']
    given = [s[n] for n in s['names']]
    if own:
        path = os.path.join(ROOT, 'nice-diffusion_amd')
        if path not in sys.path:
            sys.path.insert(0, path)
        from nicediffusion import block
        outs = _call(s, block)
        grads = torch.autograd.grad(outs, given, s['douts']) if c['train'] else ()
        return [o.detach() for o in outs], list(grads)
    dtype = _DTYPES[c['dtype']]
    wide = [t.detach().float().requires_grad_(c['train']) for t in given]
    plain = {'qk': _plain_qk, 'diff': _plain_diff, 'ffn': _plain_ffn}[c['op']]
    outs = plain(s, **dict(zip(s['names'], wide)))
    grads = torch.autograd.grad(outs, wide, [d.float() for d in s['douts']]) if c['train'] else ()
    return [o.detach().to(dtype) for o in outs], [g.to(dtype) for g in grads]


# -------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_qk(s, c):
    outs, dxs, dws = [], [], []
    R, D = c['R'], c['D']
    first = slice(0, R, 2) if c['interleaved'] else slice(0, R // 2)
    second = slice(1, R, 2) if c['interleaved'] else slice(R // 2, R)
    cos, sin = s['cos'].double().unsqueeze(1), s['sin'].double().unsqueeze(1)
    for i, (x, w) in enumerate(((s['q'], s['qw']), (s['k'], s['kw']))):
        x, w = x.detach().double(), w.detach().double()
        r = ((x * x).sum(-1, keepdim=True) / D + 1e-6) ** -0.5
        n = x * r * w
        y = n.clone()
        y[..., first] = cos * n[..., first] - sin * n[..., second]
        y[..., second] = sin * n[..., first] + cos * n[..., second]
        outs.append(y)
        if c['train']:
            dy = s['douts'][i].double()
            dn = dy.clone()
            dn[..., first] = cos * dy[..., first] + sin * dy[..., second]
            dn[..., second] = cos * dy[..., second] - sin * dy[..., first]
            dws.append((dn * x * r).sum((0, 1, 2)))
            dxs.append(r * (dn * w) - x * r ** 3 * (dn * w * x).sum(-1, keepdim=True) / D)
    return outs, dxs + dws


def _exact_diff(s, c):
    B, Tq, Tk, H, Hk, D, Dv = (c[n] for n in ('B', 'Tq', 'Tk', 'H', 'Hk', 'D', 'Dv'))
    q, k, v, a1, b1, a2, b2 = (s[n].detach().double() for n in ('q', 'k', 'v', 'lq1', 'lk1', 'lq2', 'lk2'))
    e1, e2 = torch.exp(a1 @ b1), torch.exp(a2 @ b2)
    lam, scale = e1 - e2 + 0.8, 1 / math.sqrt(D)
    out = torch.zeros(B, Tq, H, Dv, dtype=torch.float64, device='cuda')
    dq, dk, dv, dlam = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), 0.0
    for b, n in enumerate(_lengths(c)):
        for h in range(H):
            g = h * Hk // H
            if n == 0:
                continue
            kk, vv = k[b, :n, g], v[b, :n, g]
            maps = []
            for half in (slice(0, D), slice(D, 2 * D)):
                x = q[b, :, h, half] @ kk[:, half].t() * scale
                hidden = torch.ones(Tq, n, dtype=torch.bool, device='cuda').triu(n - Tq + 1) if c['causal'] else None
                if hidden is not None:
                    x = x.masked_fill(hidden, -math.inf)
                p = torch.softmax(x, -1)
                maps.append(torch.nan_to_num(p, nan=0.0))
            p1, p2 = maps
            out[b, :, h] = p1 @ vv - lam * (p2 @ vv)
            if c['train']:
                do = s['douts'][0][b, :, h].double()
                dp = do @ vv.t()
                dv[b, :n, g] += (p1 - lam * p2).t() @ do
                dlam = dlam - (p2 * dp).sum()
                for half, p, sign in ((slice(0, D), p1, 1.0), (slice(D, 2 * D), p2, -lam)):
                    ds = sign * p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                    dq[b, :, h, half] = ds @ kk[:, half]
                    dk[b, :n, g, half] += ds.t() @ q[b, :, h, half]
    if not c['train']:
        return [out], []
    return [out], [dq, dk, dv, dlam * e1 * b1, dlam * e1 * a1, -dlam * e2 * b2, -dlam * e2 * a2]


def _exact_ffn(s, c):
    F = c['F']
    t = {n: s[n].detach().double() for n in s['names']}
    x = t['x'].reshape(-1, c['C'])
    wg, wu, wo = t['w_in'][:F], t['w_in'][F:], t['w_out']
    a, u = x @ wg.t(), x @ wu.t()
    if c['bias']:
        a, u = a + t['b_in'][:F], u + t['b_in'][F:]
    if c['act'] == 'silu':
        sg = torch.sigmoid(a)
        f, df = a * sg, sg * (1 + a * (1 - sg))
    elif c['act'] == 'gelu':
        cdf = 0.5 * torch.erfc(-a / math.sqrt(2))
        f, df = a * cdf, cdf + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    else:
        z = math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
        th = torch.tanh(z)
        f, df = a * (1 + th) / 2, (1 + th) / 2 + a / 2 * (1 - th * th) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * a * a)
    h = f * u
    y = h @ wo.t()
    if c['bias']:
        y = y + t['b_out']
    y = y.reshape(t['x'].shape)
    if c['residual']:
        y = y + t['residual']
    if not c['train']:
        return [y], []
    dy = s['douts'][0].double().reshape(-1, c['C'])
    dh = dy @ wo
    da, du = dh * u * df, dh * f
    grads = {'x': (da @ wg + du @ wu).reshape(t['x'].shape), 'w_in': torch.cat([da.t() @ x, du.t() @ x]), 'w_out': dy.t() @ h,
             'b_in': torch.cat([da.sum(0), du.sum(0)]), 'b_out': dy.sum(0), 'residual': s['douts'][0].double()}
    return [y], [grads[n] for n in s['names']]


def exact(case, seed):
    s = prepare(case, seed)
    return {'qk': _exact_qk, 'diff': _exact_diff, 'ffn': _exact_ffn}[case['op']](s, case)
