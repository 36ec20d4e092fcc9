"""Transformer-block operators (nicediffusion.block, libnd_block.so) on a real MI355X against their definitions in float64.

Tolerances.  Outputs are rounded once to their dtype: half a unit, eps/2 relative.  fp32: a sum of n terms of magnitudes
a_i carries at most n eps/2 sum(a_i); the tests use norms, where roundings of random sign add as squares, with a factor of 4
over sqrt(n) eps/2.  Values rounded to bf16 on the way (stated at each kernel) add eps/2 of bf16 each."""
import math

import pytest
import torch

from nicediffusion import _hip, block

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, F32 = torch.bfloat16, torch.float32


def rnd(*shape, seed=0, dtype=F32, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype).to(DEV)


def rel(got, ref):
    """2-norm of the difference over that of the reference (0 / 0 = 0)."""
    d, n = (got.double() - ref).norm().item(), ref.norm().item()
    return d / n if n else (math.inf if d else 0.0)


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def fp32_tol(n):
    return 4 * math.sqrt(n) * half_ulp(F32)


# ----------------------------------------------------------------------------------------------- qk_norm_rope
def qk_ref(x, w, cos, sin, eps, inter):
    x = x.double()
    n = x * (x.square().mean(-1, keepdim=True) + eps) ** -0.5
    if w is not None:
        n = n * w.double()
    if cos is None:
        return n
    R = 2 * cos.shape[-1]
    cos, sin = (t.double() if t.dim() == 3 else t.double()[None] for t in (cos, sin))
    cos, sin = cos[:, :, None], sin[:, :, None]
    a, b = (n[..., 0:R:2], n[..., 1:R:2]) if inter else (n[..., :R // 2], n[..., R // 2:R])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([ya, yb], -1).flatten(-2) if inter else torch.cat([ya, yb], -1)
    return torch.cat([y, n[..., R:]], -1)


QK_CASES = [  # B, T, Hq, Hk, D, R, interleaved, packed, batch tables
    (1, 1, 1, 1, 2, 2, False, False, False), (4, 1, 12, 12, 64, 64, False, False, True), (2, 33, 6, 6, 64, 64, False, True, False),
    (3, 785, 4, 2, 96, 48, True, True, False), (2, 17, 3, 1, 40, 40, False, False, False), (2, 5, 8, 2, 128, 128, False, False, True),
    (1, 130, 2, 2, 512, 256, True, False, False), (2, 9, 5, 5, 22, 10, False, True, False), (2, 7, 3, 3, 30, 14, True, True, False),
    (1, 3, 1, 1, 510, 510, False, False, False), (2, 65, 2, 1, 256, 0, False, True, False), (1, 2100, 3, 1, 32, 32, True, True, False),
]


def qk_inputs(B, T, Hq, Hk, D, R, packed, batched, dtype, far=0):
    if packed:
        row = rnd(B, T, (Hq + 2 * Hk) * D, seed=1, dtype=dtype)
        q, k = row[..., :Hq * D].view(B, T, Hq, D), row[..., Hq * D:(Hq + Hk) * D].view(B, T, Hk, D)
    else:
        q, k = rnd(B, T, Hq, D, seed=1, dtype=dtype), rnd(B, T, Hk, D, seed=2, dtype=dtype)
    qw, kw = rnd(D, seed=3, dtype=dtype, scale=0.2, mean=1.0), rnd(D, seed=4, dtype=dtype, scale=0.2, mean=1.0)
    cos = sin = None
    if R:
        pos = torch.arange(T, device=DEV) + far
        if batched:
            pos = (pos[None] + 17 * torch.arange(B, device=DEV)[:, None])[..., None]
        cos, sin = block.rotary_table(pos, R)
    return q, k, qw, kw, cos, sin


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('B,T,Hq,Hk,D,R,inter,packed,batched', QK_CASES)
def test_qk_norm_rope_and_gradients(B, T, Hq, Hk, D, R, inter, packed, batched, dtype):
    q, k, qw, kw, cos, sin = qk_inputs(B, T, Hq, Hk, D, R, packed, batched, dtype, far=100000)
    leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
    outs = block.qk_norm_rope(*leaves, cos, sin, eps=1e-6, interleaved=inter)
    plain = block.qk_norm_rope(q, k, qw, kw, cos, sin, eps=1e-6, interleaved=inter)
    wide = [t.detach().double().requires_grad_() for t in (q, k, qw, kw)]
    refs = (qk_ref(wide[0], wide[2], cos, sin, 1e-6, inter), qk_ref(wide[1], wide[3], cos, sin, 1e-6, inter))
    # the row's sum of D squares, the reciprocal root (~2 ulp) and ~6 roundings behind it, then the store
    tol = half_ulp(dtype) + fp32_tol(D) + 8 * half_ulp(F32)
    for o, p, r in zip(outs, plain, refs):
        assert torch.equal(o, p) and o.is_contiguous() and o.dtype == dtype
        assert rel(o, r) <= tol, rel(o, r)
        assert ((o.double() - r).abs() <= 2 * tol * r.abs().amax(-1, keepdim=True)).all()
    douts = [rnd(*o.shape, seed=7 + i, dtype=dtype) for i, o in enumerate(outs)]
    grads = torch.autograd.grad(outs, leaves, douts)
    want = torch.autograd.grad(refs, wide, [d.double() for d in douts])
    for i, (g, w) in enumerate(zip(grads, want)):
        n = D if i < 2 else B * T * (Hq if i == 2 else Hk)
        t = half_ulp(dtype) + 2 * fp32_tol(D) + (fp32_tol(n) if i >= 2 else 0) + 16 * half_ulp(F32)
        if D == 2 and i < 2:
            # dx = r (g' - n (g'.n) / D) is the part of r g' across n (n = r x, |n|^2 <= D): of two channels it may be a small one,
            # while the terms' fp32 errors stay relative to |r g'| and |r n (g'.n) / D| <= |r g'|, |g'| <= max|w| |dout|.  So the
            # store's half unit stays relative to |dx|, the rest is relative to 2 r max|w| |dout|.
            r = (wide[i].detach().square().mean(-1, keepdim=True) + 1e-6) ** -0.5
            terms = (2 * r * wide[2 + i].detach().abs().max() * douts[i].double().norm(dim=-1, keepdim=True)).norm()
            t = half_ulp(dtype) + (t - half_ulp(dtype)) * max(1.0, (terms / w.norm()).item())
        assert g.dtype == dtype and rel(g, w) <= t, (i, rel(g, w), t)


def test_qk_norm_rope_gradient_against_differences():
    q, k, qw, kw, cos, sin = qk_inputs(1, 3, 2, 1, 16, 16, False, False, F32)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    dout = [rnd(1, 3, 2, 16, seed=8), rnd(1, 3, 1, 16, seed=9)]
    grads = torch.autograd.grad(block.qk_norm_rope(*leaves, cos, sin), leaves, dout)
    step = 2.0 ** -7
    for i, t in enumerate(leaves):
        d = rnd(*t.shape, seed=20 + i)
        with torch.no_grad():
            f = []
            for sgn in (1, -1):
                moved = [x + sgn * step * d if j == i else x for j, x in enumerate(leaves)]
                f.append(sum((o.double() * g.double()).sum() for o, g in zip(block.qk_norm_rope(*moved, cos, sin), dout)))
        num, ana = ((f[0] - f[1]) / (2 * step)).item(), (grads[i].double() * d.double()).sum().item()
        # central difference: third-derivative term step^2 / 6 of O(30) terms, plus fp32 rounding 100 * 2^-24 / step
        assert abs(num - ana) <= 30 * step ** 2 / 6 * 4 + 100 * 2.0 ** -24 / step + 1e-4 * abs(ana), (i, num, ana)


def test_qk_norm_rope_in_place_in_a_packed_row_and_without_weights():
    B, T, H, D = 2, 19, 3, 64
    row = rnd(B, T, 3 * H * D, seed=1, dtype=BF)
    want = row.clone()
    cos, sin = block.rotary_table(block.grid_positions(1, T, DEV), D)
    v = lambda r, i: r[..., i * H * D:(i + 1) * H * D].view(B, T, H, D)  # noqa: E731
    a, b = block.qk_norm_rope(v(row, 0), v(row, 1), None, None, cos, sin)
    got = block.qk_norm_rope(v(row, 0), v(row, 1), None, None, cos, sin, out=(v(row, 0), v(row, 1)))
    assert got[0].data_ptr() == row.data_ptr()
    assert torch.equal(v(row, 0), a) and torch.equal(v(row, 1), b) and torch.equal(v(row, 2), v(want, 2))
    assert rel(a, qk_ref(v(want, 0), None, cos, sin, 1e-6, False)) <= half_ulp(BF) + 1e-5
    # interleaved q / k / v of each head (split_qkv_first=False), channels of one head transposed: a copy is made
    w2 = rnd(B, T, H, 3, D, seed=3)
    c, d = block.qk_norm_rope(w2[:, :, :, 0], w2[:, :, :, 1].transpose(-1, -2).contiguous().transpose(-1, -2))
    assert rel(c, qk_ref(w2[:, :, :, 0], None, None, None, 1e-6, False)) <= 1e-6
    assert rel(d, qk_ref(w2[:, :, :, 1], None, None, None, 1e-6, False)) <= 1e-6


def test_qk_norm_rope_special_rows():
    """A zero row stays zero (forward and gradient finite), a NaN or infinite channel spoils its own row alone."""
    q = rnd(1, 4, 2, 64, seed=1)
    q[0, 0, 0] = 0
    q[0, 1, 1, 5] = math.nan
    q[0, 2, 0, 7] = math.inf
    q.requires_grad_()
    k = rnd(1, 4, 1, 64, seed=2)
    cos, sin = block.rotary_table(torch.arange(4, device=DEV), 64)
    o, _ = block.qk_norm_rope(q, k, None, None, cos, sin)
    g, = torch.autograd.grad(o, q, rnd(1, 4, 2, 64, seed=3))
    bad = torch.zeros(1, 4, 2, dtype=torch.bool, device=DEV)
    bad[0, 1, 1] = bad[0, 2, 0] = True
    for t in (o, g):
        assert torch.equal(torch.isfinite(t).all(-1), ~bad)
    assert (o[0, 0, 0] == 0).all()


def test_qk_norm_rope_empty_and_unaligned():
    e = block.qk_norm_rope(torch.empty(2, 0, 3, 8, device=DEV), torch.empty(2, 0, 1, 8, device=DEV))
    assert e[0].shape == (2, 0, 3, 8) and e[1].shape == (2, 0, 1, 8)
    buf = rnd(1 + 2 * 5 * 3 * 64, seed=1, dtype=BF)
    q = buf[1:].view(2, 5, 3, 64)               # 2-byte aligned rows
    a, _ = block.qk_norm_rope(q, q)
    b, _ = block.qk_norm_rope(q.clone(), q.clone())
    # lanes hold other channels, so the row sum is taken in another order: a last-place difference at most
    assert rel(a, b.double()) <= 2 * half_ulp(BF)
    assert rel(a, qk_ref(q, None, None, None, 1e-6, False)) <= half_ulp(BF) + 1e-5


# ------------------------------------------------------------------------------------------------ gated_feed_forward
def ffn_ref(x, w_in, w_out, b_in, b_out, res, act):
    F = w_out.shape[1]
    a = x @ w_in.t()
    if b_in is not None:
        a = a + b_in
    a, u = a[..., :F], a[..., F:]
    if act == 'silu':
        f = a * torch.sigmoid(a)
    elif act == 'gelu':
        f = a * 0.5 * torch.special.erfc(-a / math.sqrt(2))
    else:
        f = 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
    y = (f * u) @ w_out.t()
    if b_out is not None:
        y = y + b_out
    return y if res is None else y + res


FFN_CASES = [  # M, C, F, act, bias, residual
    (1, 8, 8, 'silu', False, False), (1, 64, 136, 'gelu', True, True), (3, 72, 24, 'gelu_tanh', True, False), (17, 1024, 512, 'silu', True, True),
    (127, 40, 200, 'gelu', False, True), (256, 256, 256, 'silu', False, False), (257, 264, 680, 'gelu', True, True),
    (2355, 264, 680, 'gelu_tanh', False, True), (700, 136, 2056, 'silu', True, False), (5000, 64, 48, 'gelu', True, True),
]


def ffn_inputs(M, C, F, bias, residual, dtype):
    x = rnd(M, C, seed=1, dtype=dtype)
    w_in, w_out = rnd(2 * F, C, seed=2, dtype=dtype, scale=C ** -0.5), rnd(C, F, seed=3, dtype=dtype, scale=F ** -0.5)
    b_in, b_out = (rnd(2 * F, seed=4, dtype=dtype, scale=0.3), rnd(C, seed=5, dtype=dtype, scale=0.3)) if bias else (None, None)
    return [x, w_in, w_out, b_in, b_out, rnd(M, C, seed=6, dtype=dtype) if residual else None]


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('M,C,F,act,bias,residual', FFN_CASES)
def test_gated_feed_forward_and_gradients(M, C, F, act, bias, residual, dtype):
    given = ffn_inputs(M, C, F, bias, residual, dtype)
    leaves = [None if t is None else t.detach().requires_grad_() for t in given]
    wide = [None if t is None else t.detach().double().requires_grad_() for t in given]
    y = block.gated_feed_forward(leaves[0], leaves[1], leaves[2], leaves[3], leaves[4], leaves[5], act)
    plain = block.gated_feed_forward(*given[:5], residual=given[5], activation=act)
    ref = ffn_ref(*wide, act)
    assert torch.equal(y, plain) and y.dtype == dtype and y.shape == (M, C)
    # roundings: the output, h (bf16), then the fp32 sums of C and of F products and ~8 roundings of the activation
    tol = half_ulp(dtype) * (2 if dtype == BF else 1) + fp32_tol(C) + fp32_tol(F) + 16 * half_ulp(F32)
    assert rel(y, ref) <= tol, (rel(y, ref), tol)
    dy = rnd(M, C, seed=9, dtype=dtype)
    present = [i for i, t in enumerate(leaves) if t is not None]
    grads = torch.autograd.grad(y, [leaves[i] for i in present], dy)
    want = torch.autograd.grad(ref, [wide[i] for i in present], dy.double())
    # bf16: the output, da / du, and the kept a and u they are made from (a's half unit passes through act' and act: their
    # relative slopes stay below 2 where the values carry weight)
    for i, g, w in zip(present, grads, want):
        k = {0: C + 2 * F, 1: C + M, 2: C + M, 3: C + M, 4: M, 5: 0}[i]
        t = half_ulp(dtype) * (5 if dtype == BF else 1) + 2 * fp32_tol(k + 1) + 32 * half_ulp(F32)
        assert g.dtype == dtype and g.shape == w.shape and rel(g, w) <= t, (i, rel(g, w), t)


def test_gated_feed_forward_columns_one_by_one():
    """Every operand order of the products with values that name their place: exact in both dtypes, so any element that lands in a
    wrong row, column or k shows."""
    for dtype in (BF, F32):
        for M, C, F in ((300, 136, 264), (72, 520, 96)):
            x = torch.zeros(M, C, device=DEV, dtype=dtype)
            rows = torch.arange(M, device=DEV)
            x[rows, rows % C] = 1
            w_in = torch.zeros(2 * F, C, device=DEV, dtype=dtype)
            b_in = torch.zeros(2 * F, device=DEV, dtype=dtype)
            w_in[:F] = torch.randint(-8, 9, (F, C), device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(dtype)
            b_in[F:] = 1
            b_in[:F] = 64          # act(a) = a to fp32 rounding at a >= 56
            eye = torch.zeros(C, F, device=DEV, dtype=dtype)
            n = min(C, F)
            eye[torch.arange(n), torch.arange(n)] = 1
            y = block.gated_feed_forward(x, w_in, eye, b_in=b_in, activation='gelu')
            want = torch.zeros(M, C, device=DEV)
            want[:, :n] = 64 + w_in[:F].t()[rows % C][:, :n].float()
            assert torch.equal(y.float(), want), (dtype, M, C, F)


def test_gated_feed_forward_views_and_empty():
    x = rnd(3, 5, 128, seed=1, dtype=BF)
    w_in, w_out = rnd(2 * 64, 72, seed=2, dtype=BF, scale=0.1), rnd(72, 64, seed=3, dtype=BF, scale=0.1)
    v = x[..., 16:88]
    want = block.gated_feed_forward(v.contiguous(), w_in, w_out, residual=v.contiguous())
    assert torch.equal(block.gated_feed_forward(v, w_in, w_out, residual=v), want)
    assert torch.equal(block.gated_feed_forward(x[..., 3:75], w_in, w_out), block.gated_feed_forward(x[..., 3:75].contiguous(), w_in, w_out))
    assert torch.equal(block.gated_feed_forward(v.transpose(0, 1), w_in.t().contiguous().t(), w_out, residual=v.transpose(0, 1)), want.transpose(0, 1))
    one = block.gated_feed_forward(v[1, 2], w_in, w_out)
    assert one.shape == (72,) and rel(one, ffn_ref(v[1, 2].double()[None], w_in.double(), w_out.double(), None, None, None, 'silu')[0]) <= 2 * half_ulp(BF) + 1e-5
    e = rnd(0, 72, dtype=BF).requires_grad_()
    wg = w_in.clone().requires_grad_()
    y = block.gated_feed_forward(e, wg, w_out)
    g = torch.autograd.grad(y, (e, wg), torch.empty_like(y))
    assert y.shape == (0, 72) and g[0].shape == (0, 72) and (g[1] == 0).all()


# -------------------------------------------------------------------------------------------- differential_attention
def diff_ref(q, k, v, lams, lam_init, scale, lengths, causal, u, dout=None):
    """Outputs and gradients in float64 with, for each, the 2-norm that its error may have when the weights, dS and the kept maps'
    outputs are rounded by at most u relative and a score's exponential by eps (fp32)."""
    B, Tq, H, _ = q.shape
    Tk, Hk, D, Dv = k.shape[1], k.shape[2], q.shape[3] // 2, v.shape[3]
    per_head = lams[0].dim() == 2
    out = torch.zeros(B, Tq, H, Dv, dtype=torch.float64, device=q.device)
    e_out = torch.zeros_like(out)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    e_q, e_k, e_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dl, e_l = [torch.zeros_like(t) for t in lams], [torch.zeros_like(t) for t in lams]
    for b in range(B):
        n = lengths[b]
        for h in range(H):
            a1, b1, a2, b2 = (t[h] if per_head else t for t in lams)
            x1, x2 = (a1 * b1).sum().exp(), (a2 * b2).sum().exp()
            lam = x1 - x2 + lam_init
            if n == 0:
                continue
            g = h // (H // Hk)
            kk, vv = k[b, :n, g], v[b, :n, g]
            ps = []
            for m in range(2):
                s = q[b, :, h, m * D:(m + 1) * D] @ kk[:, m * D:(m + 1) * D].t() * scale
                if causal:
                    s = s.masked_fill(torch.ones(Tq, n, dtype=torch.bool, device=q.device).triu(n - Tq + 1), -math.inf)
                ps.append(torch.softmax(s, -1).nan_to_num(0.0))
                smax = s[s > -math.inf].abs().max().item() if (s > -math.inf).any() else 0.0
            eps = (smax + 8) * 4 * half_ulp(F32) * math.sqrt(D)
            p1, p2 = ps
            o1, o2 = p1 @ vv, p2 @ vv
            out[b, :, h] = o1 - lam * o2
            e_out[b, :, h] = (u + eps) * ((p1 + abs(lam) * p2) @ vv.abs())
            if dout is None:
                continue
            do = dout[b, :, h]
            dp = do @ vv.t()
            pd = p1 - lam * p2
            dv[b, :n, g] += pd.t() @ do
            e_v[b, :n, g] += (u * pd.abs() + eps * (p1 + abs(lam) * p2)).t() @ do.abs()
            dlam = -(p2 * dp).sum()
            e_lam = (p2 * eps * dp.abs()).sum() + 4 * math.sqrt(Dv) * half_ulp(F32) * (p2 * (do.abs() @ vv.abs().t())).sum()
            for i, (val, o) in enumerate(((x1, b1), (x1, a1), (-x2, b2), (-x2, a2))):
                tgt, etgt = (dl[i][h], e_l[i][h]) if per_head else (dl[i], e_l[i])
                tgt += dlam * val * o
                etgt += e_lam * val.abs() * o.abs()
            for m, (p, o, f) in enumerate(((p1, o1, 1.0), (p2, o2, -lam))):
                c = (do * o).sum(-1, keepdim=True)
                e_c = (u + eps) * (do.abs() * o.abs()).sum(-1, keepdim=True)
                ds = f * p * (dp - c) * scale
                e_ds = u * ds.abs() + abs(f) * p * scale * (e_c + eps * (dp.abs() + c.abs()))
                half = slice(m * D, (m + 1) * D)
                if n > 1:
                    dq[b, :, h, half] = ds @ kk[:, half]
                    e_q[b, :, h, half] = e_ds @ kk[:, half].abs()
                    dk[b, :n, g, half] += ds.t() @ q[b, :, h, half]
                    e_k[b, :n, g, half] += e_ds.t() @ q[b, :, h, half].abs()
    return (out, e_out), [(dq, e_q), (dk, e_k), (dv, e_v)] + list(zip(dl, e_l))


DIFF_CASES = [  # B, Tq, Tk, H, Hk, D, Dv, lengths, causal, per head
    (1, 1, 1, 1, 1, 8, 8, None, False, False), (2, 64, 64, 2, 2, 32, 64, None, False, False), (2, 64, 64, 2, 2, 32, 64, None, True, False),
    (3, 49, 49, 4, 2, 32, 64, (49, 17, 0), False, True), (2, 130, 130, 2, 1, 64, 128, (130, 65), True, True), (1, 257, 300, 2, 2, 64, 128, None, True, False),
    (2, 1, 700, 8, 2, 64, 128, (700, 1), False, False), (3, 3, 1500, 4, 4, 32, 64, (1500, 2, 0), True, False), (1, 1, 5000, 16, 1, 128, 256, None, False, True),
    (2, 70, 33, 3, 3, 128, 256, None, True, False), (1, 100, 90, 2, 1, 96, 192, (64,), False, False), (2, 33, 65, 2, 2, 24, 40, (65, 31), False, True),
    (1, 40, 40, 6, 2, 128, 128, None, True, False), (1, 600, 600, 1, 1, 40, 80, None, False, False), (2, 5, 2, 2, 2, 16, 16, (1, 2), False, False),
    (1, 4, 97, 32, 4, 56, 112, None, True, False),
]


def diff_inputs(B, Tq, Tk, H, Hk, D, Dv, lengths, per_head, dtype):
    q, k, v = rnd(B, Tq, H, 2 * D, seed=1, dtype=dtype), rnd(B, Tk, Hk, 2 * D, seed=2, dtype=dtype), rnd(B, Tk, Hk, Dv, seed=3, dtype=dtype)
    k[0, Tk // 2] *= 3          # a spiky key: the running maximum moves
    lams = [rnd(*((H, D) if per_head else (D,)), seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
    return q, k, v, lams, None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)


def within(got, ref, err, dtype, slack=1.0):
    """2-norm of the difference against the derived bound plus the output's own rounding."""
    return (got.double() - ref).norm().item() <= slack * (err.norm().item() + half_ulp(dtype) * ref.norm().item()) * (1 + 1e-6) + 1e-30


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('B,Tq,Tk,H,Hk,D,Dv,lengths,causal,per_head', DIFF_CASES)
def test_differential_attention_and_gradients(B, Tq, Tk, H, Hk, D, Dv, lengths, causal, per_head, dtype):
    q, k, v, lams, ln = diff_inputs(B, Tq, Tk, H, Hk, D, Dv, lengths, per_head, dtype)
    if lengths is not None:          # what lies behind a sequence's end is not looked at
        for b, n in enumerate(lengths):
            k[b, n:] = math.nan
            v[b, n:] = math.inf
    leaves = [t.clone().requires_grad_() for t in (q, k, v, *lams)]
    out = block.differential_attention(*leaves, lambda_init=0.6, key_lengths=ln, causal=causal)
    plain = block.differential_attention(q, k, v, *lams, lambda_init=0.6, key_lengths=ln, causal=causal)
    assert torch.equal(out, plain) and out.dtype == dtype and out.shape == (B, Tq, H, Dv)
    dout = rnd(B, Tq, H, Dv, seed=11, dtype=dtype)
    u = half_ulp(BF) if dtype == BF else 0.0
    full = lengths or (Tk,) * B
    (ref, err), grads = diff_ref(*(t.double() for t in (q, k, v)), [t.double() for t in lams], 0.6, D ** -0.5, full, causal, u, dout.double())
    assert within(out, ref, err, dtype), ((out.double() - ref).norm() / ref.norm(), err.norm() / ref.norm())
    for b in range(B):                # rows that see nothing
        blind = Tq if full[b] == 0 else (max(0, Tq - full[b]) if causal else 0)
        assert (out[b, :blind] == 0).all()
    got = torch.autograd.grad(out, leaves, dout)
    for i, (g, (r, e)) in enumerate(zip(got, grads)):
        assert g.dtype == dtype and within(g, r, e, dtype), (i, (g.double() - r).norm() / r.norm(), e.norm() / r.norm())
    for b in range(B):
        assert (got[1][b, full[b]:] == 0).all() and (got[2][b, full[b]:] == 0).all()
        if full[b] <= 1:
            assert (got[0][b] == 0).all() and (got[1][b] == 0).all()


@pytest.mark.parametrize('dtype', [BF, F32])
def test_differential_attention_in_a_packed_row(dtype):
    B, T, H, D = 2, 77, 3, 32
    row = rnd(B, T, H, 3, 2 * D, seed=1, dtype=dtype)          # q, k, v of each head beside each other
    q, k, v = row.unbind(3)
    lams = [rnd(D, seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
    a = block.differential_attention(q, k, v, *lams)
    b = block.differential_attention(q.contiguous(), k.contiguous(), v.contiguous(), *lams)
    assert torch.equal(a, b)
    # rows off the 16-byte grid and transposed channels are copied
    wide = rnd(B, T, H, 2 * D + 1, seed=5, dtype=dtype)
    assert torch.equal(block.differential_attention(wide[..., 1:], k, v, *lams), block.differential_attention(wide[..., 1:].contiguous(), k, v, *lams))
    # shared keys (a batch of one, expanded) and int64 lengths
    ks, vs = k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1)
    ln = torch.tensor([77, 20], device=DEV)
    c = block.differential_attention(q, ks, vs, *lams, key_lengths=ln)
    assert torch.equal(c, block.differential_attention(q, ks.contiguous(), vs.contiguous(), *lams, key_lengths=ln.int()))
    leaf = k[:1].clone().requires_grad_()
    g, = torch.autograd.grad(block.differential_attention(q, leaf.expand(B, -1, -1, -1), vs, *lams, key_lengths=ln), leaf, a)
    assert g.shape == leaf.shape and torch.isfinite(g).all()


def test_differential_attention_splits_agree_with_one_pass():
    """The same queries alone (keys divided among waves and workgroups) and among many (one pass)."""
    for dtype in (BF, F32):
        q, k, v, lams, _ = diff_inputs(1, 512, 2048, 4, 2, 64, 128, None, False, dtype)
        many = block.differential_attention(q, k, v, *lams)
        one = block.differential_attention(q[:, 100:101], k, v, *lams)
        assert rel(one, many[:, 100:101].double()) <= (2.5 if dtype == BF else 16) * half_ulp(dtype)


def test_differential_attention_gradient_against_differences():
    q, k, v, lams, _ = diff_inputs(1, 5, 6, 2, 1, 8, 16, None, False, F32)
    leaves = [t.requires_grad_() for t in (q, k, v, *lams)]
    dout = rnd(1, 5, 2, 16, seed=8)
    grads = torch.autograd.grad(block.differential_attention(*leaves, causal=True), leaves, dout)
    step = 2.0 ** -7
    for i, t in enumerate(leaves):
        d = rnd(*t.shape, seed=20 + i, scale=0.3)
        with torch.no_grad():
            f = [(block.differential_attention(*[x + sgn * step * d if j == i else x for j, x in enumerate(leaves)], causal=True).double() * dout.double()).sum()
                 for sgn in (1, -1)]
        num, ana = ((f[0] - f[1]) / (2 * step)).item(), (grads[i].double() * d.double()).sum().item()
        # central difference: third derivatives of O(100) / 6 times step^2, rounding 100 * 2^-24 / step
        assert abs(num - ana) <= 100 / 6 * step ** 2 + 100 * 2.0 ** -24 / step + 1e-3 * abs(ana), (i, num, ana)


def test_differential_attention_empty():
    lams = [rnd(8, seed=i).requires_grad_() for i in range(4)]
    for B, Tq, Tk in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q, k, v = (torch.randn(B, t, 2, 16, device=DEV, requires_grad=True) for t in (Tq, Tk, Tk))
        o = block.differential_attention(q, k, v, *lams)
        assert o.shape == (B, Tq, 2, 16) and (o == 0).all()
        for g, t in zip(torch.autograd.grad(o.sum(), (q, k, v, *lams)), (q, k, v, *lams)):
            assert g.shape == t.shape and (g == 0).all()


def test_differential_attention_rows_that_repeat_in_memory():
    """Queries, keys and values expanded over tokens (stride 0): rows past the last are not told apart by their address."""
    for dtype in (BF, F32):
        B, T, H, D = 2, 45, 2, 32
        q, k, v = (rnd(B, 1, H, 2 * D, seed=i, dtype=dtype).expand(-1, T, -1, -1) for i in range(3))
        lams = [rnd(D, seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
        dout = rnd(B, 1, H, 2 * D, seed=9, dtype=dtype).expand(-1, T, -1, -1)
        ln = torch.tensor([45, 33], dtype=torch.int32, device=DEV)
        got = []
        for a, b, c, d in ((q, k, v, dout), [t.contiguous() for t in (q, k, v, dout)]):
            leaves = [t.detach().requires_grad_() for t in (a, b, c, *lams)]
            o = block.differential_attention(*leaves, key_lengths=ln)
            got.append((o, *torch.autograd.grad(o, leaves, d)))
        for a, b in zip(*got):
            assert torch.equal(a, b)


def test_qk_norm_rope_reciprocal_root():
    """Rows (1, t, 0, ..) with exact squares, exact mean and no weight: the first channel is the reciprocal root itself.  One correction of
    the hardware's (1 ulp) leaves its own rounding, half an ulp, and half that of m r: 3/2 half units."""
    for D in (4, 64, 512):
        t = torch.arange(1, 2048, dtype=torch.float64) / 1024
        x = torch.zeros(1, 2047, 1, D)
        x[0, :, 0, 0], x[0, :, 0, 1] = 1, t.float()
        x = x.to(DEV)
        want = ((1 + t * t) / D) ** -0.5
        got = block.qk_norm_rope(x, x, eps=0.0)[0][0, :, 0, 0].double().cpu()
        assert ((got - want).abs() <= 1.5 * half_ulp(F32) * want * (1 + 1e-6)).all(), (D, ((got - want).abs() / want).max().item() / half_ulp(F32))
        # gradient of the second channel's output 1: -x0 x1 r^3 / D, from r^2 and r, two products and the division by D
        leaf = x.clone().requires_grad_()
        o, _ = block.qk_norm_rope(leaf, x, eps=0.0)
        d = torch.zeros_like(o)
        d[..., 1] = 1
        g = torch.autograd.grad(o, leaf, d)[0][0, :, 0, 0].double().cpu()
        ref = -t * want ** 3 / D
        assert ((g - ref).abs() <= (3 * 1.5 + 4) * half_ulp(F32) * ref.abs() * (1 + 1e-6)).all(), D
    big = torch.full((1, 1, 1, 8), 1e25, device=DEV)           # the sum of squares leaves fp32: zeros, as the reciprocal root says
    assert (block.qk_norm_rope(big, big)[0] == 0).all()
    z = torch.zeros(1, 1, 1, 8, device=DEV)
    assert (block.qk_norm_rope(z, z)[0] == 0).all() and torch.isnan(block.qk_norm_rope(z, z, eps=0.0)[0]).all()
