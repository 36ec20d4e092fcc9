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
        if D == 2 and i < 2:      # x (D = 2): dx = r (g - x r^2 (g.x) / 2) cancels to its part across x; the error stays that of its terms
            t *= 50
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
