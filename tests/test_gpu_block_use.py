"""The transformer-block operators as a program uses them, on a real MI355X: together, beside the attention of nd_hip.h, on other
streams, in captured graphs, from two threads, over long caches and at the ends of their ranges."""
import math
import threading

import pytest
import torch

from nicediffusion import _hip, block
from tests.test_gpu_block import BF, DEV, F32, diff_ref, ffn_ref, fp32_tol, half_ulp, qk_ref, rel, rnd, within

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


# --------------------------------------------------------------------------------------------------------- together
def layer(p, x, height, width, heads, q_norm_rope, attention, ffn, linear):
    """One layer over the tokens of a map: packed projection, norm and rotation of both maps' queries and keys, attention, gated
    feed-forward with the residual."""
    B, T, C = x.shape
    D = C // heads // 2
    row = linear(x, p['qkv'])                                  # [B, T, heads * (2D + 2D + 2D)]
    q, k, v = (row[..., i * C:(i + 1) * C] for i in range(3))
    q, k = q_norm_rope(q.reshape(B, T, 2 * heads, D), k.reshape(B, T, 2 * heads, D), p['qw'], p['kw'])
    o = attention(q.reshape(B, T, heads, 2 * D), k.reshape(B, T, heads, 2 * D), v.reshape(B, T, heads, 2 * D), [p['l%d' % i] for i in range(4)])
    x = x + linear(o.reshape(B, T, C), p['proj'])
    return ffn(x, p['w_in'], p['w_out'])


def plain_layer(p, x, height, width, heads, store):
    """The same in float64; store(t) stands where a value is kept in the tensors' dtype."""
    B, T, C = x.shape
    D = C // heads // 2
    cos, sin = block.rotary_table(block.grid_positions(height, width, DEV), D)

    def attention(q, k, v, lams):
        lam = (lams[0] * lams[1]).sum().exp() - (lams[2] * lams[3]).sum().exp() + 0.8
        ps = []
        for m in range(2):
            a, b = (t[..., m * D:(m + 1) * D].transpose(1, 2) for t in (q, k))
            ps.append(store(torch.softmax((a @ b.transpose(2, 3).contiguous()) * D ** -0.5, -1)))
        vt = v.transpose(1, 2).contiguous()
        return store((ps[0] @ vt - lam * (ps[1] @ vt)).transpose(1, 2))

    def ffn(x, w_in, w_out):
        F = w_out.shape[1]
        a = x @ w_in.t()
        a, u = store(a[..., :F]), store(a[..., F:])
        return store(x + store(a * torch.sigmoid(a) * u) @ w_out.t())

    return layer(p, x, height, width, heads, lambda q, k, a, b: (store(qk_ref(q, a, cos, sin, 1e-6, False)), store(qk_ref(k, b, cos, sin, 1e-6, False))),
                 attention, ffn, lambda t, w: store(t @ w.t()))


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('B,height,width,C,heads,F', [(2, 8, 8, 128, 2, 336), (1, 5, 13, 192, 3, 256)])
def test_the_operators_as_one_layer(B, height, width, C, heads, F, dtype):
    T, D = height * width, C // heads // 2
    p = dict(qkv=rnd(3 * C, C, seed=1, dtype=dtype, scale=C ** -0.5), qw=rnd(D, seed=2, dtype=dtype, scale=0.1, mean=1.0),
             kw=rnd(D, seed=3, dtype=dtype, scale=0.1, mean=1.0), proj=rnd(C, C, seed=4, dtype=dtype, scale=C ** -0.5),
             w_in=rnd(2 * F, C, seed=5, dtype=dtype, scale=C ** -0.5), w_out=rnd(C, F, seed=6, dtype=dtype, scale=F ** -0.5))
    p.update({'l%d' % i: rnd(D, seed=10 + i, dtype=dtype, scale=0.2) for i in range(4)})
    x, dy = rnd(B, T, C, seed=7, dtype=dtype), rnd(B, T, C, seed=8, dtype=dtype)
    cos, sin = block.rotary_table(block.grid_positions(height, width, DEV), D)
    lin = lambda t, w: torch.nn.functional.linear(t.reshape(-1, t.shape[-1]), w).view(*t.shape[:-1], -1)  # noqa: E731
    leaves = {n: t.clone().requires_grad_() for n, t in dict(p, x=x).items()}
    y = layer(leaves, leaves['x'], height, width, heads, lambda q, k, a, b: block.qk_norm_rope(q, k, a, b, cos, sin),
              lambda q, k, v, l: block.differential_attention(q, k, v, *l), lambda t, a, b: block.gated_feed_forward(t, a, b, residual=t), lin)
    names = sorted(leaves)
    got = [y] + list(torch.autograd.grad(y, [leaves[n] for n in names], dy))

    def reference(noise):
        wide = {n: t.double().requires_grad_() for n, t in dict(p, x=x).items()}
        g = torch.Generator(DEV).manual_seed(5)

        class Store(torch.autograd.Function):          # a kept value and its gradient, each off by at most `noise` of itself
            @staticmethod
            def forward(ctx, t):
                return t * (1 + noise * (2 * torch.randint(0, 2, t.shape, device=DEV, generator=g) - 1))

            @staticmethod
            def backward(ctx, d):
                return d * (1 + noise * (2 * torch.randint(0, 2, d.shape, device=DEV, generator=g) - 1))

        out = plain_layer(wide, wide['x'], height, width, heads, Store.apply)
        return [out.detach()] + [t.detach() for t in torch.autograd.grad(out, [wide[n] for n in names], dy.double())]

    # Every stored value is off by at most half a unit; in fp32 the sums behind it add 4 sqrt(n) half units (n <= max(2F, 3C, T)).
    # The float64 layer with errors of exactly that size and random sign at each store shows what they make of the results; a
    # factor of 4 for sums that happen to agree, and the result's own half unit.
    noise = half_ulp(dtype) + fp32_tol(max(2 * F, 3 * C, T))
    exact, moved = reference(0.0), reference(noise)
    for n, a, e, m in zip(['y'] + names, got, exact, moved):
        bound = 4 * (m - e).norm().item() + noise * e.norm().item()
        assert a.dtype == dtype and (a.double() - e).norm().item() <= bound, (n, rel(a, e), bound / e.norm().item())


def test_norm_and_rotation_in_front_of_the_frameworks_attention():
    """qk_norm_rope in place in the packed row that nd_attention_nhwc / nd_attention_bf16_nhwc read."""
    B, T, H, D = 2, 64, 3, 64
    C = H * D
    cos, sin = block.rotary_table(block.grid_positions(8, 8, DEV), D)
    for dtype, name in ((F32, 'nd_attention_nhwc'), (BF, 'nd_attention_bf16_nhwc')):
        row = rnd(B, T, 3 * C, seed=1, dtype=dtype)
        part = lambda r, i: r[..., i * C:(i + 1) * C].view(B, T, H, D)  # noqa: E731
        q, k, v = (part(row.double(), i) for i in range(3))
        q, k = (qk_ref(t, None, cos, sin, 1e-6, False) for t in (q, k))
        s = torch.softmax(q.transpose(1, 2) @ k.permute(0, 2, 3, 1).contiguous() * D ** -0.5, -1)
        want = (s @ v.transpose(1, 2).contiguous()).transpose(1, 2)
        block.qk_norm_rope(part(row, 0), part(row, 1), None, None, cos, sin, out=(part(row, 0), part(row, 1)))
        out = torch.empty(B, T, C, device=DEV, dtype=dtype)
        _hip.check(getattr(_hip.load(), name)(row.data_ptr(), 3 * C, out.data_ptr(), C, B, T, H, D, 0, C, 2 * C, D, D ** -0.5, stream()))
        # normed rows have length sqrt(D), so |score| <= sqrt(D) = 8: q and k rounded by u each move it by 16 u at most, a weight by
        # as much relative to itself; the weights' and the output's own rounding add u each
        tol = half_ulp(dtype) * (2 + 2 * 8) + fp32_tol(D) * 8 + fp32_tol(T)
        assert rel(out.view(B, T, H, D), want) <= tol, (name, rel(out.view(B, T, H, D), want), tol)


# -------------------------------------------------------------------------------------- calls of each operator, for the tests below
def calls(dtype, seed=0, tokens=70):
    """name -> (function, its tensors): a serving-sized and a training-sized call of each operator."""
    T, D = tokens, 32
    cos, sin = block.rotary_table(torch.arange(T, device=DEV), D)
    lam = [rnd(D, seed=seed + 20 + i, dtype=dtype, scale=0.2) for i in range(4)]
    ln = torch.tensor([T, T // 3], dtype=torch.int32, device=DEV)
    w = [rnd(2 * 136, 64, seed=seed + 8, dtype=dtype, scale=0.125), rnd(64, 136, seed=seed + 9, dtype=dtype, scale=0.1)]
    r = lambda i, *s: rnd(*s, seed=seed + i, dtype=dtype)  # noqa: E731
    return {
        'qk': (lambda q, k, a, b: block.qk_norm_rope(q, k, a, b, cos, sin), [r(1, 2, T, 4, D), r(2, 2, T, 2, D), r(3, D), r(4, D)]),
        'diff': (lambda q, k, v, *l: block.differential_attention(q, k, v, *l, key_lengths=ln, causal=True), [r(1, 2, T, 4, 2 * D), r(2, 2, T, 2, 2 * D), r(3, 2, T, 2, 2 * D), *lam]),
        'diff_few': (lambda q, k, v, *l: block.differential_attention(q, k, v, *l), [r(1, 2, 1, 4, 2 * D), r(2, 2, 40 * T, 2, 2 * D), r(3, 2, 40 * T, 2, 2 * D), *lam]),
        'ffn': (lambda x, a, b: block.gated_feed_forward(x, a, b, residual=x), [r(1, 2, T, 64), *w]),
        'ffn_few': (lambda x, a, b: block.gated_feed_forward(x, a, b, activation='gelu'), [r(1, 3, 64), *w]),
    }


def outputs(o):
    return list(o) if isinstance(o, (tuple, list)) else [o]


def with_gradients(fn, tensors, clone=True):
    leaves = [t.detach().clone().requires_grad_() if clone else t.detach().requires_grad_() for t in tensors]
    out = outputs(fn(*leaves))
    return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out]))


NAMES = ['qk', 'diff', 'diff_few', 'ffn', 'ffn_few']


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('name', NAMES)
def test_a_call_repeats_bit_for_bit(name, dtype):
    fn, ts = calls(dtype, tokens=300)[name]
    a = with_gradients(fn, ts)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(a, with_gradients(fn, ts)))


@pytest.mark.parametrize('name', NAMES)
def test_on_another_stream(name):
    """Inputs made on a side stream, the call and its backward on it, read there: ordered without a device synchronisation."""
    fn, ts = calls(BF)[name]
    want = with_gradients(fn, [t * 2 for t in ts])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.empty(1 << 28, device=DEV)
        big.fill_(2.0)                                         # ~0.2 ms: a call on the wrong stream would read ahead of it
        got = with_gradients(fn, [t * big[-1].to(t.dtype) for t in ts])
        same = [torch.equal(a, b) for a, b in zip(got, want)]
    torch.cuda.synchronize()
    assert all(same)


def test_two_threads_at_once():
    """Each on its own stream, different operators side by side."""
    table = calls(BF)
    want = {n: with_gradients(*table[n]) for n in NAMES}
    torch.cuda.synchronize()
    bad = []

    def work(names):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                for n in names:
                    got = with_gradients(*table[n])
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[n])):
                        bad.append(n)

    threads = [threading.Thread(target=work, args=(o,)) for o in (NAMES, NAMES[::-1])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize('name', NAMES)
def test_captured_and_replayed(name):
    """Forward and backward in two graphs of the same shapes, replayed in turn between eager calls, each against the eager result of
    its own inputs."""
    fn, _ = calls(BF)[name]
    graphs = []
    for g in range(2):
        static = [t.clone() for t in calls(BF, seed=100 * g)[name][1]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            with_gradients(fn, static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = with_gradients(fn, static, clone=False)      # leaves that only this graph holds
        graphs.append((graph, static, out))
    for step in range(3):
        for i, (graph, static, out) in enumerate(graphs):
            fresh = calls(BF, seed=1000 + 10 * step + i)[name][1]
            for s, f in zip(static, fresh):
                s.copy_(f)
            for o in out:
                o.fill_(math.nan)
            graph.replay()
        for i, (graph, static, out) in enumerate(graphs):
            fresh = calls(BF, seed=1000 + 10 * step + i)[name][1]
            want = with_gradients(fn, fresh)
            torch.cuda.synchronize()
            for j, (a, b) in enumerate(zip(out, want)):
                assert torch.equal(a, b), (step, i, j)


# --------------------------------------------------------------------------------------------------- caches and long rows
def test_a_slot_of_a_cache_and_rows_behind_the_last():
    """qk_norm_rope into one slot of a longer cache leaves the others; the attention that reads it sees `length` rows only, and a
    padded batch's rows of other sequences do not enter."""
    B, H, Hk, D, room = 3, 4, 2, 32, 50
    kc = torch.full((B, room, Hk, 2 * D), math.nan, device=DEV, dtype=BF)
    vc = torch.full((B, room, Hk, 2 * D), math.nan, device=DEV, dtype=BF)
    lens, lams = [0, 0, 0], [rnd(D, seed=30 + i, dtype=BF, scale=0.2) for i in range(4)]
    for step in range(4):
        q, k, v = rnd(B, 1, 2 * H, D, seed=step, dtype=BF), rnd(B, 1, 2 * Hk, D, seed=10 + step, dtype=BF), rnd(B, 1, Hk, 2 * D, seed=20 + step, dtype=BF)
        cos, sin = block.rotary_table(torch.tensor([step], device=DEV), D)
        before = kc.clone()
        qo = torch.empty_like(q)
        block.qk_norm_rope(q, k, None, None, cos, sin, out=(qo, kc[:, step:step + 1].view(B, 1, 2 * Hk, D)))
        before[:, step] = qk_ref(k, None, cos, sin, 1e-6, False).view(B, Hk, 2 * D).to(BF)
        same = torch.isnan(before) == torch.isnan(kc)
        assert same.all() and torch.allclose(kc.nan_to_num(0.0).float(), before.nan_to_num(0.0).float(), rtol=2 * half_ulp(BF) + 1e-5, atol=1e-6)
        vc[:, step:step + 1] = v
        lens = [max(0, step + 1 - b) for b in range(B)]
        ln = torch.tensor(lens, device=DEV)
        o = block.differential_attention(qo.view(B, 1, H, 2 * D), kc, vc, *lams, key_lengths=ln)
        (ref, err), _ = diff_ref(qo.view(B, 1, H, 2 * D).double(), kc.double(), vc.double(), [t.double() for t in lams], 0.8, D ** -0.5, lens, False, half_ulp(BF))
        assert within(o, ref, err, BF) and (o[[b for b in range(B) if lens[b] == 0]] == 0).all()


def far_rows(n, cols, dtype, stride, seed):
    """[n, cols] whose rows lie `stride` elements apart (a strided cache of more than 2^32 bytes), and the same packed."""
    flat = torch.empty(n * stride, device=DEV, dtype=dtype)
    far = torch.as_strided(flat, (n, cols), (stride, 1))
    packed = rnd(n, cols, seed=seed, dtype=dtype)
    far.copy_(packed)
    return far, packed


def test_offsets_past_32_bits():
    n, H, D = 1100, 2, 64
    stride = 1 << 21
    assert (n - 1) * stride * 2 > 1 << 32
    far, packed = far_rows(n, 3 * H * 2 * D, BF, stride, 1)
    part = lambda r, i: r.unflatten(1, (3 * H, 2 * D))[None, :, i * H:(i + 1) * H]  # noqa: E731
    lams = [rnd(D, seed=4 + i, dtype=BF, scale=0.2) for i in range(4)]
    a, b = ([part(r, i) for i in range(3)] for r in (far, packed))
    assert a[1].stride(1) == stride
    for q in (slice(0, n), slice(n - 1, n)):                    # all queries, and a single token
        x = block.differential_attention(a[0][:, q], a[1], a[2], *lams, causal=True)
        y = block.differential_attention(b[0][:, q], b[1], b[2], *lams, causal=True)
        assert torch.equal(x, y) and torch.isfinite(x).all()
    gx, gy = (with_gradients(lambda q, k, v, *l: block.differential_attention(q, k, v, *l, causal=True), [*r, *lams], clone=False) for r in (a, b))
    assert all(torch.equal(s, t) for s, t in zip(gx, gy))
    cos, sin = block.rotary_table(torch.arange(n, device=DEV), 2 * D)
    gx, gy = (with_gradients(lambda q, k: block.qk_norm_rope(q, k, None, None, cos, sin), r[:2], clone=False) for r in (a, b))
    assert all(torch.equal(s, t) for s, t in zip(gx, gy))
    block.qk_norm_rope(a[0], a[1], None, None, cos, sin, out=(a[0], a[1]))
    assert torch.equal(a[0], gy[0]) and torch.equal(a[1], gy[1]) and torch.equal(a[2], b[2])
    w = [rnd(2 * 96, 128, seed=8, dtype=BF, scale=0.1), rnd(128, 96, seed=9, dtype=BF, scale=0.1)]
    x, y = far[:, :128], packed[:, :128]
    x.copy_(y)
    gx, gy = (with_gradients(lambda t, i, o: block.gated_feed_forward(t, i, o, residual=t), [r, *w], clone=False) for r in (x, y))
    assert all(torch.equal(s, t) for s, t in zip(gx, gy))


def test_feed_forward_of_more_than_2_32_bytes():
    """Intermediate rows past 4 GiB: the last rows against a call on them alone, the weights' gradients against the halves' sum."""
    M, C, F = 280000, 64, 4096
    assert M * 2 * F * 2 > 1 << 32
    x, w_in, w_out = rnd(M, C, seed=1, dtype=BF), rnd(2 * F, C, seed=2, dtype=BF, scale=C ** -0.5), rnd(C, F, seed=3, dtype=BF, scale=F ** -0.5)
    whole = with_gradients(lambda *t: block.gated_feed_forward(*t), [x, w_in, w_out], clone=False)
    halves = [with_gradients(lambda *t: block.gated_feed_forward(*t), [x[s], w_in, w_out], clone=False) for s in (slice(0, M // 2), slice(M // 2, M))]
    # the same sums in another order or split, rounded to bf16: one unit at most, in all half a unit of norm from either side
    for i in (0, 1):
        both = torch.cat([halves[0][i], halves[1][i]])
        assert rel(whole[i], both.double()) <= 2 * half_ulp(BF)
        assert rel(whole[i][-1000:], both[-1000:].double()) <= 2 * half_ulp(BF)
    for i in (2, 3):
        assert rel(whole[i], halves[0][i].double() + halves[1][i].double()) <= 3 * half_ulp(BF) * max(1.0, math.sqrt(2) * halves[0][i].double().norm().item() / whole[i].double().norm().item())


# ----------------------------------------------------------------------------------------------------- ends of the ranges
@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('B,T,Hq,Hk,D,R', [(1, 1, 1, 1, 64, 64), (3, 5, 3, 2, 64, 64), (1, 1, 1, 2, 32, 32), (2, 37, 5, 2, 32, 0), (1, 3, 1, 1, 16, 16),
                                           (5, 1, 2, 1, 64, 0), (1, 1031, 1, 1, 64, 64), (1, 67, 3, 1, 8, 8)])
def test_norm_and_rotation_of_short_rows(B, T, Hq, Hk, D, R, dtype):
    """Rows of at most 256 bytes, several to a wave: odd numbers of rows, waves that span queries and keys, eps = 0, in place."""
    q, k = rnd(B, T, Hq, D, seed=1, dtype=dtype), rnd(B, T, Hk, D, seed=2, dtype=dtype)
    w = [rnd(D, seed=3 + i, dtype=dtype, scale=0.2, mean=1.0) for i in range(2)]
    cos, sin = block.rotary_table(torch.arange(T, device=DEV), R) if R else (None, None)
    leaves = [t.clone().requires_grad_() for t in (q, k, *w)]
    wide = [t.double().requires_grad_() for t in (q, k, *w)]
    outs = block.qk_norm_rope(*leaves, cos, sin, eps=0.0)
    refs = [qk_ref(wide[i], wide[2 + i], cos, sin, 0.0, False) for i in range(2)]
    tol = half_ulp(dtype) + fp32_tol(D) + 8 * half_ulp(F32)
    for o, r in zip(outs, refs):
        assert rel(o, r) <= tol
    douts = [rnd(*o.shape, seed=7 + i, dtype=dtype) for i, o in enumerate(outs)]
    for i, (g, r) in enumerate(zip(torch.autograd.grad(outs, leaves, douts), torch.autograd.grad(refs, wide, [d.double() for d in douts]))):
        n = D if i < 2 else B * T * (Hq, Hk)[i - 2]
        assert rel(g, r) <= half_ulp(dtype) + 2 * fp32_tol(D) + fp32_tol(n) + 16 * half_ulp(F32), i
    room = torch.full((B, T + 1, Hq + Hk + 1, D), 7.0, device=DEV, dtype=dtype)      # in place in wider rows: the rest stays
    room[:, :T, :Hq], room[:, :T, Hq:Hq + Hk] = q, k
    a, b = room[:, :T, :Hq], room[:, :T, Hq:Hq + Hk]
    block.qk_norm_rope(a, b, *w, cos, sin, eps=0.0, out=(a, b))
    assert torch.equal(a, outs[0]) and torch.equal(b, outs[1]) and (room[:, T:] == 7).all() and (room[:, :, Hq + Hk:] == 7).all()


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('B,Tq,Tk,H,Hk,D,Dv,causal', [
    (2, 1, 33, 64, 1, 128, 256, False), (1, 3, 65, 64, 1, 8, 8, True), (1, 32, 32, 1, 1, 64, 128, True), (1, 33, 257, 1, 1, 64, 128, True),
    (5, 1, 255, 3, 3, 32, 64, False), (5, 1, 256, 3, 3, 32, 64, False), (2, 1, 513, 3, 3, 32, 256, False), (1, 1, 20000, 2, 1, 16, 24, False),
    (1, 8, 1000, 8, 2, 128, 8, True), (40, 1, 300, 8, 8, 40, 72, False),
    (1, 1, 40000, 3, 1, 64, 120, False), (1, 17, 5000, 1, 1, 32, 64, True), (2, 16, 2049, 2, 1, 128, 256, True),
])
def test_differential_attention_sizes(B, Tq, Tk, H, Hk, D, Dv, causal, dtype):
    q, k, v = rnd(B, Tq, H, 2 * D, seed=1, dtype=dtype), rnd(B, Tk, Hk, 2 * D, seed=2, dtype=dtype), rnd(B, Tk, Hk, Dv, seed=3, dtype=dtype)
    lams = [rnd(D, seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
    leaves = [t.clone().requires_grad_() for t in (q, k, v, *lams)]
    out = block.differential_attention(*leaves, causal=causal)
    dout = rnd(B, Tq, H, Dv, seed=9, dtype=dtype)
    u = half_ulp(BF) if dtype == BF else 0.0
    (ref, err), grads = diff_ref(*(t.double() for t in (q, k, v)), [t.double() for t in lams], 0.8, D ** -0.5, (Tk,) * B, causal, u, dout.double())
    assert within(out, ref, err, dtype)
    for i, (g, (r, e)) in enumerate(zip(torch.autograd.grad(out, leaves, dout), grads)):
        assert within(g, r, e, dtype), i


def test_differential_attention_scores_of_every_size():
    """Scores that grow, fall and jump along the keys by hundreds: the running reference moves late, early and never."""
    D, Tk = 32, 700
    for dtype in (BF, F32):
        for Tq in (1, 40):
            for ramp in (torch.linspace(-60, 60, Tk), torch.linspace(60, -60, Tk), (torch.arange(Tk) % 97 == 96) * 200.0, torch.full((Tk,), -300.0)):
                q = torch.zeros(1, Tq, 1, 2 * D, device=DEV, dtype=dtype)
                q[..., 0] = q[..., D] = 1
                k = rnd(1, Tk, 1, 2 * D, seed=1, dtype=dtype, scale=0.1)
                k[0, :, 0, 0] = ramp.to(DEV).to(dtype)
                k[0, :, 0, D] = ramp.flip(0).to(DEV).to(dtype)
                v = rnd(1, Tk, 1, 2 * D, seed=2, dtype=dtype)
                lams = [rnd(D, seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
                o = block.differential_attention(q, k, v, *lams, scale=1.0)
                (ref, err), _ = diff_ref(*(t.double() for t in (q, k, v)), [t.double() for t in lams], 0.8, 1.0, (Tk,), False, half_ulp(BF) if dtype == BF else 0.0)
                assert within(o, ref, err, dtype), (dtype, Tq, rel(o, ref), err.norm() / ref.norm())


def test_differential_attention_bad_numbers_stay_in_their_row():
    """A NaN or infinite query spoils its own row, NaN keys and values past a sequence's length none."""
    for dtype in (BF, F32):
        q, k, v = (rnd(1, 80, 1, 64, seed=i, dtype=dtype) for i in range(3))
        lams = [rnd(32, seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
        good = block.differential_attention(q, k, v, *lams, causal=True)
        q2, v2 = q.clone(), v.clone()
        q2[0, 5, 0, 3] = math.nan
        q2[0, 9, 0, 40] = math.inf
        o = block.differential_attention(q2, k, v, *lams, causal=True)
        rest = [t for t in range(80) if t not in (5, 9)]
        assert torch.equal(o[0, rest], good[0, rest]) and torch.isnan(o[0, 5]).all() and torch.isnan(o[0, 9]).all()
        v2[0, 70:] = math.nan
        k2 = k.clone()
        k2[0, 70:] = math.nan
        o = block.differential_attention(q, k2, v2, *lams, key_lengths=torch.tensor([70], device=DEV))
        assert torch.equal(o, block.differential_attention(q, k, v, *lams, key_lengths=torch.tensor([70], device=DEV)))


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('M', [1, 2, 15, 16, 17, 31, 32, 33])
@pytest.mark.parametrize('C,F', [(8, 4104), (2048, 72), (2056, 2056), (136, 520)])
def test_feed_forward_of_few_rows(M, C, F, dtype):
    x, w_in, w_out = rnd(M, C, seed=1, dtype=dtype), rnd(2 * F, C, seed=2, dtype=dtype, scale=C ** -0.5), rnd(C, F, seed=3, dtype=dtype, scale=F ** -0.5)
    b_in, b_out, res = rnd(2 * F, seed=4, dtype=dtype, scale=0.3), rnd(C, seed=5, dtype=dtype, scale=0.3), rnd(M, C, seed=6, dtype=dtype)
    y = block.gated_feed_forward(x, w_in, w_out, b_in, b_out, res, 'gelu_tanh')
    ref = ffn_ref(*(t.double() for t in (x, w_in, w_out, b_in, b_out, res)), 'gelu_tanh')
    assert rel(y, ref) <= half_ulp(dtype) * (2 if dtype == BF else 1) + fp32_tol(C) + fp32_tol(F) + 16 * half_ulp(F32)
    wide = torch.zeros(M, C + 24, device=DEV, dtype=dtype)       # rows of a wider tensor, no bias, no residual
    wide[:, 8:8 + C] = x
    assert torch.equal(block.gated_feed_forward(wide[:, 8:8 + C], w_in, w_out), block.gated_feed_forward(x, w_in, w_out))


def test_differential_attention_infinite_key_of_one_map():
    """A key that one map gives a score of -inf has no weight there and its ordinary one in the other map, alone and among many queries."""
    D, Tk = 32, 70
    for dtype in (BF, F32):
        for Tq in (1, 40):
            q, k, v = rnd(1, Tq, 2, 2 * D, seed=1, dtype=dtype), rnd(1, Tk, 2, 2 * D, seed=2, dtype=dtype), rnd(1, Tk, 2, 2 * D, seed=3, dtype=dtype)
            q[..., 0], q[..., D] = 1, 1
            k[0, 33, :, D], k[0, 5, :, 0] = -math.inf, -math.inf
            lams = [rnd(D, seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
            o = block.differential_attention(q, k, v, *lams)
            (ref, err), _ = diff_ref(*(t.double() for t in (q, k, v)), [t.double() for t in lams], 0.8, D ** -0.5, (Tk,), False, half_ulp(BF) if dtype == BF else 0.0)
            assert torch.isfinite(ref).all() and within(o, ref, err, dtype)


def test_feed_forward_bad_numbers_stay_in_their_row():
    for M in (3, 40, 300):
        for dtype in (BF, F32):
            x, w_in, w_out = rnd(M, 72, seed=1, dtype=dtype), rnd(2 * 104, 72, seed=2, dtype=dtype, scale=0.1), rnd(72, 104, seed=3, dtype=dtype, scale=0.1)
            good = block.gated_feed_forward(x, w_in, w_out)
            x[1, 70] = math.nan
            x[M - 1, 0] = math.inf
            y = block.gated_feed_forward(x, w_in, w_out)
            rest = [m for m in range(M) if m not in (1, M - 1)]
            assert torch.equal(y[rest], good[rest]) and torch.isnan(y[1]).all() and not torch.isfinite(y[M - 1]).any()


# ------------------------------------------------------------------------------------------------------------ refusals
def test_calls_refuse_on_the_gpu():
    q = rnd(2, 5, 3, 16)
    with pytest.raises(TypeError, match='one dtype'):
        block.qk_norm_rope(q, q.to(BF))
    with pytest.raises(TypeError, match='float32 or bfloat16'):
        block.qk_norm_rope(q.half(), q.half())
    with pytest.raises(ValueError, match='lives on'):
        block.qk_norm_rope(q, q.cpu())
    with pytest.raises(ValueError, match='live on'):
        block.qk_norm_rope(q, q, None, None, torch.ones(5, 8), torch.ones(5, 8))
    with pytest.raises(ValueError, match='no gradient'):
        block.qk_norm_rope(q.clone().requires_grad_(), q, out=(q.clone(), q.clone()))
    k = q.clone()
    for out in ((k, q), (q.clone().expand(2, 5, 3, 16), q), ((o := q.clone()), o), (q[:1].expand(2, 5, 3, 16), k), (q.transpose(-1, -2), k)):
        with pytest.raises(ValueError):
            block.qk_norm_rope(q, k, out=out)
    a, b, c = rnd(2, 5, 4, 32), rnd(2, 7, 2, 32), rnd(2, 7, 2, 24)
    lams = [rnd(16, seed=i) for i in range(4)]
    with pytest.raises(TypeError, match='one dtype'):
        block.differential_attention(a, b, c.to(BF), *lams)
    with pytest.raises(ValueError, match='lives on'):
        block.differential_attention(a, b, c, lams[0].cpu(), *lams[1:])
    with pytest.raises(ValueError, match='key_lengths'):
        block.differential_attention(a, b, c, *lams, key_lengths=torch.tensor([1, 2]))
    with pytest.raises(TypeError, match='one dtype'):
        block.gated_feed_forward(rnd(3, 16), rnd(48, 16, dtype=BF), rnd(16, 24))
    with pytest.raises(RuntimeError):                              # differentiable once
        t = rnd(3, 16).requires_grad_()
        g, = torch.autograd.grad(block.gated_feed_forward(t, rnd(48, 16, seed=1), rnd(16, 24, seed=2)).sum(), t, create_graph=True)
        g.sum().backward()


def test_differential_attention_without_keys_ignores_its_queries():
    lams = [rnd(8, seed=i) for i in range(4)]
    q = torch.full((2, 3, 2, 16), math.inf, device=DEV).requires_grad_()
    o = block.differential_attention(q, torch.empty(2, 0, 2, 16, device=DEV), torch.empty(2, 0, 2, 16, device=DEV), *lams)
    assert (o == 0).all() and (torch.autograd.grad(o.sum(), q)[0] == 0).all()


# ---------------------------------------------------------------------------------------------------------- many short sequences
def test_differential_attention_of_more_than_2_20_short_sequences():
    """Windows: 2^20 + 8 (sequence, key head)s of three tokens.  The first and the last sequences against the definition, the vectors'
    gradients against the sum over all of them."""
    B, T, H, D, Dv = (1 << 17) + 1, 3, 8, 8, 16
    g = torch.Generator(DEV).manual_seed(1)
    q, k, v, dout = (torch.randn(B, T, H, n, device=DEV, generator=g).to(BF) for n in (2 * D, 2 * D, Dv, Dv))
    lams = [rnd(D, seed=4 + i, dtype=BF, scale=0.2) for i in range(4)]
    leaves = [t.requires_grad_() for t in (q, k, v, *lams)]
    out = block.differential_attention(*leaves, causal=True)
    grads = torch.autograd.grad(out, leaves, dout)
    wide = [t.detach().double() for t in lams]
    for s in (slice(0, 20), slice(B - 20, B)):
        (ref, err), want = diff_ref(*(t.detach()[s].double() for t in (q, k, v)), wide, 0.8, D ** -0.5, (T,) * 20, True, half_ulp(BF), dout[s].double())
        assert within(out[s], ref, err, BF)
        for got, (r, e) in zip(grads[:3], want):
            assert within(got[s], r, e, BF)
    a, b, vv, do = (t.detach().double().transpose(1, 2) for t in (q[..., D:], k[..., D:], v, dout))
    x = (a @ b.transpose(-1, -2).contiguous()) * D ** -0.5
    smax = x.abs().max().item()
    p2 = torch.softmax(x.masked_fill(torch.ones(T, T, dtype=torch.bool, device=DEV).triu(1), -math.inf), -1)
    terms = p2 * (do @ vv.transpose(-1, -2).contiguous())
    # dlam = -sum P2 dP: P2 off by eps (as in diff_ref), dP by its sum over Dv channels, then fp32 sums whose longest chain is one of
    # 1024 threads over four waves' partials of every (sequence, head)
    eps = (smax + 8) * 4 * half_ulp(F32) * math.sqrt(D)
    size = (p2 * (do.abs() @ vv.abs().transpose(-1, -2).contiguous())).sum()
    e_lam = (eps + 4 * math.sqrt(Dv) * half_ulp(F32) + fp32_tol(4 * B * H / 1024 + 100)) * size
    x1, x2 = (wide[0] * wide[1]).sum().exp(), (wide[2] * wide[3]).sum().exp()
    for got, val, o in zip(grads[3:], (x1, x1, -x2, -x2), (wide[1], wide[0], wide[3], wide[2])):
        assert within(got, -terms.sum() * val * o, e_lam * val.abs() * o.abs(), BF)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('B,T,H,Hk,D,Dv', [(2, 70, 2, 2, 32, 64), (2, 300, 2, 1, 64, 128), (1, 40, 1, 1, 128, 256), (1, 2000, 1, 1, 64, 128), (48, 600, 8, 8, 40, 64)])
def test_gradients_past_a_sequences_end_are_zero_whatever_the_queries_hold(B, T, H, Hk, D, Dv, dtype):
    """Keys behind a sequence's end take no part: their gradients are zero beside NaN and infinite queries and output gradients too, the
    other queries' are right, and another sequence's are as they were."""
    q, k, v = rnd(B, T, H, 2 * D, seed=1, dtype=dtype), rnd(B, T, Hk, 2 * D, seed=2, dtype=dtype), rnd(B, T, Hk, Dv, seed=3, dtype=dtype)
    lams = [rnd(D, seed=4 + i, dtype=dtype, scale=0.2) for i in range(4)]
    dout = rnd(B, T, H, Dv, seed=9, dtype=dtype)
    n = T // 2 + 3
    ln = torch.tensor([n] * B, device=DEV)

    def grads(q, dout):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, *lams)]
        return torch.autograd.grad(block.differential_attention(*leaves, key_lengths=ln), leaves, dout)

    good = grads(q, dout)
    _, want = diff_ref(*(t[:1].double() for t in (q, k, v)), [t.double() for t in lams], 0.8, D ** -0.5, (n,), False, half_ulp(BF) if dtype == BF else 0.0, dout[:1].double())
    for bad in ('query', 'gradient'):
        q2, d2 = q.clone(), dout.clone()
        (q2 if bad == 'query' else d2)[0, 5, 0, 3] = math.nan
        (q2 if bad == 'query' else d2)[0, 9, 0, 7] = math.inf
        dq, dk, dv, *_ = grads(q2, d2)
        assert (dk[:, n:] == 0).all() and (dv[:, n:] == 0).all(), bad
        assert torch.isnan(dk[0, :n]).any() and torch.isnan(dq[0, 5, 0]).any()
        rest = [t for t in range(T) if t not in (5, 9)]
        # other rows of the wave may take another reference for their weights, so they agree within their own bounds
        assert within(dq[:1, rest], want[0][0][:, rest], want[0][1][:, rest], dtype)
        for a, b in zip((dq, dk, dv), good):
            assert torch.equal(a[1:], b[1:])


# ----------------------------------------------------------------------------------------------------------- partial gradients
def subsets(names):
    """Each argument alone, all but each, and the weights or the activations frozen."""
    return [[n] for n in names] + [[m for m in names if m != n] for n in names] + [[n for n in names if 'w' in n or 'b' in n], names[:1] + names[-1:]]


def check_subsets(fn, tensors, dout):
    """Gradients of some arguments are those of the call in which all require one, to the bit."""
    names = list(tensors)

    def grads(need):
        leaves = {n: t.detach().clone().requires_grad_(n in need) for n, t in tensors.items()}
        out = outputs(fn(**leaves))
        return dict(zip(need, torch.autograd.grad(out, [leaves[n] for n in need], dout)))

    whole = grads(names)
    for need in subsets(names):
        if need:
            for n, g in grads(need).items():
                assert torch.equal(g, whole[n]), (need, n)


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('M,C,F', [(3, 72, 136), (300, 136, 264), (2100, 264, 680)])
def test_some_gradients_of_the_feed_forward(M, C, F, dtype):
    t = dict(x=rnd(M, C, seed=1, dtype=dtype), w_in=rnd(2 * F, C, seed=2, dtype=dtype, scale=C ** -0.5), w_out=rnd(C, F, seed=3, dtype=dtype, scale=F ** -0.5),
             b_in=rnd(2 * F, seed=4, dtype=dtype, scale=0.3), b_out=rnd(C, seed=5, dtype=dtype, scale=0.3), residual=rnd(M, C, seed=6, dtype=dtype))
    dy = rnd(M, C, seed=9, dtype=dtype)
    check_subsets(lambda **a: block.gated_feed_forward(**a, activation='gelu'), t, [dy])
    t.pop('b_in')                                              # one bias of the two
    check_subsets(block.gated_feed_forward, t, [dy])
    t.pop('b_out')
    check_subsets(block.gated_feed_forward, t, [dy])


@pytest.mark.parametrize('dtype', [BF, F32])
@pytest.mark.parametrize('D,Dv', [(32, 64), (64, 128), (128, 256)])
def test_some_gradients_of_the_attention_and_the_norm(D, Dv, dtype):
    B, T, H = 2, 90, 2
    t = dict(q=rnd(B, T, H, 2 * D, seed=1, dtype=dtype), k=rnd(B, T, 1, 2 * D, seed=2, dtype=dtype), v=rnd(B, T, 1, Dv, seed=3, dtype=dtype))
    t.update({n: rnd(D, seed=4 + i, dtype=dtype, scale=0.2) for i, n in enumerate(block._LAMBDAS)})
    check_subsets(lambda **a: block.differential_attention(**a, causal=True), t, [rnd(B, T, H, Dv, seed=9, dtype=dtype)])
    cos, sin = block.rotary_table(torch.arange(T, device=DEV), D)
    t = dict(q=t['q'], k=t['k'], q_weight=rnd(2 * D, seed=8, dtype=dtype), k_weight=rnd(2 * D, seed=10, dtype=dtype))
    check_subsets(lambda **a: block.qk_norm_rope(**a, cos=cos, sin=sin), t, [rnd(B, T, H, 2 * D, seed=11, dtype=dtype), rnd(B, T, 1, 2 * D, seed=12, dtype=dtype)])


@pytest.mark.parametrize('dtype', [torch.int32, torch.int64])
@pytest.mark.parametrize('Tq,causal', [(1, False), (3, True), (60, True)])
def test_a_captured_step_follows_its_lengths(Tq, causal, dtype):
    """A decode step captured once and replayed while the cache fills: lengths, queries and one slot of the cache change in place."""
    B, H, Hk, D, room = 3, 4, 2, 32, 700
    q, k, v = rnd(B, Tq, H, 2 * D, seed=1, dtype=BF), rnd(B, room, Hk, 2 * D, seed=2, dtype=BF), rnd(B, room, Hk, 2 * D, seed=3, dtype=BF)
    lams = [rnd(D, seed=30 + i, dtype=BF, scale=0.2) for i in range(4)]
    ln = torch.zeros(B, dtype=dtype, device=DEV)
    call = lambda: block.differential_attention(q, k, v, *lams, key_lengths=ln, causal=causal)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step, lens in enumerate(((0, 1, 2), (700, 699, 33), (64, 65, 0), (900, -3, 350), (1, 1, 1))):
        ln.copy_(torch.tensor(lens))
        q.copy_(rnd(*q.shape, seed=10 + step, dtype=BF))
        k[:, 5 * step] = rnd(B, Hk, 2 * D, seed=20 + step, dtype=BF)
        out.fill_(math.nan)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
        held = [min(max(n, 0), room) for n in lens]
        (ref, err), _ = diff_ref(q.double(), k.double(), v.double(), [t.double() for t in lams], 0.8, D ** -0.5, held, causal, half_ulp(BF))
        assert within(out, ref, err, BF), step
