"""nicediffusion.block as autograd sees its calls, without a GPU: the launch is replaced by a record of its arguments."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from nicediffusion import _hip, block

T4 = (2, 5, 3, 16)


@pytest.fixture
def launches(monkeypatch):
    """Calls go through to the launch, which notes its name and arguments instead."""
    made = []
    monkeypatch.setattr(_hip, 'require_device', lambda t, what='tensor': None)
    monkeypatch.setattr(_hip, 'require_gfx950', lambda index: None)
    monkeypatch.setattr(block, '_call', lambda name, device, *args: made.append((name, args)))
    return made


def r(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape)))


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
QK = dict(q=r(*T4), k=r(*T4), q_weight=r(16), k_weight=r(16))
DIFF = dict(q=r(2, 5, 4, 32), k=r(2, 7, 2, 32), v=r(2, 7, 2, 24), lambda_q1=r(16), lambda_k1=r(16), lambda_q2=r(16), lambda_k2=r(16))
FFN = dict(x=r(3, 16), w_in=r(48, 16), w_out=r(16, 24), b_in=r(48), b_out=r(16), residual=r(3, 16))
EACH = [(f, d, n) for f, d in ((block.qk_norm_rope, QK), (block.differential_attention, DIFF), (block.gated_feed_forward, FFN)) for n in d]


@pytest.mark.parametrize('fn,tensors,name', EACH, ids=['{}-{}'.format(f.__name__, n) for f, _, n in EACH])
@pytest.mark.parametrize('grad', [False, True])
def test_a_forward_mode_tangent_is_refused(launches, fn, tensors, name, grad):
    """The operators have no forward-mode derivative: a tangent would be lost, that is, taken for zero."""
    fn(**tensors)
    assert launches
    launches.clear()
    with fwd.dual_level():
        given = dict(tensors, **{name: fwd.make_dual(tensors[name], torch.ones_like(tensors[name]))})
        if grad:
            given = {n: t.requires_grad_() if n != name and t.is_leaf else t for n, t in ((n, t if n == name else t.clone()) for n, t in given.items())}
        with pytest.raises(NotImplementedError, match='forward-mode'):
            fn(**given)
        with torch.no_grad(), pytest.raises(NotImplementedError, match='forward-mode'):
            fn(**given)
        fn(**tensors)                                          # a level that is open is no tangent
    assert len(launches) == 1
    fn(**tensors)


def test_a_forward_mode_tangent_is_refused_for_tables_out_and_empty_calls(launches):
    cos, sin = r(5, 8), r(5, 8)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for kw in (dict(cos=dual(cos), sin=sin), dict(cos=cos, sin=dual(sin)), dict(out=(dual(r(*T4)), r(*T4))), dict(out=(r(*T4), dual(r(*T4))))):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                block.qk_norm_rope(r(*T4), r(*T4), **kw)
        with pytest.raises(NotImplementedError, match='forward-mode'):
            block.qk_norm_rope(dual(r(2, 0, 3, 16)), r(2, 0, 3, 16))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            block.differential_attention(**dict(DIFF, q=dual(r(2, 0, 4, 32))))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            block.gated_feed_forward(dual(r(0, 16)), r(48, 16), r(16, 24))
    assert not launches


# ------------------------------------------------------------------------------------------------------- writing into out=
def test_out_is_a_write_that_autograd_sees(launches):
    """A graph that saved the memory cannot be run backward over what was written there, as after any in-place operation."""
    x = r(2, 5, 9 * 16).requires_grad_()
    row = torch.tanh(x)                                        # saved for its own backward
    q, k = row[..., :48].view(*T4), row[..., 48:96].view(*T4)
    with torch.no_grad():
        block.qk_norm_rope(q, k, out=(q, k))
    assert len(launches) == 1
    with pytest.raises(RuntimeError, match='inplace operation'):
        row.sum().backward()
    x, cache = r(*T4).requires_grad_(), r(2, 8, 3, 16)         # a slot of a cache that a product saved
    y = x * cache[:, :5]
    with torch.no_grad():
        block.qk_norm_rope(r(*T4), r(*T4), out=(r(*T4), cache[:, 3:8]))
    with pytest.raises(RuntimeError, match='inplace operation'):
        y.sum().backward()


def test_out_counts_each_output_once_per_call_and_skips_what_has_no_counter(launches):
    a, b = r(*T4), r(*T4)
    va, vb = a._version, b._version
    block.qk_norm_rope(r(*T4), r(*T4), out=(a, b))
    assert (a._version, b._version) == (va + 1, vb + 1)
    with torch.inference_mode():
        block.qk_norm_rope(r(*T4), r(*T4), out=(torch.empty(T4), torch.empty(T4)))
    block.qk_norm_rope(r(2, 0, 3, 16), r(2, 0, 3, 16), out=(r(2, 0, 3, 16), r(2, 0, 3, 16)))
    assert len(launches) == 2


def test_out_that_requires_a_gradient_is_refused_in_grad_mode(launches):
    """As torch's own out=: the write would leave the tensor's history as it was."""
    leaf, row = r(*T4).requires_grad_(), torch.tanh(r(2, 5, 9 * 16).requires_grad_())
    part = row[..., :48].view(*T4)
    for i, out in enumerate(((leaf, r(*T4)), (r(*T4), leaf), (part, r(*T4)), (r(*T4), part))):
        with pytest.raises(ValueError, match=r'out\[{}\] requires a gradient'.format(i % 2)):
            block.qk_norm_rope(r(*T4), r(*T4), out=out)
    assert not launches
    with torch.no_grad():                                      # a parameter that is set outside of any graph
        block.qk_norm_rope(r(*T4), r(*T4), out=(leaf, r(*T4)))
    assert len(launches) == 1 and leaf._version == 1


# ------------------------------------------------------------------------------------------------ what the library refuses
@pytest.fixture
def no_device(monkeypatch):
    """Calls reach the library itself, which refuses them before any launch."""
    monkeypatch.setattr(_hip, 'require_device', lambda t, what='tensor': None)
    monkeypatch.setattr(_hip, 'require_gfx950', lambda index: None)
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: None)
    monkeypatch.setattr(block, '_stream', lambda index: None)


def test_what_the_library_refuses_is_a_value_error(no_device):
    """Sizes that only the library looks at: a ValueError like every other wrong shape, and still an NdHipError."""
    heads = (1 << 18) + 8                                      # a token's heads of 16 channels: more than 2^22 elements
    q, v = torch.zeros(1, 2, heads, 16), torch.zeros(1, 2, heads, 8)
    with pytest.raises(ValueError, match='token stride') as e:
        block.differential_attention(q, q, v, r(8), r(8), r(8), r(8))
    assert isinstance(e.value, _hip.NdHipError)
    with pytest.raises(ValueError):
        _hip.check_block(-1, 'a call')
    with pytest.raises(_hip.NdHipError) as e:                  # a failed launch is no wrong argument
        _hip.check_block(-2, 'a call')
    assert not isinstance(e.value, ValueError)
    _hip.check_block(0)


def touched(base, strides, heads, B, T, D):
    """The element addresses of a [B, T, heads, D] tensor, one set per row."""
    sb, st, sh = strides
    return [set(range(base + b * sb + t * st + h * sh, base + b * sb + t * st + h * sh + D)) for b in range(B) for t in range(T) for h in range(heads)]


def test_rows_overlap_against_every_address():
    """nd_rows_overlap against the sets of addresses themselves: views of packed rows, slots, repeats and strides at random; where two
    layouts that interleave have different strides it may say yes without need, never no."""
    import random
    lib, rng, es, far = _hip.load_block(), random.Random(1), 4, 1 << 20
    seen = {(w, g): 0 for w in (0, 1) for g in (0, 1)}
    for n in range(6000):
        B, T, D = rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 4)
        Ha, Hb = rng.randint(1, 3), rng.randint(1, 3)
        sh = rng.choice([D, D, D + 1, 2 * D, 3 * D])
        st = rng.choice([3 * sh, 4 * sh, 6 * sh, sh * max(Ha, Hb) + rng.randint(0, 5), rng.randint(0, 30)])
        sb = rng.choice([T * st, (T + 2) * st, 0, rng.randint(0, 90)])
        same = rng.random() < 0.8
        sa = (sb, st, sh)
        sb2 = sa if same else (rng.randint(0, 90), rng.randint(0, 30), rng.choice([D, 2 * D]))
        off = rng.choice([0, D, Ha * sh, st, rng.randint(0, 60), rng.randint(0, 400)])
        a, b = touched(0, sa, Ha, B, T, D), touched(off, sb2, Hb, B, T, D)
        want = int(bool(set().union(*a) & set().union(*b)))
        got = lib.nd_rows_overlap(far, *sa, Ha, far + off * es, *sb2, Hb, B, T, D, es)
        assert got == lib.nd_rows_overlap(far + off * es, *sb2, Hb, far, *sa, Ha, B, T, D, es)
        assert got >= want, (sa, sb2, Ha, Hb, B, T, D, off)
        if same:
            assert got == want, (sa, Ha, Hb, B, T, D, off)
        seen[want, got] += 1
        alone = int(sum(len(s) for s in a) != len(set().union(*a)))        # rows of one tensor that meet each other
        assert lib.nd_rows_overlap(far, *sa, Ha, None, 0, 0, 0, 0, B, T, D, es) == alone, (sa, Ha, B, T, D)
    assert seen[0, 0] > 500 and seen[1, 1] > 500


def test_out_that_overlaps_is_refused(no_device):
    """Neither a shifted view of the inputs' rows nor one of the other input, a weight, a table or the other output may be written."""
    base, fresh, fresh2 = r(2, 9, 9, 16), r(*T4), r(*T4)
    part = lambda h, t=0: base[:, t:t + 5, h:h + 3]  # noqa: E731
    q, k = part(0), part(3)
    halves = base.flatten()[8:8 + 5 * 144 + 9 * 144].as_strided(T4, (9 * 144, 144, 16, 1))      # half a head further
    for out in ((part(1), fresh), (part(0, 1), part(3)), (q, part(4)), (part(2), k), (fresh, part(2)), (q, part(1)), (part(5), part(6)), (part(4), fresh),
                (halves, fresh), (fresh, part(0)), (part(3, 1), fresh)):
        with pytest.raises(ValueError, match='overlap'):
            block.qk_norm_rope(q, k, out=out)
    with pytest.raises(ValueError, match='overlap'):           # rows that meet each other
        block.qk_norm_rope(q, k, out=(torch.as_strided(r(2000), T4, (240, 48, 8, 1)), fresh))
    weight, flat = fresh[1, 2, 1], torch.cat([r(5, 8).flatten(), r(440)])
    table = flat.as_strided((5, 8), (8, 1))
    for kw, out in ((dict(q_weight=weight), (fresh, fresh2)), (dict(k_weight=weight), (fresh, fresh2)), (dict(cos=table, sin=r(5, 8)), (fresh, flat.view(T4))),
                    (dict(cos=r(5, 8), sin=table), (flat.view(T4), fresh))):
        with pytest.raises(ValueError, match='overlap'):
            block.qk_norm_rope(q, k, out=out, **kw)


def test_layouts_that_only_interleave_do_not_overlap():
    """The q and k columns of one packed row, per-head q | k | v, a cache slot beside others, a batch of one."""
    lib, D, es, far = _hip.load_block(), 16, 2, 1 << 20
    at = lambda i: far + i * es  # noqa: E731
    row = (7 * 144, 144, D)
    assert lib.nd_rows_overlap(at(0), *row, 3, at(3 * D), *row, 3, 2, 7, D, es) == 0
    assert lib.nd_rows_overlap(at(0), *row, 5, at(5 * D), *row, 2, 2, 7, D, es) == 0
    assert lib.nd_rows_overlap(at(0), *row, 5, at(4 * D), *row, 2, 2, 7, D, es) == 1
    assert lib.nd_rows_overlap(at(0), 7 * 144, 144, 3 * D, 3, at(D), 7 * 144, 144, 3 * D, 3, 2, 7, D, es) == 0
    assert lib.nd_rows_overlap(at(0), 0, 144, 0, 1, at(D), 0, 144, D, 4, 1, 7, D, es) == 0           # strides that say nothing are 0
    slot = (50 * 2 * D, 2 * D, D)
    assert lib.nd_rows_overlap(at(4 * 2 * D), *slot, 2, at(5 * 2 * D), *slot, 2, 3, 1, D, es) == 0
    assert lib.nd_rows_overlap(at(4 * 2 * D), *slot, 2, at(5 * 2 * D), *slot, 2, 3, 2, D, es) == 1
    assert lib.nd_rows_overlap(at(0), 1 << 40, 1 << 30, D, 3, at(3 * D), 1 << 40, 1 << 30, D, 3, 64, 512, D, es) == 0
    assert lib.nd_rows_overlap(at(0), -7 * 144, 144, D, 3, at(-7 * 144), 0, 144, D, 3, 2, 7, D, es) == 1      # a negative stride


# --------------------------------------------------------------------------------------------------------- partial gradients
def test_the_feed_forward_holds_only_what_its_gradients_need(launches):
    """Frozen weights, a bias alone: the pre-activations serve dx, dw_in and db_in, the hidden rows dw_out, and nothing the others."""
    names = list(FFN)
    for need, au, h in ((('x',), 1, 0), (('w_in',), 1, 0), (('b_in',), 1, 0), (('w_out',), 0, 1), (('b_out',), 0, 0), (('residual',), 0, 0), (names, 1, 1)):
        launches.clear()
        given = {n: t.clone().requires_grad_(n in need) for n, t in FFN.items()}
        y = block.gated_feed_forward(**given)
        (name, args), = launches
        assert name == 'nd_gated_ffn' and (args[11] != 0) == bool(au)
        saved = y.grad_fn.saved_tensors
        assert (saved[3] is not None) == bool(h) and (saved[4] is not None) == bool(au)
        grads = torch.autograd.grad(y, [given[n] for n in need], torch.ones_like(y))
        assert all(g.shape == given[n].shape for g, n in zip(grads, need))
        assert len(launches) == (1 if need == ('residual',) else 2)


# ----------------------------------------------------------------------------------------------------- functional transforms
@pytest.mark.parametrize('fn,tensors', [(block.qk_norm_rope, QK), (block.differential_attention, DIFF), (block.gated_feed_forward, FFN)])
def test_functional_transforms_end_in_an_error(monkeypatch, no_device, fn, tensors):
    """vmap, grad and jvp wrap the tensors, and a wrapper has no memory to launch on: no transform returns a result."""
    def launched(name, device, *args):
        raise AssertionError('launched')
    monkeypatch.setattr(block, '_call', launched)
    first = next(iter(tensors))
    rest = {n: t for n, t in tensors.items() if n != first}
    call = lambda t: (lambda o: (o[0] if isinstance(o, tuple) else o).sum())(fn(**{first: t}, **rest))  # noqa: E731
    for run in (lambda: torch.func.vmap(call)(torch.stack([tensors[first]] * 2)), lambda: torch.func.grad(call)(tensors[first]),
                lambda: torch.func.jvp(call, (tensors[first],), (torch.ones_like(tensors[first]),)), lambda: torch.func.vjp(call, tensors[first])[1](torch.ones(()))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            run()


def test_gradients_of_empty_calls(launches):
    """No rows: zero gradients of every weight, nothing launched."""
    q, k = r(2, 0, 3, 16).requires_grad_(), r(2, 0, 1, 16).requires_grad_()
    w = [r(16).requires_grad_() for _ in range(2)]
    o = block.qk_norm_rope(q, k, *w, cos=r(0, 8), sin=r(0, 8))
    g = torch.autograd.grad(o, (q, k, *w), [torch.empty_like(t) for t in o])
    assert g[0].shape == q.shape and g[1].shape == k.shape and all((t == 0).all() for t in g[2:])
    given = {n: t.clone().requires_grad_() for n, t in FFN.items() if n not in ('x', 'residual')}
    x = r(2, 0, 16).requires_grad_()
    g = torch.autograd.grad(block.gated_feed_forward(x, **given), (x, *given.values()), torch.empty(2, 0, 16))
    assert g[0].shape == x.shape and all((t == 0).all() for t in g[1:]) and not launches
