"""nicediffusion.block and libnd_block.so without a GPU: the ABI table, what calls refuse, the position tables."""
import glob
import hashlib
import math
import os
import re

import pytest
import torch

from nicediffusion import _hip, block

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF = torch.float32, torch.bfloat16


# ------------------------------------------------------------------------------------------------------------- C ABI
def test_block_library_exports_every_header_symbol():
    src = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'nd_block.h')).read(), flags=re.S)
    names = sorted(set(re.findall(r'\b(nd_[a-z0-9_]+)\s*\(', src)))
    assert names == sorted(_hip.BLOCK_SIGNATURES)
    lib = _hip.load_block()
    for n in names:
        assert hasattr(lib, n), n
        proto = re.search(r'\b' + n + r'\s*\(([^)]*)\)', src).group(1)
        want = 0 if proto.strip() == 'void' else proto.count(',') + 1
        assert len(_hip.BLOCK_SIGNATURES[n][0]) == want, n


def test_block_library_is_built_from_the_sources_in_the_tree():
    pkg = os.path.join(ROOT, 'nice-diffusion_amd')
    files = sorted(f for ext in ('*.hip', '*.h') for f in glob.glob(os.path.join(pkg, 'csrc', 'block', ext)))
    files = [os.path.join(ROOT, 'include', n) for n in ('nd_block.h', 'nd_hip.h')] + files
    got = _hip.load_block().nd_block_build_id().decode()
    make = open(os.path.join(pkg, 'Makefile')).read()
    assert re.fullmatch(r'[0-9a-f]{16}', got) and '-packed-fp32-ops' in make
    h = hashlib.sha256()
    for f in files:
        h.update(open(f, 'rb').read())
    assert got == h.hexdigest()[:16], 'libnd_block.so was not built from the sources in the tree: make -C nice-diffusion_amd'


A = 1 << 20          # an aligned address that is never followed: every call below is refused before any launch


def qk_args(**kw):
    a = dict(q=A, qs=(640, 128, 64), k=A, ks=(640, 128, 64), qw=None, kw=None, cos=A, sin=A, tb=0, qo=A, qos=(640, 128, 64), ko=A,
             kos=(640, 128, 64), B=2, T=5, Hq=2, Hk=2, D=64, R=64, eps=1e-6, flags=0, dtype=_hip.DT_BF16)
    a.update(kw)
    return (a['q'], *a['qs'], a['k'], *a['ks'], a['qw'], a['kw'], a['cos'], a['sin'], a['tb'], a['qo'], *a['qos'], a['ko'], *a['kos'], a['B'],
            a['T'], a['Hq'], a['Hk'], a['D'], a['R'], a['eps'], a['flags'], a['dtype'], None)


def refused(fn, args, what):
    lib = _hip.load_block()
    assert getattr(lib, fn)(*args) == -1 and re.search(what, lib.nd_block_last_error().decode()), lib.nd_block_last_error()
    with pytest.raises(_hip.NdHipError, match=what):
        _hip.check_block(-1, fn)


@pytest.mark.parametrize('kw,what', [
    (dict(B=0), 'positive'), (dict(Hk=-1), 'positive'), (dict(D=63), 'even'), (dict(D=514), '512'), (dict(R=66), 'rotated'), (dict(R=7), 'rotated'),
    (dict(cos=None), 'tables'), (dict(dtype=7), 'dtype'), (dict(q=None), 'null'), (dict(ko=None), 'null'), (dict(B=1 << 20, T=1 << 20), 'rows'),
])
def test_c_qk_norm_rope_refuses(kw, what):
    refused('nd_qk_norm_rope', qk_args(**kw), what)


def diff_args(**kw):
    a = dict(q=A, qs=(640, 128, 64), k=A, ks=(640, 128, 64), v=A, vs=(640, 128, 64), lam=(A,) * 4, lsh=0, init=0.8, ln=None, out=A, o1=None, o2=None,
             lse=None, ws=A, B=2, Tq=5, Tk=5, H=2, Hk=2, D=32, Dv=64, scale=0.1, flags=0, dtype=_hip.DT_BF16)
    a.update(kw)
    return (a['q'], *a['qs'], a['k'], *a['ks'], a['v'], *a['vs'], *a['lam'], a['lsh'], a['init'], a['ln'], a['out'], a['o1'], a['o2'], a['lse'],
            a['ws'], a['B'], a['Tq'], a['Tk'], a['H'], a['Hk'], a['D'], a['Dv'], a['scale'], a['flags'], a['dtype'], None)


@pytest.mark.parametrize('kw,what', [
    (dict(Tk=0), 'positive'), (dict(H=3), 'multiple'), (dict(H=130), '64'), (dict(H=1 << 21, Hk=1 << 21), 'heads'), (dict(D=36), 'multiple of 8'), (dict(D=136), '128'), (dict(Dv=12), 'value dim'),
    (dict(Dv=264), '256'), (dict(Tq=1 << 29, H=2), 'tokens'), (dict(scale=0.0), 'scale'), (dict(scale=float('nan')), 'scale'), (dict(k=None), 'null'),
    (dict(k=A + 8), 'aligned'), (dict(vs=(640, 132, 64)), 'aligned'), (dict(qs=(640, 1 << 23, 64)), 'stride'), (dict(ks=(640, -128, 64)), 'stride'),
    (dict(lam=(A, A, None, A)), 'lambda'), (dict(out=None), 'outputs'), (dict(o1=A), 'outputs'), (dict(Tk=1 << 20, B=1, Tq=1, ws=None), 'workspace'),
    (dict(dtype=2), 'dtype'),
])
def test_c_diff_attention_refuses(kw, what):
    refused('nd_diff_attention', diff_args(**kw), what)


def ffn_args(**kw):
    a = dict(x=A, ldx=64, wi=A, bi=None, wo=A, bo=None, res=None, ldr=0, y=A, ldy=64, h=A, au=None, ws=A, M=5, C=64, F=128, act=0, dtype=_hip.DT_BF16)
    a.update(kw)
    return tuple(a[n] for n in ('x', 'ldx', 'wi', 'bi', 'wo', 'bo', 'res', 'ldr', 'y', 'ldy', 'h', 'au', 'ws', 'M', 'C', 'F', 'act', 'dtype')) + (None,)


@pytest.mark.parametrize('kw,what', [
    (dict(M=0), 'positive'), (dict(C=60), 'multiples of 8'), (dict(F=4), 'multiples of 8'), (dict(C=1 << 15, F=1 << 15, ldx=1 << 15, ldy=1 << 15), '2\\^28'),
    (dict(C=8, F=1 << 21), '2\\^20'), (dict(act=3), 'activation'), (dict(act=-1), 'activation'), (dict(dtype=5), 'dtype'), (dict(h=None), 'null'),
    (dict(ldx=56), 'shorter'), (dict(ldy=68), 'aligned'), (dict(res=A + 4, ldr=64), 'aligned'), (dict(wi=A + 2), 'aligned'),
])
def test_c_gated_ffn_refuses(kw, what):
    refused('nd_gated_ffn', ffn_args(**kw), what)


def test_c_backward_calls_refuse():
    lib = _hip.load_block()
    refused('nd_gated_ffn_bwd', (None, 64, A, 64, A, A, A, A, A, A, None, A, None, A, A, 5, 64, 128, 0, _hip.DT_F32, None), 'null')
    refused('nd_gated_ffn_bwd', (A, 64, A, 64, A, A, None, A, A, A, None, A, None, A, A, 5, 64, 128, 0, _hip.DT_F32, None), 'au')
    refused('nd_gated_ffn_bwd', (A, 64, A, 64, A, A, A, A, A, A, None, A, None, A, None, 5, 64, 128, 0, _hip.DT_F32, None), 'workspace')
    t = (A, 640, 128, 64)
    refused('nd_diff_attention_bwd', (*t, *t, *t, A, A, A, A, 0, 0.8, None, A, None, A, *t, A, A, A, None, None, None, None, A, 2, 5, 5, 2, 2, 32, 64, 0.1, 0,
                                      _hip.DT_BF16, None), 'null|missing')
    refused('nd_qk_norm_rope_bwd', (*t, *t, A, A, A, A, 0, *t, *t, *t, *t, A, None, None, 2, 5, 2, 2, 64, 64, 1e-6, 0, _hip.DT_BF16, None), 'workspace')
    assert lib.nd_diff_attention_workspace_floats(1, 1, 1, 3, 2, 32, 64, _hip.DT_BF16) < 0
    assert lib.nd_gated_ffn_workspace_floats(0, 8, 8, _hip.DT_F32) < 0 and lib.nd_gated_ffn_bwd_workspace_floats(4, 0, 8, _hip.DT_F32) < 0
    assert lib.nd_diff_attention_bwd_workspace_floats(1, 0, 1, 2, 2, 32, 64, _hip.DT_BF16) < 0


def test_packed_calls_are_the_plain_ones():
    """Same refusals through nd_block_packed; a wrong count, an unknown call and an integer too large for its type are refused."""
    lib = _hip.load_block()
    plain = {'nd_qk_norm_rope': (qk_args(D=63), 'even'), 'nd_diff_attention': (diff_args(scale=0.0), 'scale'), 'nd_gated_ffn': (ffn_args(act=3), 'activation')}
    for name, (args, what) in plain.items():
        k, pack, n = _hip.BLOCK_CALLS[name]
        words = pack.pack(*[0 if a is None else a for a in args[:-1]])
        assert len(words) == 8 * n
        assert lib.nd_block_packed(k, words, n, None) == -1 and re.search(what, lib.nd_block_last_error().decode())
        assert lib.nd_block_packed(k, words, n - 1, None) == -1 and b'number' in lib.nd_block_last_error()
    assert lib.nd_block_packed(17, words, n, None) == -1 and b'unknown' in lib.nd_block_last_error()
    k, pack, n = _hip.BLOCK_CALLS['nd_gated_ffn']
    words = pack.pack(*[0 if a is None else a for a in ffn_args(M=(1 << 32) + 5)[:-1]])
    assert lib.nd_block_packed(k, words, n, None) == -1 and b'fit' in lib.nd_block_last_error()
    header = open(os.path.join(ROOT, 'include', 'nd_block.h')).read()
    for name, (k, _, _) in _hip.BLOCK_CALLS.items():
        assert re.search(r'#define ND_CALL_{} {}\b'.format(name[3:].upper(), k), header), name


def test_workspaces_are_as_large_as_the_splits_need():
    """Divided keys and contractions: one fp32 partial row per split; nothing where the chip is full without."""
    lib = _hip.load_block()
    one = lib.nd_diff_attention_workspace_floats(1, 1, 8192, 4, 4, 64, 128, _hip.DT_BF16)
    row = 1 * 1 * 4 * (2 * 128 + 4)
    assert one > 0 and one % row == 0 and 2 <= one // row <= 64
    assert lib.nd_diff_attention_workspace_floats(64, 1024, 1024, 8, 8, 64, 128, _hip.DT_BF16) == 0
    assert lib.nd_diff_attention_workspace_floats(4, 1, 200, 4, 4, 64, 128, _hip.DT_BF16) == 0
    assert lib.nd_gated_ffn_workspace_floats(65536, 512, 1024, _hip.DT_BF16) == 0 == lib.nd_gated_ffn_workspace_floats(1, 512, 1024, _hip.DT_F32)


# ------------------------------------------------------------------------------------------------------------ Python calls
def z(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


T4 = (2, 5, 3, 16)


@pytest.mark.parametrize('args,kw,exc,what', [
    ((z(5, 3, 16), z(*T4)), {}, ValueError, 'q has shape'), ((z(*T4), z(5, 3, 16)), {}, ValueError, 'k has shape'),
    ((z(*T4), z(2, 6, 3, 16)), {}, ValueError, 'k has shape'), ((z(2, 5, 3, 15), z(2, 5, 3, 15)), {}, ValueError, 'even'),
    ((z(2, 5, 3, 514), z(2, 5, 3, 514)), {}, ValueError, '512'), ((z(2, 5, 0, 16), z(*T4)), {}, ValueError, 'head'),
    ((z(*T4), z(*T4)), {'eps': -1e-6}, ValueError, 'eps'), ((z(*T4), z(*T4)), {'eps': float('nan')}, ValueError, 'eps'),
    ((z(*T4), z(*T4), z(8)), {}, ValueError, 'q_weight'), ((z(*T4), z(*T4), None, z(1, 16)), {}, ValueError, 'k_weight'),
    ((z(*T4), z(*T4), None, None, z(5, 8)), {}, ValueError, 'together'), ((z(*T4), z(*T4), None, None, z(5, 8), z(5, 7)), {}, ValueError, 'sin'),
    ((z(*T4), z(*T4), None, None, z(4, 8), z(4, 8)), {}, ValueError, 'cos has shape'), ((z(*T4), z(*T4), None, None, z(5, 9), z(5, 9)), {}, ValueError, '18 channels'),
    ((z(*T4), z(*T4), None, None, z(3, 5, 8), z(3, 5, 8)), {}, ValueError, 'cos has shape'), ((z(*T4), z(*T4), None, None, z(5, 8, dtype=BF), z(5, 8, dtype=BF)), {}, TypeError, 'float32'),
    ((z(*T4), z(*T4), None, None, z(5, 8).requires_grad_(), z(5, 8)), {}, ValueError, 'constants'), ((z(*T4), z(*T4)), {}, _hip.NdHipError, 'no CPU'),
])
def test_qk_norm_rope_refuses(args, kw, exc, what):
    with pytest.raises(exc, match=what):
        block.qk_norm_rope(*args, **kw)


def diff_tensors(**kw):
    d = dict(q=z(2, 5, 4, 32), k=z(2, 7, 2, 32), v=z(2, 7, 2, 24), lambda_q1=z(16), lambda_k1=z(16), lambda_q2=z(16), lambda_k2=z(16))
    d.update(kw)
    return d


@pytest.mark.parametrize('kw,exc,what', [
    (dict(q=z(2, 5, 4, 33)), ValueError, 'q has shape'), (dict(q=z(5, 4, 32)), ValueError, 'q has shape'), (dict(k=z(2, 7, 32)), ValueError, 'k has shape'),
    (dict(k=z(2, 8, 2, 32)), ValueError, 'k has shape'), (dict(v=z(1, 7, 2, 24)), ValueError, 'v has shape'), (dict(lambda_q1=z(8)), ValueError, 'lambda_q1'),
    (dict(lambda_k2=z(4, 16)), ValueError, 'lambda_k2'), (dict(q=z(2, 5, 4, 24), k=z(2, 7, 2, 24), **{n: z(12) for n in block._LAMBDAS}), ValueError, 'multiples of 8'),
    (dict(v=z(2, 7, 2, 20)), ValueError, 'multiples of 8'), (dict(v=z(2, 7, 2, 264)), ValueError, '256'), (dict(q=z(2, 5, 3, 32)), ValueError, 'divide'),
    (dict(q=z(2, 5, 130, 32)), ValueError, '64'), (dict(scale=0.0), ValueError, 'scale'), (dict(scale=-1.0), ValueError, 'scale'),
    (dict(scale=float('inf')), ValueError, 'scale'), (dict(scale=float('nan')), ValueError, 'scale'), (dict(key_lengths=z(3).int()), ValueError, 'key_lengths'),
    (dict(key_lengths=z(2)), TypeError, 'int32'), ({}, _hip.NdHipError, 'no CPU'),
])
def test_differential_attention_refuses(kw, exc, what):
    with pytest.raises(exc, match=what):
        block.differential_attention(**diff_tensors(**kw))


def ffn_tensors(**kw):
    d = dict(x=z(3, 16), w_in=z(48, 16), w_out=z(16, 24))
    d.update(kw)
    return d


@pytest.mark.parametrize('kw,exc,what', [
    (dict(activation='relu'), ValueError, 'activation'), (dict(x=torch.tensor(1.0)), ValueError, 'channel'), (dict(w_in=z(47, 16)), ValueError, 'w_in'),
    (dict(w_in=z(48, 8)), ValueError, 'w_in'), (dict(w_out=z(24, 16)), ValueError, 'w_out'), (dict(b_in=z(24)), ValueError, 'b_in'),
    (dict(b_out=z(24)), ValueError, 'b_out'), (dict(residual=z(1, 16)), ValueError, 'residual'), (dict(x=z(3, 12), w_in=z(48, 12), w_out=z(12, 24)), ValueError, 'multiples'),
    (dict(w_in=z(24, 16), w_out=z(16, 12)), ValueError, 'multiples'), (dict(x=z(1, 8), w_in=z(1, 8).expand(2 << 21, 8), w_out=z(8, 1).expand(8, 1 << 21)), ValueError, '2\\^20'),
    ({}, _hip.NdHipError, 'no CPU'),
])
def test_gated_feed_forward_refuses(kw, exc, what):
    with pytest.raises(exc, match=what):
        block.gated_feed_forward(**ffn_tensors(**kw))


# ------------------------------------------------------------------------------------------------------------ tables
def test_grid_positions_are_the_tokens_of_a_map():
    p = block.grid_positions(3, 4)
    assert p.shape == (12, 2) and p[7].tolist() == [1, 3] and p[0].tolist() == [0, 0] and p[11].tolist() == [2, 3]


def test_rotary_table_values():
    cos, sin = block.rotary_table(torch.tensor([0, 5, 131071]), 8, theta=100.0)
    for i, pos in enumerate((0, 5, 131071)):
        for j in range(4):
            a = pos * 100.0 ** (-j / 4)
            assert abs(cos[i, j].item() - math.cos(a)) <= 2 ** -24 + 1e-10 and abs(sin[i, j].item() - math.sin(a)) <= 2 ** -24 + 1e-10
    assert cos.dtype == F32 and cos.shape == (3, 4)
    c2, s2 = block.rotary_table(block.grid_positions(3, 4), 8)        # two axes: the first half of the pairs turns by the row
    cy, sy = block.rotary_table(torch.arange(3), 4)
    cx, sx = block.rotary_table(torch.arange(4), 4)
    assert torch.equal(c2.view(3, 4, 4)[:, 1, :2], cy) and torch.equal(s2.view(3, 4, 4)[2, :, 2:], sx)
    cb, _ = block.rotary_table(torch.arange(6).view(2, 3, 1), 4)
    assert torch.equal(cb.view(6, 2), block.rotary_table(torch.arange(6), 4)[0])
    assert block.rotary_table(torch.empty(0, dtype=torch.long), 4)[0].shape == (0, 2)


@pytest.mark.parametrize('pos,ch', [(torch.arange(4), 7), (torch.arange(4), 0), (block.grid_positions(2, 2), 6), (torch.zeros(2, 9), 8), (torch.tensor(3), 8)])
def test_rotary_table_refuses(pos, ch):
    with pytest.raises(ValueError):
        block.rotary_table(pos, ch)


def diff_bwd_args(**kw):
    d = diff_args(**dict(dict(o1=A, o2=A, lse=A), **kw))
    tensors, (out1, out2, lse, ws), sizes = d[:19], d[20:24], d[24:]
    dout = (A, *kw.get('dos', (640, 128, 64)))
    return (*tensors, out1, out2, lse, *dout, A, A, A, None, None, None, None, ws, *sizes)


@pytest.mark.parametrize('kw,what', [
    (dict(B=1 << 21, H=8, Hk=8, Tq=1, Tk=1), 'workgroups'), (dict(B=1 << 12, H=1, Hk=1, D=8, Dv=8, Tq=1, Tk=1 << 20), 'workgroups'),
    (dict(B=1, H=1 << 17, Hk=1 << 17, D=8, Dv=64, Tq=2, Tk=1, qs=(0, 1 << 21, 16)), 'gradient'),
])
def test_a_forward_pass_that_is_kept_refuses_what_its_backward_pass_would(kw, what):
    refused('nd_diff_attention_bwd', diff_bwd_args(**kw), what)
    refused('nd_diff_attention', diff_args(o1=A, o2=A, lse=A, **kw), what)


def test_sizes_past_what_a_launch_can_count_are_refused():
    """Few rows run in workgroups of 512 threads: 2^23 of them are 2^32 threads.  A feed-forward row index and its step stay in 32 bits."""
    refused('nd_diff_attention', diff_args(B=1 << 20, H=8, Hk=8, Tq=1, Tk=1), 'workgroups')
    refused('nd_gated_ffn', ffn_args(M=(1 << 30) + 1), '2\\^30 rows')
    refused('nd_gated_ffn_bwd', (A, 64, A, 64, A, A, A, A, A, A, None, A, None, A, A, (1 << 30) + 1, 64, 128, 0, _hip.DT_F32, None), '2\\^30 rows')
    with pytest.raises(ValueError, match='2\\^30 rows'):
        block.gated_feed_forward(torch.zeros(1, 8).expand((1 << 30) + 1, 8), z(16, 8), z(8, 8))


@pytest.mark.skipif(torch.cuda.is_available(), reason='the call would be launched')
@pytest.mark.parametrize('C,F', [(8, 8), (64, 256), (256, 64), (72, 24)])
@pytest.mark.parametrize('M', [(1 << 26) + 1, 1 << 30])
def test_every_accepted_row_count_has_a_tile_that_fits_a_launch(M, C, F):
    lib = _hip.load_block()
    for dtype in (_hip.DT_BF16, _hip.DT_F32):
        assert lib.nd_gated_ffn(*ffn_args(M=M, C=C, F=F, ldx=C, ldy=C, dtype=dtype)) == -2, lib.nd_block_last_error()
        assert lib.nd_gated_ffn_bwd_workspace_floats(M, C, F, dtype) > 0


def test_the_key_kernels_rows_are_divided_for_the_workgroups_that_fit():
    """256-byte rows: one workgroup a CU.  192 of them, 16096 rows each: four parts are three full rounds of the chip, eight only more
    partials (measured 1071 us for 1108)."""
    lib, (B, T, H, Hk, D, Dv) = _hip.load_block(), (6, 4024, 4, 1, 64, 128)
    rows_part, keys_part = B * T * Hk * (2 * D + Dv), B * T * H * 2 * D      # floats of one part of dk | dv, and of dq
    small = 2 * B * T * H + (1 << 16)                          # row statistics, shares of lambda's gradient
    assert lib.nd_diff_attention_bwd_workspace_floats(B, T, T, H, Hk, D, Dv, _hip.DT_BF16) <= 4 * rows_part + 2 * keys_part + small
