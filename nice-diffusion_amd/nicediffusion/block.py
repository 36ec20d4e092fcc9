"""Operators of a transformer block over image tokens, as hand-written HIP kernels (``libnd_block.so``) on an MI355X (gfx950).

They stand beside the attention and 1x1-convolution launches of the UNet plan and take the rows those produce: an NHWC map
is a [batch, token, channel] tensor here, and the q / k / v parts of a packed qkv row are passed as views.

* ``qk_norm_rope``: RMS norm of every query / key head and rotation by position, in one pass.
* ``differential_attention``: difference of two softmax maps with a learned weight.
* ``gated_feed_forward``: both projections, the activation and the product in one kernel, then the output projection.

Conventions.  Tensors live on an AMD GPU (there is no CPU path: ``NdHipError``) and share one dtype, float32 or bfloat16;
sums, softmax statistics and products are fp32.  Work is queued on the current stream of the tensors' device, nothing
synchronises, scratch memory comes from torch's allocator, so a call may be captured into a hipGraph.  Wrong shapes or dtypes
raise ``ValueError`` / ``TypeError`` before anything is launched.  All three are differentiable (once): gradients flow to
every floating argument except the tables.  To capture a backward pass, do it on leaves that no graph built outside the
capture still holds (torch ties a leaf's gradient accumulation to the stream of its first graph).
"""
import torch
from torch.autograd.function import once_differentiable

from . import _hip

_DT = {torch.float32: _hip.DT_F32, torch.bfloat16: _hip.DT_BF16}


# ------------------------------------------------------------------------------------------------------------ plumbing
def _check(first, **others):
    """Device and dtype of a call: every tensor on ``first``'s GPU, in its dtype (float32 / bfloat16).  None is skipped."""
    name, t = first
    _hip.require_device(t, name)
    if t.dtype not in _DT:
        raise TypeError('{} is {}: float32 or bfloat16 expected'.format(name, t.dtype))
    for n, o in others.items():
        if o is None:
            continue
        if o.device != t.device:
            raise ValueError('{} lives on {}, {} on {}'.format(n, o.device, name, t.device))
        if o.dtype != t.dtype:
            raise TypeError('{} is {}, {} is {}: one dtype per call'.format(n, o.dtype, name, t.dtype))
    _hip.require_gfx950(t.device.index)


def _shape(t, name, *want):
    if t.dim() != len(want) or any(w is not None and s != w for s, w in zip(t.shape, want)):
        raise ValueError('{} has shape {}, expected {}'.format(name, tuple(t.shape), tuple('?' if w is None else w for w in want)))


def _rows(t):
    """``t`` with its last dimension contiguous (a copy only if it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t):
    """Element strides of the leading dimensions; 0 for a dimension of one element, whose stride says nothing."""
    return [0 if n == 1 else s for n, s in zip(t.shape[:-1], t.stride()[:-1])]


def _call(name, device, *args):
    """Launch ``name`` on the current stream of ``device`` (made the current device for the call)."""
    fn = getattr(_hip.load_block(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    _hip.check_block(rc, name)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------- query / key norm with rotation
def grid_positions(height, width, device=None):
    """[height * width, 2] (row, column) of the tokens of an NHWC map, in token order."""
    y, x = torch.meshgrid(torch.arange(height, device=device), torch.arange(width, device=device), indexing='ij')
    return torch.stack([y.reshape(-1), x.reshape(-1)], -1)


def rotary_table(positions, channels, theta=10000.0):
    """cos and sin tables for ``qk_norm_rope``: fp32 [..., channels / 2] each.

    ``positions`` [...] (one axis) or [..., axes]: the pairs are divided evenly among the axes; pair i of an axis' n turns by
    ``position * theta ** (-i / n)``.  Angles are formed in float64: far positions keep their phase.  A 2-D tensor is read as
    [..., axes] when its last dimension is at most 3; give a [B, T] batch of one-axis positions as [B, T, 1]."""
    if channels <= 0 or channels % 2:
        raise ValueError('channels must be positive and even, got {}'.format(channels))
    p = positions.double()
    if p.dim() == 1 or p.shape[-1] > 3:
        p = p[..., None]
    axes, pairs = p.shape[-1], channels // 2
    if pairs % axes:
        raise ValueError('{} pairs do not divide among {} axes'.format(pairs, axes))
    n = pairs // axes
    f = float(theta) ** (-torch.arange(n, dtype=torch.float64, device=p.device) / n)
    a = (p[..., :, None] * f).flatten(-2)
    return torch.cos(a).float(), torch.sin(a).float()


def _table(t, name, B, T):
    if t.dtype != torch.float32:
        raise TypeError('{} is {}: float32 tables expected'.format(name, t.dtype))
    if t.requires_grad:
        raise ValueError('{} requires a gradient: the tables are constants'.format(name))
    if t.dim() == 2:
        t = t[None]
    if t.dim() != 3 or t.shape[0] not in (1, B) or t.shape[1] != T:
        raise ValueError('{} has shape {}, expected [{}, pairs] or [{}, {}, pairs]'.format(name, tuple(t.shape), T, B, T))
    if t.stride(2) != 1 or t.stride(1) != t.shape[2]:
        t = t.contiguous()
    return t


def _launch_qk(q, k, qw, kw, cos, sin, eps, interleaved, qo, ko):
    B, T, Hq, D = q.shape
    R = 0 if cos is None else 2 * cos.shape[-1]
    tb = 0 if cos is None or cos.shape[0] == 1 else cos.stride(0)
    _call('nd_qk_norm_rope', q.device, q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), _hip.ptr(qw), _hip.ptr(kw), _hip.ptr(cos),
          _hip.ptr(sin), tb, qo.data_ptr(), *_strides(qo), ko.data_ptr(), *_strides(ko), B, T, Hq, k.shape[2], D, R, eps,
          _hip.ROPE_INTERLEAVED if interleaved else 0, _DT[q.dtype])


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, eps, interleaved):
        qo, ko = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
        if q.numel():
            _launch_qk(q, k, qw, kw, cos, sin, eps, interleaved, qo, ko)
        ctx.save_for_backward(q, k, qw, kw, cos, sin)
        ctx.eps, ctx.interleaved = eps, interleaved
        return qo, ko

    @staticmethod
    @once_differentiable
    def backward(ctx, dqo, dko):
        q, k, qw, kw, cos, sin = ctx.saved_tensors
        B, T, Hq, D = q.shape
        Hk = k.shape[2]
        dqo, dko = _rows(dqo), _rows(dko)
        dq, dk = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dqw = torch.empty_like(qw, memory_format=torch.contiguous_format) if qw is not None and ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(kw, memory_format=torch.contiguous_format) if kw is not None and ctx.needs_input_grad[3] else None
        if q.numel():
            ws = None
            if dqw is not None or dkw is not None:
                n = _hip.load_block().nd_qk_norm_rope_bwd_workspace_floats(B, T, Hq, Hk, D)
                ws = torch.empty(n, dtype=torch.float32, device=q.device)
            R = 0 if cos is None else 2 * cos.shape[-1]
            tb = 0 if cos is None or cos.shape[0] == 1 else cos.stride(0)
            _call('nd_qk_norm_rope_bwd', q.device, q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), _hip.ptr(qw), _hip.ptr(kw),
                  _hip.ptr(cos), _hip.ptr(sin), tb, dqo.data_ptr(), *_strides(dqo), dko.data_ptr(), *_strides(dko), dq.data_ptr(),
                  *_strides(dq), dk.data_ptr(), *_strides(dk), _hip.ptr(dqw), _hip.ptr(dkw), _hip.ptr(ws), B, T, Hq, Hk, D, R, ctx.eps,
                  _hip.ROPE_INTERLEAVED if ctx.interleaved else 0, _DT[q.dtype])
        else:
            for g in (dqw, dkw):
                if g is not None:
                    g.zero_()
        return dq, dk, dqw, dkw, None, None, None, None


def qk_norm_rope(q, k, q_weight=None, k_weight=None, cos=None, sin=None, eps=1e-6, interleaved=False, out=None):
    """RMS norm of every query and key head, scaled by the weights, then rotated by position: one pass over both.

    q [B, T, Hq, D], k [B, T, Hk, D]: any strides (views of a packed qkv row); D even, at most 512.  q_weight, k_weight [D] or
    None (ones).  cos, sin: fp32 tables of ``rotary_table`` for these tokens, [T, R/2] or [B, T, R/2]; the first R channels are
    rotated, the rest only normed; None: norm alone.  Pairs are channels (i, i + R/2), or (2i, 2i + 1) if ``interleaved``.

    Returns new contiguous (q, k).  ``out=(q_out, k_out)`` writes there instead and records no gradient: the inputs themselves
    (in place in the packed row that ``nd_attention_nhwc`` reads) or memory that does not overlap them (a slot of a cache)."""
    if q.dim() != 4:
        raise ValueError('q has shape {}, expected [B, T, heads, D]'.format(tuple(q.shape)))
    B, T, Hq, D = q.shape
    _shape(k, 'k', B, T, None, D)
    _check(('q', q), k=k, q_weight=q_weight, k_weight=k_weight)
    if D == 0 or D % 2 or D > 512:
        raise ValueError('head dim must be even and at most 512, got {}'.format(D))
    if Hq == 0 or k.shape[2] == 0:
        raise ValueError('q and k need at least one head')
    for n, w in (('q_weight', q_weight), ('k_weight', k_weight)):
        if w is not None:
            _shape(w, n, D)
    if (cos is None) != (sin is None):
        raise ValueError('cos and sin come together')
    if cos is not None:
        if cos.device != q.device or sin.device != q.device:
            raise ValueError('the tables live on {}, q on {}'.format(cos.device, q.device))
        if cos.shape != sin.shape:
            raise ValueError('cos has shape {}, sin {}'.format(tuple(cos.shape), tuple(sin.shape)))
        cos, sin = _table(cos, 'cos', B, T), _table(sin, 'sin', B, T)
        if cos.shape[0] > 1 and cos.stride(0) != sin.stride(0):
            cos, sin = cos.contiguous(), sin.contiguous()
        if not 0 < 2 * cos.shape[-1] <= D:
            raise ValueError('tables for {} channels, head dim is {}'.format(2 * cos.shape[-1], D))
    q, k = _rows(q), _rows(k)
    q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    if out is not None:
        if _wants_grad(q, k, q_weight, k_weight):
            raise ValueError('out= records no gradient: call under torch.no_grad() or without out')
        qo, ko = out
        for n, o, t in (('out[0]', qo, q), ('out[1]', ko, k)):
            _shape(o, n, *t.shape)
            if o.stride(-1) != 1:
                raise ValueError('{} must have contiguous channels'.format(n))
        _check(('q', q), **{'out[0]': qo, 'out[1]': ko})
        if q.numel():
            _launch_qk(q, k, q_weight, k_weight, cos, sin, eps, interleaved, qo, ko)
        return qo, ko
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, eps, interleaved)
    qo, ko = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if q.numel():
        _launch_qk(q, k, q_weight, k_weight, cos, sin, eps, interleaved, qo, ko)
    return qo, ko


# ------------------------------------------------------------------------------------------------ gated feed-forward
_ACTS = {'silu': _hip.ACT_SILU, 'gelu': _hip.ACT_GELU, 'gelu_tanh': _hip.ACT_GELU_TANH}


def _matrix(t, cols):
    """``t`` [..., cols] as 16-byte aligned rows [M, cols] (a copy only where it does not lie like that)."""
    m = t.reshape(-1, cols)
    if m.stride(1) != 1 or (m.shape[0] > 1 and not cols <= m.stride(0) <= 1 << 21) or m.stride(0) * m.element_size() % 16 or m.data_ptr() % 16:
        m = m.contiguous() if not m.is_contiguous() else m.clone()
    return m


def _ld(m):
    return m.shape[1] if m.shape[0] == 1 else m.stride(0)


def _aligned(t):
    """A contiguous parameter on a 16-byte boundary."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _floats(n, device):
    return torch.empty(n, dtype=torch.float32, device=device) if n > 0 else None


def _launch_ffn(x, w_in, b_in, w_out, b_out, res, act, keep):
    M, C = x.shape
    F = w_out.shape[1]
    new = dict(dtype=x.dtype, device=x.device)
    y, h = torch.empty(M, C, **new), torch.empty(M, F, **new)
    au = torch.empty(M, 2 * F, **new) if keep else None
    ws = _floats(_hip.load_block().nd_gated_ffn_workspace_floats(M, C, F, _DT[x.dtype]), x.device)
    _call('nd_gated_ffn', x.device, x.data_ptr(), _ld(x), w_in.data_ptr(), _hip.ptr(b_in), w_out.data_ptr(), _hip.ptr(b_out), _hip.ptr(res),
          0 if res is None else _ld(res), y.data_ptr(), C, h.data_ptr(), _hip.ptr(au), _hip.ptr(ws), M, C, F, act, _DT[x.dtype])
    return y, h, au


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, b_in, w_out, b_out, res, act):
        C = x.shape[-1]
        xm, wi, wo = _matrix(x, C), _aligned(w_in), _aligned(w_out)
        rm = None if res is None else _matrix(res, C)
        if xm.shape[0]:
            y, h, au = _launch_ffn(xm, wi, _aligned(b_in), wo, _aligned(b_out), rm, act, True)
        else:
            y, h, au = xm.new_empty(0, C), None, None
        ctx.save_for_backward(xm, wi, wo, h, au)
        ctx.act, ctx.shape = act, x.shape
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_in, w_out, h, au = ctx.saved_tensors
        M, C = x.shape
        F = w_out.shape[1]
        need = ctx.needs_input_grad
        new = dict(dtype=x.dtype, device=x.device)
        dx = torch.empty(M, C, **new) if need[0] else None
        dwi = torch.empty(2 * F, C, **new) if need[1] else None
        dbi = torch.empty(2 * F, **new) if need[2] else None
        dwo = torch.empty(C, F, **new) if need[3] else None
        dbo = torch.empty(C, **new) if need[4] else None
        if M:
            if any(need[:5]):
                g = _matrix(dy, C)
                dau = torch.empty(M, 2 * F, **new) if any(need[:3]) else None
                ws = _floats(_hip.load_block().nd_gated_ffn_bwd_workspace_floats(M, C, F, _DT[x.dtype]), x.device)
                _call('nd_gated_ffn_bwd', x.device, g.data_ptr(), _ld(g), x.data_ptr(), _ld(x), w_in.data_ptr(), w_out.data_ptr(), au.data_ptr(),
                      h.data_ptr(), _hip.ptr(dx), _hip.ptr(dwi), _hip.ptr(dbi), _hip.ptr(dwo), _hip.ptr(dbo), _hip.ptr(dau), _hip.ptr(ws), M, C,
                      F, ctx.act, _DT[x.dtype])
        else:
            for t in (dwi, dbi, dwo, dbo):
                if t is not None:
                    t.zero_()
        return None if dx is None else dx.view(ctx.shape), dwi, dbi, dwo, dbo, dy if need[5] else None, None


def gated_feed_forward(x, w_in, w_out, b_in=None, b_out=None, residual=None, activation='silu'):
    """``residual + (act(x Wg^T + bg) * (x Wu^T + bu)) w_out^T + b_out``: the block's gated feed-forward half.

    x [..., C]; w_in [2F, C]: the gate's rows Wg, then the up projection's Wu; w_out [C, F]; b_in [2F], b_out [C], residual
    (x's shape) or None.  C and F multiples of 8.  activation: 'silu', 'gelu' (error function) or 'gelu_tanh'.  Returns a new
    contiguous tensor of x's shape.  In bfloat16 the hidden row is rounded once between the two products; a backward pass keeps
    it and the pre-activations (3 F values a token)."""
    if activation not in _ACTS:
        raise ValueError('activation is {!r}, expected one of {}'.format(activation, sorted(_ACTS)))
    if x.dim() < 1:
        raise ValueError('x has no channel dimension')
    C = x.shape[-1]
    if w_in.dim() != 2 or w_in.shape[0] % 2:
        raise ValueError('w_in has shape {}, expected [2 F, {}]'.format(tuple(w_in.shape), C))
    F = w_in.shape[0] // 2
    _shape(w_in, 'w_in', 2 * F, C)
    _shape(w_out, 'w_out', C, F)
    if C == 0 or F == 0 or C % 8 or F % 8:
        raise ValueError('channels ({}) and hidden channels ({}) must be positive multiples of 8'.format(C, F))
    if C * F > 1 << 28:
        raise ValueError('weights of more than 2^28 elements')
    if b_in is not None:
        _shape(b_in, 'b_in', 2 * F)
    if b_out is not None:
        _shape(b_out, 'b_out', C)
    if residual is not None:
        _shape(residual, 'residual', *x.shape)
    _check(('x', x), w_in=w_in, w_out=w_out, b_in=b_in, b_out=b_out, residual=residual)
    if x.numel() // C >= 1 << 31:
        raise ValueError('too many rows')
    act = _ACTS[activation]
    if _wants_grad(x, w_in, b_in, w_out, b_out, residual):
        return _GatedFfn.apply(x, w_in, b_in, w_out, b_out, residual, act)
    if x.numel() == 0:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    res = None if residual is None else _matrix(residual, C)
    return _launch_ffn(_matrix(x, C), _aligned(w_in), _aligned(b_in), _aligned(w_out), _aligned(b_out), res, act, False)[0].view(x.shape)
