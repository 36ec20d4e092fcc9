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
every floating argument except the tables.  A forward-mode tangent raises ``NotImplementedError``; ``torch.func`` transforms
(vmap, grad, jvp) are not supported and end in torch's own error.  To capture a backward pass, do it on leaves that no graph
built outside the capture still holds (torch ties a leaf's gradient accumulation to the stream of its first graph).
"""
import torch
import torch.autograd.forward_ad as _fwd
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _hip

_DT = {torch.float32: _hip.DT_F32, torch.bfloat16: _hip.DT_BF16}


# ------------------------------------------------------------------------------------------------------------ plumbing
# (a decode step is a few microseconds of kernels: what runs per call below is kept short)
def _check(name, t, names, others):
    """Device and dtype of a call: every tensor on the first one's GPU, in its dtype (float32 / bfloat16).  None is skipped."""
    _hip.require_device(t, name)
    dev, dtype = t.device, t.dtype
    if dtype not in _DT:
        raise TypeError('{} is {}: float32 or bfloat16 expected'.format(name, dtype))
    for n, o in zip(names, others):
        if o is not None and (o.dtype is not dtype or o.device != dev):
            if o.device != dev:
                raise ValueError('{} lives on {}, {} on {}'.format(n, o.device, name, dev))
            raise TypeError('{} is {}, {} is {}: one dtype per call'.format(n, o.dtype, name, dtype))
    if getattr(_fwd, '_current_level', 0) >= 0:                # a level is open, or this torch does not say
        _no_tangent((name, *names), (t, *others))
    _hip.require_gfx950(dev.index)


def _no_tangent(names, tensors):
    """The operators have no forward-mode derivative, and a launch would drop a tangent as if it were zero."""
    for n, t in zip(names, tensors):
        if t is not None and _fwd.unpack_dual(t).tangent is not None:
            raise NotImplementedError('{} carries a forward-mode tangent: these operators have reverse-mode gradients only'.format(n))


class _Nothing(torch.autograd.Function):
    """A result without work: zeros of ``shape`` that every input gets a zero gradient from."""
    @staticmethod
    def forward(ctx, shape, *tensors):
        ctx.tensors = [(t.shape, t.dtype, t.device) for t in tensors]
        return tensors[0].new_zeros(shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, _):
        return (None, *(torch.zeros(s, dtype=d, device=v) for s, d, v in ctx.tensors))


def _shape(t, name, *want):
    if t.shape != want:
        raise ValueError('{} has shape {}, expected {}'.format(name, tuple(t.shape), want))


def _rows(t):
    """``t`` with its last dimension contiguous (a copy only if it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t):
    """Element strides of the first three of four dimensions; 0 for a dimension of one element, whose stride says nothing."""
    (a, b, c, _), (i, j, k, _) = t.stride(), t.shape
    return (0 if i == 1 else a, 0 if j == 1 else b, 0 if k == 1 else c)


_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _stream(index):
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _call(name, device, *args):
    """Launch ``name`` on the current stream of ``device`` (made the current device for the call)."""
    call, pack, n = _hip.BLOCK_CALLS[name]
    fn, words, index = _hip.load_block().nd_block_packed, pack.pack(*args), device.index
    if torch.cuda.current_device() == index:
        rc = fn(call, words, n, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(call, words, n, _stream(index))
    if rc:
        _hip.check_block(rc, name)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _aligned(t):
    """A contiguous parameter on a 16-byte boundary."""
    if t is None:
        return None
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _floats(n, device):
    return torch.empty(n, dtype=torch.float32, device=device) if n > 0 else None


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ------------------------------------------------------------------------------------- query / key norm with rotation
def grid_positions(height, width, device=None):
    """[height * width, 2] (row, column) of the tokens of an NHWC map, in token order."""
    y, x = torch.meshgrid(torch.arange(height, device=device), torch.arange(width, device=device), indexing='ij')
    return torch.stack([y.reshape(-1), x.reshape(-1)], -1)


def rotary_table(positions, channels, theta=10000.0):
    """cos and sin tables for ``qk_norm_rope``: fp32 [..., channels / 2] each.

    ``positions`` [...] (one axis) or [..., axes]: the pairs are divided evenly among the axes; pair i of an axis' n turns by
    ``position * theta ** (-i / n)``.  Angles are formed in float64: far positions keep their phase.  Tensors of two and
    more dimensions end in the axes (at most 3): a [B, T] batch of one-axis positions is given as [B, T, 1]."""
    if channels <= 0 or channels % 2:
        raise ValueError('channels must be positive and even, got {}'.format(channels))
    p = positions.double()
    if p.dim() == 1:
        p = p[:, None]
    if p.dim() == 0 or not 1 <= p.shape[-1] <= 3:
        raise ValueError('positions have shape {}, expected [T] or [..., axes] with at most 3 axes'.format(tuple(positions.shape)))
    axes, pairs = p.shape[-1], channels // 2
    if pairs % axes:
        raise ValueError('{} pairs do not divide among {} axes'.format(pairs, axes))
    n = pairs // axes
    f = float(theta) ** (-torch.arange(n, dtype=torch.float64, device=p.device) / n)
    a = (p[..., :, None] * f).flatten(-2)
    return torch.cos(a).float(), torch.sin(a).float()


def _table(t, name, B, T):
    """A table [T, pairs] or [1 or B, T, pairs] with contiguous token rows (the batch may have a stride of its own)."""
    if t.dtype is not torch.float32:
        raise TypeError('{} is {}: float32 tables expected'.format(name, t.dtype))
    if t.requires_grad:
        raise ValueError('{} requires a gradient: the tables are constants'.format(name))
    shape = t.shape
    n = len(shape)
    if n not in (2, 3) or shape[n - 2] != T or (n == 3 and shape[0] not in (1, B)):
        raise ValueError('{} has shape {}, expected [{}, pairs] or [{}, {}, pairs]'.format(name, tuple(shape), T, B, T))
    if t.is_contiguous():
        return t
    return t if t.stride(-1) == 1 and t.stride(-2) == shape[-1] else t.contiguous()


def _table_stride(t):
    return t.stride(0) if t is not None and t.dim() == 3 and t.shape[0] > 1 else 0


def _launch_qk(q, k, qw, kw, cos, sin, eps, interleaved, qo, ko):
    B, T, Hq, D = q.shape
    R, tb = 0 if cos is None else 2 * cos.shape[-1], _table_stride(cos)
    _call('nd_qk_norm_rope', q.device, q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), _ptr(qw), _ptr(kw), _ptr(cos),
          _ptr(sin), tb, qo.data_ptr(), *_strides(qo), ko.data_ptr(), *_strides(ko), B, T, Hq, k.shape[2], D, R, eps,
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
            R, tb = 0 if cos is None else 2 * cos.shape[-1], _table_stride(cos)
            _call('nd_qk_norm_rope_bwd', q.device, q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), _ptr(qw), _ptr(kw),
                  _ptr(cos), _ptr(sin), tb, dqo.data_ptr(), *_strides(dqo), dko.data_ptr(), *_strides(dko), dq.data_ptr(),
                  *_strides(dq), dk.data_ptr(), *_strides(dk), _ptr(dqw), _ptr(dkw), _ptr(ws), B, T, Hq, Hk, D, R, ctx.eps,
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
    (in place in the packed row that ``nd_attention_nhwc`` reads) or memory that shares no address with them, the tables, the
    weights or each other (a slot of a cache; where address ranges interleave, equal strides are needed to tell): else ValueError."""
    if q.dim() != 4:
        raise ValueError('q has shape {}, expected [B, T, heads, D]'.format(tuple(q.shape)))
    B, T, Hq, D = q.shape
    if k.dim() != 4:
        raise ValueError('k has shape {}, expected [B, T, heads, D]'.format(tuple(k.shape)))
    _shape(k, 'k', B, T, k.shape[2], D)
    if D == 0 or D % 2 or D > 512:
        raise ValueError('head dim must be even and at most 512, got {}'.format(D))
    if Hq == 0 or k.shape[2] == 0:
        raise ValueError('q and k need at least one head')
    if not 0 <= eps < float('inf'):
        raise ValueError('eps must be finite and not negative, got {}'.format(eps))
    if q_weight is not None:
        _shape(q_weight, 'q_weight', D)
        q_weight = _aligned(q_weight)
    if k_weight is not None:
        _shape(k_weight, 'k_weight', D)
        k_weight = _aligned(k_weight)
    if (cos is None) != (sin is None):
        raise ValueError('cos and sin come together')
    if cos is not None:
        if cos.device != q.device or sin.device != q.device:
            raise ValueError('the tables live on {}, q on {}'.format(cos.device, q.device))
        if cos.shape != sin.shape:
            raise ValueError('cos has shape {}, sin {}'.format(tuple(cos.shape), tuple(sin.shape)))
        cos, sin = _table(cos, 'cos', B, T), _table(sin, 'sin', B, T)
        if _table_stride(cos) != _table_stride(sin):
            cos, sin = cos.contiguous(), sin.contiguous()
        if not 0 < 2 * cos.shape[-1] <= D:
            raise ValueError('tables for {} channels, head dim is {}'.format(2 * cos.shape[-1], D))
        if getattr(_fwd, '_current_level', 0) >= 0:
            _no_tangent(('cos', 'sin'), (cos, sin))
    _check('q', q, ('k', 'q_weight', 'k_weight'), (k, q_weight, k_weight))
    q, k = _rows(q), _rows(k)
    if out is not None:
        if _wants_grad(q, k, q_weight, k_weight):
            raise ValueError('out= records no gradient: call under torch.no_grad() or without out')
        qo, ko = out
        for n, o, t in (('out[0]', qo, q), ('out[1]', ko, k)):
            _shape(o, n, *t.shape)
            if o.requires_grad and torch.is_grad_enabled():
                raise ValueError('{} requires a gradient, and out= records none: call under torch.no_grad()'.format(n))
            if o.stride(-1) != 1 or 0 in [a for a, z in zip(o.stride(), o.shape) if z > 1]:
                raise ValueError('{} must have contiguous channels and no rows that repeat'.format(n))
        _check('q', q, ('out[0]', 'out[1]'), (qo, ko))
        if q.numel():
            _launch_qk(q, k, q_weight, k_weight, cos, sin, eps, interleaved, qo, ko)
            increment_version((qo, ko))                        # a graph that saved this memory must not be run backward over it
        return qo, ko
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, eps, interleaved)
    qo, ko = q.new_empty(q.shape), k.new_empty(k.shape)
    if q.numel():
        _launch_qk(q, k, q_weight, k_weight, cos, sin, eps, interleaved, qo, ko)
    return qo, ko


# -------------------------------------------------------------------------------------------- differential attention
def _attn_rows(t):
    """``t`` [B, T, heads, channels] as the kernels read it: contiguous channels, every row on a 16-byte boundary (else a copy)."""
    per = 16 // t.element_size()
    a, b, c = _strides(t)
    if t.stride(-1) != 1 or t.data_ptr() % 16 or (a | b | c) % per or b > 1 << 22:
        t = t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def _diff_args(q, k, v, lams, lambda_init, lengths):
    per_head = lams[0].dim() == 2
    lq1, lk1, lq2, lk2 = lams
    return (q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v), lq1.data_ptr(), lk1.data_ptr(), lq2.data_ptr(),
            lk2.data_ptr(), lq1.shape[-1] if per_head else 0, lambda_init, _ptr(lengths))


def _diff_sizes(q, k, v):
    B, Tq, H, D2 = q.shape
    _, Tk, Hk, Dv = v.shape
    return (B, Tq, Tk, H, Hk, D2 // 2, Dv)


def _launch_diff(q, k, v, lams, lambda_init, scale, lengths, causal, keep):
    B, Tq, Tk, H, Hk, D, Dv = sizes = _diff_sizes(q, k, v)
    out = q.new_empty(B, Tq, H, Dv)
    o1, o2, lse = (torch.empty_like(out), torch.empty_like(out), _floats(2 * B * Tq * H, q.device)) if keep else (None,) * 3
    ws = _floats(_hip.load_block().nd_diff_attention_workspace_floats(*sizes, _DT[q.dtype]), q.device)
    _call('nd_diff_attention', q.device, *_diff_args(q, k, v, lams, lambda_init, lengths), out.data_ptr(), _ptr(o1), _ptr(o2),
          _ptr(lse), _ptr(ws), *sizes, scale, _hip.ATTN_CAUSAL if causal else 0, _DT[q.dtype])
    return out, o1, o2, lse


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lq1, lk1, lq2, lk2, lambda_init, scale, lengths, causal):
        q, k, v = _attn_rows(q), _attn_rows(k), _attn_rows(v)
        lams = [_aligned(t) for t in (lq1, lk1, lq2, lk2)]
        out, o1, o2, lse = _launch_diff(q, k, v, lams, lambda_init, scale, lengths, causal, True)
        ctx.save_for_backward(q, k, v, *lams, lengths, o1, o2, lse)
        ctx.lambda_init, ctx.scale, ctx.causal = lambda_init, scale, causal
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lq1, lk1, lq2, lk2, lengths, o1, o2, lse = ctx.saved_tensors
        lams = [lq1, lk1, lq2, lk2]
        sizes = _diff_sizes(q, k, v)
        dout = _attn_rows(dout)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dl = [torch.empty_like(t) if n else None for t, n in zip(lams, ctx.needs_input_grad[3:7])]
        ws = _floats(_hip.load_block().nd_diff_attention_bwd_workspace_floats(*sizes, _DT[q.dtype]), q.device)
        _call('nd_diff_attention_bwd', q.device, *_diff_args(q, k, v, lams, ctx.lambda_init, lengths), o1.data_ptr(), o2.data_ptr(),
              lse.data_ptr(), dout.data_ptr(), *_strides(dout), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *(_ptr(t) for t in dl),
              ws.data_ptr(), *sizes, ctx.scale, _hip.ATTN_CAUSAL if ctx.causal else 0, _DT[q.dtype])
        return (dq, dk, dv, *dl, None, None, None, None)


_LAMBDAS = ('lambda_q1', 'lambda_k1', 'lambda_q2', 'lambda_k2')
_DIFF_NAMES = ('k', 'v') + _LAMBDAS


def differential_attention(q, k, v, lambda_q1, lambda_k1, lambda_q2, lambda_k2, lambda_init=0.8, scale=None, key_lengths=None, causal=False):
    """``(softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v`` with ``lam = exp(lq1.lk1) - exp(lq2.lk2) + lambda_init``.

    q [B, Tq, H, 2 D], k [B, Tk, Hk, 2 D]: the first D channels of a head are the first map's, the rest the second's; v
    [B, Tk, Hk, Dv].  Query head h reads key head h // (H / Hk).  D and Dv multiples of 8, at most 128 and 256.  Any strides (views
    of a packed qkv row); a cache that is longer than its contents is passed whole with ``key_lengths``.  The lambda vectors are [D]
    (one layer's) or [H, D] (each head its own).  scale defaults to D ** -0.5 and must be positive.

    key_lengths [B] (int32 or int64, on the GPU): keys at or past it take no part, whatever their memory holds, and get zero
    gradients; values are held to 0 .. Tk.  causal: query t sees the keys up to t + length - Tq (the queries are the sequence's
    last); it hides by weights of zero, so a NaN or infinite key or value may spoil rows before it too.  A query that sees no key
    gives a zero row and no gradient.  This is the difference of the maps alone: a norm of each head's output and a factor
    (1 - lambda_init), where a model has them, are the caller's.  Returns [B, Tq, H, Dv], contiguous.  Few query rows
    (Tq H / Hk <= 32, single tokens) have a form of their own that divides the keys."""
    if q.dim() != 4 or q.shape[3] % 2:
        raise ValueError('q has shape {}, expected [B, Tq, H, 2 D]'.format(tuple(q.shape)))
    B, Tq, H, D = q.shape
    D //= 2
    if k.dim() != 4 or v.dim() != 4:
        raise ValueError('k has shape {}, v {}, expected [B, Tk, Hk, 2 D] and [B, Tk, Hk, Dv]'.format(tuple(k.shape), tuple(v.shape)))
    _, Tk, Hk, Dv = v.shape
    _shape(k, 'k', B, Tk, Hk, 2 * D)
    _shape(v, 'v', B, Tk, Hk, Dv)
    lams = (lambda_q1, lambda_k1, lambda_q2, lambda_k2)
    if lambda_q1.shape not in ((D,), (H, D)):
        raise ValueError('lambda_q1 has shape {}, expected [{}] or [{}, {}]'.format(tuple(lambda_q1.shape), D, H, D))
    for n, t in zip(_LAMBDAS, lams):
        _shape(t, n, *lambda_q1.shape)
    if D == 0 or D % 8 or D > 128 or Dv == 0 or Dv % 8 or Dv > 256:
        raise ValueError('D ({}) and Dv ({}) must be positive multiples of 8, at most 128 and 256'.format(D, Dv))
    if H == 0 or Hk == 0 or H % Hk or H // Hk > 64 or H > 1 << 20:
        raise ValueError('{} query heads do not divide among {} key heads (at most 64 each, 2^20 in all)'.format(H, Hk))
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float('inf'):
        raise ValueError('scale must be positive, got {}'.format(scale))
    if key_lengths is not None:
        _shape(key_lengths, 'key_lengths', B)
        if key_lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError('key_lengths is {}: int32 or int64 expected'.format(key_lengths.dtype))
        if key_lengths.device != q.device:
            raise ValueError('key_lengths lives on {}, q on {}'.format(key_lengths.device, q.device))
    _check('q', q, _DIFF_NAMES, (k, v) + lams)
    if key_lengths is not None:
        key_lengths = (key_lengths.clamp(0, Tk) if key_lengths.dtype == torch.int64 else key_lengths).to(torch.int32).contiguous()
    if B == 0 or Tq == 0 or Tk == 0:        # nothing to see: zeros that every input's gradient (zero) flows through
        return _Nothing.apply((B, Tq, H, Dv), q, k, v, *lams)
    if _wants_grad(q, k, v, *lams):
        return _DiffAttention.apply(q, k, v, *lams, float(lambda_init), scale, key_lengths, bool(causal))
    return _launch_diff(_attn_rows(q), _attn_rows(k), _attn_rows(v), [_aligned(t) for t in lams], float(lambda_init), scale, key_lengths,
                        bool(causal), False)[0]


# ------------------------------------------------------------------------------------------------ gated feed-forward
_ACTS = {'silu': _hip.ACT_SILU, 'gelu': _hip.ACT_GELU, 'gelu_tanh': _hip.ACT_GELU_TANH}


def _matrix(t, cols):
    """``t`` [..., cols] as 16-byte aligned rows [M, cols] (a copy only where it does not lie like that)."""
    m = t if t.dim() == 2 else t.reshape(-1, cols)
    if m.stride(1) != 1 or (m.shape[0] > 1 and not cols <= m.stride(0) <= 1 << 21) or m.stride(0) * m.element_size() % 16 or m.data_ptr() % 16:
        m = m.contiguous() if not m.is_contiguous() else m.clone()
    return m


def _ld(m):
    return m.shape[1] if m.shape[0] == 1 else m.stride(0)


def _launch_ffn(x, w_in, b_in, w_out, b_out, res, act, keep, shape):
    M, C = x.shape
    F = w_out.shape[1]
    y, h = x.new_empty(shape), x.new_empty(M, F)
    au = x.new_empty(M, 2 * F) if keep else None
    ws = _floats(_hip.load_block().nd_gated_ffn_workspace_floats(M, C, F, _DT[x.dtype]), x.device)
    _call('nd_gated_ffn', x.device, x.data_ptr(), _ld(x), w_in.data_ptr(), _ptr(b_in), w_out.data_ptr(), _ptr(b_out), _ptr(res),
          0 if res is None else _ld(res), y.data_ptr(), C, h.data_ptr(), _ptr(au), _ptr(ws), M, C, F, act, _DT[x.dtype])
    return y, h, au


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, b_in, w_out, b_out, res, act):
        C = x.shape[-1]
        xm, wi, wo = _matrix(x, C), _aligned(w_in), _aligned(w_out)
        rm = xm if res is x else (None if res is None else _matrix(res, C))
        if xm.shape[0]:
            need = ctx.needs_input_grad
            y, h, au = _launch_ffn(xm, wi, _aligned(b_in), wo, _aligned(b_out), rm, act, any(need[:3]), x.shape)
            h = h if need[3] else None                         # what no gradient wanted here is made from is not held
        else:
            y, h, au = xm.new_empty(x.shape), None, None
        ctx.save_for_backward(xm, wi, wo, h, au)
        ctx.act, ctx.shape = act, x.shape
        return y

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
                _call('nd_gated_ffn_bwd', x.device, g.data_ptr(), _ld(g), x.data_ptr(), _ld(x), w_in.data_ptr(), w_out.data_ptr(), _ptr(au),
                      _ptr(h), _ptr(dx), _ptr(dwi), _ptr(dbi), _ptr(dwo), _ptr(dbo), _ptr(dau), _ptr(ws), M, C,
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
    it for w_out's gradient and the pre-activations for those of x, w_in and b_in (3 F values a token for all)."""
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
    if C * F > 1 << 28 or C > 1 << 20 or F > 1 << 20:
        raise ValueError('weights of more than 2^28 elements, or more than 2^20 channels')
    if b_in is not None:
        _shape(b_in, 'b_in', 2 * F)
    if b_out is not None:
        _shape(b_out, 'b_out', C)
    if residual is not None:
        _shape(residual, 'residual', *x.shape)
    if x.numel() // C > 1 << 30:
        raise ValueError('more than 2^30 rows')
    _check('x', x, ('w_in', 'w_out', 'b_in', 'b_out', 'residual'), (w_in, w_out, b_in, b_out, residual))
    act = _ACTS[activation]
    if _wants_grad(x, w_in, b_in, w_out, b_out, residual):
        return _GatedFfn.apply(x, w_in, b_in, w_out, b_out, residual, act)
    if x.numel() == 0:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    xm = _matrix(x, C)
    res = xm if residual is x else (None if residual is None else _matrix(residual, C))
    return _launch_ffn(xm, _aligned(w_in), _aligned(b_in), _aligned(w_out), _aligned(b_out), res, act, False, x.shape)[0]
