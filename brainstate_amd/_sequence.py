"""Operators of sequence layers over the C ABI (torch device tensors in, device tensors out): the
gated delta rule, the norms around a block, the 8-bit integer product.  They have no counterpart
in brainstate; :mod:`brainstate_amd.ops` exports them.
"""
import struct

import torch

from . import _native as N

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # enum bs_dtype
_CHUNK = 64
_DELTA_IN = struct.Struct('5P15q7if')      # bs_delta_in
_NORM_IN = struct.Struct('6P4q5i2f')       # bs_norm_in


def _floating(name, t, dtype=None):
    if not torch.is_tensor(t):
        raise TypeError(f'{name} must be a tensor, not {type(t).__name__}')
    if t.dtype not in _DTYPES:
        raise TypeError(f'{name}: dtype {t.dtype} not supported (float32, bfloat16, float16)')
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f'{name} is {t.dtype}, expected {dtype}')
    if not t.is_cuda:
        raise ValueError(f'{name} must be on the GPU')


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ------------------------------------------------------------------------- gated delta rule
def _delta_operands(q, k, v, g, beta, scale):
    """Checked operands as (views, bytes of bs_delta_in, sizes).  A head's values have to lie
    side by side; any other strides are taken as they are."""
    _floating('q', q)
    for name, t in (('k', k), ('v', v)):
        _floating(name, t, q.dtype)
    for name, t in (('g', g), ('beta', beta)):
        _floating(name, t)
    if q.dim() != 4 or q.shape != k.shape or v.dim() != 4 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f'q, k [batch, tokens, key heads, dk] and v [batch, tokens, heads, dv]: '
                         f'got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    b, t, hk, dk = q.shape
    hv, dv = v.shape[2:]
    if hk < 1 or hv < 1 or hv % hk:
        raise ValueError(f'{hv} value heads for {hk} key heads')
    if not 1 <= dk <= 128 or not 1 <= dv <= 128:
        raise ValueError(f'head sizes {dk}, {dv} outside 1..128')
    if g.shape != v.shape[:3] or beta.shape != v.shape[:3]:
        raise ValueError(f'g and beta must be {tuple(v.shape[:3])}: got {tuple(g.shape)}, '
                         f'{tuple(beta.shape)}')
    dev = q.device
    if any(x.device != dev for x in (k, v, g, beta)):
        raise ValueError('q, k, v, g and beta must be on one device')
    q, k, v = (x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous() for x in (q, k, v))
    q, k, v = (x if x.stride(1) < 1 << 23 else x.contiguous() for x in (q, k, v))
    scale = dk ** -0.5 if scale is None else float(scale)
    packed = _DELTA_IN.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride(), *beta.stride(),
        _DTYPES[q.dtype], _DTYPES[g.dtype], _DTYPES[beta.dtype], hk, hv, dk, dv, scale)
    return (q, k, v, g, beta), packed, (b, t, hk, hv, dk, dv)


def _states(name, s, n, hv, dk, dv, device):
    if not torch.is_tensor(s) or s.dtype != torch.float32:
        raise TypeError(f'{name} must be a float32 tensor')
    if s.dim() != 4 or tuple(s.shape[1:]) != (hv, dk, dv) or n is not None and s.shape[0] != n:
        raise ValueError(f'{name} must be [{"n" if n is None else n}, {hv}, {dk}, {dv}]: got '
                         f'{tuple(s.shape)}')
    if s.device != device:
        raise ValueError(f'{name} must be on {device}')


def gated_delta_step(q, k, v, g, beta, state, slots=None, scale=None):
    """Tokens of running sequences through the gated delta rule, ``state`` updated in place.

    Per head ``S' = exp(g) S``, ``u = beta (v - S'^T k)``, ``S = S' + k u^T``,
    ``o = scale S^T q`` (``scale`` None: dk^-0.5), in 32 bits.

    ``q``, ``k`` [batch, key heads, dk], ``v`` [batch, heads, dv], ``g`` (log decay) and ``beta``
    [batch, heads]; each may have a dimension of tokens after the batch, which are taken in
    order.  ``state`` [n, heads, dk, dv] float32, contiguous.  ``slots`` [batch] int32 names each
    row's state; a negative one (or one from n on) marks an idle row, whose output is 0.  Without
    it row b has state b.  Not differentiable."""
    N.require_gpu()
    if _wants_grad(q, k, v, g, beta, state):
        raise ValueError('gated_delta_step updates its state in place and has no gradient: use '
                         'gated_delta_rule, or torch.no_grad()')
    one = torch.is_tensor(q) and q.dim() == 3
    if one:
        if v.dim() != 3 or k.dim() != 3 or g.dim() != 2 or beta.dim() != 2:
            raise ValueError('q, k, v, g and beta must all have a dimension of tokens, or none')
        q, k, v, g, beta = (x.unsqueeze(1) for x in (q, k, v, g, beta))
    keep, packed, (b, t, _, hv, dk, dv) = _delta_operands(q, k, v, g, beta, scale)
    _states('state', state, None, hv, dk, dv, q.device)
    if not state.is_contiguous():
        raise ValueError('state must be contiguous (it is updated in place)')
    if slots is None:
        if state.shape[0] != b:
            raise ValueError(f'{state.shape[0]} states for {b} rows without slots')
    elif slots.dtype != torch.int32 or slots.shape != (b,) or slots.device != q.device:
        raise ValueError(f'slots must be int32 [{b}] on {q.device}')
    else:
        slots = slots.contiguous()
    o = torch.empty((b, t, hv, dv), dtype=q.dtype, device=q.device)
    N.check(N.lib().bs_gated_delta_step(packed, b, t, state.data_ptr(), state.shape[0],
                                        N.ptr(slots), o.data_ptr(), N.raw_stream(q.device)),
            'bs_gated_delta_step')
    return o.squeeze(1) if one else o


def _delta_forward(q, k, v, g, beta, scale, initial_state, seq_offsets, keep):
    """(o, final state, what the backward pass needs of it or None)."""
    held, packed, (b, t, hk, hv, dk, dv) = _delta_operands(q, k, v, g, beta, scale)
    dev = q.device
    n = b
    if seq_offsets is not None:
        if b != 1:
            raise ValueError(f'packed sequences lie in one batch row, not {b}')
        if seq_offsets.dtype != torch.int32 or seq_offsets.dim() != 1 or \
                seq_offsets.numel() < 1 or seq_offsets.device != dev:
            raise ValueError(f'seq_offsets must be int32 [sequences + 1] on {dev}')
        seq_offsets = seq_offsets.contiguous()
        n = seq_offsets.numel() - 1
    if initial_state is not None:
        _states('initial_state', initial_state, n, hv, dk, dv, dev)
        initial_state = initial_state.contiguous()
    o = torch.empty((b, t, hv, dv), dtype=q.dtype, device=dev)
    final = torch.empty((n, hv, dk, dv), dtype=torch.float32, device=dev)
    kept = (None, None)
    if keep:
        slots = t // _CHUNK + n if seq_offsets is not None else n * -(-t // _CHUNK)
        dvp = -(-dv // 32) * 32
        kept = (torch.empty((slots, hv, 64 if dk <= 64 else 128, dvp), dtype=torch.float32,
                            device=dev),
                torch.empty((slots, hv, _CHUNK, dvp), dtype=torch.float32, device=dev))
    lib = N.lib()
    nbytes = lib.bs_gated_delta_workspace_size(packed, n, t, seq_offsets is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    N.check(lib.bs_gated_delta_rule(
        packed, n, t, N.ptr(seq_offsets), N.ptr(initial_state), final.data_ptr(), o.data_ptr(),
        N.ptr(kept[0]), N.ptr(kept[1]), ws.data_ptr(), nbytes, N.raw_stream(dev)),
        'bs_gated_delta_rule')
    return o, final, kept


class _DeltaRule(torch.autograd.Function):
    """gated_delta_rule with its gradients; the states before every chunk and the values written
    are kept for them."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state, scale, seq_offsets):
        o, final, kept = _delta_forward(q, k, v, g, beta, scale, initial_state, seq_offsets, True)
        ctx.save_for_backward(q, k, v, g, beta, seq_offsets, *kept)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go, gstate):
        *x, seq_offsets, kept_s, kept_u = ctx.saved_tensors
        held, packed, (b, t, hk, hv, dk, dv) = _delta_operands(*x, ctx.scale)
        dev = x[0].device
        n = b
        if seq_offsets is not None:
            seq_offsets, n = seq_offsets.contiguous(), seq_offsets.numel() - 1
        go = torch.zeros(x[2].shape, dtype=x[2].dtype, device=dev) if go is None else \
            go.contiguous()
        gstate = None if gstate is None else gstate.contiguous()
        grads = [torch.empty(y.shape, dtype=y.dtype, device=dev) for y in x]
        ds = torch.empty((n, hv, dk, dv), dtype=torch.float32, device=dev) \
            if ctx.needs_input_grad[5] else None
        lib = N.lib()
        nbytes = lib.bs_gated_delta_grad_workspace_size(packed, n, t, seq_offsets is not None)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        N.check(lib.bs_gated_delta_rule_grad(
            packed, n, t, N.ptr(seq_offsets), go.data_ptr(), N.ptr(gstate), kept_s.data_ptr(),
            kept_u.data_ptr(), *(y.data_ptr() for y in grads), N.ptr(ds), ws.data_ptr(), nbytes,
            N.raw_stream(dev)), 'bs_gated_delta_rule_grad')
        return (*grads, ds, None, None)


def gated_delta_rule(q, k, v, g, beta, scale=None, initial_state=None, seq_offsets=None):
    """Whole sequences through the gated delta rule (see :func:`gated_delta_step`), in chunks of
    64 tokens -> (o [batch, tokens, heads, dv], final states [sequences, heads, dk, dv] float32).

    ``q``, ``k`` [batch, tokens, key heads, dk], ``v`` [batch, tokens, heads, dv], ``g`` and
    ``beta`` [batch, tokens, heads]; ``initial_state`` float32, None for zeros.  With
    ``seq_offsets`` (int32 [sequences + 1], ascending) the sequences are packed end to end into
    one batch row; tokens outside all of them give 0.  Differentiable in everything but
    ``seq_offsets``."""
    N.require_gpu()
    if _wants_grad(q, k, v, g, beta, initial_state):
        return _DeltaRule.apply(q, k, v, g, beta, initial_state, scale, seq_offsets)
    o, final, _ = _delta_forward(q, k, v, g, beta, scale, initial_state, seq_offsets, False)
    return o, final


# ------------------------------------------------------------------------- norms around a block
def _rows(t, dim):
    """``t`` [.., dim] as rows with their values side by side."""
    t = t.reshape(-1, dim)
    return t if t.stride(1) == 1 or dim == 1 else t.contiguous()


def _norm_operands(y, post, gate, scale, residual, pre, eps):
    """Checked operands as (row views, bytes of bs_norm_in, rows, dim)."""
    _floating('y', y)
    if y.dim() < 1 or not 1 <= y.shape[-1] <= 16384:
        raise ValueError(f'y [.., dim] with dim in 1..16384: got {tuple(y.shape)}')
    dim, dev = y.shape[-1], y.device
    for name, t in (('gate', gate), ('residual', residual)):
        if t is not None:
            _floating(name, t, y.dtype)
            if t.shape != y.shape or t.device != dev:
                raise ValueError(f'{name} must be {tuple(y.shape)} on {dev}: got '
                                 f'{tuple(t.shape)} on {t.device}')
    value = 1.0
    if scale is not None and not torch.is_tensor(scale):
        scale, value = None, float(scale)
    weights = []
    for name, t in (('post_weight', post), ('scale', scale), ('pre_weight', pre)):
        if t is not None:
            _floating(name, t)
            if t.shape != (dim,) or t.device != dev:
                raise ValueError(f'{name} must be [{dim}] on {dev}: got {tuple(t.shape)} on '
                                 f'{t.device}')
            t = t.contiguous()
        weights.append(t)
    acts = [t if t is None else _rows(t, dim) for t in (y, gate, residual)]
    rows = acts[0].shape[0]
    at = [0 if t is None else t.data_ptr() for t in acts + weights]
    packed = _NORM_IN.pack(
        at[0], at[3], at[1], at[4], at[2], at[5],
        *(0 if t is None else t.stride(0) for t in acts), rows, dim, _DTYPES[y.dtype],
        *(0 if t is None else _DTYPES[t.dtype] for t in weights), eps, value)
    return (acts, weights), packed, rows, dim


def _norm_forward(y, post, gate, scale, residual, pre, eps):
    held, packed, _, _ = _norm_operands(y, post, gate, scale, residual, pre, eps)
    stream = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    normed = torch.empty_like(stream) if pre is not None else None
    N.check(N.lib().bs_norm_gate_residual(packed, stream.data_ptr(), N.ptr(normed),
                                          N.raw_stream(y.device)), 'bs_norm_gate_residual')
    return stream, normed


class _NormGateResidual(torch.autograd.Function):
    """norm_gate_residual with its gradients, formed from the operands alone."""

    @staticmethod
    def forward(ctx, y, post, gate, scale, residual, pre, eps):
        ctx.eps = eps
        ctx.value = None if torch.is_tensor(scale) else scale
        ctx.save_for_backward(y, post, gate, scale if ctx.value is None else None, residual, pre)
        ctx.set_materialize_grads(False)
        return _norm_forward(y, post, gate, scale, residual, pre, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gs, gn):
        y, post, gate, scale, residual, pre = x = ctx.saved_tensors
        held, packed, rows, dim = _norm_operands(
            y, post, gate, scale if ctx.value is None else ctx.value, residual, pre, ctx.eps)
        dev = y.device
        gs, gn = (None if t is None else t.contiguous() for t in (gs, gn))
        grads = [torch.empty(t.shape, dtype=t.dtype, device=dev) if need else None
                 for t, need in zip(x, ctx.needs_input_grad)]
        lib = N.lib()
        nbytes, ws = 0, None
        if any(grads[i] is not None for i in (1, 3, 5)):
            nbytes = lib.bs_norm_grad_workspace_size(rows, dim)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        N.check(lib.bs_norm_gate_residual_grad(
            packed, N.ptr(gs), N.ptr(gn), *(N.ptr(t) for t in grads), N.ptr(ws), nbytes,
            N.raw_stream(dev)), 'bs_norm_gate_residual_grad')
        return (*grads, None)


def norm_gate_residual(y, post_weight=None, gate=None, scale=None, residual=None,
                       pre_weight=None, eps=1e-6):
    """What stands between a block's output and the next block, in one pass over rows [.., dim]:

    ``stream = residual + scale * silu(gate) * (r(y) * post_weight)`` and
    ``normed = r(stream) * pre_weight`` with ``r(x) = x / sqrt(mean(x^2) + eps)``
    -> (stream, normed), (stream, None) without ``pre_weight``.

    ``y``, ``gate`` and ``residual`` have one shape and type; ``post_weight``, ``scale`` and
    ``pre_weight`` are [dim] of any floating type, ``scale`` may be a number.  Any of them may be
    left out, with its norm or factor.  Sums are in 32 bits; ``normed`` is formed before
    ``stream`` is rounded.  Differentiable in every tensor."""
    N.require_gpu()
    if _wants_grad(y, post_weight, gate, scale if torch.is_tensor(scale) else None, residual,
                   pre_weight):
        return _NormGateResidual.apply(y, post_weight, gate, scale, residual, pre_weight, eps)
    return _norm_forward(y, post_weight, gate, scale, residual, pre_weight, eps)


# ------------------------------------------------------------------------- 8-bit integer product
def _no_grad(who, *ts):
    if _wants_grad(*ts):
        raise ValueError(f'{who} has no gradient: detach its operands or use torch.no_grad()')


def _channels(name, t, n, dev):
    if not torch.is_tensor(t) or t.dtype != torch.float32 or t.shape != (n,) or t.device != dev:
        raise ValueError(f'{name} must be float32 [{n}] on {dev}')
    return t.contiguous()


def int8_quantize(x):
    """Rows of ``x`` [.., k] in 8 bits -> (int8 [.., k], float32 scales [..]): scale
    ``max|x| / 127``, integers ``127 x / max|x|`` rounded to nearest (ties to even).  A row of zeros
    has scale 0.  Not differentiable."""
    N.require_gpu()
    _floating('x', x)
    _no_grad('int8_quantize', x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 65536:
        raise ValueError(f'x [.., k] with k in 1..65536: got {tuple(x.shape)}')
    k = x.shape[-1]
    rows = _rows(x, k)
    x8 = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    N.check(N.lib().bs_int8_quantize(rows.data_ptr(), _DTYPES[x.dtype], rows.shape[0], k,
                                     rows.stride(0), x8.data_ptr(), scale.data_ptr(),
                                     N.raw_stream(x.device)), 'bs_int8_quantize')
    return x8, scale


def _int8_product(x, x_scale, w8, w_scale, bias, out_dtype):
    dev = x.device
    if not torch.is_tensor(w8) or w8.dtype != torch.int8 or w8.dim() != 2 or w8.device != dev:
        raise ValueError(f'w8 must be int8 [channels, k] on {dev}')
    n, k = w8.shape
    if x.dim() < 1 or x.shape[-1] != k or not 1 <= k <= 65536:
        raise ValueError(f'tokens [.., {k}] with k in 1..65536 expected: got {tuple(x.shape)}')
    w8 = w8.contiguous()
    w_scale = _channels('w_scale', w_scale, n, dev)
    if bias is not None:
        _floating('bias', bias)
        if bias.shape != (n,) or bias.device != dev:
            raise ValueError(f'bias must be [{n}] on {dev}: got {tuple(bias.shape)}')
        bias = bias.contiguous()
    if x_scale is None:
        rows = _rows(x, k)
    else:
        if x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:-1] or \
                x_scale.device != dev:
            raise ValueError(f'x_scale must be float32 {tuple(x.shape[:-1])} on {dev}')
        rows, x_scale = x.reshape(-1, k).contiguous(), x_scale.contiguous()
    m = rows.shape[0]
    y = torch.empty(x.shape[:-1] + (n,), dtype=out_dtype, device=dev)
    nbytes = m * (-(-k // 128) * 128 + 4)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    N.check(N.lib().bs_int8_linear(
        rows.data_ptr(), _DTYPES.get(x.dtype, 0), rows.stride(0), N.ptr(x_scale), m, k, n,
        w8.data_ptr(), w_scale.data_ptr(), N.ptr(bias),
        0 if bias is None else _DTYPES[bias.dtype], y.data_ptr(), _DTYPES[out_dtype],
        ws.data_ptr(), nbytes, N.raw_stream(dev)), 'bs_int8_linear')
    return y


def int8_matmul(x8, x_scale, w8, w_scale, bias=None, out_dtype=torch.float32):
    """``x_scale[m] * w_scale[n] * sum_k x8[m, k] * w8[n, k] + bias[n]`` with exact sums: tokens
    ``x8`` int8 [.., k] with a scale each (:func:`int8_quantize`), weights ``w8`` int8 [n, k] with
    a scale for each channel.  Not differentiable."""
    N.require_gpu()
    if not torch.is_tensor(x8) or x8.dtype != torch.int8 or not x8.is_cuda:
        raise TypeError('x8 must be an int8 tensor on the GPU')
    if out_dtype not in _DTYPES:
        raise TypeError(f'out_dtype {out_dtype} not supported (float32, bfloat16, float16)')
    _no_grad('int8_matmul', x_scale, w_scale, bias)
    return _int8_product(x8, x_scale, w8, w_scale, bias, out_dtype)


def int8_linear(x, w8, w_scale, bias=None):
    """``x`` [.., k] times 8-bit weights ``w8`` [n, k] with a scale for each channel -> [.., n] of
    the type of ``x``: its rows are quantized on the way (:func:`int8_quantize`), the sums are
    exact, ``bias`` [n] is added in 32 bits.  Not differentiable."""
    N.require_gpu()
    _floating('x', x)
    _no_grad('int8_linear', x, w_scale, bias)
    return _int8_product(x, None, w8, w_scale, bias, x.dtype)
