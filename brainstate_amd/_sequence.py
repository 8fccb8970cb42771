"""Operators of sequence layers over the C ABI (torch device tensors in, device tensors out): the
gated delta rule, the norms around a block, the 8-bit integer product.  They have no counterpart
in brainstate; :mod:`brainstate_amd.ops` exports them.
"""
import struct

import torch
from torch.autograd import forward_ad

from . import _native as N
from . import _trace

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # enum bs_dtype
_CHUNK = 64
_DELTA_IN = struct.Struct('5P15q7if')      # bs_delta_in
_NORM_IN = struct.Struct('6P4q5i2f4x')     # bs_norm_in, to its whole 8 bytes


def _floating(name, t, dtype=None):
    """Number of the type of ``t`` (enum bs_dtype); raises for what is no floating GPU tensor."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{name} must be a tensor, not {type(t).__name__}')
    number = _DTYPES.get(t.dtype)
    if number is None:
        raise TypeError(f'{name}: dtype {t.dtype} not supported (float32, bfloat16, float16)')
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f'{name} is {t.dtype}, expected {dtype}')
    if not t.is_cuda:
        N.require_gpu()
        raise ValueError(f'{name} must be on the GPU')
    return number


def _wants_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return True
    return False


# a torch that cannot tell whether a transform is active has every operand looked at
_transforms_active = getattr(torch._C, '_are_functorch_transforms_active', lambda: True)


def _tangent(*ts):
    """Whether one of the operands carries a forward-mode tangent or is wrapped by a torch.func
    transform: there is no rule for either here, and the kernels would drop it."""
    inside = _transforms_active()
    if not inside and getattr(forward_ad, '_current_level', 0) < 0:
        return False
    for t in ts:
        if isinstance(t, torch.Tensor):
            if inside and torch._C._functorch.is_functorch_wrapped_tensor(t):
                return True
            if forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False


def _recorded(who, *ts):
    """Whether autograd records a call on the tensors ``ts``."""
    if _tangent(*ts):
        raise NotImplementedError(f'{who} has neither a forward-mode derivative nor a rule for '
                                  f'torch.func transforms: use torch.autograd')
    return _wants_grad(*ts)


def _address(t):
    if t is None:
        return None
    try:
        return t.data_ptr()
    except RuntimeError:        # a new tensor inside a torch.func transform, or a batched gradient
        if not torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise NotImplementedError('no rule for batched gradients: take them one by one')
        return N.ptr(t).value


# ------------------------------------------------------------------------- gated delta rule
def _delta_operands(q, k, v, g, beta, scale):
    """Checked operands as (views, bytes of bs_delta_in, sizes)."""
    qt = _floating('q', q)
    _floating('k', k, q.dtype)
    _floating('v', v, q.dtype)
    gt, bt = _floating('g', g), _floating('beta', beta)
    shape, vshape = q.shape, v.shape
    if len(shape) != 4 or shape != k.shape or len(vshape) != 4 or vshape[:2] != shape[:2]:
        raise ValueError(f'q, k [batch, tokens, key heads, dk] and v [batch, tokens, heads, dv]: '
                         f'got {tuple(shape)}, {tuple(k.shape)}, {tuple(vshape)}')
    b, t, hk, dk = shape
    hv, dv = vshape[2:]
    if hk < 1 or hv < 1 or hv % hk:
        raise ValueError(f'{hv} value heads for {hk} key heads')
    if not 1 <= dk <= 128 or not 1 <= dv <= 128:
        raise ValueError(f'head sizes {dk}, {dv} outside 1..128')
    if g.shape != vshape[:3] or beta.shape != vshape[:3]:
        raise ValueError(f'g and beta must be {tuple(vshape[:3])}: got {tuple(g.shape)}, '
                         f'{tuple(beta.shape)}')
    dev = q.device
    if not (dev == k.device == v.device == g.device == beta.device):
        raise ValueError('q, k, v, g and beta must be on one device')
    return _delta_pack(q, k, v, g, beta, scale, qt, gt, bt) + ((b, t, hk, hv, dk, dv),)


def _heads(x):
    """``x`` with a head's values side by side; any other strides are taken as they are."""
    at = x.stride()
    if (at[3] == 1 or x.shape[3] == 1) and at[1] < 1 << 23:
        return x
    # of one token the stride does not count, and contiguous() alone would leave it
    return x.squeeze(1).contiguous().unsqueeze(1) if x.shape[1] == 1 else x.contiguous()


def _delta_pack(q, k, v, g, beta, scale, qt, gt, bt):
    q, k, v = _heads(q), _heads(k), _heads(v)
    dk = q.shape[3]
    packed = _DELTA_IN.pack(
        _address(q), _address(k), _address(v), _address(g), _address(beta),
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride(), *beta.stride(),
        qt, gt, bt, q.shape[2], v.shape[2], dk, v.shape[3],
        dk ** -0.5 if scale is None else float(scale))
    return (q, k, v, g, beta), packed


def _states(name, s, n, hv, dk, dv, device):
    if not isinstance(s, torch.Tensor) or s.dtype != torch.float32:
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
    row's state, each its own; a negative one (or one from n on) marks an idle row, whose output is
    0.  Without it row b has state b.  Not differentiable."""
    if _trace.active() is not None:      # a for_loop's recording pass: state must not advance in it
        _trace.not_fusable()
    if _wants_grad(q, k, v, g, beta, state) or _tangent(q, k, v, g, beta, state, slots):
        raise ValueError('gated_delta_step updates its state in place and has no gradient: use '
                         'gated_delta_rule, or torch.no_grad()')
    one = isinstance(q, torch.Tensor) and q.dim() == 3
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
    N.check(N.lib().bs_gated_delta_step(packed, b, t, _address(state), state.shape[0],
                                        _address(slots), _address(o), N.raw_stream(q.device)),
            'bs_gated_delta_step')
    torch.autograd.graph.increment_version(state)     # autograd does not see the kernel's stores
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
        slots = n * -(-t // _CHUNK) if seq_offsets is None else t // _CHUNK + n if n else 0
        dvp = -(-dv // 32) * 32
        kept = (torch.empty((slots, hv, 64 if dk <= 64 else 128, dvp), dtype=torch.float32,
                            device=dev),
                torch.empty((slots, hv, _CHUNK, dvp), dtype=torch.float32, device=dev))
    lib = N.lib()
    nbytes = lib.bs_gated_delta_workspace_size(packed, n, t, seq_offsets is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    N.check(lib.bs_gated_delta_rule(
        packed, n, t, _address(seq_offsets), _address(initial_state), _address(final), _address(o),
        _address(kept[0]), _address(kept[1]), _address(ws), nbytes, N.raw_stream(dev)),
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
        _recorded('gated_delta_rule', go, gstate)
        *x, seq_offsets, kept_s, kept_u = ctx.saved_tensors
        held, packed = _delta_pack(*x, ctx.scale, *(_DTYPES[x[i].dtype] for i in (0, 3, 4)))
        (b, t, hk, dk), (hv, dv) = x[0].shape, x[2].shape[2:]
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
            packed, n, t, _address(seq_offsets), _address(go), _address(gstate), _address(kept_s),
            _address(kept_u), *(_address(y) for y in grads), _address(ds), _address(ws), nbytes,
            N.raw_stream(dev)), 'bs_gated_delta_rule_grad')
        return (*grads, ds, None, None)


def gated_delta_rule(q, k, v, g, beta, scale=None, initial_state=None, seq_offsets=None):
    """Whole sequences through the gated delta rule (see :func:`gated_delta_step`), in chunks of
    64 tokens -> (o [batch, tokens, heads, dv], final states [sequences, heads, dk, dv] float32).

    ``q``, ``k`` [batch, tokens, key heads, dk], ``v`` [batch, tokens, heads, dv], ``g`` and
    ``beta`` [batch, tokens, heads]; ``initial_state`` float32, None for zeros.  With
    ``seq_offsets`` (int32 [sequences + 1], ascending) the sequences are packed end to end into
    one batch row; tokens outside all of them give 0.  Differentiable in everything but
    ``seq_offsets``, in reverse mode."""
    if _recorded('gated_delta_rule', q, k, v, g, beta, initial_state, seq_offsets):
        return _DeltaRule.apply(q, k, v, g, beta, initial_state, scale, seq_offsets)
    o, final, _ = _delta_forward(q, k, v, g, beta, scale, initial_state, seq_offsets, False)
    return o, final


# ------------------------------------------------------------------------- norms around a block
def _rows(t, dim):
    """``t`` [.., dim] as rows with their values side by side."""
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    return t if t.stride(1) == 1 or dim == 1 else t.contiguous()


def _norm_operands(y, post, gate, scale, residual, pre, eps):
    """Checked operands as (row views, bytes of bs_norm_in, rows, dim)."""
    _floating('y', y)
    shape, dtype, dev = y.shape, y.dtype, y.device
    if len(shape) < 1 or not 1 <= shape[-1] <= 16384:
        raise ValueError(f'y [.., dim] with dim in 1..16384: got {tuple(shape)}')
    dim = shape[-1]
    for name, t in (('gate', gate), ('residual', residual)):
        if t is not None:
            _floating(name, t, dtype)
            if t.shape != shape or t.device != dev:
                raise ValueError(f'{name} must be {tuple(shape)} on {dev}: got '
                                 f'{tuple(t.shape)} on {t.device}')
    if scale is not None and not isinstance(scale, torch.Tensor):
        scale = float(scale)
    for name, t in (('post_weight', post), ('scale', scale), ('pre_weight', pre)):
        if t is not None and t.__class__ is not float:
            _floating(name, t)
            if t.shape != (dim,) or t.device != dev:
                raise ValueError(f'{name} must be [{dim}] on {dev}: got {tuple(t.shape)} on '
                                 f'{t.device}')
    return _norm_pack(y, post, gate, scale, residual, pre, eps)


def _norm_pack(y, post, gate, scale, residual, pre, eps):
    dim, value = y.shape[-1], 1.0
    if scale.__class__ is float:
        scale, value = None, scale
    acts = [t if t is None else _rows(t, dim) for t in (y, gate, residual)]
    weights = [t if t is None else t.contiguous() for t in (post, scale, pre)]
    y_at, gate_at, residual_at = [_address(t) or 0 for t in acts]
    post_at, scale_at, pre_at = [_address(t) or 0 for t in weights]
    rows = acts[0].shape[0]
    packed = _NORM_IN.pack(
        y_at, post_at, gate_at, scale_at, residual_at, pre_at,
        *[0 if t is None else t.stride(0) for t in acts], rows, dim, _DTYPES[y.dtype],
        *[0 if t is None else _DTYPES[t.dtype] for t in weights], eps, value)
    return (acts, weights), packed, rows, dim


def _norm_forward(y, post, gate, scale, residual, pre, eps):
    held, packed, _, _ = _norm_operands(y, post, gate, scale, residual, pre, eps)
    stream = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    normed = torch.empty_like(stream) if pre is not None else None
    N.check(N.lib().bs_norm_gate_residual(packed, _address(stream), _address(normed),
                                          N.raw_stream(y.device)), 'bs_norm_gate_residual')
    return stream, normed


class _NormGateResidual(torch.autograd.Function):
    """norm_gate_residual with its gradients, formed from the operands alone."""

    @staticmethod
    def forward(ctx, y, post, gate, scale, residual, pre, eps):
        ctx.eps = eps
        ctx.value = None if scale is None or isinstance(scale, torch.Tensor) else float(scale)
        ctx.save_for_backward(y, post, gate, scale if ctx.value is None else None, residual, pre)
        ctx.set_materialize_grads(False)
        return _norm_forward(y, post, gate, scale, residual, pre, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gs, gn):
        _recorded('norm_gate_residual', gs, gn)
        y, post, gate, scale, residual, pre = x = ctx.saved_tensors
        held, packed, rows, dim = _norm_pack(
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
            packed, _address(gs), _address(gn), *(_address(t) for t in grads), _address(ws), nbytes,
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
    ``stream`` is rounded.  Differentiable in every tensor, in reverse mode."""
    if _recorded('norm_gate_residual', y, post_weight, gate, scale, residual, pre_weight):
        return _NormGateResidual.apply(y, post_weight, gate, scale, residual, pre_weight, eps)
    return _norm_forward(y, post_weight, gate, scale, residual, pre_weight, eps)


# ------------------------------------------------------------------------- 8-bit integer product
def _no_grad(who, *ts):
    if _wants_grad(*ts) or _tangent(*ts):
        raise ValueError(f'{who} has no gradient, nor a rule for torch.func transforms: detach its '
                         f'operands or use torch.no_grad()')


def _channels(name, t, n, dev):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (n,) or t.device != dev:
        raise ValueError(f'{name} must be float32 [{n}] on {dev}')
    return t.contiguous()


def int8_quantize(x):
    """Rows of ``x`` [.., k] in 8 bits -> (int8 [.., k], float32 scales [..]): scale
    ``max|x| / 127``, integers ``127 x / max|x|`` rounded to nearest (ties to even).  A row of zeros
    has scale 0.  Not differentiable."""
    _floating('x', x)
    _no_grad('int8_quantize', x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 65536:
        raise ValueError(f'x [.., k] with k in 1..65536: got {tuple(x.shape)}')
    k = x.shape[-1]
    rows = _rows(x, k)
    x8 = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    N.check(N.lib().bs_int8_quantize(_address(rows), _DTYPES[x.dtype], rows.shape[0], k,
                                     rows.stride(0), _address(x8), _address(scale),
                                     N.raw_stream(x.device)), 'bs_int8_quantize')
    return x8, scale


def _int8_product(x, x_scale, w8, w_scale, bias, out_dtype):
    dev = x.device
    if not isinstance(w8, torch.Tensor) or w8.dtype != torch.int8 or w8.dim() != 2 or w8.device != dev:
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
        _address(rows), _DTYPES.get(x.dtype, 0), rows.stride(0), _address(x_scale), m, k, n,
        _address(w8), _address(w_scale), _address(bias),
        0 if bias is None else _DTYPES[bias.dtype], _address(y), _DTYPES[out_dtype],
        _address(ws), nbytes, N.raw_stream(dev)), 'bs_int8_linear')
    return y


def int8_matmul(x8, x_scale, w8, w_scale, bias=None, out_dtype=torch.float32):
    """``x_scale[m] * w_scale[n] * sum_k x8[m, k] * w8[n, k] + bias[n]`` with exact sums: tokens
    ``x8`` int8 [.., k] with a scale each (:func:`int8_quantize`), weights ``w8`` int8 [n, k] with
    a scale for each channel.  Not differentiable."""
    if not isinstance(x8, torch.Tensor) or x8.dtype != torch.int8 or not x8.is_cuda:
        N.require_gpu()
        raise TypeError('x8 must be an int8 tensor on the GPU')
    if out_dtype not in _DTYPES:
        raise TypeError(f'out_dtype {out_dtype} not supported (float32, bfloat16, float16)')
    _no_grad('int8_matmul', x8, x_scale, w8, w_scale, bias)
    return _int8_product(x8, x_scale, w8, w_scale, bias, out_dtype)


def int8_linear(x, w8, w_scale, bias=None):
    """``x`` [.., k] times 8-bit weights ``w8`` [n, k] with a scale for each channel -> [.., n] of
    the type of ``x``: its rows are quantized on the way (:func:`int8_quantize`), the sums are
    exact, ``bias`` [n] is added in 32 bits.  Not differentiable."""
    _floating('x', x)
    _no_grad('int8_linear', x, w8, w_scale, bias)
    return _int8_product(x, None, w8, w_scale, bias, x.dtype)
