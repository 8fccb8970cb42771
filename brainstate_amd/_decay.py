"""Decay attention over the C ABI: linear attention whose state fades at a rate of its own for each
head (no counterpart in brainstate); :mod:`brainstate_amd.ops` exports it.
"""
import torch

from . import _native as N
from . import _trace
from ._sequence import (_DELTA_IN, _DTYPES, _address, _fits, _floating, _heads, _like, _once,
                        _recorded, _states, _tangent, _wants_grad)


def _operands(q, k, v, g, scale):
    """Checked operands as (tensors to hold, bytes of bs_delta_in, sizes)."""
    _floating('q', q)
    _floating('k', k, q.dtype)
    _floating('v', v, q.dtype)
    _floating('g', g)
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
    if g.shape != vshape[:3] and g.shape != (hv,):
        raise ValueError(f'g must be {tuple(vshape[:3])} or [{hv}]: got {tuple(g.shape)}')
    _fits(b, 'batch rows')
    _fits(t, 'tokens')
    dev = q.device
    if not (dev == k.device == v.device == g.device):
        raise ValueError('q, k, v and g must be on one device')
    return _pack(q, k, v, g, scale) + ((b, t, hk, hv, dk, dv),)


def _pack(q, k, v, g, scale):
    q, k, v = _heads(q), _heads(k), _heads(v)
    dk, g_stride = q.shape[3], g.stride() if g.dim() == 3 else (0, 0, g.stride(0))
    packed = _DELTA_IN.pack(
        _address(q), _address(k), _address(v), _address(g), 0, *q.stride()[:3], *k.stride()[:3],
        *v.stride()[:3], *g_stride, 0, 0, 0, _DTYPES[q.dtype], _DTYPES[g.dtype], 0, q.shape[2],
        v.shape[2], dk, v.shape[3], dk ** -0.5 if scale is None else float(scale))
    return (q, k, v, g), packed


def decay_attention_step(q, k, v, g, state, slots=None, scale=None):
    """Tokens of running sequences through decay attention, ``state`` updated in place.

    Per head ``S = exp(g) S + k v^T``, ``o = scale S^T q`` (``scale`` None: dk^-0.5), in 32 bits.

    ``q``, ``k`` [batch, key heads, dk], ``v`` [batch, heads, dv], ``g`` (log decay) [batch, heads]
    or [heads]; each but a [heads] ``g`` may have a dimension of tokens after the batch, which are
    taken in order.  ``state`` [n, heads, dk, dv] float32, contiguous.  ``slots`` [batch] int32 names
    each row's state, each its own; a negative one (or one from n on) marks an idle row, whose
    output is 0.  Without it row b has state b.  Not differentiable."""
    if _trace.active() is not None:      # a for_loop's recording pass: state must not advance in it
        _trace.not_fusable()
    if _wants_grad(q, k, v, g, state) or _tangent(q, k, v, g, state, slots):
        raise ValueError('decay_attention_step updates its state in place and has no gradient: use '
                         'decay_attention, or torch.no_grad()')
    one = isinstance(q, torch.Tensor) and q.dim() == 3
    if one:
        if v.dim() != 3 or k.dim() != 3 or g.dim() not in (1, 2):
            raise ValueError('q, k, v and g must all have a dimension of tokens, or none')
        q, k, v = (x.unsqueeze(1) for x in (q, k, v))
        g = g.unsqueeze(1) if g.dim() == 2 else g
    keep, packed, (b, t, _, hv, dk, dv) = _operands(q, k, v, g, scale)
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
    N.call('bs_decay_attention_step', q.device, packed, b, t, _address(state), state.shape[0],
           _address(slots), _address(o))
    torch.autograd.graph.increment_version(state)     # autograd does not see the kernel's stores
    return o.squeeze(1) if one else o


def _forward(q, k, v, g, scale, initial_state, seq_offsets, keep):
    """(o, final state, what the backward pass needs of it: ``keep`` 0 nothing, 1 without the
    gradient of g, 2 with it)."""
    held, packed, (b, t, hk, hv, dk, dv) = _operands(q, k, v, g, scale)
    dev = q.device
    n = b
    if seq_offsets is not None:
        if b != 1:
            raise ValueError(f'packed sequences lie in one batch row, not {b}')
        if seq_offsets.dtype != torch.int32 or seq_offsets.dim() != 1 or \
                seq_offsets.numel() < 1 or seq_offsets.device != dev:
            raise ValueError(f'seq_offsets must be int32 [sequences + 1] on {dev}')
        n = seq_offsets.numel() - 1
        _fits(n, 'sequences')
        seq_offsets = seq_offsets.contiguous()
    if initial_state is not None:
        _states('initial_state', initial_state, n, hv, dk, dv, dev)
        initial_state = initial_state.contiguous()
    o = torch.empty((b, t, hv, dv), dtype=q.dtype, device=dev)
    final = torch.empty((n, hv, dk, dv), dtype=torch.float32, device=dev)
    lib, is_packed = N.lib(), seq_offsets is not None
    nbytes = lib.bs_decay_attention_kept_size(packed, n, t, is_packed, keep)
    kept = torch.empty(nbytes, dtype=torch.uint8, device=dev) if keep else None
    nbytes = lib.bs_decay_attention_workspace_size(packed, n, t, is_packed, keep)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    N.call('bs_decay_attention', dev, packed, n, t, _address(seq_offsets), _address(initial_state),
           _address(final), _address(o), _address(kept), keep, _address(ws), nbytes)
    return o, final, kept


class _DecayAttention(torch.autograd.Function):
    """decay_attention with its gradients, formed from the operands and the states between the
    forward pass's segments."""

    @staticmethod
    def forward(ctx, q, k, v, g, initial_state, scale, seq_offsets):
        o, final, kept = _forward(q, k, v, g, scale, initial_state, seq_offsets,
                                  2 if ctx.needs_input_grad[3] else 1)
        ctx.save_for_backward(q, k, v, g, initial_state, seq_offsets, kept)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @_once
    def backward(ctx, go, gstate):
        _recorded('decay_attention', go, gstate)
        *x, initial_state, seq_offsets, kept = ctx.saved_tensors
        held, packed = _pack(*x, ctx.scale)
        (b, t, hk, dk), (hv, dv) = x[0].shape, x[2].shape[2:]
        dev = x[0].device
        n = b
        if seq_offsets is not None:
            seq_offsets, n = seq_offsets.contiguous(), seq_offsets.numel() - 1
        if initial_state is not None:
            initial_state = initial_state.contiguous()
        go = _like(x[2]).zero_() if go is None else go.contiguous()
        gstate = None if gstate is None else gstate.contiguous()
        decays = ctx.needs_input_grad[3]
        grads = [_like(y) for y in x[:3 + decays]]
        ds = torch.empty((n, hv, dk, dv), dtype=torch.float32, device=dev) \
            if ctx.needs_input_grad[4] else None
        nbytes = N.lib().bs_decay_attention_grad_workspace_size(
            packed, n, t, seq_offsets is not None, decays)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        if not decays:
            grads.append(None)
        N.call('bs_decay_attention_grad', dev, packed, n, t, _address(seq_offsets), _address(go),
               _address(gstate), _address(initial_state), _address(kept),
               *(_address(y) for y in grads), x[3].dim() == 1, _address(ds), _address(ws), nbytes)
        return (*grads, ds, None, None)


def decay_attention(q, k, v, g, scale=None, initial_state=None, seq_offsets=None):
    """Whole sequences through decay attention (see :func:`decay_attention_step`), in chunks of 64
    tokens -> (o [batch, tokens, heads, dv], final states [sequences, heads, dk, dv] float32).

    ``q``, ``k`` [batch, tokens, key heads, dk], ``v`` [batch, tokens, heads, dv], ``g`` (log decay)
    [batch, tokens, heads], or [heads] for one rate a head; ``initial_state`` float32, None for
    zeros.  With ``seq_offsets`` (int32 [sequences + 1], ascending) the sequences are packed end to
    end into one batch row; tokens outside all of them give 0.  Differentiable in everything but
    ``seq_offsets``, in reverse mode."""
    if _recorded('decay_attention', q, k, v, g, initial_state, seq_offsets):
        return _DecayAttention.apply(q, k, v, g, initial_state, scale, seq_offsets)
    o, final, _ = _forward(q, k, v, g, scale, initial_state, seq_offsets, False)
    return o, final
