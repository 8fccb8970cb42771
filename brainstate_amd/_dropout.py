"""Dropout and layer norm over the C ABI (no counterpart in brainstate's spiking step);
:mod:`brainstate_amd.ops` exports them.
"""
import struct

import torch

from . import _native as N
from ._sequence import _DTYPES, _address, _fits, _floating, _like, _once, _recorded, _rows

_NORM_IN = struct.Struct('5P3qQ4i2I2f')      # bs_layer_norm_in


def _chance(p, seed, site, dev):
    """(drop, scale of what is kept, seed, tensor that holds it or None) of checked arguments."""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f'p must be in [0, 1): got {p}')
    if not isinstance(site, int) or not 0 <= site < 1 << 32:
        raise ValueError(f'site must be an integer in 0..2^32 - 1: got {site!r}')
    held, drop = None, int(p * 2.0 ** 32)
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != dev:
            raise ValueError(f'a tensor seed must be one int64 on {dev}')
        held, seed = seed, 0
    elif isinstance(seed, bool) or not isinstance(seed, int):
        if seed is not None or drop:
            raise TypeError(f'seed must be an integer or an int64 tensor, not '
                            f'{type(seed).__name__}')
        seed = 0
    elif not 0 <= seed < 1 << 63:
        raise ValueError(f'seed must be in 0..2^63 - 1: got {seed}')
    return drop, 1.0 / (1.0 - p), seed, held


def _dropout(x, drop, scale, seed, held, site):
    y, n = _like(x), x.numel()
    if n:
        dim = x.shape[-1]
        rows, stride = (x, dim) if x.is_contiguous() else (None, 0)
        if rows is None:
            rows = _rows(x, dim)
            stride = rows.stride(0)
        N.call('bs_dropout', x.device, _address(rows), _DTYPES[x.dtype], n // dim, dim, stride, seed,
               _address(held), site, drop, scale, _address(y))
    return y


class _Dropout(torch.autograd.Function):
    """dropout with its gradient, whose mask is computed again."""

    @staticmethod
    def forward(ctx, x, drop, scale, seed, held, site):
        ctx.args = (drop, scale, seed, site)
        ctx.save_for_backward(held)
        return _dropout(x, drop, scale, seed, held, site)

    @staticmethod
    @_once
    def backward(ctx, gy):
        _recorded('dropout', gy)
        drop, scale, seed, site = ctx.args
        return (_dropout(gy, drop, scale, seed, ctx.saved_tensors[0], site),) + (None,) * 5


def dropout(x, p, seed, site=0):
    """``x`` [.., dim], dim below 2^31, with each element dropped, to 0, with probability ``p`` in
    [0, 1) and the others times 1 / (1 - p).

    Element (row, column) of the rows [.., dim] is kept where word column % 4 of the Philox 4x32-10
    generator with counter (column // 4, site, row) and key ``seed`` is at least p 2^32: the same
    everywhere, so no mask is stored.  ``seed`` is an integer, or an int64 tensor of one element on the
    GPU that is read when the kernel runs (a recorded graph then drops others at each replay once it
    is changed, which has to wait until the backward pass has run); ``site`` tells the places of a
    model apart that share one.  What is dropped is 0 whatever it was.  Differentiable in ``x``, in
    reverse mode."""
    _floating('x', x)
    if x.dim() < 1:
        raise ValueError('x must have a dimension')
    _fits(x.shape[-1], 'values of a row (dim)')
    args = _chance(p, seed, site, x.device)
    if _recorded('dropout', x):
        return _Dropout.apply(x, *args, site)
    return _dropout(x, *args, site)


# ------------------------------------------------------------------------- layer norm
def _operands(x, residual, weight, bias):
    _floating('x', x)
    shape, dev = x.shape, x.device
    if len(shape) < 1 or not 1 <= shape[-1] <= 16384:
        raise ValueError(f'x [.., dim] with dim in 1..16384: got {tuple(shape)}')
    if residual is not None:
        _floating('residual', residual, x.dtype)
        if residual.shape != shape or residual.device != dev:
            raise ValueError(f'residual must be {tuple(shape)} on {dev}: got '
                             f'{tuple(residual.shape)} on {residual.device}')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None:
            _floating(name, t)
            if t.shape != (shape[-1],) or t.device != dev:
                raise ValueError(f'{name} must be [{shape[-1]}] on {dev}: got {tuple(t.shape)} on '
                                 f'{t.device}')


def _pack(x, residual, weight, bias, chance, site, eps):
    """(tensors to hold, bytes of bs_layer_norm_in, rows, dim)."""
    dim = x.shape[-1]
    drop, scale, seed, held = chance
    acts = [t if t is None else _rows(t, dim) for t in (x, residual)]
    weights = [t if t is None else t.contiguous() for t in (weight, bias)]
    rows = acts[0].shape[0]
    packed = _NORM_IN.pack(
        *[_address(t) or 0 for t in (*acts, *weights, held)],
        *[0 if t is None else t.stride(0) for t in acts], rows, seed, dim, _DTYPES[x.dtype],
        *[0 if t is None else _DTYPES[t.dtype] for t in weights], site, drop, scale, eps)
    return (acts, weights, held), packed, rows, dim


def _forward(x, residual, weight, bias, chance, site, eps, keep):
    """(stream or None, normed, statistics or None)."""
    hold, packed, rows, _ = _pack(x, residual, weight, bias, chance, site, eps)
    normed = _like(x)
    stream = _like(x) if residual is not None else None
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if keep else None
    N.call('bs_layer_norm', x.device, packed, _address(stream), _address(normed), _address(stats))
    return stream, normed, stats


class _LayerNorm(torch.autograd.Function):
    """layer_norm and add_layer_norm with their gradients, formed from the operands and each row's
    mean and scale."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, drop, scale, seed, held, site, eps):
        ctx.args = (drop, scale, seed, site, eps)
        stream, normed, stats = _forward(x, residual, weight, bias, (drop, scale, seed, held),
                                         site, eps, True)
        ctx.save_for_backward(x, residual, weight, bias, held, stats)
        ctx.set_materialize_grads(False)
        return stream, normed

    @staticmethod
    @_once
    def backward(ctx, gs, gn):
        _recorded('layer_norm', gs, gn)
        x, residual, weight, bias, held, stats = ctx.saved_tensors
        drop, scale, seed, site, eps = ctx.args
        hold, packed, rows, dim = _pack(x, residual, weight, bias, (drop, scale, seed, held), site,
                                        eps)
        gs, gn = (None if t is None else t.contiguous() for t in (gs, gn))
        dev = x.device
        grads = [_like(t) if need else None
                 for t, need in zip((x, residual, weight, bias), ctx.needs_input_grad)]
        if not drop and grads[0] is not None:      # one gradient for both
            grads[1] = None
        nbytes, ws = 0, None
        if grads[2] is not None or grads[3] is not None:
            nbytes = N.lib().bs_layer_norm_grad_workspace_size(rows, dim)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        N.call('bs_layer_norm_grad', dev, packed, _address(gs), _address(gn), _address(stats),
               *(_address(t) for t in grads), _address(ws), nbytes)
        if grads[1] is None and ctx.needs_input_grad[1]:
            grads[1] = grads[0]
        return (*grads,) + (None,) * 6


_KEEP_ALL = (0, 1.0, 0, None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over rows [.., dim] of ``x``: ``(x - mean) / sqrt(variance + eps) * weight + bias``.

    ``weight`` and ``bias`` [dim] are of any floating type and may be left out.  Sums are in 32 bits.
    Differentiable in every tensor, in reverse mode."""
    _operands(x, None, weight, bias)
    if _recorded('layer_norm', x, weight, bias):
        return _LayerNorm.apply(x, None, weight, bias, *_KEEP_ALL, 0, eps)[1]
    return _forward(x, None, weight, bias, _KEEP_ALL, 0, eps, False)[1]


def add_layer_norm(x, residual, weight=None, bias=None, p=0.0, seed=None, site=0, eps=1e-5):
    """What stands between a block's output ``x`` and the next block, in one pass over rows
    [.., dim]: ``stream = residual + dropout(x, p, seed, site)`` (:func:`dropout`) and
    ``normed = layer_norm(stream, weight, bias, eps)`` -> (stream, normed).

    ``x`` and ``residual`` have one shape and type.  ``normed`` is formed before ``stream`` is
    rounded.  Differentiable in every tensor but ``seed``, in reverse mode."""
    _operands(x, residual, weight, bias)
    if residual is None:
        raise TypeError('residual must be a tensor, not NoneType')
    chance = _chance(p, seed, site, x.device)
    if _recorded('add_layer_norm', x, residual, weight, bias):
        return _LayerNorm.apply(x, residual, weight, bias, *chance, site, eps)
    return _forward(x, residual, weight, bias, chance, site, eps, False)[:2]
