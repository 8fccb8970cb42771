"""Products with 4-bit weights over the C ABI (no counterpart in brainstate);
:mod:`brainstate_amd.ops` exports them.
"""
import torch

from . import _native as N
from ._sequence import _DTYPES, _address, _fits, _floating, _no_grad, _rows

_GROUPS = (32, 64, 128)


def _group(group):
    if group not in _GROUPS:
        raise ValueError(f'group must be one of {_GROUPS}: got {group!r}')
    return int(group)


def int4_quantize(w, group=128):
    """Weights ``w`` [n, k] in 4 bits with a scale for each channel and ``group`` (32, 64 or 128)
    input values -> (uint8 [n, ceil(k / 2)], float32 scales [n, ceil(k / group)]).

    Of a group the scale is ``max|w| / 7`` and the integers are ``7 w / max|w|`` rounded to nearest
    (ties to even), in -7..7; each is stored plus 8, the one of an even place in the byte's low
    half.  A group of zeros has scale 0.  Not differentiable."""
    _floating('w', w)
    _no_grad('int4_quantize', w)
    group = _group(group)
    if w.dim() != 2 or not 1 <= w.shape[1] <= 65536:
        raise ValueError(f'w [n, k] with k in 1..65536: got {tuple(w.shape)}')
    n, k = w.shape
    rows, dev = _rows(w, k), w.device
    w4 = torch.empty((n, (k + 1) // 2), dtype=torch.uint8, device=dev)
    scale = torch.empty((n, -(-k // group)), dtype=torch.float32, device=dev)
    N.call('bs_int4_quantize', dev, _address(rows), _DTYPES[w.dtype], n, k, rows.stride(0), group,
           _address(w4), _address(scale))
    return w4, scale


def int4_linear(x, w4, w_scale, bias=None, group=128):
    """``x`` [.., k] times 4-bit weights (:func:`int4_quantize`) -> [.., n] of the type of ``x``:
    ``sum_k x[.., k] * (u[n, k] - 8) * w_scale[n, k // group] + bias[n]`` with integers u in 0..15
    from ``w4`` uint8 [n, ceil(k / 2)].  Products are exact and sums in 32 bits, scales are applied
    to a group's sum and ``bias`` [n] is added in 32 bits.  Not differentiable."""
    _floating('x', x)
    _no_grad('int4_linear', x, w4, w_scale, bias)
    group, dev = _group(group), x.device
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 65536:
        raise ValueError(f'x [.., k] with k in 1..65536: got {tuple(x.shape)}')
    k = x.shape[-1]
    if not isinstance(w4, torch.Tensor) or w4.dtype != torch.uint8 or w4.dim() != 2 or \
            w4.shape[1] != (k + 1) // 2 or w4.device != dev:
        raise ValueError(f'w4 must be uint8 [channels, {(k + 1) // 2}] on {dev}')
    n, groups = w4.shape[0], -(-k // group)
    _fits(n, 'channels')
    if not isinstance(w_scale, torch.Tensor) or w_scale.dtype != torch.float32 or \
            w_scale.shape != (n, groups) or w_scale.device != dev:
        raise ValueError(f'w_scale must be float32 [{n}, {groups}] on {dev}')
    if bias is not None:
        _floating('bias', bias)
        if bias.shape != (n,) or bias.device != dev:
            raise ValueError(f'bias must be [{n}] on {dev}: got {tuple(bias.shape)}')
        bias = bias.contiguous()
    w4, w_scale = w4.contiguous(), w_scale.contiguous()
    rows, dtype = _rows(x, k), _DTYPES[x.dtype]
    m, at = rows.shape[0], _address(rows)
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
    nbytes = N.lib().bs_int4_workspace_size(at, dtype, rows.stride(0), m, k, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    N.call('bs_int4_linear', dev, at, dtype, rows.stride(0), m, k, n, group, _address(w4),
           _address(w_scale), _address(bias), 0 if bias is None else _DTYPES[bias.dtype],
           _address(y), _address(ws), nbytes)
    return y
