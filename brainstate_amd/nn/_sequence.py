"""Sequence layers on the operators of :mod:`brainstate_amd.ops` (no counterpart in brainstate)."""
import torch
import torch.nn.functional as F

from .. import ops
from .._state import HiddenState, ParamState
from ._event import _device
from ._module import Dynamics

__all__ = ['DecayAttention', 'GatedDelta']


class _Projections(Dynamics):
    """A recurrent layer with a projection of its input and one of its output, ``weight_in`` and
    ``weight_out``, which serve in fewer bits after ``quantize()``."""
    __module__ = 'brainstate_amd.nn'
    _packed = None

    def quantize(self, bits=8, group=128):
        """Both projections in 8 bits with a scale a channel, or in 4 bits with one a channel and
        ``group`` input values, from here on, without gradient (a copy: later changes of the weights
        need another call)."""
        if bits not in (4, 8):
            raise ValueError(f'bits must be 4 or 8: got {bits!r}')
        self._packed = tuple(
            (ops.int8_linear, ops.int8_quantize(w), {}) if bits == 8 else
            (ops.int4_linear, ops.int4_quantize(w, group), {'group': group})
            for w in (self.weight_in.value.detach(), self.weight_out.value.detach()))

    def _project(self, x, which):
        if self._packed is not None:
            linear, weights, kw = self._packed[which]
            return linear(x, *weights, **kw)
        return F.linear(x, (self.weight_in, self.weight_out)[which].value)

    def _check(self, normed, stream):
        if normed.dim() not in (2, 3) or normed.shape[-1] != self.in_size[-1] or \
                normed.shape != stream.shape:
            raise ValueError(f'normed and stream must both be [batch, {self.in_size[-1]}] or '
                             f'[batch, tokens, {self.in_size[-1]}]: got {tuple(normed.shape)}, '
                             f'{tuple(stream.shape)}')


def _normal(rng, dtype, device):
    return lambda n, k: (torch.randn(n, k, generator=rng) * k ** -0.5).to(device, dtype)


class GatedDelta(_Projections):
    """A gated delta rule layer between two norms, as a recurrent module: its state is one matrix
    [key_size, head_size] a head and row (``S``, a HiddenState in 32 bits).

    ``layer(normed, stream)`` takes the normed input and the residual stream and returns the next
    ``(normed, stream)``, ready for a following layer:

        q, k, v, z, a, b = normed weight_in^T
        g = -exp(log_decay) softplus(a + decay_bias),  beta = sigmoid(b)
        o = gated delta rule of q / |q|, k / |k|, v, g, beta from S
        y = (norm(o) head_norm silu(z)) weight_out^T
        stream + scale y,  norm(stream + scale y) next_norm

    [batch, in_size] is one token of every row and advances ``S`` in place (no gradient: for serving,
    one by one or in a ``for_loop`` under ``torch.no_grad()``); [batch, tokens, in_size] runs whole sequences in
    chunks, is differentiable in the parameters and both inputs, and leaves the last states in
    ``S`` (with their graph where one is recorded: ``init_state`` starts the next sequence).

    ``quantize()`` takes both projections into 8 bits, a scale a channel; from then on they run as
    8-bit integer products of tokens quantized on the way, without gradient.  ``quantize(bits=4)``
    takes them into 4 bits, a scale a channel and group of inputs; tokens then stay as they are.
    """
    __module__ = 'brainstate_amd.nn'

    def __init__(self, in_size, num_heads, head_size, num_key_heads=None, key_size=None,
                 eps=1e-6, dtype=torch.bfloat16, seed=0, name=None, param_type=ParamState):
        super().__init__(in_size, name=name)
        d = self.in_size[-1]
        hk, dk = num_key_heads or num_heads, key_size or head_size
        if hk < 1 or num_heads % hk:
            raise ValueError(f'{num_heads} heads for {hk} key heads')
        if not 1 <= dk <= 128 or not 1 <= head_size <= 128:
            raise ValueError(f'head sizes {dk}, {head_size} outside 1..128')
        self.num_heads, self.head_size, self.num_key_heads, self.key_size = \
            num_heads, head_size, hk, dk
        self.eps, self.dtype = eps, dtype
        self._split = (2 * hk * dk, num_heads * head_size, num_heads * head_size, num_heads,
                       num_heads)
        dev, rng = _device(), torch.Generator().manual_seed(seed)
        normal = _normal(rng, dtype, dev)
        self.weight_in = param_type(normal(sum(self._split), d))
        self.weight_out = param_type(normal(d, num_heads * head_size))
        self.head_norm = param_type(torch.ones(head_size, device=dev))
        self.next_norm = param_type(torch.ones(d, device=dev))
        self.scale = param_type(torch.ones(d, device=dev))
        self.log_decay = param_type(torch.rand(num_heads, generator=rng).mul(4).log().to(dev))
        self.decay_bias = param_type(torch.full((num_heads,), -4.0, device=dev))
        self._unit = torch.full((dk,), dk ** -0.5, device=dev)

    def init_state(self, batch_size=None, **kwargs):
        shape = (batch_size or 1, self.num_heads, self.key_size, self.head_size)
        self.S = HiddenState(torch.zeros(shape, device=_device()))

    def update(self, normed, stream):
        self._check(normed, stream)
        lead, hk = normed.shape[:-1], self.num_key_heads
        qk, v, z, a, b = self._project(normed, 0).split(self._split, dim=-1)
        # one norm for queries and keys: x / |x| is x / rms(x) over the root of its length
        qk, _ = ops.norm_gate_residual(qk.reshape(*lead, 2 * hk, self.key_size), self._unit,
                                       eps=self.eps / self.key_size)
        q, k = qk.split(hk, dim=-2)
        v, z = (x.reshape(*lead, self.num_heads, self.head_size) for x in (v, z))
        g = -self.log_decay.value.exp() * F.softplus(a.float() + self.decay_bias.value)
        beta = b.sigmoid()
        if len(lead) == 1:
            o = ops.gated_delta_step(q, k, v, g, beta, self.S.value)
        else:
            o, self.S.value = ops.gated_delta_rule(q, k, v, g, beta, initial_state=self.S.value)
        o, _ = ops.norm_gate_residual(o, self.head_norm.value, gate=z, eps=self.eps)
        y = self._project(o.reshape(*lead, -1), 1)
        stream, normed = ops.norm_gate_residual(y, scale=self.scale.value, residual=stream,
                                                pre_weight=self.next_norm.value, eps=self.eps)
        return normed, stream


class DecayAttention(_Projections):
    """A decay attention layer between two layer norms, as a recurrent module: its state is one
    matrix [key_size, head_size] a head and row (``S``, a HiddenState in 32 bits).

    ``layer(normed, stream)`` takes the normed input and the residual stream and returns the next
    ``(normed, stream)``, ready for a following layer:

        q, k, v = normed weight_in^T
        o = decay attention of q, k, v and the log decays -exp(log_rate) from S
        y = layer_norm(o, each head by itself) weight_out^T
        stream + dropout(y),  layer_norm(stream + dropout(y), next_weight, next_bias)

    [batch, in_size] is one token of every row and advances ``S`` in place (no gradient: for serving,
    one by one or in a ``for_loop`` under ``torch.no_grad()``); [batch, tokens, in_size] runs whole
    sequences in chunks, is differentiable in the parameters and both inputs, and leaves the last
    states in ``S`` (with their graph where one is recorded: ``init_state`` starts the next sequence).

    ``dropout`` is the chance that an element of ``y`` is dropped, in calls that are given a ``seed``
    (:func:`brainstate_amd.ops.dropout`; layers of one model that share a seed have a ``site`` each).
    ``quantize()`` takes both projections into 8 or 4 bits, without gradient from then on.
    """
    __module__ = 'brainstate_amd.nn'

    def __init__(self, in_size, num_heads, head_size, num_key_heads=None, key_size=None,
                 dropout=0.0, site=0, eps=1e-5, dtype=torch.bfloat16, seed=0, name=None,
                 param_type=ParamState):
        super().__init__(in_size, name=name)
        d = self.in_size[-1]
        hk, dk = num_key_heads or num_heads, key_size or head_size
        if hk < 1 or num_heads % hk:
            raise ValueError(f'{num_heads} heads for {hk} key heads')
        if not 1 <= dk <= 128 or not 1 <= head_size <= 128:
            raise ValueError(f'head sizes {dk}, {head_size} outside 1..128')
        if not 0.0 <= dropout < 1.0:
            raise ValueError(f'dropout must be in [0, 1): got {dropout}')
        self.num_heads, self.head_size, self.num_key_heads, self.key_size = \
            num_heads, head_size, hk, dk
        self.dropout, self.site, self.eps, self.dtype = dropout, site, eps, dtype
        self._split = (hk * dk, hk * dk, num_heads * head_size)
        dev, rng = _device(), torch.Generator().manual_seed(seed)
        normal = _normal(rng, dtype, dev)
        self.weight_in = param_type(normal(sum(self._split), d))
        self.weight_out = param_type(normal(d, num_heads * head_size))
        self.next_weight = param_type(torch.ones(d, device=dev))
        self.next_bias = param_type(torch.zeros(d, device=dev))
        # half-lives from a few tokens to thousands
        self.log_rate = param_type(torch.linspace(-8.0, -1.0, num_heads).to(dev))

    def init_state(self, batch_size=None, **kwargs):
        shape = (batch_size or 1, self.num_heads, self.key_size, self.head_size)
        self.S = HiddenState(torch.zeros(shape, device=_device()))

    def update(self, normed, stream, seed=None):
        self._check(normed, stream)
        lead = normed.shape[:-1]
        q, k, v = self._project(normed, 0).split(self._split, dim=-1)
        q, k = (x.unflatten(-1, (self.num_key_heads, self.key_size)) for x in (q, k))
        v = v.unflatten(-1, (self.num_heads, self.head_size))
        g = -self.log_rate.value.exp()
        if len(lead) == 1:
            o = ops.decay_attention_step(q, k, v, g, self.S.value)
        else:
            o, self.S.value = ops.decay_attention(q, k, v, g, initial_state=self.S.value)
        y = self._project(ops.layer_norm(o, eps=self.eps).flatten(-2), 1)
        p = 0.0 if seed is None else self.dropout
        stream, normed = ops.add_layer_norm(y, stream, self.next_weight.value,
                                            self.next_bias.value, p=p, seed=seed, site=self.site,
                                            eps=self.eps)
        return normed, stream
