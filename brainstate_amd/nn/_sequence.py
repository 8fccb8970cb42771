"""Sequence layers on the operators of :mod:`brainstate_amd.ops` (no counterpart in brainstate)."""
import torch
import torch.nn.functional as F

from .. import ops
from .._state import HiddenState, ParamState
from ._event import _device
from ._module import Dynamics

__all__ = ['GatedDelta']


class GatedDelta(Dynamics):
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
    8-bit integer products of tokens quantized on the way, without gradient.
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

        def normal(n, k):
            return (torch.randn(n, k, generator=rng) * k ** -0.5).to(dev, dtype)

        self.weight_in = param_type(normal(sum(self._split), d))
        self.weight_out = param_type(normal(d, num_heads * head_size))
        self.head_norm = param_type(torch.ones(head_size, device=dev))
        self.next_norm = param_type(torch.ones(d, device=dev))
        self.scale = param_type(torch.ones(d, device=dev))
        self.log_decay = param_type(torch.rand(num_heads, generator=rng).mul(4).log().to(dev))
        self.decay_bias = param_type(torch.full((num_heads,), -4.0, device=dev))
        self._unit = torch.full((dk,), dk ** -0.5, device=dev)
        self._int8 = None

    def init_state(self, batch_size=None, **kwargs):
        shape = (batch_size or 1, self.num_heads, self.key_size, self.head_size)
        self.S = HiddenState(torch.zeros(shape, device=_device()))

    def quantize(self):
        """Both projections in 8 bits from here on (a copy: later changes of the weights need
        another call)."""
        self._int8 = tuple(ops.int8_quantize(w.value.detach())
                           for w in (self.weight_in, self.weight_out))

    def _project(self, x, which):
        if self._int8 is not None:
            return ops.int8_linear(x, *self._int8[which])
        return F.linear(x, (self.weight_in, self.weight_out)[which].value)

    def update(self, normed, stream):
        if normed.dim() not in (2, 3) or normed.shape[-1] != self.in_size[-1] or \
                normed.shape != stream.shape:
            raise ValueError(f'normed and stream must both be [batch, {self.in_size[-1]}] or '
                             f'[batch, tokens, {self.in_size[-1]}]: got {tuple(normed.shape)}, '
                             f'{tuple(stream.shape)}')
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
