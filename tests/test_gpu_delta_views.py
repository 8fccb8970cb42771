"""The gated delta rule on views whose dimension of tokens has a stride past 32-bit addressing."""
import numpy as np
import pytest
import torch

from brainstate_amd import ops

pytestmark = pytest.mark.gpu


def _operands(b, t, hk, h, dk, dv, dtype, seed):
    rs = np.random.RandomState(seed)
    k = rs.randn(b, t, hk, dk) + 0.2
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    # decays of a hundred tokens, so that chunks reach far
    arrays = [rs.randn(b, t, hk, dk), k, rs.randn(b, t, h, dv), -0.02 * rs.rand(b, t, h),
              rs.rand(b, t, h)]
    types = [dtype, dtype, dtype, torch.float32, dtype]
    return [torch.tensor(a).to(d).cuda() for a, d in zip(arrays, types)]


def _pass(x, s0, do, ds, **kw):
    leaves = [y.detach().requires_grad_() for y in (*x, s0)]
    o, s1 = ops.gated_delta_rule(*leaves[:5], initial_state=leaves[5], **kw)
    return (o.detach(), s1.detach(), *torch.autograd.grad((o, s1), leaves, (do, ds)))


def test_one_token_of_a_time_major_batch():
    """The stride of a dimension of one token does not matter."""
    h, d = 2, 16
    x = _operands(3, 2, h, h, d, d, torch.float32, 4)
    wide = [torch.zeros(2 * (1 << 23), device='cuda') for _ in range(3)]
    views = []
    for flat, y in zip(wide, x[:3]):       # the second token 2^23 elements after the first
        view = flat.as_strided((3, 2, h, d), (h * d, 1 << 23, d, 1))
        view.copy_(y)
        views.append(view)
    want = ops.gated_delta_rule(*(y[:, 1:] for y in x))
    got = ops.gated_delta_rule(*(y[:, 1:] for y in views), *(y[:, 1:] for y in x[3:]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = _pass([y[:, 1:] for y in views] + [y[:, 1:] for y in x[3:]], want[1], want[0], want[1])
    again = _pass([y[:, 1:] for y in x], want[1], want[0], want[1])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    both = ops.gated_delta_rule(*views, *x[3:])
    assert all(torch.equal(a, b) for a, b in zip(both, ops.gated_delta_rule(*x)))
