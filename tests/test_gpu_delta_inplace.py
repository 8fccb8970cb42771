"""The token step of the gated delta rule writes its state in place: autograd is told."""
import pytest
import torch

import brainstate_amd as bs
from brainstate_amd import ops

pytestmark = pytest.mark.gpu


def _delta():
    rng = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=rng).cuda()                       # noqa: E731
    return [r(2, 5, 2, 16), r(2, 5, 2, 16), r(2, 5, 4, 16), -r(2, 5, 4).abs(), r(2, 5, 4)]


def test_a_state_saved_for_gradients_is_guarded():
    """A step in place changes a state that a recorded pass saved: its backward pass says so."""
    x = [a[:, 0] for a in _delta()]
    state = torch.randn(2, 4, 16, 16, generator=torch.Generator().manual_seed(3)).cuda()
    w = torch.ones((), device='cuda', requires_grad=True)
    loss = (state * w).sum()                         # saves the state
    before = state._version
    ops.gated_delta_step(*x, state)
    assert state._version > before
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_steps_in_inference_mode():
    x = [a[:, 0] for a in _delta()]
    want = torch.zeros(2, 4, 16, 16, device='cuda')
    o = ops.gated_delta_step(*x, want)
    with torch.inference_mode():
        state = torch.zeros(2, 4, 16, 16, device='cuda')
        assert torch.equal(ops.gated_delta_step(*x, state), o) and torch.equal(state, want)


def test_the_layer_steps_on_after_a_recorded_pass():
    """Its states after a recorded pass are not needed by that pass's gradients."""
    layer = bs.nn.GatedDelta(32, 2, 16, dtype=torch.float32, seed=3)
    rng = torch.Generator().manual_seed(5)
    x = torch.randn(2, 70, 32, generator=rng).cuda().requires_grad_()
    grads = []
    for steps in (0, 3):
        layer.init_state(2)
        normed, stream = layer(x, x)
        with torch.no_grad():
            for _ in range(steps):
                layer(x[:, -1], x[:, -1])
        grads.append(torch.autograd.grad(normed.sum() + stream.sum(), x)[0])
    assert torch.equal(*grads)
