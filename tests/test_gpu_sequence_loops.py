"""The sequence-layer operators in the framework's loop."""
import pytest
import torch

import brainstate_amd as bs
from brainstate_amd import ops

pytestmark = pytest.mark.gpu


def _tokens(b=2, seed=1, dtype=torch.float32):
    rng = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=rng)                               # noqa: E731
    x = [r(b, 2, 16), r(b, 2, 16) / 4, r(b, 4, 24), -r(b, 4).abs(), r(b, 4).sigmoid()]
    return [y.to('cuda', dtype) for y in x]


def test_a_loop_advances_a_state_once_a_step():
    """Recording the step function does not count as a step of its own."""
    x = _tokens()
    state, want = (torch.zeros(2, 4, 16, 24, device='cuda') for _ in range(2))
    outs = torch.stack([ops.gated_delta_step(*x, want) for _ in range(5)])
    got = bs.transform.for_loop(lambda: ops.gated_delta_step(*x, state), length=5)
    assert torch.equal(got, outs) and torch.equal(state, want)
    hidden = bs.HiddenState(torch.zeros(2, 4, 16, 24, device='cuda'))
    got = bs.transform.for_loop(lambda: ops.gated_delta_step(*x, hidden.value), length=5)
    assert torch.equal(got, outs) and torch.equal(hidden.value, want)


def test_a_loop_over_tokens():
    xs = [torch.stack(y) for y in zip(*(_tokens(seed=i) for i in range(6)))]
    state, want = (torch.zeros(2, 4, 16, 24, device='cuda') for _ in range(2))
    outs = torch.stack([ops.gated_delta_step(*(y[i] for y in xs), want) for i in range(6)])
    got = bs.transform.for_loop(lambda *t: ops.gated_delta_step(*t, state), *xs)
    assert torch.equal(got, outs) and torch.equal(state, want)


def test_the_layer_in_a_loop():
    layer = bs.nn.GatedDelta(64, 4, 24, num_key_heads=2, key_size=16, dtype=torch.float32, seed=3)
    rng = torch.Generator().manual_seed(5)
    normed, stream = (torch.randn(7, 3, 64, generator=rng).cuda() for _ in range(2))
    with torch.no_grad():
        layer.init_state(3)
        want = [layer(normed[i], stream[i]) for i in range(7)]
        last = layer.S.value.clone()
        layer.init_state(3)
        n, s = bs.transform.for_loop(layer, normed, stream)
    assert bs.transform.last_loop == 'eager'
    assert torch.equal(n, torch.stack([w[0] for w in want]))
    assert torch.equal(s, torch.stack([w[1] for w in want]))
    assert torch.equal(layer.S.value, last)
