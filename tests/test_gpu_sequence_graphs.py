"""The sequence-layer operators recorded into graphs, replayed on new inputs."""
import pytest
import torch

from brainstate_amd import ops

pytestmark = pytest.mark.gpu


def _tokens(b=2, seed=1, dtype=torch.float32):
    rng = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=rng)                               # noqa: E731
    x = [r(b, 2, 16), r(b, 2, 16) / 4, r(b, 4, 24), -r(b, 4).abs(), r(b, 4).sigmoid()]
    return [y.to('cuda', dtype) for y in x]


def _recorded(f):
    """f() recorded into a graph after two calls ahead of it -> (graph, its outputs)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = f()
    return graph, outs


def _replays(f, inputs, held=()):
    """Replays on new inputs, eager calls of the same and synchronizations between them; ``held`` is
    what f changes in place."""
    graph, outs = _recorded(f)
    for i in range(4):
        rng = torch.Generator().manual_seed(20 + i)
        for t in inputs:
            with torch.no_grad():
                t.copy_(torch.randn(t.shape, generator=rng).abs() / -4)
        start = [t.clone() for t in held]
        graph.replay()
        got = [t.clone() for t in (*outs, *held)]
        torch.cuda.synchronize()
        for t, s in zip(held, start):
            t.copy_(s)
        want = f()
        assert all(torch.equal(a, b) for a, b in zip(got, (*want, *held))), i


def test_recorded_prompts():
    x = [y.unsqueeze(0).contiguous() for y in _tokens(200)]
    offsets = torch.tensor([3, 3, 70, 198], dtype=torch.int32, device='cuda')
    s0 = torch.zeros(3, 4, 16, 24, device='cuda')
    _replays(lambda: ops.gated_delta_rule(*x, initial_state=s0, seq_offsets=offsets), [*x[:4], s0])


def test_recorded_steps():
    x = _tokens(3)
    state = torch.zeros(4, 4, 16, 24, device='cuda')
    slots = torch.tensor([2, -1, 0], dtype=torch.int32, device='cuda')
    _replays(lambda: (ops.gated_delta_step(*x, state, slots=slots),), x[:4], [state])


def test_recorded_gradients():
    x = [y.unsqueeze(0).contiguous().requires_grad_() for y in _tokens(130)]
    do = torch.ones(1, 130, 4, 24, device='cuda')
    w = torch.ones(24, device='cuda', requires_grad=True)

    def f():
        o = ops.norm_gate_residual(ops.gated_delta_rule(*x)[0], w)[0]
        return (o.detach(), *torch.autograd.grad(o, [*x, w], do))
    _replays(f, [*x[:4], do])


@pytest.mark.parametrize('tokens', [2, 300])
def test_recorded_norms_and_projections(tokens):
    y, gate, residual = (torch.ones(tokens, 200, device='cuda') for _ in range(3))
    w = torch.ones(200, device='cuda')
    w8, ws = ops.int8_quantize(torch.randn(90, 200, generator=torch.Generator().manual_seed(1)).cuda())

    def f():
        stream, normed = ops.norm_gate_residual(y, w, gate, 0.5, residual, w)
        x8, a = ops.int8_quantize(normed)
        return stream, normed, ops.int8_linear(normed, w8, ws), ops.int8_matmul(x8, a, w8, ws)
    _replays(f, [y, gate, residual, w])
