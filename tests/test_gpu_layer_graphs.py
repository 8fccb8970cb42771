"""Decay attention, layer norm, dropout and the 4-bit product recorded into graphs, replayed on new
inputs, with eager calls and synchronizations between the replays."""
import pytest
import torch

from brainstate_amd import ops

pytestmark = pytest.mark.gpu


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


def _replays(f, inputs, held=(), between=lambda i: None):
    """Replays on new inputs against eager calls of the same; ``held`` is what f changes in place."""
    graph, outs = _recorded(f)
    seen = []
    for i in range(4):
        rng = torch.Generator().manual_seed(20 + i)
        for t in inputs:
            with torch.no_grad():
                t.copy_(torch.randn(t.shape, generator=rng).abs() / -4)
        between(i)
        start = [t.clone() for t in held]
        graph.replay()
        got = [t.clone() for t in (*outs, *held)]
        torch.cuda.synchronize()
        for t, s in zip(held, start):
            t.copy_(s)
        want = f()
        assert all(torch.equal(a, b) for a, b in zip(got, (*want, *held))), i
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def _prompt(t, hk=2, h=4, dk=16, dv=24):
    shapes = [(1, t, hk, dk), (1, t, hk, dk), (1, t, h, dv), (1, t, h)]
    return [torch.ones(s, device='cuda') for s in shapes]


@pytest.mark.parametrize('t', [200, 1500])
def test_prompts(t):
    x = _prompt(t)
    offsets = torch.tensor([3, 3, 70, t - 2], dtype=torch.int32, device='cuda')
    s0 = torch.zeros(3, 4, 16, 24, device='cuda')
    _replays(lambda: ops.decay_attention(*x, initial_state=s0, seq_offsets=offsets), [*x, s0])


def test_two_graphs_have_workspaces_of_their_own():
    a, b = _prompt(1500), _prompt(1400)
    fa, fb = (lambda x=x: ops.decay_attention(*x) for x in (a, b))
    for x in (a, b):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(1)).abs() / -4)
    ga, oa = _recorded(fa)
    gb, ob = _recorded(fb)
    wa, wb = fa(), fb()
    for _ in range(3):
        ga.replay()
        gb.replay()
        ga.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((*oa, *ob), (*wa, *wb)))


def test_steps():
    x = [t[0, :3] for t in _prompt(3)]
    state = torch.zeros(4, 4, 16, 24, device='cuda')
    slots = torch.tensor([2, -1, 0], dtype=torch.int32, device='cuda')
    _replays(lambda: (ops.decay_attention_step(*x, state, slots=slots),), x, [state])


def test_gradients_with_a_new_mask_at_each_replay():
    x = [t.requires_grad_() for t in _prompt(700)]
    w = torch.ones(24, device='cuda', requires_grad=True)
    do = torch.ones(1, 700, 4, 24, device='cuda')
    seed = torch.zeros(1, dtype=torch.int64, device='cuda')

    def f():
        y = ops.dropout(ops.decay_attention(*x)[0], 0.3, seed)
        s, n = ops.add_layer_norm(y, x[2], w, None, p=0.1, seed=seed, site=1)
        return (n.detach(), *torch.autograd.grad([s, n], [*x, w], [do, do]))
    _replays(f, [*x, do], between=lambda i: seed.fill_(i))


@pytest.mark.parametrize('tokens', [2, 300])
def test_norms_and_projections(tokens):
    y, residual = (torch.ones(tokens, 200, device='cuda') for _ in range(2))
    w = torch.ones(200, device='cuda')
    weights = torch.randn(90, 200, generator=torch.Generator().manual_seed(1)).cuda()

    def f():
        w4, scale = ops.int4_quantize(weights, 64)
        stream, normed = ops.add_layer_norm(y, residual, w, w, p=0.2, seed=3)
        return stream, ops.layer_norm(normed, w), ops.int4_linear(normed, w4, scale, group=64)
    _replays(f, [y, residual, w, weights])


def test_large_products():
    x = torch.ones(4100, 256, device='cuda')
    w4 = torch.randint(0, 256, (2100, 128), dtype=torch.uint8,
                       generator=torch.Generator().manual_seed(1)).cuda()
    scale = torch.rand(2100, 2, generator=torch.Generator().manual_seed(2)).cuda()
    for dtype in (torch.bfloat16, torch.float32):
        _replays(lambda: (ops.int4_linear(x.to(dtype), w4, scale),), [x])
