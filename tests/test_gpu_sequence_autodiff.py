"""Derivatives that the sequence-layer operators do not have are refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from brainstate_amd import ops

pytestmark = pytest.mark.gpu


def _delta():
    rng = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=rng).cuda()                       # noqa: E731
    return [r(2, 5, 2, 16), r(2, 5, 2, 16), r(2, 5, 4, 16), -r(2, 5, 4).abs(), r(2, 5, 4)]


def _calls():
    """(name, call of one operand, operand, what it raises) for every operand that may carry a
    derivative."""
    x = _delta()
    state = torch.zeros(2, 4, 16, 16, device='cuda')
    for i, name in enumerate(('q', 'k', 'v', 'g', 'beta')):
        def rule(t, i=i):
            return ops.gated_delta_rule(*x[:i], t, *x[i + 1:])[0]

        def step(t, i=i):
            y = [a[:, 0] for a in x]
            y[i] = t
            return ops.gated_delta_step(*y, state.clone())
        yield f'rule {name}', rule, x[i], NotImplementedError
        yield f'step {name}', step, x[i][:, 0], ValueError
    yield 'rule state', lambda t: ops.gated_delta_rule(*x, initial_state=t)[0], state, \
        NotImplementedError
    yield 'step state', lambda t: ops.gated_delta_step(*[a[:, 0] for a in x], t), state, ValueError
    y, w = torch.ones(3, 32, device='cuda'), torch.ones(32, device='cuda')
    args = dict(post_weight=w, gate=y, scale=w, residual=y, pre_weight=w)
    yield 'norm y', lambda t: ops.norm_gate_residual(t, **args)[0], y, NotImplementedError
    for name in args:
        yield f'norm {name}', lambda t, n=name: ops.norm_gate_residual(y, **{**args, n: t})[0], \
            args[name], NotImplementedError
    w8, ws = torch.ones(8, 32, dtype=torch.int8, device='cuda'), torch.ones(8, device='cuda')
    x8, xs = torch.ones(3, 32, dtype=torch.int8, device='cuda'), torch.ones(3, device='cuda')
    yield 'quantize', lambda t: ops.int8_quantize(t)[1], y, ValueError
    yield 'linear x', lambda t: ops.int8_linear(t, w8, ws), y, ValueError
    yield 'linear scale', lambda t: ops.int8_linear(y, w8, t), ws, ValueError
    yield 'linear bias', lambda t: ops.int8_linear(y, w8, ws, bias=t), ws, ValueError
    yield 'matmul scale', lambda t: ops.int8_matmul(x8, t, w8, ws), xs, ValueError


@pytest.mark.parametrize('grad_mode', [True, False])
def test_forward_mode_is_refused(grad_mode):
    for name, f, t, error in _calls():
        with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(error):
                f(dual)
                print(name, 'went through')


def test_transforms_are_refused():
    for name, f, t, error in _calls():
        for run in (lambda: torch.func.grad(lambda a: f(a).sum())(t),
                    lambda: torch.func.jvp(f, (t,), (torch.ones_like(t),)),
                    lambda: torch.func.vmap(f)(torch.stack([t, t]))):
            with pytest.raises(error):
                run()
                print(name, 'went through')


def test_constants_inside_levels_and_transforms():
    """Operands without a derivative are computed as ever."""
    x = _delta()
    y = torch.randn(3, 32, generator=torch.Generator().manual_seed(2)).cuda()
    w = torch.ones(32, device='cuda')
    o, n = ops.gated_delta_rule(*x)[0], ops.norm_gate_residual(y, w)[0]
    x8 = ops.int8_quantize(y)[0]

    def inside(a):
        assert torch.equal(ops.gated_delta_rule(*x)[0], o)
        assert torch.equal(ops.norm_gate_residual(y, w)[0], n)
        assert torch.equal(ops.int8_quantize(y)[0], x8)
        return (a * a).sum()

    with forward_ad.dual_level():
        inside(w)
    assert torch.equal(torch.func.grad(inside)(w), 2 * w)


def test_reverse_mode_inside_a_dual_level():
    x = _delta()
    q = x[0].clone().requires_grad_()
    want = torch.autograd.grad(ops.gated_delta_rule(q, *x[1:])[0].sum(), q)[0]
    with forward_ad.dual_level():
        got = torch.autograd.grad(ops.gated_delta_rule(q, *x[1:])[0].sum(), q)[0]
    assert torch.equal(got, want)


def test_batched_gradients_are_refused():
    x = _delta()
    q = x[0].clone().requires_grad_()
    y = torch.ones(3, 32, device='cuda', requires_grad=True)
    for o, t in ((ops.gated_delta_rule(q, *x[1:])[0], q),
                 (ops.norm_gate_residual(y, torch.ones(32, device='cuda'))[0], y)):
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(o, t, torch.ones(2, *o.shape, device='cuda'), is_grads_batched=True)
