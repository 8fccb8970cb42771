"""Derivatives that decay attention, layer norm, dropout and the 4-bit product do not have are
refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from brainstate_amd import ops

pytestmark = pytest.mark.gpu


def _operands():
    rng = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=rng).cuda()                       # noqa: E731
    return [r(2, 5, 2, 16), r(2, 5, 2, 16), r(2, 5, 4, 16), -r(2, 5, 4).abs()]


def _calls():
    """(name, call of one operand, operand, what it raises) for every operand that may carry a
    derivative."""
    x = _operands()
    state = torch.zeros(2, 4, 16, 16, device='cuda')
    for i, name in enumerate(('q', 'k', 'v', 'g')):
        def rule(t, i=i):
            return ops.decay_attention(*x[:i], t, *x[i + 1:])[0]

        def step(t, i=i):
            y = [a[:, 0] for a in x]
            y[i] = t
            return ops.decay_attention_step(*y, state.clone())
        yield f'rule {name}', rule, x[i], NotImplementedError
        yield f'step {name}', step, x[i][:, 0], ValueError
    yield 'rule state', lambda t: ops.decay_attention(*x, initial_state=t)[0], state, \
        NotImplementedError
    yield 'step state', lambda t: ops.decay_attention_step(*[a[:, 0] for a in x], t), state, \
        ValueError
    y, w = torch.ones(3, 32, device='cuda'), torch.ones(32, device='cuda')
    yield 'norm x', lambda t: ops.layer_norm(t, w, w), y, NotImplementedError
    yield 'norm weight', lambda t: ops.layer_norm(y, t, w), w, NotImplementedError
    yield 'norm bias', lambda t: ops.layer_norm(y, w, t), w, NotImplementedError
    yield 'add x', lambda t: ops.add_layer_norm(t, y)[1], y, NotImplementedError
    yield 'add residual', lambda t: ops.add_layer_norm(y, t)[1], y, NotImplementedError
    yield 'dropout', lambda t: ops.dropout(t, 0.5, 1), y, NotImplementedError
    w4, ws = torch.ones(8, 16, dtype=torch.uint8, device='cuda'), torch.ones(8, 1, device='cuda')
    yield 'quantize', lambda t: ops.int4_quantize(t)[1], y, ValueError
    yield 'linear x', lambda t: ops.int4_linear(t, w4, ws), y, ValueError
    yield 'linear scale', lambda t: ops.int4_linear(y, w4, t), ws, ValueError
    yield 'linear bias', lambda t: ops.int4_linear(y, w4, ws, bias=t), ws[:, 0], ValueError


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
    x = _operands()
    y = torch.randn(3, 32, generator=torch.Generator().manual_seed(2)).cuda()
    w = torch.ones(32, device='cuda')
    w4, ws = ops.int4_quantize(y, 32)

    def all_of_them():
        return [ops.decay_attention(*x)[0], ops.layer_norm(y, w), *ops.add_layer_norm(y, y, w),
                ops.dropout(y, 0.5, 1), ops.int4_quantize(y, 32)[0],
                ops.int4_linear(y, w4, ws, group=32)]
    want = all_of_them()

    def inside(a):
        assert all(torch.equal(p, q) for p, q in zip(all_of_them(), want))
        return (a * a).sum()

    with forward_ad.dual_level():
        inside(w)
    assert torch.equal(torch.func.grad(inside)(w), 2 * w)


def test_second_derivatives_are_refused():
    x = _operands()
    q = x[0].clone().requires_grad_()
    y = torch.randn(3, 32, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    for o, t in ((ops.decay_attention(q, *x[1:])[0], q), (ops.layer_norm(y), y),
                 (ops.dropout(y, 0.5, 1), y)):
        up = torch.ones_like(o).requires_grad_()
        first = torch.autograd.grad(o, t, up, create_graph=True)[0]
        with pytest.raises(RuntimeError, match='once_differentiable'):
            first.sum().backward()


def test_batched_gradients_are_refused():
    x = _operands()
    q = x[0].clone().requires_grad_()
    y = torch.randn(3, 32, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    for o, t in ((ops.decay_attention(q, *x[1:])[0], q), (ops.layer_norm(y), y),
                 (ops.dropout(y, 0.5, 1), y)):
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(o, t, torch.ones(2, *o.shape, device='cuda'), is_grads_batched=True)
