"""The 64-bit definitions of the sequence-layer operators: gradients against differences (CPU)."""
import numpy as np
import pytest

from oracle import sequence


def _difference(f, x, d, h=1e-6):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


def test_gated_delta_gradients_against_differences():
    rs = np.random.RandomState(1)
    T, hk, h, dk, dv = 5, 2, 4, 3, 6
    args = [rs.randn(T, hk, dk), rs.randn(T, hk, dk) * 0.5, rs.randn(T, h, dv),
            -rs.rand(T, h), rs.rand(T, h), rs.randn(h, dk, dv)]
    do, ds = rs.randn(T, h, dv), rs.randn(h, dk, dv)

    def loss(a):
        o, s = sequence.gated_delta(*a[:5], state=a[5])
        return (o * do).sum() + (s * ds).sum()

    grads = sequence.gated_delta(*args[:5], state=args[5], grad_o=do, grad_state=ds)[1]
    for i, gr in enumerate(grads):
        d = rs.randn(*args[i].shape)
        num = _difference(lambda x: loss(args[:i] + [x] + args[i + 1:]), args[i], d)
        # central differences of step 1e-6 on sums of O(10): truncation 1e-12, rounding 1e-9
        assert abs(num - (gr * d).sum()) < 1e-7 * max(1.0, abs(num))


@pytest.mark.parametrize('parts', [('post', 'gate', 'scale', 'residual', 'pre'), ('post', 'gate'),
                                   ('residual', 'pre'), ('pre',), ()])
def test_norm_gradients_against_differences(parts):
    rs = np.random.RandomState(2)
    R, D = 3, 7
    shape = dict(post=(D,), gate=(R, D), scale=(D,), residual=(R, D), pre=(D,))
    args = {'y': rs.randn(R, D), **{n: rs.randn(*shape[n]) for n in parts}}
    d1, d2 = rs.randn(R, D), rs.randn(R, D) if 'pre' in parts else None

    def loss(a):
        s, n = sequence.norm_gate_residual(**a)
        return (s * d1).sum() + ((n * d2).sum() if n is not None else 0)

    grads = sequence.norm_gate_residual(**args, grad_stream=d1, grad_normed=d2)[1]
    assert set(grads) == set(args)
    for n in args:
        d = rs.randn(*args[n].shape)
        num = _difference(lambda x: loss({**args, n: x}), args[n], d)
        assert abs(num - (grads[n] * d).sum()) < 1e-7 * max(1.0, abs(num))


def test_int8_quantize_rows():
    x8, a = sequence.int8_quantize([[0.0, 0.0], [127.0, -0.5], [1e-30, -1e-30]])
    assert np.array_equal(x8, [[0, 0], [127, 0], [127, -127]]) and a[0] == 0
