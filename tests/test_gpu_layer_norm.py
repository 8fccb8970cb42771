"""Layer norm, alone and behind a dropped-out branch and its residual, against 64 bits.

Tolerances are of the norm of the difference over the norm of the result: 32-bit sums over a row
by a tree of lanes, a dozen dependent roundings of 2^-24 a value, so 32 x 2^-24; sums over R rows
for the weights' gradients walk up to R / 256 of them in a row, whose roundings add like their
root, well inside the same.  16-bit outputs add their rounding.
"""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

F32 = 32 * 2.0 ** -24
TOL = {torch.float32: F32, torch.bfloat16: F32 + 2.0 ** -8, torch.float16: F32 + 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SEED = 0x1234567890ABCDEF


def operands(rows, dim, dtype, w_dtype=torch.float32, seed=0):
    """x, residual, weight, bias and the two outputs' gradients."""
    rs = np.random.RandomState(seed)
    r = lambda *s: torch.tensor(rs.randn(*s))                                   # noqa: E731
    act = lambda: r(rows, dim).to(dtype).cuda()                                 # noqa: E731
    return [act(), act(), (1 + 0.3 * r(dim)).to(w_dtype).cuda(), r(dim).to(w_dtype).cuda(), act(),
            act()]


def numbers(*ts):
    return [t.detach().double().cpu().numpy() for t in ts]


def near(got, want, tol):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want) + 1e-30, \
        np.linalg.norm(got - want) / np.linalg.norm(want)


SIZES = [(3, 2), (3, 5), (3, 128), (70, 129), (5, 513), (2, 1000), (4, 2050), (3, 4096), (2, 5001),
         (600, 8192), (2, 16384)]


@pytest.mark.parametrize('p', [0.0, 0.3])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_add_layer_norm(size, dtype, p):
    rows, dim = size
    x, residual, w, b, gs, gn = operands(rows, dim, dtype, seed=dim)
    args = [t.requires_grad_() for t in (x, residual, w, b)]
    outs = ops.add_layer_norm(*args, p=p, seed=SEED, site=3)
    grads = torch.autograd.grad(outs, args, [gs, gn])
    mask = sequence.dropout_mask(SEED, 3, rows, dim, p)
    want, want_g = sequence.layer_norm(*numbers(x, residual, w, b), mask=mask,
                                       grad_stream=numbers(gs)[0], grad_normed=numbers(gn)[0])
    for got, ref in zip(outs, want):
        assert got.dtype == dtype
        near(got, ref, TOL[dtype])
    # of two values each normalised one is +-1, and what reaches x is all but their difference,
    # which cancels: the sums' roundings stay, against the terms' size
    scale = 1.0 if dim > 4 else 64.0
    for got, ref, t in zip(grads, want_g, (x, residual, w, b)):
        assert got.dtype == t.dtype
        near(got, ref, scale * TOL[got.dtype])
    with torch.no_grad():
        again = ops.add_layer_norm(x, residual, w, b, p=p, seed=SEED, site=3)
    assert all(torch.equal(a, o) for a, o in zip(again, outs))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(1, 1), (2, 64), (9, 500), (2, 4096)])
def test_layer_norm(size, dtype):
    x, _, w, b, _, gn = operands(*size, dtype, w_dtype=dtype, seed=1)
    for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
        args = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
        y = ops.layer_norm(args[0], args[1] if weight is not None else None,
                           args[-1] if bias is not None else None)
        given = numbers(*(t for t in (x, weight, bias) if t is not None))
        kw = dict(weight=given[1] if weight is not None else None,
                  bias=given[-1] if bias is not None else None)
        want, want_g = sequence.layer_norm(given[0], grad_normed=numbers(gn)[0], **kw)
        near(y, want[1], TOL[dtype])
        if size[1] == 1:
            assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y, args, gn))
            continue
        for got, ref in zip(torch.autograd.grad(y, args, gn),
                            [want_g[0]] + [g for g, t in zip(want_g[2:], (weight, bias))
                                           if t is not None]):
            near(got, ref, TOL[dtype])


def test_large_means_and_constant_rows():
    """The variance is taken about the mean: a mean of 1e4 leaves it whole, and a row of one value
    normalises to the bias."""
    rs = np.random.RandomState(0)
    x = torch.tensor(rs.randn(8, 1000) + 1e4, dtype=torch.float32).cuda()
    a = numbers(x)[0]
    # x itself is rounded before either side sees it; its mean in 32 bits is off by 2^-24 of 1e4,
    # against a standard deviation of 1
    near(ops.layer_norm(x), sequence.layer_norm(a)[1], 1e4 * 4 * 2.0 ** -24)
    b = torch.randn(64, generator=torch.Generator().manual_seed(0)).cuda()
    assert torch.equal(ops.layer_norm(torch.full((3, 64), 7.0, device='cuda'), None, b),
                       b.expand(3, 64))


def test_one_gradient_alone():
    x, residual, w, b, gs, gn = operands(5, 300, torch.float32)
    args = [t.requires_grad_() for t in (x, residual, w, b)]
    a = numbers(x, residual, w, b)
    mask = sequence.dropout_mask(SEED, 0, 5, 300, 0.2)
    stream, normed = ops.add_layer_norm(*args, p=0.2, seed=SEED)
    got = torch.autograd.grad(stream, args, gs, retain_graph=True)
    near(got[0], numbers(gs)[0] * mask, F32)
    assert torch.equal(got[1], gs) and (got[2] == 0).all() and (got[3] == 0).all()
    want = sequence.layer_norm(*a, mask=mask, grad_normed=numbers(gn)[0])[1]
    for i, (g, r) in enumerate(zip(torch.autograd.grad(normed, args, gn), want)):
        near(g, r, F32)
    for i in range(4):               # one operand alone wants a gradient
        y = [t.detach() for t in args]
        y[i].requires_grad_()
        outs = ops.add_layer_norm(*y, p=0.2, seed=SEED)
        near(torch.autograd.grad(outs[1], y[i], gn)[0], want[i], F32)


def test_gradients_against_differences():
    x, residual, w, b, gs, gn = operands(4, 70, torch.float32, seed=2)
    args = [x, residual, w, b]
    leaves = [t.clone().requires_grad_() for t in args]
    grads = torch.autograd.grad(ops.add_layer_norm(*leaves, p=0.25, seed=5), leaves, [gs, gn])

    def loss(*a):
        o = ops.add_layer_norm(*a, p=0.25, seed=5)
        return (o[0].double() * gs).sum() + (o[1].double() * gn).sum()
    for i, g in enumerate(grads):
        d = torch.randn(g.shape, generator=torch.Generator().manual_seed(i)).cuda()
        d = d * args[i].norm() / d.norm()
        at = lambda e: loss(*(t + e * d if j == i else t for j, t in enumerate(args)))  # noqa: E731
        num = (8 * (at(5e-3) - at(-5e-3)) - (at(1e-2) - at(-1e-2))) / 6e-2
        want = (g.double() * d).sum()
        assert abs(num - want) < 1e-3 * max(abs(want), g.double().norm()), i


def test_strided_unaligned_and_leading_dimensions():
    x, residual, w, b, _, _ = operands(12, 250, torch.bfloat16, seed=3)
    want = ops.add_layer_norm(x, residual, w, b, p=0.1, seed=1)
    wide = torch.zeros(12, 257, dtype=torch.bfloat16, device='cuda')
    wide[:, 3:253] = x
    got = ops.add_layer_norm(wide[:, 3:253], residual.t().contiguous().t(), w, b, p=0.1, seed=1)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    got = ops.add_layer_norm(x.view(3, 4, 250), residual.view(3, 4, 250), w, b, p=0.1, seed=1)
    assert all(torch.equal(a.view(12, 250), c) for a, c in zip(got, want))
    assert ops.layer_norm(x[:0], w, b).shape == (0, 250)
    y = x[:0].clone().requires_grad_()
    wg = w.clone().requires_grad_()
    g = torch.autograd.grad(ops.layer_norm(y, wg), [y, wg], torch.zeros_like(y))
    assert g[0].shape == (0, 250) and (g[1] == 0).all()


def test_what_is_dropped_does_not_count():
    """NaN and infinity in dropped places reach neither the outputs nor the gradients."""
    x, residual, w, b, gs, gn = operands(6, 200, torch.float32, seed=4)
    keep = torch.tensor(sequence.dropout_mask(9, 1, 6, 200, 0.5) > 0).cuda()
    bad = torch.where(keep, x, torch.full_like(x, float('nan')))
    bad[3] = torch.where(keep[3], x[3], torch.full_like(x[3], float('inf')))

    def run(a):
        args = [t.detach().requires_grad_() for t in (a, residual, w, b)]
        outs = ops.add_layer_norm(*args, p=0.5, seed=9, site=1)
        return [*outs, *torch.autograd.grad(outs, args, [gs, gn])]
    for got, want in zip(run(bad), run(x)):
        assert torch.equal(got, want)


def test_refusals():
    x, residual, w, b, _, _ = operands(3, 64, torch.float32)
    with pytest.raises(ValueError, match='1..16384'):
        ops.layer_norm(torch.zeros(2, 16385, device='cuda'))
    with pytest.raises(ValueError, match='1..16384'):
        ops.layer_norm(torch.zeros(2, 0, device='cuda'))
    with pytest.raises(ValueError, match='weight must be'):
        ops.layer_norm(x, w[:5])
    with pytest.raises(ValueError, match='bias must be'):
        ops.layer_norm(x, w, b.view(1, 64))
    with pytest.raises(TypeError, match='residual'):
        ops.add_layer_norm(x, None, w)
    with pytest.raises(TypeError, match='residual is'):
        ops.add_layer_norm(x, residual.half())
    with pytest.raises(ValueError, match='residual must be'):
        ops.add_layer_norm(x, residual[:2])
    with pytest.raises(ValueError, match='p must be'):
        ops.add_layer_norm(x, residual, p=1.0, seed=1)
    with pytest.raises(TypeError, match='seed'):
        ops.add_layer_norm(x, residual, p=0.1)
    with pytest.raises(TypeError, match='not supported'):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match='on the GPU'):
        ops.layer_norm(x.cpu())
