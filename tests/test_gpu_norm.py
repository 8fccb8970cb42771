"""The norms, gate and residual around a block, and their gradients, against 64 bits.

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
NAMES = ('y', 'post', 'gate', 'scale', 'residual', 'pre')
FORMS = [('post', 'gate', 'scale', 'residual', 'pre'), ('post', 'gate'), ('residual', 'pre'),
         ('pre',), ('post',), ('gate', 'scale'), ()]


def _operands(rows, dim, parts, dtype, w_dtype=torch.float32, seed=0):
    rs = np.random.RandomState(seed)
    r = lambda *s: torch.tensor(rs.randn(*s))                                   # noqa: E731
    x = {'y': r(rows, dim).to(dtype).cuda()}
    for n in parts:
        x[n] = r(rows, dim).to(dtype).cuda() if n in ('gate', 'residual') else \
            (1 + 0.3 * r(dim)).to(w_dtype).cuda()
    return x


def _call(x, **kw):
    return ops.norm_gate_residual(x['y'], post_weight=x.get('post'), gate=x.get('gate'),
                                  scale=x.get('scale'), residual=x.get('residual'),
                                  pre_weight=x.get('pre'), **kw)


def _np(x):
    return {n: t.detach().double().cpu().numpy() for n, t in x.items()}


def _near(got, want, tol):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want), \
        np.linalg.norm(got - want) / np.linalg.norm(want)


SIZES = [(1, 1), (3, 128), (70, 129), (5, 513), (2, 1000), (4, 2050), (3, 4096), (2, 5001),
         (2, 16384)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('size', SIZES)
def test_forward_and_gradients(size, dtype):
    rows, dim = size
    x = _operands(rows, dim, FORMS[0], dtype, seed=dim)
    for t in x.values():
        t.requires_grad_()
    gen = torch.Generator().manual_seed(dim)
    gs, gn = (torch.randn(rows, dim, generator=gen).to(dtype).cuda() for _ in range(2))
    outs = _call(x)
    grads = torch.autograd.grad(outs, list(x.values()), (gs, gn))
    a = _np({**x, 'grad_stream': gs, 'grad_normed': gn})
    want, wg = sequence.norm_gate_residual(**a)
    for o, w in zip(outs, want):
        assert o.dtype == dtype
        _near(o, w, TOL[dtype])
    for n, g in zip(x, grads):
        assert g.dtype == x[n].dtype
        # a row's gradient is what its projection off the row leaves; with one value a row that
        # is eps / x^2 of it, and nothing is left to compare
        if dim > 1 or n not in ('y', 'post', 'gate', 'scale', 'residual'):
            _near(g, wg[n], 4 * F32 + TOL[g.dtype])


# rows of 5 and 6 waves' runs, and so many of them that a workgroup takes several
@pytest.mark.parametrize('size', [(700, 2049), (1100, 2568), (600, 3070), (5, 3080), (1300, 640)])
def test_many_rows_forward_and_gradients(size):
    test_forward_and_gradients(size, torch.bfloat16)


@pytest.mark.parametrize('w_dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('parts', FORMS)
def test_parts_left_out(parts, w_dtype):
    rows, dim = 300, 200
    x = _operands(rows, dim, parts, torch.bfloat16, w_dtype, seed=3)
    stream, normed = _call(x, eps=1e-3)
    want = sequence.norm_gate_residual(**_np(x), eps=1e-3)
    _near(stream, want[0], TOL[torch.bfloat16])
    assert (normed is None) == ('pre' not in parts)
    if normed is not None:
        _near(normed, want[1], TOL[torch.bfloat16])
    for t in x.values():
        t.requires_grad_()
    outs = [o for o in _call(x, eps=1e-3) if o is not None]
    gen = torch.Generator().manual_seed(1)
    ups = [torch.randn(rows, dim, generator=gen).bfloat16().cuda() for _ in outs]
    grads = torch.autograd.grad(outs, list(x.values()), ups)
    a = _np({**x, **dict(zip(('grad_stream', 'grad_normed'), ups))})
    wg = sequence.norm_gate_residual(**a, eps=1e-3)[1]
    for n, g in zip(x, grads):
        _near(g, wg[n], 4 * F32 + TOL[g.dtype])


def test_gradient_of_one_output_and_some_operands():
    x = _operands(40, 96, FORMS[0], torch.float32, seed=5)
    d = torch.randn(40, 96, generator=torch.Generator().manual_seed(2)).cuda()
    a = _np({**x, 'd': d})
    d64 = a.pop('d')
    for which in (0, 1):
        x['gate'].requires_grad_()
        x['post'].requires_grad_()
        got = torch.autograd.grad(_call(x)[which], [x['gate'], x['post']], d)
        wg = sequence.norm_gate_residual(**a, **{('grad_stream', 'grad_normed')[which]: d64})[1]
        _near(got[0], wg['gate'], 4 * F32)
        _near(got[1], wg['post'], 4 * F32)


def test_gradients_against_differences():
    x = _operands(6, 33, FORMS[0], torch.float32, seed=6)
    d1, d2 = (torch.randn(6, 33, generator=torch.Generator().manual_seed(i)).cuda()
              for i in (1, 2))
    for t in x.values():
        t.requires_grad_()
    grads = torch.autograd.grad(_call(x), list(x.values()), (d1, d2))
    for (n, t), g in zip(x.items(), grads):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(9)).cuda()

        def loss(e):
            with torch.no_grad():
                s, m = _call({**x, n: t + e * d})
            return (s.double() * d1).sum() + (m.double() * d2).sum()

        num = (8 * (loss(5e-3) - loss(-5e-3)) - (loss(1e-2) - loss(-1e-2))) / 6e-2
        want = (g.double() * d).sum()
        # a fourth-order difference of step 5e-3 over 32-bit values
        assert abs(num - want) < 1e-3 * max(abs(want), g.double().norm()), n


def test_strides_shapes_and_a_number_as_scale():
    x = _operands(60, 72, ('post', 'gate', 'residual', 'pre'), torch.bfloat16, seed=8)
    s, n = _call(x)
    wide = torch.zeros(60, 3 * 72 + 1, dtype=torch.bfloat16, device='cuda')
    y = wide[:, 1:73]
    y.copy_(x['y'])
    gate = x['gate'].t().contiguous().t()
    s2, n2 = _call({**x, 'y': y, 'gate': gate})
    assert torch.equal(s, s2) and torch.equal(n, n2)
    s3, n3 = _call({k: v.reshape(3, 4, 5, 72) if v.dim() == 2 else v for k, v in x.items()})
    assert s3.shape == (3, 4, 5, 72) and torch.equal(s3.reshape(60, 72), s)
    a = _np(x)
    s4, n4 = _call({**x, 'scale': 0.25})
    want = sequence.norm_gate_residual(**a, scale=np.full(72, 0.25))
    _near(s4, want[0], TOL[torch.bfloat16])
    _near(n4, want[1], TOL[torch.bfloat16])


def test_rows_of_zeros_and_no_rows():
    x = _operands(4, 64, FORMS[0], torch.float32)
    x['y'][1] = 0
    x['residual'][1] = 0
    s, n = _call(x)
    assert (s[1] == 0).all() and (n[1] == 0).all() and torch.isfinite(n).all()
    e = {k: (v[:0] if v.dim() == 2 else v).clone().requires_grad_() for k, v in x.items()}
    s, n = _call(e)
    assert s.shape == n.shape == (0, 64)
    grads = torch.autograd.grad((s, n), list(e.values()), (s, n))
    assert all((g == 0).all() for g in grads) and grads[1].shape == (64,)


def test_the_same_bits_every_time():
    x = _operands(3000, 260, FORMS[0], torch.bfloat16, seed=2)
    for t in x.values():
        t.requires_grad_()
    first = torch.autograd.grad(_call(x), list(x.values()), (x['y'].detach(), x['gate'].detach()))
    again = torch.autograd.grad(_call(x), list(x.values()), (x['y'].detach(), x['gate'].detach()))
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals():
    y = torch.zeros(4, 32, device='cuda')
    with pytest.raises(TypeError, match='not supported'):
        ops.norm_gate_residual(y.double())
    with pytest.raises(TypeError, match='gate is'):
        ops.norm_gate_residual(y, gate=y.half())
    with pytest.raises(ValueError, match='residual must be'):
        ops.norm_gate_residual(y, residual=y[:2])
    with pytest.raises(ValueError, match='pre_weight must be'):
        ops.norm_gate_residual(y, pre_weight=y[0, :5])
    with pytest.raises(ValueError, match='1..16384'):
        ops.norm_gate_residual(torch.zeros(1, 16385, device='cuda'))
    with pytest.raises(ValueError, match='on the GPU'):
        ops.norm_gate_residual(y.cpu())
