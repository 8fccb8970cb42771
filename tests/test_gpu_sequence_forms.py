"""The forms of the sequence-layer kernels that only larger calls reach: tiles of 128 and 256 of the
integer product with several steps of k, gradients of norms whose lanes have two runs and whose
workgroups several rows.

Tolerances as in the operators' own tests: 32 x 2^-24 of the norm for results of the norms (4 times
that more for gradients), exact integer sums with four roundings of 2^-24; 16-bit results add their
rounding.
"""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _near(got, want, tol, name):
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    off = ((got.double() - want).norm() / want.norm()).item()
    assert off <= tol, (name, off)


# ------------------------------------------------------------------- integer product
# tiles of 128 and of 256, steps of 128 values even, odd and cut, weights that start on 16 bytes
# and that do not, rows of whole and of cut groups of 4
@pytest.mark.parametrize('size', [(2048, 272, 4100), (2050, 200, 4097), (2048, 640, 4096),
                                  (4100, 400, 4200), (4100, 272, 4097), (4100, 401, 4200)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_large_integer_products(size, dtype):
    m, k, n = size
    rs = np.random.RandomState(k)
    x = torch.tensor(rs.randn(m, k) * (0.1 + rs.rand(m, 1))).to(dtype).cuda()
    w8 = torch.tensor(rs.randint(-128, 128, (n, k)), dtype=torch.int8).cuda()
    ws = torch.tensor(0.01 * (0.5 + rs.rand(n)), dtype=torch.float32).cuda()
    bias = torch.tensor(rs.randn(n)).to(dtype).cuda()
    x8, a = ops.int8_quantize(x)
    s = (x8.double() @ w8.double().t()) * a.double()[:, None] * ws.double()
    want = s + bias.double()
    tol = 4 * 2.0 ** -24 * (s.abs() + bias.double().abs()) + UNIT[dtype] * want.abs()
    y = ops.int8_linear(x, w8, ws, bias=bias)
    assert ((y.double() - want).abs() <= tol).all()
    assert torch.equal(ops.int8_matmul(x8, a, w8, ws, bias=bias, out_dtype=dtype), y)


# ------------------------------------------------------------------- norms
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', [(600, 5001), (600, 8192), (600, 16384), (700, 9000)])
def test_gradients_of_wide_rows(size, dtype):
    """Two runs a lane; each workgroup takes several rows."""
    rows, dim = size
    rng = torch.Generator().manual_seed(dim)
    r = lambda *s: torch.randn(*s, generator=rng).cuda()                        # noqa: E731
    x = dict(y=r(rows, dim).to(dtype), post=1 + 0.3 * r(dim), gate=r(rows, dim).to(dtype),
             scale=1 + 0.3 * r(dim), residual=r(rows, dim).to(dtype), pre=1 + 0.3 * r(dim))
    gs, gn = r(rows, dim).to(dtype), r(rows, dim).to(dtype)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    stream, normed = ops.norm_gate_residual(
        leaves['y'], leaves['post'], leaves['gate'], leaves['scale'], leaves['residual'],
        leaves['pre'])
    grads = torch.autograd.grad((stream, normed), list(leaves.values()), (gs, gn))
    a = {n: t.double().cpu().numpy() for n, t in x.items()}
    want, wg = sequence.norm_gate_residual(**a, grad_stream=gs.double().cpu().numpy(),
                                           grad_normed=gn.double().cpu().numpy())
    tol = 32 * 2.0 ** -24
    for name, got, w, extra in [('stream', stream, want[0], tol + UNIT[dtype]),
                                ('normed', normed, want[1], tol + UNIT[dtype])] + \
            [(n, g, wg[n], 5 * tol + UNIT[g.dtype]) for n, g in zip(x, grads)]:
        _near(got.detach(), torch.tensor(w).cuda(), extra, name)
