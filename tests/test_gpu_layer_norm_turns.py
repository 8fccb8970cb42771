"""Layer norm where every workgroup goes over several groups of rows, the last of them not whole:
each of its forms, with the weights' gradients that it sums over them.

Tolerances are of the norm of the difference over the norm of the result: 32-bit sums over a row by a
tree of lanes, a dozen dependent roundings of 2^-24 a value, so 32 x 2^-24; sums over R rows for the
weights' gradients walk up to R / 256 of them in a row, whose roundings add like their root.  16-bit
outputs add their rounding.
"""
import pytest
import torch

from brainstate_amd import ops

pytestmark = pytest.mark.gpu

F32 = 32 * 2.0 ** -24
TOL = {torch.float32: F32, torch.bfloat16: F32 + 2.0 ** -8, torch.float16: F32 + 2.0 ** -11}

# rows x dim: rows shorter than a vector, 16 lanes a row, a wave a row, a workgroup of up to 512 and up
# to 1,024 threads a row, two vectors a lane; whole vectors and odd ends
SIZES = [(40001, 5), (40003, 100), (40003, 104), (9001, 512), (9003, 509), (5003, 513), (2100, 2048),
         (2100, 2050), (1100, 4096), (1100, 4099), (1100, 8192), (1100, 8191), (600, 16384),
         (800, 9001)]


def near(got, want, tol, name):
    assert got.shape == want.shape and got.isfinite().all(), name
    err = (got.double() - want).norm() / want.norm()
    assert err <= tol, (name, err.item())


@pytest.mark.parametrize('p', [0.0, 0.3])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', SIZES)
def test_rows_in_turns(size, dtype, p):
    rows, dim = size
    gen = torch.Generator(device='cuda').manual_seed(dim)
    randn = lambda *s: torch.randn(s, generator=gen, device='cuda')             # noqa: E731
    x, residual, gs, gn = (randn(rows, dim).to(dtype) for _ in range(4))
    w, b = 1 + 0.3 * randn(dim), randn(dim)
    args = [t.requires_grad_() for t in (x, residual, w, b)]
    outs = ops.add_layer_norm(*args, p=p, seed=77, site=3)
    grads = torch.autograd.grad(outs, args, [gs, gn])
    x, residual, w, b, gs, gn = (t.detach().double() for t in (x, residual, w, b, gs, gn))
    m = (ops.dropout(torch.ones(rows, dim, device='cuda'), p, 77, site=3) != 0).double() / (1 - p)
    stream = residual + x * m
    d = stream - stream.mean(1, keepdim=True)
    r = (d.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    h, dh = d * r, gn * w
    ds = gs + r * (dh - dh.mean(1, keepdim=True) - h * (dh * h).mean(1, keepdim=True))
    near(outs[0], stream, TOL[dtype], 'stream')
    near(outs[1], h * w + b, TOL[dtype], 'normed')
    near(grads[0], ds * m, TOL[dtype], 'dx')
    near(grads[1], ds, TOL[dtype], 'dresidual')
    near(grads[2], (gn * h).sum(0), F32, 'dweight')
    near(grads[3], gn.sum(0), F32, 'dbias')
