"""The 8-bit integer product with token and channel scales, against 64 bits.

Integers are equal to the definition's (a quotient that 32 bits round across a half would differ
by one: the seeds here have none).  The products' sums are exact and three roundings of 2^-24
follow, so 32-bit results are within 4 x 2^-24 of each value's own size plus the bias's; 16-bit
ones add their rounding.
"""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _operands(m, k, n, dtype=torch.float32, seed=0):
    rs = np.random.RandomState(seed)
    x = torch.tensor(rs.randn(m, k) * (0.1 + rs.rand(m, 1))).to(dtype).cuda()
    w8 = torch.tensor(rs.randint(-128, 128, (n, k)), dtype=torch.int8).cuda()
    ws = torch.tensor(0.01 * (0.5 + rs.rand(n)), dtype=torch.float32).cuda()
    bias = torch.tensor(rs.randn(n)).to(dtype).cuda()
    return x, w8, ws, bias


def _np(t):
    return t.double().cpu().numpy()


def _close(y, x8, a, w8, ws, bias=None):
    """y against exact sums of the given integers."""
    s = _np(x8) @ _np(w8).T * _np(a)[:, None] * _np(ws)
    b = 0 if bias is None else _np(bias)
    got = _np(y)
    tol = (4 * 2.0 ** -24) * (np.abs(s) + np.abs(b)) + UNIT[y.dtype] * np.abs(s + b) + 1e-7 * (
        y.dtype == torch.float16)      # float16 below 6e-5 is spaced 6e-8 apart
    assert got.shape == s.shape and (np.abs(got - (s + b)) <= tol).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('size', [(1, 1), (3, 7), (70, 129), (2, 4096), (5, 9001)])
def test_quantize(size, dtype):
    x = _operands(*size, 1, dtype, seed=size[1])[0]
    x[0, 0] = 0
    x8, a = ops.int8_quantize(x)
    w8, wa = sequence.int8_quantize(_np(x))
    assert np.array_equal(x8.cpu().numpy(), w8)
    assert np.abs(_np(a) - wa).max() <= 2.0 ** -24 * wa.max()


SIZES = [(1, 1, 1), (1, 4096, 300), (16, 129, 17), (17, 64, 100), (33, 1000, 45), (77, 300, 300),
         (130, 256, 70), (200, 513, 129), (300, 1024, 2000), (1030, 272, 1100), (513, 100, 4100),
         (4100, 48, 4200)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('size', SIZES)
def test_product(size, dtype):
    m, k, n = size
    x, w8, ws, bias = _operands(m, k, n, dtype, seed=m)
    x8, a = ops.int8_quantize(x)
    _close(ops.int8_linear(x, w8, ws, bias=bias), x8, a, w8, ws, bias)
    y = ops.int8_matmul(x8, a, w8, ws, out_dtype=dtype)
    _close(y, x8, a, w8, ws)
    assert torch.equal(y, ops.int8_linear(x, w8, ws))


# tokens around the counts where another form of the product takes over, few and many channels
@pytest.mark.parametrize('size', [(32, 200, 300), (33, 200, 2100), (64, 1000, 300), (65, 64, 1000),
                                  (96, 272, 4100), (129, 130, 520), (257, 384, 300),
                                  (500, 1000, 260), (1000, 128, 17), (4100, 33, 5)])
def test_product_between_forms(size):
    m, k, n = size
    x, w8, ws, bias = _operands(m, k, n, torch.bfloat16, seed=m)
    x8, a = ops.int8_quantize(x)
    _close(ops.int8_linear(x, w8, ws, bias=bias), x8, a, w8, ws, bias)


def test_against_the_definition():
    x, w8, ws, bias = _operands(90, 500, 210, seed=4)
    y = ops.int8_linear(x, w8, ws, bias=bias)
    want = sequence.int8_linear(_np(x), _np(w8), _np(ws), _np(bias))
    assert np.abs(_np(y) - want).max() <= 1e-6 * np.abs(want).max()


def test_extreme_integers_do_not_overflow():
    m, k, n = 20, 65536, 20
    x8 = torch.full((m, k), -128, dtype=torch.int8, device='cuda')
    w8 = torch.full((n, k), -128, dtype=torch.int8, device='cuda')
    one = torch.ones(20, device='cuda')
    assert (ops.int8_matmul(x8, one, w8, one) == 2.0 ** 30).all()


@pytest.mark.parametrize('m', [4, 300])
def test_rows_of_zeros_nan_and_infinity(m):
    """Each is its own row's matter."""
    x, w8, ws, bias = _operands(m, 200, 70, seed=5)
    clean = ops.int8_linear(x, w8, ws, bias=bias)
    x[0] = 0
    x[1, 7], x[2, 9] = float('nan'), float('-inf')
    y = ops.int8_linear(x, w8, ws, bias=bias)
    assert torch.equal(y[0], bias) and torch.isnan(y[1:3]).all() and torch.equal(y[3:], clean[3:])
    assert (ops.int8_quantize(x)[0][:3] == 0).all()


def test_strides_unaligned_weights_and_shapes():
    x, w8, ws, bias = _operands(150, 96, 130, torch.bfloat16, seed=6)
    y = ops.int8_linear(x, w8, ws, bias=bias)
    wide = torch.zeros(150, 200, dtype=torch.bfloat16, device='cuda')
    wide[:, 3:99] = x
    flat = torch.zeros(130 * 96 + 1, dtype=torch.int8, device='cuda')
    flat[1:] = w8.reshape(-1)
    assert torch.equal(y, ops.int8_linear(wide[:, 3:99], flat[1:].view(130, 96), ws, bias=bias))
    assert torch.equal(y, ops.int8_linear(x.t().contiguous().t(), w8.t().contiguous().t(), ws,
                                          bias=bias))
    assert torch.equal(y.view(3, 50, 130), ops.int8_linear(x.view(3, 50, 96), w8, ws, bias=bias))
    assert torch.equal(y[0], ops.int8_linear(x[0], w8, ws, bias=bias))
    assert ops.int8_linear(x[:0], w8, ws).shape == (0, 130)
    assert ops.int8_linear(x, w8[:0], ws[:0]).shape == (150, 0)


def test_refusals():
    x, w8, ws, bias = _operands(4, 32, 8)
    with pytest.raises(TypeError, match='not supported'):
        ops.int8_linear(x.double(), w8, ws)
    with pytest.raises(ValueError, match='w8 must be int8'):
        ops.int8_linear(x, w8.float(), ws)
    with pytest.raises(ValueError, match='tokens'):
        ops.int8_linear(x[:, :31], w8, ws)
    with pytest.raises(ValueError, match='w_scale must be'):
        ops.int8_linear(x, w8, ws[:7])
    with pytest.raises(ValueError, match='bias must be'):
        ops.int8_linear(x, w8, ws, bias=bias[:7])
    with pytest.raises(ValueError, match='no gradient'):
        ops.int8_linear(x.clone().requires_grad_(), w8, ws)
    with pytest.raises(ValueError, match='x_scale must be'):
        ops.int8_matmul(w8, ws[:7], w8, ws)
    with pytest.raises(TypeError, match='x8 must be'):
        ops.int8_matmul(x, ws[:4], w8, ws)
    with pytest.raises(ValueError, match='1..65536'):
        ops.int8_quantize(torch.zeros(1, 65537, device='cuda'))
