"""Products with 4-bit weights against 64 bits.

Tolerances are of the norm of the difference over the norm of the result: products are exact, sums
over k of 32-bit roundings by tiles of 16 or 32 products add up like their root (at most 2,048 of
them, 45), and each group's sum is rounded twice more: 64 x 2^-24.  16-bit outputs add their
rounding.  Weights' integers and scales are compared bit for bit.
"""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

F32 = 64 * 2.0 ** -24
TOL = {torch.float32: F32, torch.bfloat16: F32 + 2.0 ** -8, torch.float16: F32 + 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def operands(m, k, n, group, dtype, seed=0):
    """Tokens, the integers, their bytes, scales and a bias; integers over the whole 0..15."""
    rs = np.random.RandomState(seed)
    x = torch.tensor(rs.randn(m, k)).to(dtype).cuda()
    u = rs.randint(0, 16, (n, k))
    scale = torch.tensor((0.5 + rs.rand(n, -(-k // group))) * 0.1, dtype=torch.float32).cuda()
    bias = torch.tensor(rs.randn(n)).to(dtype).cuda()
    return x, u, torch.tensor(sequence.int4_pack(u)).cuda(), scale, bias


def near(got, want, tol):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want) + 1e-30, \
        np.linalg.norm(got - want) / np.linalg.norm(want)


def want_of(x, u, scale, group, bias=None):
    f = lambda t: t.double().cpu().numpy()                                      # noqa: E731
    return sequence.int4_linear(f(x), u, f(scale), group, None if bias is None else f(bias))


SIZES = [(1, 1, 1), (1, 4096, 4096), (2, 127, 17), (16, 128, 16), (17, 130, 33), (33, 1000, 300),
         (64, 4224, 50), (65, 64, 64), (77, 1001, 300), (128, 256, 128), (300, 515, 1000),
         (1030, 384, 4100)]


@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_linear(size, dtype, group):
    x, u, w4, scale, bias = operands(*size, group, dtype, seed=size[1])
    y = ops.int4_linear(x, w4, scale, bias=bias, group=group)
    assert y.dtype == dtype
    near(y, want_of(x, u, scale, group, bias), TOL[dtype])
    near(ops.int4_linear(x, w4, scale, group=group), want_of(x, u, scale, group), TOL[dtype])


@pytest.mark.parametrize('dtype', TYPES)
def test_large_tiles(dtype):
    """Enough tiles of 256 x 128 for every CU, none of them whole at the edges."""
    x, u, w4, scale, bias = operands(4099, 256, 2100, 128, dtype)
    y = ops.int4_linear(x, w4, scale, bias=bias)
    near(y, want_of(x, u, scale, 128, bias), TOL[dtype])


@pytest.mark.parametrize('m', [1, 20, 90])
def test_exact_where_every_number_is(m):
    """Small whole tokens and scales of powers of two: every sum is exact, so is the result."""
    rs = np.random.RandomState(0)
    x = torch.tensor(rs.randint(-3, 4, (m, 777)), dtype=torch.float32).cuda()
    u = rs.randint(0, 16, (90, 777))
    scale = torch.tensor(2.0 ** rs.randint(-3, 3, (90, 25)), dtype=torch.float32).cuda()
    w4 = torch.tensor(sequence.int4_pack(u)).cuda()
    want = torch.tensor(want_of(x, u, scale, 32)).cuda()
    for dtype in TYPES:
        assert torch.equal(ops.int4_linear(x.to(dtype), w4, scale, group=32),
                           want.to(torch.float32).to(dtype)), dtype


@pytest.mark.parametrize('m', [3, 100])
@pytest.mark.parametrize('dtype', TYPES)
def test_sums_that_cancel(m, dtype):
    """A pair of tokens' values 2^12 times the others' whose weights cancel leaves the others' sum,
    with the roundings of the large ones' products only."""
    x, u, w4, scale, _ = operands(m, 512, 40, 128, dtype, seed=3)
    x[:, 5], x[:, 9] = 4096.0, 4096.0
    u[:, 5], u[:, 9] = 15, 1
    w4 = torch.tensor(sequence.int4_pack(u)).cuda()
    want = want_of(x, u, scale, 128)
    got = ops.int4_linear(x, w4, scale).double().cpu().numpy()
    size = 4096 * 7 * scale.max().item()
    step = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert (np.abs(got - want) <= 16 * 2.0 ** -24 * size + step * np.abs(want) + F32 * 10).all()


def test_rows_do_not_depend_on_what_runs_beside_them():
    x, u, w4, scale, bias = operands(50, 1000, 60, 64, torch.bfloat16, seed=7)
    y = ops.int4_linear(x, w4, scale, bias, 64)
    z = x.clone()
    z[::2] = float('nan')
    got = ops.int4_linear(z, w4, scale, bias, 64)
    assert torch.equal(got[1::2], y[1::2]) and got[::2].isnan().all()


def test_strides_leading_dimensions_and_nothing():
    x, u, w4, scale, bias = operands(70, 256, 96, 128, torch.bfloat16, seed=2)
    want = ops.int4_linear(x, w4, scale, bias)
    wide = torch.full((70, 300), float('nan'), dtype=torch.bfloat16, device='cuda')
    wide[:, 3:259] = x
    for rows in (slice(0, 70), slice(0, 9)):
        assert torch.equal(ops.int4_linear(wide[rows, 3:259], w4, scale, bias),
                           ops.int4_linear(x[rows], w4, scale, bias))
    assert torch.equal(ops.int4_linear(x.t().contiguous().t(), w4, scale, bias), want)
    assert torch.equal(ops.int4_linear(x.view(7, 10, 256), w4, scale, bias).view(70, 96), want)
    assert torch.equal(ops.int4_linear(x, w4.t().contiguous().t(), scale.t().contiguous().t(),
                                       bias), want)
    pad = torch.zeros(96 * 128 + 1, dtype=torch.uint8, device='cuda')
    pad[1:] = w4.flatten()                              # bytes that start anywhere
    assert torch.equal(ops.int4_linear(x, pad[1:].view(96, 128), scale, bias), want)
    assert ops.int4_linear(x[:0], w4, scale).shape == (0, 96)
    assert ops.int4_linear(x, w4[:0], scale[:0]).shape == (70, 0)


@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(1, 1), (3, 33), (20, 129), (300, 1000)])
def test_quantize(size, dtype, group):
    rs = np.random.RandomState(size[1])
    w = torch.tensor(rs.randn(*size)).to(dtype).cuda()
    w[0] = 0
    w4, scale = ops.int4_quantize(w, group)
    # in the kernel's own 32-bit operations: a quotient near a half may round to its other side
    g = torch.nn.functional.pad(w.float(), (0, -size[1] % group)).unflatten(1, (-1, group))
    top = g.abs().amax(2, keepdim=True)
    u = torch.where(top > 0, (7 * g / top).round(), torch.zeros_like(g)) + 8
    u = u.flatten(1)[:, :size[1]].cpu().numpy()
    assert torch.equal(w4, torch.tensor(sequence.int4_pack(u)).cuda())
    # (53 bits hold a quotient of 24-bit numbers well enough that rounding it again is exact)
    assert torch.equal(scale, (top[..., 0].double() / 7).float())
    want = sequence.int4_quantize(w.double().cpu().numpy(), group)[0]
    assert (np.abs(u - want) <= 1).all() and (u != want).mean() < 1e-3


def test_quantize_then_multiply():
    """Rounding each weight by at most half a step of its group."""
    w = torch.randn(100, 300, generator=torch.Generator().manual_seed(0)).cuda()
    w4, scale = ops.int4_quantize(w)
    eye = torch.eye(300, device='cuda')
    back = ops.int4_linear(eye, w4, scale).t()
    half = 0.5 * scale.repeat_interleave(128, 1)[:, :300]
    assert ((back - w).abs() <= half * (1 + 1e-5)).all()


def test_quantize_extremes():
    big = torch.finfo(torch.float32).max
    w = torch.tensor([[big, -big, big / 2] + [0.0] * 29, [float('inf')] + [1.0] * 31,
                      [float('nan')] + [1.0] * 31, [1e-42, -1e-42] + [0.0] * 30], device='cuda')
    w4, scale = ops.int4_quantize(w, 32)
    assert w4[0, 0] == 15 | 1 << 4 and (w4[1:3] == 0x88).all()
    assert scale[1, 0] == float('inf') and scale[2, 0].isnan()
    y = ops.int4_linear(torch.ones(1, 32, device='cuda'), w4, scale, group=32)
    assert y[0, 1].isnan() and y[0, 2].isnan() and y[0, 3] == 0


def test_refusals():
    x, u, w4, scale, bias = operands(3, 100, 8, 32, torch.float32)
    for group in (16, 48, 256, 0):
        with pytest.raises(ValueError, match='group must be'):
            ops.int4_linear(x, w4, scale, group=group)
    with pytest.raises(ValueError, match='w4 must be'):
        ops.int4_linear(x[:, :98], w4, scale, group=32)
    with pytest.raises(ValueError, match='w4 must be'):
        ops.int4_linear(x, w4.to(torch.int8), scale, group=32)
    with pytest.raises(ValueError, match='w_scale must be'):
        ops.int4_linear(x, w4, scale[:, :3], group=32)
    with pytest.raises(ValueError, match='w_scale must be'):
        ops.int4_linear(x, w4, scale)
    with pytest.raises(ValueError, match='bias must be'):
        ops.int4_linear(x, w4, scale, bias[:3], 32)
    with pytest.raises(ValueError, match='no gradient'):
        ops.int4_linear(x.requires_grad_(), w4, scale, group=32)
    with pytest.raises(ValueError, match='65536'):
        ops.int4_quantize(torch.zeros(1, 65537, device='cuda'))
    with pytest.raises(ValueError, match='on the GPU'):
        ops.int4_quantize(x.detach().cpu())
    with pytest.raises(TypeError, match='not supported'):
        ops.int4_quantize(x.detach().double())
