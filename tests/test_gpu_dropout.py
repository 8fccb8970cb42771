"""Dropout: which elements are kept, bit for bit, from the generator in numpy's integers; what is
kept is one 32-bit product away from x, rounded once more to x's type."""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
SEED = 0x7F3456789ABCDEF0


def randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to('cuda', dtype)


def want_of(x, p, seed=SEED, site=0):
    """The operator in 32-bit torch arithmetic from the oracle's mask."""
    rows = x.reshape(-1, x.shape[-1])
    mask = torch.tensor(sequence.dropout_mask(seed, site, *rows.shape, p) > 0).cuda()
    scale = torch.tensor(1 / (1 - p), dtype=torch.float32, device='cuda')
    y = torch.where(mask, rows.float() * scale, torch.zeros((), device='cuda'))
    return y.to(x.dtype).view(x.shape)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(1,), (3, 2), (5, 7), (4, 8), (3, 9), (2, 3, 130), (70, 217),
                                   (2, 4097)])
@pytest.mark.parametrize('p', [0.1, 0.5])
def test_forward_and_gradient(shape, dtype, p):
    x = randn(*shape, dtype=dtype).requires_grad_()
    g = randn(*shape, dtype=dtype, seed=1)
    y = ops.dropout(x, p, SEED, site=2)
    assert torch.equal(y, want_of(x.detach(), p, site=2))
    assert torch.equal(torch.autograd.grad(y, x, g)[0], want_of(g, p, site=2))


def test_known_words():
    """The published answer for a counter and key of zeros."""
    assert [hex(w) for w in sequence.philox(0, 0, [0], 4)[0]] == \
        ['0x6627e8d5', '0xe169c58d', '0xbc57ac4c', '0x9b00dbd8']


@pytest.mark.parametrize('p', [0.0, 0.03, 0.9])
def test_share_of_what_is_kept(p):
    """n independent draws of chance 1 - p lie within 5 standard deviations of their mean."""
    x = torch.ones(1024, 1024, device='cuda')
    kept = (ops.dropout(x, p, 77) != 0).double().mean().item()
    assert abs(kept - (1 - p)) <= 5 * (p * (1 - p) / x.numel()) ** 0.5


def test_seeds_and_sites_tell_apart():
    x = torch.ones(64, 64, device='cuda')
    a = ops.dropout(x, 0.5, 1)
    for b in (ops.dropout(x, 0.5, 2), ops.dropout(x, 0.5, 1, site=1), ops.dropout(x, 0.5, 1 << 40)):
        assert 0.4 < (a == b).double().mean().item() < 0.6
    assert torch.equal(a[:10], ops.dropout(x[:10], 0.5, 1))


def test_seed_in_a_tensor():
    x = randn(9, 100).requires_grad_()
    seed = torch.tensor([SEED], device='cuda')
    y = ops.dropout(x, 0.3, seed)
    assert torch.equal(y, ops.dropout(x, 0.3, SEED))
    g = torch.ones_like(x)
    assert torch.equal(torch.autograd.grad(y, x, g)[0], want_of(g, 0.3))
    y = ops.dropout(x, 0.3, seed)
    seed += 1                    # another mask: the backward pass of the first one is refused
    with pytest.raises(RuntimeError, match='inplace'):
        torch.autograd.grad(y, x, g)


def test_what_is_dropped_is_zero():
    x = randn(7, 333)
    keep = torch.tensor(sequence.dropout_mask(4, 0, 7, 333, 0.5) > 0).cuda()
    x[~keep] = float('nan')
    x[0][~keep[0]] = float('inf')
    assert torch.equal(ops.dropout(x, 0.5, 4), want_of(torch.nan_to_num(x), 0.5, seed=4))


def test_strides_and_nothing():
    x = randn(6, 50, dtype=torch.bfloat16)
    want = ops.dropout(x, 0.2, 3)
    wide = torch.zeros(6, 55, dtype=torch.bfloat16, device='cuda')
    wide[:, 1:51] = x
    assert torch.equal(ops.dropout(wide[:, 1:51], 0.2, 3), want)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.2, 3), want)
    assert ops.dropout(x[:0], 0.2, 3).shape == (0, 50) and ops.dropout(x[:, :0], 0.2, 3).shape == (6, 0)


def test_rows_past_32_bits_are_counted_whole():
    """The row's upper half is part of the counter."""
    a, b = sequence.philox(SEED, 0, [5, 5 + (1 << 32)], 8)
    assert not (a == b).any()


def test_refusals():
    x = randn(3, 4)
    for p in (-0.1, 1.0, float('nan')):
        with pytest.raises(ValueError, match='p must be'):
            ops.dropout(x, p, 1)
    with pytest.raises(TypeError, match='seed'):
        ops.dropout(x, 0.1, None)
    with pytest.raises(TypeError, match='seed'):
        ops.dropout(x, 0.1, 1.5)
    with pytest.raises(ValueError, match='seed'):
        ops.dropout(x, 0.1, -1)
    with pytest.raises(ValueError, match='seed'):
        ops.dropout(x, 0.1, torch.tensor([1]))
    with pytest.raises(ValueError, match='seed'):
        ops.dropout(x, 0.1, torch.tensor([1, 2], device='cuda'))
    with pytest.raises(ValueError, match='site'):
        ops.dropout(x, 0.1, 1, site=-1)
    with pytest.raises(ValueError, match='dimension'):
        ops.dropout(x[0, 0], 0.1, 1)
    with pytest.raises(TypeError, match='not supported'):
        ops.dropout(x.long(), 0.1, 1)
