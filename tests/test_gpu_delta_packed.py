"""Packed sequences of the gated delta rule whose first one begins chunks after the row's start,
and no sequence at all: rows outside all sequences give 0, and so do their gradients.

Tolerances: 64 x 2^-24 of the norm for 32-bit sums, 8 times that for dg (a difference of sums over 64
tokens) and, in gradients, for the terms' spread over a sequence; 16-bit results add 2^-8.
"""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

F32 = 64 * 2.0 ** -24
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}
H, DK, DV = 4, 40, 48


def _operands(total, dtype, seed):
    rs = np.random.RandomState(seed)
    k = rs.randn(1, total, 2, DK) + 0.3
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    arrays = [rs.randn(1, total, 2, DK), k, rs.randn(1, total, H, DV), -rs.rand(1, total, H),
              rs.rand(1, total, H)]
    x = [torch.tensor(a).to(dtype).cuda() for a in arrays]
    return x, torch.tensor(rs.randn(1, total, H, DV)).to(dtype).cuda()


def _near(got, want, tol):
    got = got.detach().double().cpu().numpy()
    assert np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


# first offsets on a chunk's edge, inside one and past several; tails of more than a chunk
@pytest.mark.parametrize('dtype', list(UNIT))
@pytest.mark.parametrize('cuts', [[64, 100, 264, 300], [100, 200, 300], [130, 131, 131, 259],
                                  [640, 645], [63, 127, 128], [128, 128, 128]])
def test_late_first_sequences(cuts, dtype):
    n, total = len(cuts) - 1, cuts[-1] + 80
    x, do = _operands(total, dtype, seed=cuts[0])
    s0 = torch.randn(n, H, DK, DV, generator=torch.Generator().manual_seed(2)).cuda()
    offsets = torch.tensor(cuts, dtype=torch.int32).cuda()
    leaves = [y.requires_grad_() for y in (*x, s0)]
    o, s1 = ops.gated_delta_rule(*x, initial_state=s0, seq_offsets=offsets)
    grads = torch.autograd.grad(o, leaves, do)
    a = [y.detach().double().cpu().numpy() for y in (*x, s0, do)]
    want_o, want_s, want = np.zeros(o.shape), np.zeros(s1.shape), [np.zeros(y.shape) for y in a[:6]]
    for i, (p, e) in enumerate(zip(cuts, cuts[1:])):
        (want_o[0, p:e], want_s[i]), r = sequence.gated_delta(
            *(y[0, p:e] for y in a[:5]), state=a[5][i], grad_o=a[6][0, p:e])
        for j in range(5):
            want[j][0, p:e] = r[j]
        want[5][i] = r[5]
    _near(o, want_o, F32 + UNIT[dtype])
    _near(s1, want_s, F32)
    for got, w in zip(grads, want):
        _near(got, w, 8 * F32 + UNIT[got.dtype])
    for got in (o, *grads[:5]):
        assert (got[:, :cuts[0]] == 0).all() and (got[:, cuts[-1]:] == 0).all()


@pytest.mark.parametrize('tokens', [0, 10, 100])
def test_no_sequence_at_all(tokens):
    """Offsets of one entry: every token is outside."""
    x, do = _operands(tokens, torch.float32, seed=1)
    s0 = torch.zeros(0, H, DK, DV, device='cuda')
    offsets = torch.tensor([min(tokens, 3)], dtype=torch.int32).cuda()
    o, s1 = ops.gated_delta_rule(*x, seq_offsets=offsets)
    assert o.shape == (1, tokens, H, DV) and (o == 0).all() and s1.shape == (0, H, DK, DV)
    leaves = [y.requires_grad_() for y in (*x, s0)]
    o, s1 = ops.gated_delta_rule(*x, initial_state=s0, seq_offsets=offsets)
    assert (o == 0).all()
    for got, y in zip(torch.autograd.grad((o, s1), leaves, (do, s1.detach())), leaves):
        assert got.shape == y.shape and (got == 0).all()
