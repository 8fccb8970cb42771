"""Decay attention, chunked and token by token, against its definition in 64 bits.

Tolerances are of the norm of the difference over the norm of the result.  32-bit outputs: sums
of at most 128 + 64 products and a handful of dependent 32-bit roundings a chunk, 2^-24 each,
which add up like their root: 64 x 2^-24 = 4e-6 leaves room for a hundred chunks.  Outputs in 16
bits add their own rounding, 2^-8 (bfloat16) or 2^-11 (float16) at most.
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


def operands(lead, hk, h, dk, dv, dtype, seed=0, each=True, decay=0.3):
    rs = np.random.RandomState(seed)
    arrays = [rs.randn(*lead, hk, dk), rs.randn(*lead, hk, dk) + 0.3, rs.randn(*lead, h, dv)]
    g = -decay * rs.rand(*(lead if each else ()), h)
    return [torch.tensor(a).to(dtype).cuda() for a in arrays] + [
        torch.tensor(g, dtype=torch.float32).cuda()]


def numbers(*ts):
    return [t.detach().double().cpu().numpy() for t in ts]


def near(got, want, tol):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= tol * norm + 1e-30, np.linalg.norm(got - want) / norm


def rows(x, i, lead=1):
    """Row i of every operand; a rate for each head is every row's."""
    return [y[i] if y.ndim > lead else y for y in x]


SIZES = [(1, 1, 1, 1, 1, 1), (2, 64, 1, 1, 64, 64), (1, 65, 2, 4, 128, 128),
         (3, 63, 1, 3, 33, 17), (1, 200, 2, 2, 65, 96), (2, 130, 1, 2, 16, 128),
         (1, 7, 3, 3, 127, 1), (2, 700, 1, 2, 48, 33), (1, 1500, 2, 2, 128, 128)]


@pytest.mark.parametrize('each', [True, False])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_chunked_forward(size, dtype, each):
    b, t, hk, h, dk, dv = size
    x = operands((b, t), hk, h, dk, dv, dtype, seed=t, each=each)
    s0 = torch.randn(b, h, dk, dv, generator=torch.Generator().manual_seed(t)).cuda()
    o, s1 = ops.decay_attention(*x, initial_state=s0)
    assert o.dtype == dtype and s1.dtype == torch.float32
    a, s0 = numbers(*x), numbers(s0)[0]
    want = [sequence.decay_attention(*rows(a, i), state=s0[i]) for i in range(b)]
    near(o, np.stack([w[0] for w in want]), TOL[dtype])
    near(s1, np.stack([w[1] for w in want]), F32)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_packed_sequences(dtype):
    """Empty sequences, single tokens, ends inside a chunk, several segments, and tokens that are no
    sequence's."""
    offsets = [3, 3, 4, 68, 68, 197, 325, 330, 1200, 1200]
    n, total = len(offsets) - 1, 1207
    x = operands((1, total), 2, 4, 48, 40, dtype, seed=3)
    s0 = torch.randn(n, 4, 48, 40, generator=torch.Generator().manual_seed(1)).cuda()
    o, s1 = ops.decay_attention(*x, initial_state=s0,
                                seq_offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
    *a, s0 = numbers(*x, s0)
    want_o, want_s = np.zeros((total, 4, 40)), np.zeros((n, 4, 48, 40))
    for i, (p, e) in enumerate(zip(offsets, offsets[1:])):
        want_o[p:e], want_s[i] = sequence.decay_attention(*(y[0, p:e] for y in a), state=s0[i])
    near(o, want_o[None], TOL[dtype])
    assert (o[0, :3] == 0).all() and (o[0, 1200:] == 0).all()
    near(s1, want_s, F32)


def test_empty_sequences_only():
    x = operands((1, 0), 1, 2, 16, 16, torch.float32)
    s0 = torch.randn(2, 2, 16, 16).cuda()
    o, s1 = ops.decay_attention(*x, initial_state=s0,
                                seq_offsets=torch.zeros(3, dtype=torch.int32).cuda())
    assert o.shape == (1, 0, 2, 16) and torch.equal(s1, s0)
    o, s1 = ops.decay_attention(*x)
    assert s1.shape == (1, 2, 16, 16) and (s1 == 0).all()
    x = operands((1, 9), 1, 2, 16, 16, torch.float32)
    o, s1 = ops.decay_attention(*x, seq_offsets=torch.zeros(1, dtype=torch.int32).cuda())
    assert (o == 0).all() and s1.shape == (0, 2, 16, 16)


@pytest.mark.parametrize('low', [float('-inf'), torch.finfo(torch.float32).min])
def test_decays_that_empty_the_state(low):
    """g of -inf or the type's lowest value starts afresh inside a chunk; what follows keeps its
    own decays."""
    x = operands((1, 150), 1, 2, 32, 32, torch.float32, seed=5)
    g = x[3]
    g[:, 10], g[:, 64], g[:, 100:103], g[:, 20:30] = low, low, low, -60.0
    o, s1 = ops.decay_attention(*x)
    wo, ws = sequence.decay_attention(*(y[0] for y in numbers(*x)))
    near(o, wo[None], F32)
    near(s1, ws[None], F32)


def test_strided_and_unaligned_operands():
    """Views into one projection, a transposed layout, and rows that start at odd elements."""
    b, t, hk, h, dk, dv = 2, 70, 2, 4, 32, 24
    x = operands((b, t), hk, h, dk, dv, torch.bfloat16, seed=9)
    o, s1 = ops.decay_attention(*x)
    flat = torch.zeros(b, t, 2 * hk * dk + h * dv + 3, dtype=torch.bfloat16, device='cuda')
    views, at = [], 1
    for y in x[:3]:
        w = y.shape[2] * y.shape[3]
        view = flat[..., at:at + w].unflatten(-1, y.shape[2:])
        view.copy_(y)
        views.append(view)
        at += w
    heads_first = x[3].transpose(1, 2).contiguous().transpose(1, 2)
    o2, s2 = ops.decay_attention(*views, heads_first)
    assert torch.equal(o, o2) and torch.equal(s1, s2)
    v = x[2].transpose(2, 3).contiguous().transpose(2, 3)      # a head's values not side by side
    o3, s3 = ops.decay_attention(x[0], x[1], v, x[3])
    assert torch.equal(o, o3) and torch.equal(s1, s3)


@pytest.mark.parametrize('each', [True, False])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(1, 1, 1, 1, 1), (5, 2, 4, 128, 128), (3, 1, 3, 33, 17),
                                  (2, 3, 3, 64, 127), (9, 1, 1, 100, 36)])
def test_step(size, dtype, each):
    b, hk, h, dk, dv = size
    x = operands((b, 3), hk, h, dk, dv, dtype, seed=b, each=each)
    rs = np.random.RandomState(4)
    state = torch.tensor(rs.randn(b + 3, h, dk, dv), dtype=torch.float32).cuda()
    slots = torch.tensor(rs.permutation(b + 3)[:b], dtype=torch.int32)
    if b > 2:
        slots[1], slots[2] = -1, b + 3
    before, s = state.clone(), state.cpu().double().numpy()
    o = ops.decay_attention_step(*x, state, slots=slots.cuda())
    one = before.clone()
    for t in range(3):            # the same tokens one by one
        token = [y[:, t] for y in x[:3]] + [x[3][:, t] if each else x[3]]
        assert torch.equal(ops.decay_attention_step(*token, one, slots=slots.cuda()), o[:, t])
    assert torch.equal(one, state)
    a = numbers(*x)
    want = np.zeros((b, 3, h, dv))
    for i, at in enumerate(slots.tolist()):
        if 0 <= at < b + 3:
            want[i], s[at] = sequence.decay_attention(*rows(a, i), state=s[at])
        else:
            assert (o[i] == 0).all()
    near(o, want, TOL[dtype])
    near(state, s, F32)
    idle = [i for i in range(b + 3) if i not in slots.tolist()]
    assert torch.equal(state[idle], before[idle])


def test_step_continues_the_chunked_form():
    x = operands((2, 101), 1, 2, 64, 64, torch.float32, seed=6)
    o, s = ops.decay_attention(*x)
    _, state = ops.decay_attention(*(y[:, :97] for y in x))
    tail = ops.decay_attention_step(*(y[:, 97:] for y in x), state)
    near(tail, numbers(o[:, 97:])[0], F32)
    near(state, numbers(s)[0], F32)
