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


def grads_of(x, s0, do, dstate=None, **kw):
    x = [y.detach().requires_grad_() for y in x]
    s0 = None if s0 is None else s0.detach().requires_grad_()
    o, s1 = ops.decay_attention(*x, initial_state=s0, **kw)
    outs, ups = ([o, s1], [do, dstate]) if dstate is not None else ([o], [do])
    return torch.autograd.grad(outs, x + ([s0] if s0 is not None else []), ups)


# Gradients are sums of the same kind as the outputs.  dg is a difference of sums over the tokens of
# a chunk: errors of 64 terms add up like their root, 8 times one term's; 16 with those of the states'
# product that the sum starts from.
@pytest.mark.parametrize('each', [True, False])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_gradients(size, dtype, each):
    b, t, hk, h, dk, dv = size
    x = operands((b, t), hk, h, dk, dv, dtype, seed=t + 1, each=each)
    gen = torch.Generator().manual_seed(t)
    s0 = torch.randn(b, h, dk, dv, generator=gen).cuda()
    do = torch.randn(b, t, h, dv, generator=gen).to(dtype).cuda()
    dstate = torch.randn(b, h, dk, dv, generator=gen).cuda()
    got = grads_of(x, s0, do, dstate)
    a, (s0, do, dstate) = numbers(*x), numbers(s0, do, dstate)
    want = [sequence.decay_attention(*rows(a, i), state=s0[i], grad_o=do[i], grad_state=dstate[i])
            [1] for i in range(b)]
    for i, name in enumerate(('dq', 'dk', 'dv', 'dg', 'dstate')):
        w = np.stack([r[i] for r in want])
        tol = 16 * F32 if name == 'dg' else F32 if name == 'dstate' else TOL[dtype]
        near(got[i], w.sum(0) if name == 'dg' and not each else w, tol)
        assert got[i].dtype == (torch.float32 if name in ('dg', 'dstate') else dtype)


def test_gradients_without_states():
    x = operands((2, 300), 2, 2, 64, 64, torch.float32, seed=2)
    do = torch.randn(2, 300, 2, 64, generator=torch.Generator().manual_seed(1)).cuda()
    got = grads_of(x, None, do)
    a, do = numbers(*x), numbers(do)[0]
    want = [sequence.decay_attention(*rows(a, i), grad_o=do[i])[1] for i in range(2)]
    for i in range(4):
        near(got[i], np.stack([r[i] for r in want]), 16 * F32)


def test_gradients_with_fixed_decays():
    """Without a gradient of g the others have the same bits, and fewer states are kept."""
    x = operands((2, 300), 1, 2, 64, 96, torch.bfloat16, seed=2)
    do = torch.randn(2, 300, 2, 96, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = grads_of(x, None, do)
    y = [t.detach().requires_grad_() for t in x[:3]]
    o = ops.decay_attention(*y, x[3])[0]
    for a, b in zip(torch.autograd.grad(o, y, do), want):
        assert torch.equal(a, b)


def test_gradients_of_the_final_state_alone():
    x = operands((1, 600), 1, 2, 32, 48, torch.float32, seed=2)
    y = [t.requires_grad_() for t in x]
    ds = torch.randn(1, 2, 32, 48, generator=torch.Generator().manual_seed(1)).cuda()
    got = torch.autograd.grad(ops.decay_attention(*y)[1], y[1:], ds)
    a = [t[0] for t in numbers(*x)]
    want = sequence.decay_attention(*a, grad_o=np.zeros((600, 2, 48)), grad_state=numbers(ds)[0][0])
    for i in range(3):
        near(got[i], want[1][i + 1][None], 16 * F32)


def test_gradients_against_differences():
    """Of the operator itself, along random directions: central differences of a loss whose
    terms are 32-bit, so the step is large (1e-2) and the agreement 1e-3."""
    x = operands((1, 290), 1, 2, 16, 16, torch.float32, seed=12)
    s0 = torch.randn(1, 2, 16, 16, generator=torch.Generator().manual_seed(0)).cuda()
    do = torch.randn(1, 290, 2, 16, generator=torch.Generator().manual_seed(1)).cuda()
    got = grads_of(x, s0, do)
    args = x + [s0]
    for i, gr in enumerate(got):
        d = torch.randn(gr.shape, generator=torch.Generator().manual_seed(2 + i)).cuda()
        d = d * args[i].norm() / d.norm()

        def loss(e):
            y = list(args)
            y[i] = y[i] + e * d
            return (ops.decay_attention(*y[:4], initial_state=y[4])[0].double() * do).sum()

        num = (8 * (loss(5e-3) - loss(-5e-3)) - (loss(1e-2) - loss(-1e-2))) / 6e-2
        want = (gr.double() * d).sum()
        assert abs(num - want) < 1e-3 * max(abs(want), gr.double().norm()), i


@pytest.mark.parametrize('each', [True, False])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_packed_gradients(dtype, each):
    offsets = [2, 2, 3, 70, 70, 134, 300, 301, 1100, 1100]
    total = 1107
    x = operands((1, total), 2, 4, 40, 48, dtype, seed=4, each=each)
    gen = torch.Generator().manual_seed(1)
    do = torch.randn(1, total, 4, 48, generator=gen).to(dtype).cuda()
    s0, ds = (torch.randn(9, 4, 40, 48, generator=gen).cuda() for _ in range(2))
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    got = grads_of(x, s0, do, ds, seq_offsets=off)
    a, (s0, do, ds) = numbers(*x), numbers(s0, do, ds)
    want = [np.zeros(y.shape) for y in a]
    dstate = np.zeros(s0.shape)
    for i, (p, e) in enumerate(zip(offsets, offsets[1:])):
        r = sequence.decay_attention(*(y[0, p:e] for y in a[:3]), a[3][0, p:e] if each else a[3],
                                     state=s0[i], grad_o=do[0, p:e], grad_state=ds[i])[1]
        for j in range(3):
            want[j][0, p:e] = r[j]
        if each:
            want[3][0, p:e] = r[3]
        else:
            want[3] += r[3]
        dstate[i] = r[4]
    for i in range(4):
        near(got[i], want[i], 16 * F32 if i == 3 else TOL[dtype])
        if i < 3 or each:
            assert (got[i][0, :2] == 0).all() and (got[i][0, 1100:] == 0).all()
    near(got[4], dstate, F32)


def test_gradients_with_decays_that_empty_the_state():
    x = operands((1, 340), 1, 2, 32, 32, torch.float32, seed=5)
    low = float('-inf')
    x[3][:, 10], x[3][:, 64], x[3][:, 256], x[3][:, 100:103] = low, low, low, -1e30
    do = torch.randn(1, 340, 2, 32, generator=torch.Generator().manual_seed(1)).cuda()
    got = grads_of(x, None, do)
    *a, do = numbers(*x, do)
    want = sequence.decay_attention(*(y[0] for y in a), grad_o=do[0])[1]
    for i in range(4):
        near(got[i], want[i][None], 16 * F32)
    assert (got[3][:, [10, 64, 100, 101, 102, 256]] == 0).all()


def test_gradients_of_nothing():
    x = operands((1, 0), 1, 2, 16, 16, torch.float32)
    s0, ds = torch.randn(1, 2, 16, 16).cuda(), torch.randn(1, 2, 16, 16).cuda()
    do = torch.zeros(1, 0, 2, 16, device='cuda')
    assert torch.equal(grads_of(x, s0, do, ds)[4], ds)
    x = operands((1, 70), 1, 2, 16, 16, torch.float32, each=False)
    off = torch.tensor([5], dtype=torch.int32).cuda()
    got = grads_of(x, None, torch.ones(1, 70, 2, 16, device='cuda'), seq_offsets=off)
    assert all((g == 0).all() for g in got)


def test_same_bits_beside_other_sequences():
    """A sequence's results and gradients do not change with what runs beside it."""
    offsets = [0, 100, 400, 401]
    x = operands((1, 401), 2, 4, 64, 64, torch.bfloat16, seed=3)
    do = torch.randn(1, 401, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    o, s = ops.decay_attention(*x, seq_offsets=off)
    grads = grads_of(x, None, do, seq_offsets=off)
    for seed in (5, 6):
        y = [t.clone() for t in x]
        for t, r in zip(y, operands((1, 401), 2, 4, 64, 64, torch.bfloat16, seed=seed)):
            t[:, :100], t[:, 400:] = r[:, :100], r[:, 400:]
        o2, s2 = ops.decay_attention(*y, seq_offsets=off)
        assert torch.equal(o[:, 100:400], o2[:, 100:400]) and torch.equal(s[1], s2[1])
        for a, b in zip(grads, grads_of(y, None, do, seq_offsets=off)):
            assert torch.equal(a[:, 100:400], b[:, 100:400])


def test_on_another_stream():
    x = operands((1, 530), 2, 2, 64, 64, torch.bfloat16, seed=8)
    o, s = ops.decay_attention(*x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o2, s2 = ops.decay_attention(*x)
    st.synchronize()
    assert torch.equal(o, o2) and torch.equal(s, s2)


def test_refusals():
    x = operands((2, 5), 2, 4, 16, 16, torch.float32)
    q, k, v, g = x
    state = torch.zeros(2, 4, 16, 16, device='cuda')
    with pytest.raises(TypeError, match='k is'):
        ops.decay_attention(q, k.half(), v, g)
    with pytest.raises(TypeError, match='not supported'):
        ops.decay_attention(q.double(), k.double(), v.double(), g)
    with pytest.raises(ValueError, match='on the GPU'):
        ops.decay_attention(q.cpu(), k, v, g)
    with pytest.raises(ValueError, match='value heads'):
        ops.decay_attention(q, k, v[:, :, :3], g[:, :, :3])
    with pytest.raises(ValueError, match='g must be'):
        ops.decay_attention(q, k, v, g[:, :4])
    with pytest.raises(ValueError, match='g must be'):
        ops.decay_attention(q, k, v, g[0, 0, :2])
    with pytest.raises(ValueError, match='outside 1..128'):
        big = torch.zeros(1, 2, 1, 129, device='cuda')
        ops.decay_attention(big, big, v[:1, :2, :1], g[:1, :2, :1])
    with pytest.raises(ValueError, match='one batch row'):
        ops.decay_attention(*x, seq_offsets=torch.zeros(2, dtype=torch.int32, device='cuda'))
    with pytest.raises(ValueError, match='seq_offsets must be int32'):
        ops.decay_attention(*(y[:1] for y in x), seq_offsets=torch.zeros(2, device='cuda'))
    with pytest.raises(TypeError, match='float32'):
        ops.decay_attention(*x, initial_state=state.half())
    with pytest.raises(ValueError, match='initial_state must be'):
        ops.decay_attention(*x, initial_state=state[:1])
    with pytest.raises(ValueError, match='states for'):
        ops.decay_attention_step(*x, torch.cat([state, state]))
    with pytest.raises(ValueError, match='contiguous'):
        ops.decay_attention_step(*x, state.transpose(2, 3))
    with pytest.raises(ValueError, match='slots must be'):
        ops.decay_attention_step(*x, state, slots=torch.zeros(2, device='cuda'))
    with pytest.raises(ValueError, match='no gradient'):
        ops.decay_attention_step(q.requires_grad_(), k, v, g, state)
