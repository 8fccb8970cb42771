"""The gated delta rule, chunked and token by token, against its definition in 64 bits.

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


def _operands(lead, hk, h, dk, dv, dtype, seed=0, g_dtype=torch.float32, decay=1.0):
    rs = np.random.RandomState(seed)
    k = rs.randn(*lead, hk, dk) + 0.3
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    arrays = [rs.randn(*lead, hk, dk), k, rs.randn(*lead, h, dv),
              -decay * rs.rand(*lead, h), rs.rand(*lead, h)]
    types = [dtype, dtype, dtype, g_dtype, dtype]
    return [torch.tensor(a).to(t).cuda() for a, t in zip(arrays, types)]


def _np(*ts):
    return [t.detach().double().cpu().numpy() for t in ts]


def _near(got, want, tol):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= tol * norm + 1e-30, np.linalg.norm(got - want) / norm


SIZES = [(1, 1, 1, 1, 1, 1), (2, 64, 1, 1, 64, 64), (1, 65, 2, 4, 128, 128),
         (3, 63, 1, 3, 33, 17), (1, 200, 2, 2, 65, 96), (2, 130, 1, 2, 16, 128),
         (1, 7, 3, 3, 127, 1)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('size', SIZES)
def test_chunked_forward(size, dtype):
    b, t, hk, h, dk, dv = size
    x = _operands((b, t), hk, h, dk, dv, dtype, seed=t)
    s0 = torch.randn(b, h, dk, dv, generator=torch.Generator().manual_seed(t)).cuda()
    o, s1 = ops.gated_delta_rule(*x, initial_state=s0)
    assert o.dtype == dtype and s1.dtype == torch.float32
    a = _np(*x, s0)
    want = [sequence.gated_delta(*(y[i] for y in a[:5]), state=a[5][i]) for i in range(b)]
    _near(o, np.stack([w[0] for w in want]), TOL[dtype])
    _near(s1, np.stack([w[1] for w in want]), F32)


def test_chunked_long_without_decay():
    """40 chunks whose state never decays: roundings are carried to the end."""
    x = _operands((1, 2550), 1, 1, 64, 32, torch.float32, decay=0.0)
    o, s1 = ops.gated_delta_rule(*x, scale=0.25)
    wo, ws = sequence.gated_delta(*(y[0] for y in _np(*x)), scale=0.25)
    _near(o, wo[None], F32)
    _near(s1, ws[None], F32)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_packed_sequences(dtype):
    """Empty sequences, single tokens, ends inside a chunk, and tokens that are no sequence's."""
    offsets = [3, 3, 4, 68, 68, 197, 325, 330]
    n, total = len(offsets) - 1, 333
    x = _operands((1, total), 2, 4, 48, 40, dtype, seed=3)
    s0 = torch.randn(n, 4, 48, 40, generator=torch.Generator().manual_seed(1)).cuda()
    o, s1 = ops.gated_delta_rule(*x, initial_state=s0,
                                 seq_offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
    a = _np(*x, s0)
    want_o, want_s = np.zeros((total, 4, 40)), np.zeros((n, 4, 48, 40))
    for i, (p, e) in enumerate(zip(offsets, offsets[1:])):
        want_o[p:e], want_s[i] = sequence.gated_delta(*(y[0, p:e] for y in a[:5]), state=a[5][i])
    _near(o, want_o[None], TOL[dtype])
    assert (o[0, :3] == 0).all() and (o[0, 330:] == 0).all()
    _near(s1, want_s, F32)


def test_empty_sequences_only():
    x = _operands((1, 0), 1, 2, 16, 16, torch.float32)
    s0 = torch.randn(2, 2, 16, 16).cuda()
    o, s1 = ops.gated_delta_rule(*x, initial_state=s0,
                                 seq_offsets=torch.zeros(3, dtype=torch.int32).cuda())
    assert o.shape == (1, 0, 2, 16) and torch.equal(s1, s0)
    o, s1 = ops.gated_delta_rule(*x)
    assert s1.shape == (1, 2, 16, 16) and (s1 == 0).all()


@pytest.mark.parametrize('decay', ['-inf', 'lowest', 'mixed'])
def test_decays_that_empty_the_state(decay):
    """g of -inf or the type's lowest value starts afresh inside a chunk; what follows keeps its
    own decays."""
    x = _operands((1, 150), 1, 2, 32, 32, torch.float32, seed=5)
    g = x[3]
    low = float('-inf') if decay != 'lowest' else torch.finfo(torch.float32).min
    g[:, 10], g[:, 64], g[:, 100:103] = low, low, low
    if decay == 'mixed':
        g[:, 20:30] = -60.0
    o, s1 = ops.gated_delta_rule(*x)
    wo, ws = sequence.gated_delta(*(y[0] for y in _np(*x)))
    _near(o, wo[None], F32)
    _near(s1, ws[None], F32)


def test_strided_and_unaligned_operands():
    """Views into one projection, a transposed layout, and rows that start at odd elements."""
    b, t, hk, h, dk, dv = 2, 70, 2, 4, 32, 24
    x = _operands((b, t), hk, h, dk, dv, torch.bfloat16, seed=9)
    o, s1 = ops.gated_delta_rule(*x)
    flat = torch.zeros(b, t, 2 * hk * dk + h * dv + 3, dtype=torch.bfloat16, device='cuda')
    views, at = [], 1
    for y in x[:3]:
        w = y.shape[2] * y.shape[3]
        view = flat[..., at:at + w].unflatten(-1, y.shape[2:])
        view.copy_(y)
        views.append(view)
        at += w
    heads_first = [y.transpose(1, 2).contiguous().transpose(1, 2) for y in x[3:]]
    o2, s2 = ops.gated_delta_rule(*views, *heads_first)
    assert torch.equal(o, o2) and torch.equal(s1, s2)
    v = x[2].transpose(2, 3).contiguous().transpose(2, 3)      # a head's values not side by side
    o3, s3 = ops.gated_delta_rule(x[0], x[1], v, x[3], x[4])
    assert torch.equal(o, o3) and torch.equal(s1, s3)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('size', [(1, 1, 1, 1, 1), (5, 2, 4, 128, 128), (3, 1, 3, 33, 17),
                                  (2, 3, 3, 64, 127), (9, 1, 1, 100, 36)])
def test_step(size, dtype):
    b, hk, h, dk, dv = size
    x = _operands((b, 3), hk, h, dk, dv, dtype, seed=b)
    rs = np.random.RandomState(4)
    state = torch.tensor(rs.randn(b + 3, h, dk, dv), dtype=torch.float32).cuda()
    slots = torch.tensor(rs.permutation(b + 3)[:b], dtype=torch.int32)
    if b > 2:
        slots[1], slots[2] = -1, b + 3
    before, s = state.clone(), state.cpu().double().numpy()
    o = ops.gated_delta_step(*x, state, slots=slots.cuda())
    one = before.clone()
    for t in range(3):            # the same tokens one by one
        ot = ops.gated_delta_step(*(y[:, t] for y in x), one, slots=slots.cuda())
        assert torch.equal(ot, o[:, t])
    assert torch.equal(one, state)
    a = _np(*x)
    want = np.zeros((b, 3, h, dv))
    for i, at in enumerate(slots.tolist()):
        if 0 <= at < b + 3:
            want[i], s[at] = sequence.gated_delta(*(y[i] for y in a), state=s[at])
        else:
            assert (o[i] == 0).all()
    _near(o, want, TOL[dtype])
    _near(state, s, F32)
    idle = [i for i in range(b + 3) if i not in slots.tolist()]
    assert torch.equal(state[idle], before[idle])


def test_step_continues_the_chunked_form():
    x = _operands((2, 101), 1, 2, 64, 64, torch.float32, seed=6)
    o, s = ops.gated_delta_rule(*x)
    _, state = ops.gated_delta_rule(*(y[:, :97] for y in x))
    tail = ops.gated_delta_step(*(y[:, 97:] for y in x), state)
    _near(tail, _np(o[:, 97:])[0], F32)
    _near(state, _np(s)[0], F32)


GRADS = ('dq', 'dk', 'dv', 'dg', 'dbeta', 'dstate')


def _grads(x, s0, do, dstate=None, **kw):
    x = [y.detach().requires_grad_() for y in x]
    s0 = None if s0 is None else s0.detach().requires_grad_()
    o, s1 = ops.gated_delta_rule(*x, initial_state=s0, **kw)
    outs, ups = ([o, s1], [do, dstate]) if dstate is not None else ([o], [do])
    return torch.autograd.grad(outs, x + ([s0] if s0 is not None else []), ups)


# Gradients are sums of the same kind as the outputs; dg is what is left of sums up to its
# count of tokens times larger, so it gets that factor's root (8 for a chunk of 64).
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('size', SIZES)
def test_gradients(size, dtype):
    b, t, hk, h, dk, dv = size
    x = _operands((b, t), hk, h, dk, dv, dtype, seed=t + 1)
    gen = torch.Generator().manual_seed(t)
    s0 = torch.randn(b, h, dk, dv, generator=gen).cuda()
    do = torch.randn(b, t, h, dv, generator=gen).to(dtype).cuda()
    dstate = torch.randn(b, h, dk, dv, generator=gen).cuda()
    got = _grads(x, s0, do, dstate)
    a = _np(*x, s0, do, dstate)
    want = [sequence.gated_delta(*(y[i] for y in a[:5]), state=a[5][i], grad_o=a[6][i],
                                 grad_state=a[7][i])[1] for i in range(b)]
    for i, name in enumerate(GRADS):
        print(name, flush=True)
        tol = F32 if name == 'dstate' else 8 * F32 if name == 'dg' else TOL[dtype]
        assert got[i].dtype == (torch.float32 if name in ('dg', 'dstate') else dtype)
        _near(got[i], np.stack([w[i] for w in want]), tol)


def test_gradients_against_differences():
    """Of the operator itself, along random directions: central differences of a loss whose
    terms are 32-bit, so the step is large (1e-2) and the agreement 1e-3."""
    x = _operands((1, 90), 1, 2, 16, 16, torch.float32, seed=12)
    s0 = torch.randn(1, 2, 16, 16, generator=torch.Generator().manual_seed(0)).cuda()
    do = torch.randn(1, 90, 2, 16, generator=torch.Generator().manual_seed(1)).cuda()
    got = _grads(x, s0, do)
    args = x + [s0]
    for i, gr in enumerate(got):
        d = torch.randn(gr.shape, generator=torch.Generator().manual_seed(2 + i)).cuda()
        d = d * args[i].norm() / d.norm()

        def loss(e):
            y = list(args)
            y[i] = y[i] + e * d
            return (ops.gated_delta_rule(*y[:5], initial_state=y[5])[0].double() * do).sum()

        num = (8 * (loss(5e-3) - loss(-5e-3)) - (loss(1e-2) - loss(-1e-2))) / 6e-2
        want = (gr.double() * d).sum()
        assert abs(num - want) < 1e-3 * max(abs(want), gr.double().norm()), GRADS[i]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_packed_gradients(dtype):
    offsets = [2, 2, 3, 70, 70, 134, 300, 301]
    n, total = len(offsets) - 1, 305
    x = _operands((1, total), 2, 4, 40, 48, dtype, seed=4, g_dtype=dtype)
    do = torch.randn(1, total, 4, 48, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    got = _grads(x, None, do, seq_offsets=off)
    a = _np(*x, do)
    want = [np.zeros(y.shape) for y in a[:5]]
    for p, e in zip(offsets, offsets[1:]):
        r = sequence.gated_delta(*(y[0, p:e] for y in a[:5]), grad_o=a[5][0, p:e])[1]
        for w, gr in zip(want, r):
            w[0, p:e] = gr
    for i in range(5):
        _near(got[i], want[i], 8 * F32 + TOL[dtype])
        assert (got[i][0, :2] == 0).all() and (got[i][0, 301:] == 0).all()


def test_gradients_with_decays_that_empty_the_state():
    x = _operands((1, 140), 1, 2, 32, 32, torch.float32, seed=5)
    x[3][:, 10], x[3][:, 64], x[3][:, 100:103] = float('-inf'), float('-inf'), -1e30
    do = torch.randn(1, 140, 2, 32, generator=torch.Generator().manual_seed(1)).cuda()
    got = _grads(x, None, do)
    a = _np(*x, do)
    want = sequence.gated_delta(*(y[0] for y in a[:5]), grad_o=a[5][0])[1]
    for i in range(5):
        _near(got[i], want[i][None], 8 * F32)


def test_zero_write_strengths():
    """beta = 0 writes nothing, but its own gradient is there."""
    x = _operands((1, 70), 1, 1, 16, 16, torch.float32, seed=7)
    x[4][:] = 0
    s0 = torch.randn(1, 1, 16, 16, generator=torch.Generator().manual_seed(3)).cuda()
    do = torch.randn(1, 70, 1, 16, generator=torch.Generator().manual_seed(1)).cuda()
    got = _grads(x, s0, do)
    a = _np(*x, s0, do)
    want = sequence.gated_delta(*(y[0] for y in a[:5]), state=a[5][0], grad_o=a[6][0])[1]
    for i in range(6):
        _near(got[i], want[i][None], 8 * F32)


def test_on_another_stream():
    x = _operands((1, 130), 2, 2, 64, 64, torch.bfloat16, seed=8)
    o, s = ops.gated_delta_rule(*x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o2, s2 = ops.gated_delta_rule(*x)
    st.synchronize()
    assert torch.equal(o, o2) and torch.equal(s, s2)


def test_refusals():
    x = _operands((2, 5), 2, 4, 16, 16, torch.float32)
    q, k, v, g, beta = x
    state = torch.zeros(2, 4, 16, 16, device='cuda')
    with pytest.raises(TypeError, match='k is'):
        ops.gated_delta_rule(q, k.half(), v, g, beta)
    with pytest.raises(TypeError, match='not supported'):
        ops.gated_delta_rule(q.double(), k.double(), v.double(), g, beta)
    with pytest.raises(ValueError, match='on the GPU'):
        ops.gated_delta_rule(q.cpu(), k, v, g, beta)
    with pytest.raises(ValueError, match='value heads'):
        ops.gated_delta_rule(q, k, v[:, :, :3], g[:, :, :3], beta[:, :, :3])
    with pytest.raises(ValueError, match='g and beta'):
        ops.gated_delta_rule(q, k, v, g[:, :4], beta)
    with pytest.raises(ValueError, match='outside 1..128'):
        ops.gated_delta_rule(torch.zeros(1, 2, 1, 129, device='cuda'),
                             torch.zeros(1, 2, 1, 129, device='cuda'), v[:1, :2, :1],
                             g[:1, :2, :1], beta[:1, :2, :1])
    with pytest.raises(ValueError, match='one batch row'):
        ops.gated_delta_rule(*x, seq_offsets=torch.zeros(2, dtype=torch.int32, device='cuda'))
    with pytest.raises(ValueError, match='seq_offsets must be int32'):
        ops.gated_delta_rule(*(y[:1] for y in x), seq_offsets=torch.zeros(2, device='cuda'))
    with pytest.raises(TypeError, match='float32'):
        ops.gated_delta_rule(*x, initial_state=state.half())
    with pytest.raises(ValueError, match='initial_state must be'):
        ops.gated_delta_rule(*x, initial_state=state[:1])
    with pytest.raises(ValueError, match='states for'):
        ops.gated_delta_step(*x, torch.cat([state, state]))
    with pytest.raises(ValueError, match='contiguous'):
        ops.gated_delta_step(*x, state.transpose(2, 3))
    with pytest.raises(ValueError, match='slots must be'):
        ops.gated_delta_step(*x, state, slots=torch.zeros(2, device='cuda'))
    with pytest.raises(ValueError, match='no gradient'):
        ops.gated_delta_step(q.requires_grad_(), k, v, g, beta, state)
