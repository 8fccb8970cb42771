"""The gated delta rule where there are more heads and sequences than CUs: recurrences over 32 value
columns a workgroup, over eleven chunks and more.

Tolerances as in the operator's own tests: 64 x 2^-24 of the norm for 32-bit results (a hundred
chunks), 8 times that for dg, a difference of sums over 64 tokens; 16-bit results add their rounding.
A sequence's results do not depend on what runs beside it, in any bit.
"""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 64 * 2.0 ** -24


def _operands(b, t, hk, h, dk, dv, dtype, seed):
    rs = np.random.RandomState(seed)
    k = rs.randn(b, t, hk, dk) + 0.2
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    # decays of a hundred tokens, so that chunks reach far
    arrays = [rs.randn(b, t, hk, dk), k, rs.randn(b, t, h, dv), -0.02 * rs.rand(b, t, h),
              rs.rand(b, t, h)]
    types = [dtype, dtype, dtype, torch.float32, dtype]
    return [torch.tensor(a).to(d).cuda() for a, d in zip(arrays, types)]


def _plain(q, k, v, g, beta, state, do, dstate):
    """Token by token in 64 bits on the GPU, [B, T, H, ..] -> (o, state, the six gradients)."""
    b, t, hk, dk = q.shape
    group, scale = v.shape[2] // hk, dk ** -0.5
    q, k, v, g, beta, state, do, ds = (x.detach().double() for x in
                                       (q, k, v, g, beta, state, do, dstate))
    q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    o, kept = torch.empty_like(v), []
    for i in range(t):
        kept.append(state)
        s = g[:, i].exp()[..., None, None] * state
        ki = k[:, i, :, :, None]
        u = beta[:, i, :, None] * (v[:, i] - (s * ki).sum(2))
        state = s + ki * u[:, :, None]
        o[:, i] = scale * (state * q[:, i, :, :, None]).sum(2)
    gq, gk, gv, gg, gb = (torch.empty_like(x) for x in (q, k, v, g, beta))
    for i in reversed(range(t)):
        decay = g[:, i].exp()[..., None, None]
        ki, oi = k[:, i, :, :, None], do[:, i, :, None]
        s = decay * kept.pop()
        miss = v[:, i] - (s * ki).sum(2)
        u = beta[:, i, :, None] * miss
        gq[:, i] = scale * ((s + ki * u[:, :, None]) * oi).sum(3)
        ds = ds + scale * q[:, i, :, :, None] * oi
        du = (ds * ki).sum(2)
        gb[:, i] = (du * miss).sum(2)
        gv[:, i] = du = beta[:, i, :, None] * du
        gk[:, i] = (ds * u[:, :, None]).sum(3) - (s * du[:, :, None]).sum(3)
        ds = ds - ki * du[:, :, None]
        gg[:, i] = (ds * s).sum((2, 3))
        ds = decay * ds
    gq, gk = (x.unflatten(2, (hk, group)).sum(3) for x in (gq, gk))
    return o, state, gq, gk, gv, gg, gb, ds


def _near(got, want, tol, name):
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    off = ((got.double() - want).norm() / want.norm()).item()
    assert off <= tol, (name, off)


def test_the_plain_form_is_the_definition():
    x = _operands(1, 9, 2, 4, 5, 7, torch.float32, 0)
    rng = torch.Generator().manual_seed(1)
    s0, ds = (torch.randn(1, 4, 5, 7, generator=rng).cuda() for _ in range(2))
    do = torch.randn(1, 9, 4, 7, generator=rng).cuda()
    got = _plain(*x, s0, do, ds)
    a = [y.double().cpu().numpy()[0] for y in (*x, s0, do, ds)]
    (o, s), grads = sequence.gated_delta(*a[:5], state=a[5], grad_o=a[6], grad_state=a[7])
    for y, w in zip(got, (o, s, *grads)):
        assert np.abs(y.cpu().numpy()[0] - w).max() < 1e-12 * max(1, np.abs(w).max())


# sequences x heads x columns / 16 past the 256 workgroups of a round, over eleven chunks
WIDE = [(6, 650, 4, 8, 40, 90), (5, 700, 2, 8, 100, 128), (70, 65, 1, 2, 128, 17)]


def _pass(x, s0, do, ds, **kw):
    leaves = [y.detach().requires_grad_() for y in (*x, s0)]
    o, s1 = ops.gated_delta_rule(*leaves[:5], initial_state=leaves[5], **kw)
    return (o.detach(), s1.detach(), *torch.autograd.grad((o, s1), leaves, (do, ds)))


NAMES = ('o', 'state', 'dq', 'dk', 'dv', 'dg', 'dbeta', 'dstate')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', WIDE)
def test_many_heads_and_chunks(size, dtype):
    b, t, hk, h, dk, dv = size
    x = _operands(*size, dtype, seed=t)
    rng = torch.Generator().manual_seed(t)
    s0, ds = (torch.randn(b, h, dk, dv, generator=rng).cuda() for _ in range(2))
    do = torch.randn(b, t, h, dv, generator=rng).to(dtype).cuda()
    got = _pass(x, s0, do, ds)
    for name, y, w in zip(NAMES, got, _plain(*x, s0, do, ds)):
        tol = F32 if name in ('state', 'dstate') else 8 * F32 if name == 'dg' else \
            F32 + UNIT[dtype]
        _near(y, w, tol, name)
    # without gradients the same outputs, and a sequence alone the same bits
    with torch.no_grad():
        o, s1 = ops.gated_delta_rule(*x, initial_state=s0)
        assert torch.equal(o, got[0]) and torch.equal(s1, got[1])
    one = _pass([y[1:2] for y in x], s0[1:2], do[1:2], ds[1:2])
    assert all(torch.equal(a, y[1:2]) for a, y in zip(one, got))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dims', [(48, 64), (128, 100)])
def test_many_packed_heads_and_chunks(dims, dtype):
    """What each sequence gives alone, where it is short of a round of workgroups."""
    cuts = [5, 5, 6, 70, 134, 800, 801, 1500, 1563]
    n, total, (hk, h), (dk, dv) = len(cuts) - 1, 1570, (4, 8), dims
    x = _operands(1, total, hk, h, dk, dv, dtype, seed=3)
    rng = torch.Generator().manual_seed(1)
    s0, ds = (torch.randn(n, h, dk, dv, generator=rng).cuda() for _ in range(2))
    do = torch.randn(1, total, h, dv, generator=rng).to(dtype).cuda()
    got = _pass(x, s0, do, ds, seq_offsets=torch.tensor(cuts, dtype=torch.int32).cuda())
    for i, (p, e) in enumerate(zip(cuts, cuts[1:])):
        one = _pass([y[:, p:e] for y in x], s0[i:i + 1], do[:, p:e], ds[i:i + 1])
        for name, a, y in zip(NAMES, one, got):
            assert torch.equal(a, y[i:i + 1] if 'state' in name else y[:, p:e]), (name, i)
    for name, y in zip(NAMES, got):
        if 'state' not in name:
            assert (y[:, :5] == 0).all() and (y[:, 1563:] == 0).all(), name
