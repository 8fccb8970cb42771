"""Decay attention where a workgroup walks 3 chunks and more of a sequence, or several whole
sequences, against its definition in 64 bits.

Tolerances are of the norm of the difference over the norm of the result, as in the operator's other
tests: sums of at most 128 + 64 products and a handful of dependent 32-bit roundings a chunk, 2^-24
each, which add up like their root: 64 x 2^-24 leaves room for a hundred chunks.  Outputs in 16 bits
add their own rounding, 2^-8 (bfloat16) or 2^-11 (float16) at most.  dg is a difference of sums over
the tokens of a chunk: 16 times as much.
"""
import pytest
import torch

from brainstate_amd import _decay, ops
from brainstate_amd import _native as N

pytestmark = pytest.mark.gpu

F32 = 64 * 2.0 ** -24
TOL = {torch.float32: F32, torch.bfloat16: F32 + 2.0 ** -8, torch.float16: F32 + 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def definition(q, k, v, g, s, do, ds):
    """[B, T, H, d] token by token in 64 bits -> (o, final state), (dq, dk, dv, dg, dstate) for the
    keys of every value head."""
    t, scale = q.shape[1], q.shape[-1] ** -0.5
    o, kept = torch.empty_like(v), []
    for i in range(t):
        kept.append(s)
        s = g[:, i].exp()[..., None, None] * s + k[:, i, :, :, None] * v[:, i, :, None]
        o[:, i] = scale * (s * q[:, i, :, :, None]).sum(2)
    final = s
    dq, dk, dv, dg = (torch.empty_like(x) for x in (q, k, v, g))
    for i in reversed(range(t)):
        ki, vi, doi = k[:, i, :, :, None], v[:, i, :, None], do[:, i, :, None]
        decay = g[:, i].exp()[..., None, None]
        old = decay * kept[i]
        dq[:, i] = scale * ((old + ki * vi) * doi).sum(3)
        ds = ds + scale * q[:, i, :, :, None] * doi
        dk[:, i], dv[:, i] = (ds * vi).sum(3), (ds * ki).sum(2)
        dg[:, i] = (ds * old).sum((2, 3))
        ds = decay * ds
    return (o, final), (dq, dk, dv, dg, ds)


def want_of(x, s0, do, ds, each, offsets=None):
    """Outputs and gradients by the definition, laid out as the operator's."""
    q, k, v, g, s0, do, ds = (t.double() for t in (*x, s0, do, ds))
    (b, t, hk, dk), h = q.shape, v.shape[2]
    qh, kh = (y.repeat_interleave(h // hk, 2) for y in (q, k))
    gh = g.expand(b, t, h)
    if offsets is None:
        outs, grads = definition(qh, kh, v, gh, s0, do, ds)
        grads = list(grads)
    else:
        outs = [torch.zeros_like(v), torch.empty_like(s0)]
        grads = [torch.zeros_like(y) for y in (qh, kh, v, gh)] + [torch.empty_like(s0)]
        for i, (p, e) in enumerate(zip(offsets, offsets[1:])):
            cut = [y[:, p:e] for y in (qh, kh, v, gh)]
            (o, s), gr = definition(*cut, s0[i:i + 1], do[:, p:e], ds[i:i + 1])
            outs[0][:, p:e], outs[1][i] = o, s[0]
            for y, z in zip(grads, gr[:4]):
                y[:, p:e] = z
            grads[4][i] = gr[4][0]
    for i in range(2):
        grads[i] = grads[i].unflatten(2, (hk, h // hk)).sum(3)
    if not each:
        grads[3] = grads[3].sum((0, 1))
    return outs, grads


def near(got, want, tol, name):
    assert got.shape == want.shape and got.isfinite().all(), name
    err = (got.double() - want).norm() / want.norm()
    assert err <= tol, (name, err.item())


def check(x, s0, do, ds, each, offsets=None):
    dtype = x[0].dtype
    leaves = [t.detach().requires_grad_() for t in (*x, s0)]
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda()
    outs = ops.decay_attention(*leaves[:4], initial_state=leaves[4], seq_offsets=off)
    grads = torch.autograd.grad(outs, leaves, [do, ds])
    want, want_g = want_of(x, s0, do, ds, each, offsets)
    near(outs[0], want[0], TOL[dtype], 'o')
    near(outs[1], want[1], F32, 'state')
    for name, a, w in zip(('dq', 'dk', 'dv', 'dg', 'dstate'), grads, want_g):
        near(a, w, 16 * F32 if name == 'dg' else F32 if name == 'dstate' else TOL[dtype], name)
    with torch.no_grad():        # nothing kept: the states between segments lie in the workspace
        again = ops.decay_attention(*x, initial_state=s0, seq_offsets=off)
    assert all(torch.equal(a, o) for a, o in zip(again, outs))


def operands(b, t, hk, h, dk, dv, n, dtype, each, seed):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen).cuda()                    # noqa: E731
    q, k, v, do = randn(b, t, hk, dk), randn(b, t, hk, dk) + 0.3, randn(b, t, h, dv), randn(b, t, h, dv)
    g = -0.3 * torch.rand(*((b, t) if each else ()), h, generator=gen).cuda()
    x = [y.to(dtype) for y in (q, k, v)] + [g]
    return x, randn(n, h, dk, dv), do.to(dtype), randn(n, h, dk, dv)


def segments(x, n, packed):
    """(segments that the states are carried over, 0 for none, slots of chunks, workgroups at a
    time)."""
    (b, t, _, dk), (h, dv) = x[0].shape, x[2].shape[2:]
    kept = N.lib().bs_decay_attention_kept_size(_decay._pack(*x, None)[1], n, t, packed, 1)
    slots = t // 64 + n if packed else n * -(-t // 64)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return kept // (h * dk * dv * 4), slots, cus * (2 if x[0].dtype == torch.bfloat16 else 1)


# batch, tokens, key heads, heads, dk, dv: segments that begin inside a sequence, a short last one, and
# states wider than 64 rows
CARRIED = [(4, 1100, 12, 24, 16, 16), (1, 3000, 64, 64, 16, 20), (2, 1100, 48, 48, 72, 100)]


@pytest.mark.parametrize('each', [True, False])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', CARRIED)
def test_segments_of_more_chunks(size, dtype, each):
    b, t, hk, h, dk, dv = size
    x, s0, do, ds = operands(*size, b, dtype, each, seed=t)
    segs, slots, _ = segments(x, b, False)
    assert segs > 1 and slots > 2 * segs, (segs, slots)
    check(x, s0, do, ds, each)


# a segment has 2 whole sequences of 3 chunks and more; 4 in the types that take half the workgroups
@pytest.mark.parametrize('each', [True, False])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(48, 130, 24, 24, 16, 16), (40, 190, 8, 32, 40, 24)])
def test_segments_of_several_sequences(size, dtype, each):
    b, t, hk, h, dk, dv = size
    x, s0, do, ds = operands(*size, b, dtype, each, seed=t)
    segs, slots, at_once = segments(x, b, False)
    assert segs == 0 and slots * h > 6 * at_once, (slots, at_once)
    check(x, s0, do, ds, each)


LONG = [2, 2, 3, 70, 70, 134, 1500, 1501, 3900, 3900]
SHORT = [0] + [i * 61 + i * i % 37 for i in range(1, 61)]


@pytest.mark.parametrize('each', [True, False])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('offsets', [LONG, SHORT])
def test_packed_segments_of_more_chunks(offsets, dtype, each):
    n, total = len(offsets) - 1, offsets[-1] + 7
    assert sorted(offsets) == offsets
    x, s0, do, ds = operands(1, total, 12, 24, 24, 16, n, dtype, each, seed=n)
    segs, slots, _ = segments(x, n, True)
    assert segs > 1 and slots > 2 * segs, (segs, slots)
    check(x, s0, do, ds, each, offsets)


def test_gradient_of_decays_head_by_head():
    """Heads that hardly fade beside heads of which a token leaves nothing.  Of token t of a chunk that
    ends before token e, dg is the sum of <S_e, dS_e>, less every write's part in it from t on, and of
    what the outputs from t on take from writes before t.  Each term is an inner product of 32-bit
    results, off by 64 x 2^-24 of its factors' norms at most, so that is its bound, token by token; fast
    heads' dg is the difference that is left, and its bound relative to it the larger."""
    b, t, h, d = 2, 300, 8, 32
    rates = torch.logspace(-2.5, 1.2, h)
    gen = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(b, t, h, d, generator=gen).cuda() for _ in range(4))
    g = (-rates * (0.5 + torch.rand(b, t, h, generator=gen))).cuda()
    leaves = [y.requires_grad_() for y in (q, k, v, g)]
    got = torch.autograd.grad(ops.decay_attention(*leaves)[0], g, do)[0].double()
    q, k, v, g, do = (y.detach().double() for y in (q, k, v, g, do))
    zero = torch.zeros(b, h, d, d, dtype=torch.float64, device='cuda')
    want = definition(q, k, v, g, zero, do, zero)[1][3]
    scale, size = d ** -0.5, lambda y: y.norm(dim=-1)                           # noqa: E731
    s_in, ds_out = zero, {}
    for at in reversed(range(0, t, 64)):           # dS after each chunk
        ds_out[at] = s_in
        for i in reversed(range(at, min(at + 64, t))):
            s_in = s_in + scale * q[:, i, :, :, None] * do[:, i, :, None]
            s_in = g[:, i].exp()[..., None, None] * s_in
    s = zero
    for at in range(0, t, 64):
        rows = slice(at, min(at + 64, t))
        before, run = s.flatten(2).norm(dim=-1), g[:, rows].cumsum(1)
        for i in range(rows.start, rows.stop):
            s = g[:, i].exp()[..., None, None] * s + k[:, i, :, :, None] * v[:, i, :, None]
        ds, n = ds_out[at].flatten(2).norm(dim=-1), run.shape[1]
        write, read = size(k[:, rows]) * size(v[:, rows]), scale * size(q[:, rows]) * size(do[:, rows])
        behind = write * (run[:, -1:] - run).exp() * ds[:, None]
        taken = read * run.exp() * before[:, None]
        i = torch.arange(n, device='cuda')
        pair = read[:, :, None] * write[:, None] * (run[:, :, None] - run[:, None]).clamp(max=0).exp()
        pair = pair * (i[:, None] > i)[None, :, :, None]          # what i takes from a write of j < i
        cross = torch.stack([pair[:, x:, :x].sum((1, 2)) for x in range(n)], 1)
        total = s.flatten(2).norm(dim=-1)[:, None] * ds[:, None] + cross + \
            (behind + taken).flip(1).cumsum(1).flip(1)
        err = (got[:, rows] - want[:, rows]).abs()
        bound = F32 * total + 2.0 ** -24 * want[:, rows].abs() + 1e-37
        assert (err <= bound).all(), (at, (err / bound).amax((0, 1)))
    # and what that leaves of a head's gradient: where a token fades by 1 at most, 16 times a sum's bound
    per = (got - want).norm(dim=(0, 1)) / want.norm(dim=(0, 1))
    assert (per[rates * 1.5 <= 1] <= 16 * F32).all(), per
