"""Infinities and NaN in decay attention's operands: what the definition does not take from them keeps
its bits.  A run whose operands are finite there is the measure."""
import pytest
import torch

from brainstate_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAN, INF = float('nan'), float('inf')


def operands(t, dtype, b=2, hk=2, h=4, dk=40, dv=72, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen).cuda()                    # noqa: E731
    x = [randn(b, t, n, d).to(dtype) for n, d in ((hk, dk), (hk, dk), (h, dv))]
    return x + [-0.3 * torch.rand(b, t, h, generator=gen).cuda()]


def changed(t, at, value):
    t = t.clone()
    t[at] = value
    return t


@pytest.mark.parametrize('value', [INF, -INF, NAN])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('t', [50, 200, 1500])
def test_a_key_value_reaches_its_own_row_of_the_state(t, dtype, value):
    """Value 6 of a key is row 6 of the state that is left, whatever lies beside it, and the tokens from
    it on."""
    x = operands(t, dtype)
    at = t - 10
    o, s = ops.decay_attention(*x)
    o2, s2 = ops.decay_attention(x[0], changed(x[1], (1, at, 0, 6), value), *x[2:])
    other = torch.arange(40, device='cuda') != 6
    assert torch.equal(s2[:, :, other], s[:, :, other])
    assert torch.equal(s2[0], s[0]) and torch.equal(s2[1, 2:], s[1, 2:])
    assert not s2[1, :2, 6].isfinite().any()
    assert torch.equal(o2[0], o[0]) and torch.equal(o2[1, :, 2:], o[1, :, 2:])
    assert torch.equal(o2[1, :at], o[1, :at])
    assert not o2[1, at:, :2].isfinite().any()


# tokens where a chunk begins, inside it, at its end, and behind the first segments
PLACES = [(50, [20]), (200, [0, 63, 130]), (1500, [64, 700, 705])]


@pytest.mark.parametrize('value', [INF, -INF, NAN])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('t, at', PLACES)
def test_a_value_reaches_its_own_column_from_its_token_on(t, at, dtype, value):
    """Whatever stands behind a token, in the same chunk too, leaves it as it is."""
    x = operands(t, dtype)
    o, s = ops.decay_attention(*x)
    for first in at:
        o2, s2 = ops.decay_attention(*x[:2], changed(x[2], (1, first, 1, 37), value), x[3])
        clean = torch.ones_like(o, dtype=torch.bool)
        clean[1, first:, 1, 37] = False
        assert torch.equal(o2[clean], o[clean])
        assert not o2[~clean].isfinite().any()
        clean = torch.ones_like(s, dtype=torch.bool)
        clean[1, 1, :, 37] = False
        assert torch.equal(s2[clean], s[clean])
        assert not s2[~clean].isfinite().any()


@pytest.mark.parametrize('dtype', TYPES)
def test_values_behind_the_end_of_a_prompt(dtype):
    """Rows that are padded with what lies in memory: many columns, heads and tokens at once."""
    x = operands(300, dtype, seed=1)
    o, _ = ops.decay_attention(*x)
    ends = [170, 5]
    bad = [y.clone() for y in x]
    for row, end in enumerate(ends):
        for y in bad:
            junk = torch.tensor([NAN, INF, 1.0, -INF, 0.0], device='cuda').to(y.dtype)
            flat = y[row, end:].reshape(-1)
            y[row, end:] = junk[torch.arange(flat.numel(), device='cuda') % 5].view_as(y[row, end:])
    o2, _ = ops.decay_attention(*bad)
    for row, end in enumerate(ends):
        assert torch.equal(o2[row, :end], o[row, :end])


@pytest.mark.parametrize('dtype', TYPES)
def test_a_state_column_that_is_lost_already(dtype):
    x = operands(150, dtype, seed=2)
    s0 = torch.randn(2, 4, 40, 72, generator=torch.Generator().manual_seed(1)).cuda()
    o, s = ops.decay_attention(*x, initial_state=s0)
    lost = changed(s0, (0, 3, slice(None), 5), NAN)
    o2, s2 = ops.decay_attention(*x[:2], changed(x[2], (0, 100, 3, 6), INF), x[3],
                                 initial_state=lost)
    clean = torch.ones_like(o, dtype=torch.bool)
    clean[0, :, 3, 5] = clean[0, 100:, 3, 6] = False
    assert torch.equal(o2[clean], o[clean]) and not o2[~clean].isfinite().any()
    clean = torch.ones_like(s, dtype=torch.bool)
    clean[0, 3, :, 5:7] = False
    assert torch.equal(s2[clean], s[clean])


@pytest.mark.parametrize('value', [INF, NAN])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('t, at', PLACES)
def test_gradients_from_tokens_that_do_not_meet_it(t, at, dtype, value):
    """An output's gradient reaches dq of its own token, dk and dv of the tokens up to it; a value
    reaches dk of its own token and dq of the tokens from it on."""
    x = operands(t, dtype, hk=4)
    do = operands(t, dtype, seed=5)[2]

    def grads(x, do):
        leaves = [y.detach().requires_grad_() for y in x]
        return torch.autograd.grad(ops.decay_attention(*leaves)[0], leaves[:3], do)
    want = grads(x, do)
    for p in at:
        dq, dk, dv = grads(x, changed(do, (1, p, 1, 37), value))
        for got, ref, rows in ((dq, want[0], slice(p, p + 1)), (dk, want[1], slice(0, p + 1)),
                               (dv, want[2], slice(0, p + 1))):
            clean = torch.ones_like(ref, dtype=torch.bool)
            clean[1, rows, 1] = False
            assert torch.equal(got[clean], ref[clean])
        y = list(x)
        y[2] = changed(x[2], (1, p, 1, 37), value)
        dq, dk, dv = grads(y, do)
        assert torch.equal(dv, want[2])
        for got, ref, rows in ((dq, want[0], slice(p, t)), (dk, want[1], slice(p, p + 1))):
            clean = torch.ones_like(ref, dtype=torch.bool)
            clean[1, rows, 1] = False
            assert torch.equal(got[clean], ref[clean])
