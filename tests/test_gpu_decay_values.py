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
