"""Outputs of the gated delta rule whose terms cancel: a key of length 1 written over in full and
read back gives the value just written, however large what the state held there was.

Terms are of the old state's size, in 32 bits: an output is off by 64 x 2^-24 of that (the bound of
the other outputs' sums) and by its own rounding.
"""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

F32 = 64 * 2.0 ** -24
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZE = 4096.0


@pytest.mark.parametrize('dk', [32, 128])
@pytest.mark.parametrize('dtype', list(UNIT))
def test_written_values_come_back(dtype, dk):
    t, h, dv = 70, 2, 40
    rs = np.random.RandomState(dk)
    k = np.zeros((1, t, 1, dk))
    for row in k.reshape(-1, dk):          # four entries of a half: of length 1 in every type
        row[rs.permutation(dk)[:4]] = 0.5 * rs.choice([-1, 1], 4)
    arrays = [k, k, rs.randn(1, t, h, dv), np.zeros((1, t, h)), np.ones((1, t, h))]
    x = [torch.tensor(a).to(dtype).cuda() for a in arrays]
    s0 = torch.tensor(SIZE * rs.randn(1, h, dk, dv), dtype=torch.float32).cuda()
    o, _ = ops.gated_delta_rule(*x, scale=1.0, initial_state=s0)
    a = [y.double().cpu().numpy()[0] for y in (*x, s0)]
    want, _ = sequence.gated_delta(*a[:5], scale=1.0, state=a[5])
    assert np.abs(want - a[2]).max() < 1e-9                  # the values just written
    off = np.linalg.norm(o[0].double().cpu().numpy() - want)
    assert off <= F32 * SIZE * want.size ** 0.5 + UNIT[dtype] * np.linalg.norm(want), off
