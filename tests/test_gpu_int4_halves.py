"""Weights whose quotient 7 w / max|w| lies beside a half: the nearest integer is a matter of the last
bit of 32-bit weights, and of ties to even where the quotient is one exactly."""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu


def weights(dtype, size=1.0):
    """Groups of 32 whose first value is the largest; the others are multiples of a half of a seventh of
    it in 32 bits, and the numbers next to them."""
    rs = np.random.RandomState(0)
    top = (size * (0.5 + rs.rand(400, 8, 1))).astype(np.float32)
    half = (rs.randint(0, 7, (400, 8, 31)) + 0.5) * rs.choice([-1, 1], (400, 8, 31))
    w = torch.tensor((top.astype(np.float64) * half / 7).astype(np.float32))
    w = torch.nextafter(w, torch.tensor(rs.choice([-np.inf, np.inf], w.shape).astype(np.float32))
                        ).where(torch.tensor(rs.rand(*w.shape) < 0.3), w)
    w = torch.cat([torch.tensor(top), w], 2).reshape(400, 256)
    return w.to(dtype).cuda()


@pytest.mark.parametrize('dtype, size', [(t, s) for t in (torch.float32, torch.bfloat16)
                                         for s in (1.0, 2.0 ** 126.5, 2.0 ** -126)] +
                         [(torch.float16, 1.0)])
def test_the_nearest_integer(dtype, size):
    w = weights(dtype, size)
    w4, scale = ops.int4_quantize(w, 32)
    # 53 bits hold 7 w, and a quotient of 27 bits by 24 that is no half is 2^-28 away from one
    u, a = sequence.int4_quantize(w.double().cpu().numpy(), 32)
    assert torch.equal(w4, torch.tensor(sequence.int4_pack(u)).cuda())
    assert torch.equal(scale, torch.tensor(a).float().cuda())


def test_the_smallest_numbers():
    """A scale that rounds to 0 leaves the integers what they are."""
    step = 2.0 ** -149
    w = torch.tensor([[step, -step] + [0.0] * 30, [7 * step, 3 * step, -4 * step] + [0.0] * 29],
                     dtype=torch.float64).float().cuda()
    w4, scale = ops.int4_quantize(w, 32)
    assert w4[0, 0] == 15 | 1 << 4 and (w4[0, 1:] == 0x88).all() and scale[0, 0] == 0
    assert w4[1, 0] == 15 | 11 << 4 and w4[1, 1] == 4 | 8 << 4 and scale[1, 0].double() == step
