"""The tiles that the 4-bit product chooses among, each at sizes that the choice gives it, with edges
in tokens, channels and k; tolerances as in the operator's other tests."""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu

F32 = 64 * 2.0 ** -24
TOL = {torch.float32: F32, torch.bfloat16: F32 + 2.0 ** -8, torch.float16: F32 + 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TILES = {(128, 256): 75, (64, 256): 46, (64, 128): 34, (64, 64): 25}     # us a round


def tile_of(m, n, dtype, group, cus):
    """The tile that costs least, the larger one where two do."""
    whole = dtype != torch.float32
    fits = {(128, 256): whole and group == 128, (64, 256): whole or group > 32}
    cost = {t: us * -(-(-(-m // t[0]) * -(-n // t[1])) // cus) for t, us in TILES.items()
            if fits.get(t, True)}
    return min(cost, key=lambda t: (cost[t], -t[0] * t[1]))


# tokens, k, channels, group, tile in 16 bits and in 32
CASES = [(1030, 385, 4100, 128, (128, 256), (64, 256)),      # an odd k, tokens in padded rows
         (1030, 515, 4100, 128, (128, 256), (64, 256)),
         (4000, 400, 4000, 128, (128, 256), (64, 256)),      # two rounds of workgroups
         (4000, 256, 4000, 128, (128, 256), (64, 256)),      # and tokens read where they are
         (700, 333, 4100, 128, (64, 256), (64, 256)),
         (700, 333, 4100, 64, (64, 256), (64, 256)),
         (700, 333, 4100, 32, (64, 256), (64, 128)),
         (500, 201, 4090, 128, (64, 128), (64, 128)),
         (250, 201, 4090, 64, (64, 64), (64, 64))]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('case', CASES)
def test_tiles(case, dtype):
    m, k, n, group = case[:4]
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    if cus == 256:           # the sizes are chosen for a whole card
        assert tile_of(m, n, dtype, group, cus) == case[5 if dtype == torch.float32 else 4]
    rs = np.random.RandomState(k)
    x = torch.tensor(rs.randn(m, k)).to(dtype).cuda()
    u = rs.randint(0, 16, (n, k))
    scale = torch.tensor((0.5 + rs.rand(n, -(-k // group))) * 0.1, dtype=torch.float32).cuda()
    bias = torch.tensor(rs.randn(n)).to(dtype).cuda()
    y = ops.int4_linear(x, torch.tensor(sequence.int4_pack(u)).cuda(), scale, bias=bias, group=group)
    w = (torch.tensor(u - 8).cuda() *
         scale.double().repeat_interleave(group, 1)[:, :k])
    want = x.double() @ w.t() + bias.double()
    assert y.dtype == dtype and y.isfinite().all()
    # by edges too: the last tile's rows, channels, and the whole
    for cut in (np.s_[:, :], np.s_[m // 64 * 64 - 1:, :], np.s_[:, n // 64 * 64 - 1:]):
        assert (y[cut].double() - want[cut]).norm() <= TOL[dtype] * want[cut].norm(), cut
