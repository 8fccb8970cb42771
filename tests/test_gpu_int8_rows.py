"""More rows of tokens than one launch has workgroups for."""
import numpy as np
import pytest
import torch

from brainstate_amd import ops
from oracle import sequence

pytestmark = pytest.mark.gpu


def test_more_rows_than_one_launch_of_threads():
    m, k = (1 << 24) + 3, 4
    x = torch.randn(m, k, generator=torch.Generator('cuda').manual_seed(1), device='cuda').half()
    x8, a = ops.int8_quantize(x)
    for at in (slice(0, 5), slice((1 << 23) - 3, (1 << 23) + 3), slice(m - 5, m)):
        w8, wa = sequence.int8_quantize(x[at].double().cpu().numpy())
        assert np.array_equal(x8[at].cpu().numpy(), w8)
        assert np.abs(a[at].double().cpu().numpy() - wa).max() <= 2.0 ** -24 * wa.max()
    w = torch.tensor([[1, -2, 3, 4]], dtype=torch.int8, device='cuda')
    one = torch.ones(1, device='cuda')
    want = (x8.int() * w.int()).sum(1, keepdim=True).float()
    assert torch.equal(ops.int8_matmul(x8, torch.ones_like(a), w, one), want)
    y = ops.int8_linear(x, w, one)
    assert torch.equal(y, (want * a[:, None]).half())
