"""Sizes that do not fit the 32-bit arguments of the entry points are refused by name, not cut off
(CPU: the checks come before any device work)."""
import ctypes
import os

import pytest
import torch

from brainstate_amd import _decay, _dropout, _int4, _sequence
from brainstate_amd import _native as N

AT = ctypes.c_void_p(4096)            # an address that nothing reads
SIZES = [1 << 31, (1 << 32) + 8, (1 << 33) + 1]


@pytest.fixture
def anywhere(monkeypatch):
    """The checks of operands on tensors without storage, of any size."""
    for module in (_sequence, _decay, _dropout, _int4):
        monkeypatch.setattr(module, '_floating', lambda name, t, dtype=None: 0)


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device='meta')


@pytest.mark.parametrize('n', SIZES)
def test_a_row_to_drop_from(n, anywhere):
    with pytest.raises(ValueError, match=f'{n} values of a row.*exceed'):
        _dropout.dropout(meta(n), 0.5, 1)
    with pytest.raises(ValueError, match=f'{n} values of a row.*exceed'):
        _dropout.dropout(meta(2, n).requires_grad_(), 0.5, 1)


@pytest.mark.parametrize('n', SIZES)
def test_rows_at_the_entry_point(n):
    if not os.path.exists(N.LIB_PATH):
        pytest.skip('library not built')
    lib = N.load_library()
    assert lib.bs_dropout(AT, 0, 1, n, n, 1, None, 0, 1 << 31, 2.0, AT, None) == N.BS_ERR_INVALID
    assert str(n).encode() in lib.bs_last_error()


@pytest.mark.parametrize('n', SIZES)
def test_batches_tokens_and_sequences(n, anywhere):
    for b, t in ((n, 1), (1, n)):
        q, g = meta(b, t, 1, 1), meta(b, t, 1)
        with pytest.raises(ValueError, match=f'{n}.*exceed'):
            _decay.decay_attention(q, q, q, g)
        with pytest.raises(ValueError, match=f'{n}.*exceed'):
            _decay.decay_attention_step(q, q, q, g, meta(b, 1, 1, 1, dtype=torch.float32))
        with pytest.raises(ValueError, match=f'{n}.*exceed'):
            _sequence.gated_delta_rule(q, q, q, g, g)
        with pytest.raises(ValueError, match=f'{n}.*exceed'):
            _sequence.gated_delta_step(q, q, q, g, g, meta(b, 1, 1, 1, dtype=torch.float32))
    q, g = meta(1, 8, 1, 1), meta(1, 8, 1)
    offsets = meta(n + 1, dtype=torch.int32)
    with pytest.raises(ValueError, match=f'{n} sequences exceed'):
        _decay.decay_attention(q, q, q, g, seq_offsets=offsets)
    with pytest.raises(ValueError, match=f'{n} sequences exceed'):
        _sequence.gated_delta_rule(q, q, q, g, g, seq_offsets=offsets)


@pytest.mark.parametrize('n', SIZES)
def test_channels(n, anywhere):
    with pytest.raises(ValueError, match=f'{n} channels exceed'):
        _int4.int4_linear(meta(3, 2), meta(n, 1, dtype=torch.uint8),
                          meta(n, 1, dtype=torch.float32))
    with pytest.raises(ValueError, match=f'{n} channels exceed'):
        _sequence.int8_linear(meta(3, 2), meta(n, 2, dtype=torch.int8),
                              meta(n, dtype=torch.float32))
