"""Checks of the sequence-layer entry points that come before any device work (CPU)."""
import ctypes
import os

import pytest

from brainstate_amd import _native as N
from brainstate_amd import _sequence

F32 = 0


@pytest.fixture
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.skip('library not built')
    return N.load_library()


def _delta_in(hk=1, hv=1, dk=16, dv=16, stride=16, at=4096):
    """Operands of float32 at addresses that nothing reads."""
    return _sequence._DELTA_IN.pack(*[at] * 5, *[stride] * 15, F32, F32, F32, hk, hv, dk, dv, 1.0)


def test_kept_matrices_are_both_given_or_neither(lib):
    at = ctypes.c_void_p(4096)
    need = lib.bs_gated_delta_workspace_size(_delta_in(), 1, 64, 0)
    for kept in ((at, None), (None, at)):
        rc = lib.bs_gated_delta_rule(_delta_in(), 1, 64, None, None, at, at, *kept, at, need, None)
        assert rc == N.BS_ERR_INVALID and b'kept_u' in lib.bs_last_error()
