"""Checks of the sequence-layer entry points that come before any device work (CPU)."""
import ctypes
import os
import struct

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


def test_packed_operands_are_the_compiled_headers_structs(tmp_path):
    """Sizes, padding included, and where the fields past the pointers lie."""
    import shutil
    import subprocess
    cc = shutil.which('gcc')
    if cc is None:
        pytest.skip('no host C compiler')
    fields = {'bs_delta_in': ['q_stride', 'beta_stride', 'dtype', 'hk', 'dv', 'scale'],
              'bs_norm_in': ['y_stride', 'rows', 'dim', 'pre_dtype', 'eps', 'scale_value']}
    src = tmp_path / 'sizes.c'
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "brainstate_amd.h"\n'
                   'int main(void) {\n' + ''.join(
                       f'printf("%zu ", sizeof({s}));' + ''.join(
                           f'printf("%zu ", offsetof({s}, {f}));' for f in fs)
                       for s, fs in fields.items()) + 'return 0; }\n')
    exe = tmp_path / 'sizes'
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([cc, '-I', os.path.join(root, 'include'), str(src), '-o', str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    delta, norm = struct.calcsize('@5P'), struct.calcsize('@6P')
    assert got == [_sequence._DELTA_IN.size, delta, delta + 12 * 8, delta + 15 * 8,
                   delta + 15 * 8 + 12, delta + 15 * 8 + 24, delta + 15 * 8 + 28,
                   _sequence._NORM_IN.size, norm, norm + 3 * 8, norm + 4 * 8, norm + 4 * 8 + 16,
                   norm + 4 * 8 + 20, norm + 4 * 8 + 24]


def test_launches_of_too_many_threads_are_refused(lib):
    """A grid of 2^32 threads or more wraps: what would need one is an invalid argument."""
    at = ctypes.c_void_p(4096)

    def refused(rc):
        return rc == N.BS_ERR_INVALID and b'exceed' in lib.bs_last_error()

    one = _delta_in(hv=1, dv=128)              # 4 workgroups of 256 a row
    assert refused(lib.bs_gated_delta_step(one, 1 << 22, 1, at, 1 << 22, None, at, None))
    assert lib.bs_gated_delta_workspace_size(one, 1 << 21, 1, 0) == 0
    assert refused(lib.bs_gated_delta_rule(one, 1 << 21, 1, None, None, at, at, None, None, at,
                                           1 << 62, None))
    assert lib.bs_gated_delta_workspace_size(one, (1 << 21) - 16, 1, 0) > 0
    assert lib.bs_gated_delta_grad_workspace_size(_delta_in(), 1, 1 << 29, 0) == 0
    assert lib.bs_gated_delta_grad_workspace_size(_delta_in(), 1, (1 << 29) - 128, 0) > 0
    linear = (at, F32, 8, None, 1 << 30, 8, 1 << 20, at, at, None, F32, at, F32, at, 1 << 62, None)
    assert refused(lib.bs_int8_linear(*linear))
    assert lib.bs_int8_linear(at, F32, 8, None, 1, 8, 1 << 28, at, at, None, F32, at, F32, at,
                              1 << 62, None) == N.BS_ERR_INVALID
