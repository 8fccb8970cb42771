"""Checks of the decay-attention, layer-norm, dropout and 4-bit entry points that come before any
device work (CPU)."""
import ctypes
import os
import shutil
import struct
import subprocess

import pytest

from brainstate_amd import _dropout, _sequence
from brainstate_amd import _native as N

F32, BF16 = 0, 1
AT = ctypes.c_void_p(4096)            # an address that nothing reads


@pytest.fixture
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.skip('library not built')
    return N.load_library()


def _in(hk=1, hv=1, dk=16, dv=16, stride=16, at=4096, dtype=F32):
    return _sequence._DELTA_IN.pack(*[at] * 4, 0, *[stride] * 12, 0, 0, 0, dtype, F32, 0, hk, hv,
                                    dk, dv, 1.0)


def _refused(lib, rc, *words):
    text = lib.bs_last_error()
    return rc == N.BS_ERR_INVALID and all(w in text for w in words)


def test_layer_norm_operands_are_the_compiled_headers_struct(tmp_path):
    cc = shutil.which('gcc')
    if cc is None:
        pytest.skip('no host C compiler')
    fields = ['seed_at', 'x_stride', 'seed', 'dim', 'site', 'eps']
    src = tmp_path / 'sizes.c'
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "brainstate_amd.h"\n'
                   'int main(void) { printf("%zu ", sizeof(bs_layer_norm_in));' +
                   ''.join(f'printf("%zu ", offsetof(bs_layer_norm_in, {f}));' for f in fields) +
                   'return 0; }\n')
    exe = tmp_path / 'sizes'
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([cc, '-I', os.path.join(root, 'include'), str(src), '-o', str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    p, q = struct.calcsize('P'), 8
    assert got == [_dropout._NORM_IN.size, 4 * p, 5 * p, 5 * p + 3 * q, 5 * p + 4 * q,
                   5 * p + 4 * q + 16, 5 * p + 4 * q + 28]


def test_decay_attention_refusals(lib):
    assert _refused(lib, lib.bs_decay_attention_step(_in(hk=2, hv=3), 1, 1, AT, 1, None, AT, None),
                    b'value heads')
    assert _refused(lib, lib.bs_decay_attention_step(_in(dk=129), 1, 1, AT, 1, None, AT, None),
                    b'outside')
    assert _refused(lib, lib.bs_decay_attention_step(_in(at=0), 1, 1, AT, 1, None, AT, None),
                    b'NULL')
    assert _refused(lib, lib.bs_decay_attention_step(_in(dv=128), 1 << 22, 1, AT, 1 << 22, None,
                                                     AT, None), b'exceeds')
    one = _in(dk=128, dv=128)
    need = lib.bs_decay_attention_workspace_size(one, 1, 4096, 0, 0)
    assert need > 0
    assert _refused(lib, lib.bs_decay_attention(one, 1, 4096, None, None, AT, AT, None, 0, AT,
                                                need - 1, None), b'workspace')
    kept = lib.bs_decay_attention_kept_size(one, 1, 4096, 0, 2)
    assert kept >= 64 * 128 * 128 * 4
    assert lib.bs_decay_attention_kept_size(one, 1, 4096, 0, 1) < kept
    assert _refused(lib, lib.bs_decay_attention(one, 1, 4096, None, None, AT, AT, None, 2, AT, need,
                                                None), b'kept')
    assert _refused(lib, lib.bs_decay_attention(one, 1, 4096, None, None, AT, AT, AT, 3, AT, need,
                                                None), b'keep 3')
    assert _refused(lib, lib.bs_decay_attention_grad(one, 1, 4096, None, AT, None, None, None, AT,
                                                     AT, AT, AT, 0, None, AT, 1 << 62, None),
                    b'kept')
    assert lib.bs_decay_attention_workspace_size(one, 1, 1 << 28, 0, 0) == 0
    assert b'exceed' in lib.bs_last_error()
    wide = _in(stride=1 << 23)
    assert lib.bs_decay_attention_workspace_size(wide, 1, 64, 0, 0) == 0
    assert b'token to token' in lib.bs_last_error()


def test_layer_norm_and_dropout_refusals(lib):
    def norm(rows=2, dim=8, dtype=F32, x=4096, weight=0):
        return _dropout._NORM_IN.pack(x, 0, weight, 0, 0, dim, dim, rows, 0, dim, dtype, F32, F32,
                                      0, 0, 1.0, 1e-5)
    assert _refused(lib, lib.bs_layer_norm(norm(dim=16385), None, AT, None, None), b'16384')
    assert _refused(lib, lib.bs_layer_norm(norm(dtype=7), None, AT, None, None), b'dtype')
    assert _refused(lib, lib.bs_layer_norm(norm(x=0), None, AT, None, None), b'NULL')
    assert _refused(lib, lib.bs_layer_norm(norm(), None, None, None, None), b'output')
    assert _refused(lib, lib.bs_layer_norm_grad(norm(), AT, AT, None, AT, None, None, None, None, 0,
                                                None), b'stats')
    assert _refused(lib, lib.bs_layer_norm_grad(norm(), AT, AT, AT, AT, AT, None, None, None, 0,
                                                None), b'not given')
    assert _refused(lib, lib.bs_layer_norm_grad(norm(weight=4096), AT, AT, AT, AT, None, AT, None,
                                                None, 0, None), b'workspace')
    assert lib.bs_layer_norm(norm(rows=0), None, None, None, None) == N.BS_OK
    assert _refused(lib, lib.bs_dropout(AT, 9, 1, 1, 1, 0, None, 0, 0, 1.0, AT, None), b'dtype')
    assert _refused(lib, lib.bs_dropout(None, F32, 1, 1, 1, 0, None, 0, 0, 1.0, AT, None), b'NULL')
    assert lib.bs_dropout(None, F32, 0, 1, 1, 0, None, 0, 0, 1.0, None, None) == N.BS_OK


def test_int4_channels_of_one_launch(lib):
    # 16 channels to a workgroup of 512 threads: from 2^27 on a launch would have 2^32 threads
    assert _refused(lib, lib.bs_int4_linear(AT, F32, 1, 1, 1, 1 << 27, 32, AT, AT, None, F32, AT, None, 0,
                                            None), b'channels')


def test_int4_refusals(lib):
    def linear(m=1, k=64, n=8, group=32, w4=AT, ws=AT, nbytes=1 << 40, dtype=BF16):
        return lib.bs_int4_linear(AT, dtype, k, m, k, n, group, w4, AT, None, F32, AT, ws, nbytes,
                                  None)
    assert _refused(lib, linear(group=16), b'groups')
    assert _refused(lib, linear(k=65537), b'65536')
    assert _refused(lib, linear(w4=None), b'NULL')
    assert _refused(lib, linear(dtype=5), b'dtype')
    assert _refused(lib, linear(m=1 << 26, n=1 << 20), b'exceed')
    need = lib.bs_int4_workspace_size(AT, F32, 64, 100, 64, 8)
    assert need == 100 * 128 * 2 * 3            # three parts in rows of whole steps
    assert _refused(lib, linear(m=100, dtype=F32, ws=None), b'workspace')
    assert lib.bs_int4_workspace_size(AT, BF16, 128, 100, 128, 8) == 0
    assert lib.bs_int4_workspace_size(AT, BF16, 1 << 22, 100, 128, 8) > 0   # rows too far apart
    assert lib.bs_int4_workspace_size(AT, F32, 64, 16, 64, 8) == 0
    assert _refused(lib, lib.bs_int4_quantize(AT, F32, 1, 64, 64, 48, AT, AT, None), b'groups')
    assert lib.bs_int4_quantize(None, F32, 0, 64, 64, 32, None, None, None) == N.BS_OK
