"""Index arithmetic of the channel-mixing kernels, compiled for the CPU (tests/emu/linear_emu.cu)."""
import ctypes
import os
import subprocess

import pytest

from tests import conftest


@pytest.fixture(scope='module')
def emu():
    from kerops_b200 import build

    src = os.path.join(conftest.ROOT, 'tests', 'emu', 'linear_emu.cu')
    so = os.path.join(os.path.dirname(src), 'liblinear_emu.so')
    if not os.path.exists(so) or any(os.path.getmtime(d) > os.path.getmtime(so) for d in [src] + build.HEADERS):
        r = subprocess.run([build.find_nvcc(), '-std=c++17', '-O2', '-Xcompiler', '-fPIC', '-shared', '-gencode',
                            'arch=compute_100a,code=sm_100a', '-o', so, src], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
    lib = ctypes.CDLL(so)
    i64, ci = ctypes.c_int64, ctypes.c_int
    lib.emu_lin_out_offset.argtypes, lib.emu_lin_out_offset.restype = [i64, ci, ci], i64
    return lib


@pytest.mark.parametrize('cols', [1, 24, 2 ** 30 - 8, 2 ** 30 + 8, 2 ** 31 - 1025])
def test_offsets_of_any_accepted_size(emu, cols):
    """Every size that the argument checks accept: up to 2^31 - 1025 rows, and as many columns."""
    for row in (0, 1, 17, 2 ** 20, 2 ** 31 - 1026):
        for col in {0, cols // 2, max(0, cols - 32), cols - 1}:
            assert emu.emu_lin_out_offset(row, col, cols) == 2 * (row * cols + col)
