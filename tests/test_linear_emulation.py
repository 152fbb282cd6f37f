"""Index arithmetic of the channel-mixing kernels, compiled for the CPU (tests/emu/linear_emu.cu)."""
import ctypes
import os
import subprocess

import numpy as np
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
    lib.emu_scaled_sum.argtypes, lib.emu_scaled_sum.restype = [ci, ctypes.c_float, ctypes.c_float], ctypes.c_float
    lib.emu_lin_div_misses.argtypes, lib.emu_lin_div_misses.restype = [ctypes.c_void_p, ctypes.c_void_p, i64, ci], i64
    lib.emu_few_channels.argtypes = [i64, i64, ci]
    return lib


@pytest.mark.parametrize('cols', [1, 24, 2 ** 30 - 8, 2 ** 30 + 8, 2 ** 31 - 1025])
def test_offsets_of_any_accepted_size(emu, cols):
    """Every size that the argument checks accept: up to 2^31 - 1025 rows, and as many columns."""
    for row in (0, 1, 17, 2 ** 20, 2 ** 31 - 1026):
        for col in {0, cols // 2, max(0, cols - 32), cols - 1}:
            assert emu.emu_lin_out_offset(row, col, cols) == 2 * (row * cols + col)


def test_a_sum_with_scales_of_any_size(emu):
    """Three roundings of the exact product wherever it lies inside fp32's normal range, however large the row's scale or
    small the channel's; and the plain sum * rs * cs to the bit wherever that does not overflow on its way."""
    rng = np.random.default_rng(0)
    f32 = np.float32
    sums = [0, 1, -1, 127 * 127, -(2 ** 14) * 131071, *rng.integers(-2 ** 31 + 1, 2 ** 31, 40).tolist()]
    row = [0.0, 1.0, 2.0 ** 90, np.nextafter(f32(2.0 ** 90), f32(0)), f32(3.4e38), f32(1e-38), f32(1e-44), -2.0 ** 100, *np.exp(rng.uniform(-85, 88, 40))]
    col = [0.0, 1.0, f32(3.4e38), f32(1e-38), f32(1e-45), -1e-30, *np.exp(rng.uniform(-85, 88, 40))]
    inside = 0
    for s in sums:
        for rs in map(f32, row):
            for cs in map(f32, col):
                got = f32(emu.emu_scaled_sum(s, rs, cs))
                exact = float(s) * float(rs) * float(cs)
                with np.errstate(all='ignore'):
                    step = f32(s) * rs
                    plain = step * cs
                if np.isfinite(step):
                    assert got == plain, (s, rs, cs)
                if 2.0 ** -126 <= abs(exact) < 2.0 ** 127:
                    inside += not np.isfinite(plain)
                    assert abs(float(got) - exact) <= 3.1 * 2.0 ** -24 * abs(exact), (s, rs, cs)
    assert inside > 100  # results that the plain order loses


@pytest.mark.parametrize('ulps', [-1, 0, 1])
def test_division_by_a_reciprocal(emu, ulps):
    """The quotient that finds units: exact for every pair, with the hardware's reciprocal off by up to its documented unit."""
    rng, top = np.random.default_rng(ulps + 1), 2 ** 31 - 1
    edges = np.unique(np.clip([v + k for e in range(32) for v in (2 ** e, 3 * 2 ** e // 2) for k in range(-2, 3)], 0, top))
    pairs = [np.meshgrid(edges, edges[edges > 0])]
    for hi in (100, 10 ** 4, 2 ** 20, 2 ** 24, top):
        for dhi in (2, 17, 300, 5000, 2 ** 20, top):
            n, d = rng.integers(0, hi, 100000), rng.integers(1, dhi, 100000)
            pairs += [(n, d), (np.clip(n // d * d + rng.integers(-1, 2, n.shape), 0, top), d)]
    pairs.append((np.full(100000, top), np.arange(1, 100001)))
    for n, d in pairs:
        n, d = (np.ascontiguousarray(np.ravel(a), np.int32) for a in (n, d))
        assert emu.emu_lin_div_misses(n.ctypes.data, d.ctypes.data, len(n), ulps) == 0


@pytest.mark.parametrize('sms', [18, 74, 132, 148])
def test_channels_of_a_few_rows_cta_follow_the_device(emu, sms):
    """CTAs of 16 channels as long as two to an SM hold all of them, on a device (or a part of one) of any size."""
    for groups in (1, 8, 16):
        n = 2 * sms // groups * 16
        assert emu.emu_few_channels(n, groups, sms) == 16 and emu.emu_few_channels(n + 1, groups, sms) == 32
    assert emu.emu_few_channels(2 ** 31 - 1025, 1, sms) == 32
