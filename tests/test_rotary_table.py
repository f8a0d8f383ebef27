"""The host's table of rotary angles against its formulas in the widest floats of
numpy, and what it refuses. Runs without a GPU."""
import ctypes

import numpy as np
import pytest

import qwen_b200
from qwen_b200 import _lib

F = np.longdouble


def table(positions, rotated, scaling=_lib.ROTARY_PLAIN, theta=1e6, factor=1.0, fast=32.0, slow=1.0, size=0.0, trained=32768):
    a = qwen_b200.RotaryAngles(theta, factor, fast, slow, size, rotated, scaling, trained)
    out = np.full(positions * rotated, np.nan, np.float32)
    assert qwen_b200.lib().qwen_b200_rotary_table(ctypes.byref(a), positions, _lib.ptr(out, ctypes.c_float)) == 0
    return out.reshape(positions, rotated)


def formula(positions, rotated, scaling, theta=1e6, factor=1.0, fast=32.0, slow=1.0, size=0.0, trained=32768):
    i = np.arange(rotated // 2).astype(F)
    if scaling == _lib.ROTARY_NTK:
        theta = F(theta) * F(factor) ** (F(rotated) / (rotated - 2))
    f = F(theta) ** (-2 * i / rotated)
    if scaling == _lib.ROTARY_LINEAR:
        f = f / F(factor)
    if scaling == _lib.ROTARY_YARN:
        turns = F(trained) * f / (2 * np.pi)
        # i as a real number at which a pair turns n times, by bisection over the pairs' falling turns
        at = [np.interp(-np.log(n), -np.log(turns.astype(float)), i.astype(float), left=-1e9, right=1e9) for n in (fast, slow)]
        exact = [rotated * np.log(trained / (n * 2 * np.pi)) / (2 * np.log(theta)) for n in (fast, slow)]
        for a, e in zip(at, exact):
            assert abs(a) > 1e8 or abs(a - e) < 1e-6
        low, high = max(np.floor(exact[0]), 0), min(np.ceil(exact[1]), rotated - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        f = f * (1 - ramp) + f / F(factor) * ramp
        size = size or (0.1 * np.log(factor) + 1 if factor > 1 else 1.0)
    a = np.arange(positions).astype(F)[:, None] * f
    return np.concatenate([np.cos(a), np.sin(a)], 1) * (size or 1.0)


@pytest.mark.parametrize('scaling', [_lib.ROTARY_PLAIN, _lib.ROTARY_LINEAR, _lib.ROTARY_NTK, _lib.ROTARY_YARN])
@pytest.mark.parametrize('rotated', [16, 64, 96, 128, 512])
@pytest.mark.parametrize('factor', [1.0, 4.0, 7.3])
def test_angles(scaling, rotated, factor):
    kw = dict(scaling=scaling, factor=1.0 if scaling == _lib.ROTARY_PLAIN else factor)
    got, exact = table(3000, rotated, **kw), formula(3000, rotated, **kw)
    # an angle below 3000 in 64 bits: some 4 roundings of 2^-53 of it (power, ramp, product), then one of fp32 (2^-24 of a value up to 1.21)
    assert np.abs(got - exact).max() <= 1.25 * 2.0 ** -24 + 3000 * 16 * 2.0 ** -53


def test_far_positions_and_size():
    got, exact = table(1 << 18, 16, size=0.5), formula(1 << 18, 16, _lib.ROTARY_PLAIN, size=0.5)
    assert np.abs(got[-1000:] - exact[-1000:]).max() <= 2.0 ** -25 + (1 << 18) * 16 * 2.0 ** -53


def test_the_models_own_table():
    """64 dims, theta 1e6: the angles of qwen_b200_rope_table, which forms them its own way."""
    own = np.zeros((300, 64), np.float32)
    qwen_b200.lib().qwen_b200_rope_table(300, _lib.ptr(own, ctypes.c_float))
    assert np.abs(table(300, 64) - own).max() < 1e-4


@pytest.mark.parametrize('change', [
    dict(rotated=0), dict(rotated=8), dict(rotated=72), dict(rotated=528), dict(scaling=4), dict(theta=1.0),
    dict(theta=float('nan')), dict(theta=float('inf')), dict(factor=0.0, scaling=1), dict(factor=-1.0, scaling=2),
    dict(factor=float('inf'), scaling=3), dict(trained=0, scaling=3), dict(fast=1.0, slow=1.0, scaling=3),
    dict(slow=0.0, scaling=3), dict(fast=float('inf'), scaling=3), dict(size=-1.0), dict(size=float('nan')),
], ids=str)
def test_refused(change):
    d = dict(theta=1e6, factor=2.0, fast=32.0, slow=1.0, size=0.0, rotated=64, scaling=0, trained=4096) | change
    a = qwen_b200.RotaryAngles(**d)
    out = np.zeros(64 * 4, np.float32)
    assert qwen_b200.lib().qwen_b200_rotary_table(ctypes.byref(a), 4, _lib.ptr(out, ctypes.c_float)) == _lib.EINVAL
    assert not out.any()


def test_refused_pointers_and_positions():
    L = qwen_b200.lib()
    a = qwen_b200.RotaryAngles(1e6, 1.0, 32.0, 1.0, 0.0, 64, 0, 0)
    out = np.zeros(64, np.float32)
    p = _lib.ptr(out, ctypes.c_float)
    assert L.qwen_b200_rotary_table(None, 1, p) == _lib.EINVAL
    assert L.qwen_b200_rotary_table(ctypes.byref(a), 1, None) == _lib.EINVAL
    assert L.qwen_b200_rotary_table(ctypes.byref(a), 0, p) == _lib.EINVAL
    assert L.qwen_b200_rotary_table(ctypes.byref(a), (1 << 24) + 1, p) == _lib.EINVAL
