"""Settings at the ends of their ranges that the host's table of rotary angles takes
or refuses: a table that it returns has no NaN or infinity in it. Runs without a GPU."""
import ctypes

import numpy as np
import pytest

import qwen_b200
from qwen_b200 import _lib


def table(positions=5, **change):
    d = dict(theta=1e4, factor=1.0, fast=32.0, slow=1.0, size=0.0, rotated=64, scaling=_lib.ROTARY_PLAIN, trained=4096) | change
    out = np.full((positions, d['rotated']), 7, np.float32)
    rc = qwen_b200.lib().qwen_b200_rotary_table(ctypes.byref(qwen_b200.RotaryAngles(**d)), positions, _lib.ptr(out, ctypes.c_float))
    return rc, out


@pytest.mark.parametrize('change', [
    dict(scaling=_lib.ROTARY_LINEAR, factor=1e-308),            # the fourth position at 4 / 1e-308
    dict(scaling=_lib.ROTARY_YARN, factor=5e-324),              # f / factor
    dict(scaling=_lib.ROTARY_NTK, factor=5e-323, rotated=512),  # theta is some 5e-320, its last power 1e318
    dict(size=3.5e38), dict(size=1e300)], ids=str)
def test_settings_whose_table_would_have_infinities_or_nan_are_refused(change):
    rc, out = table(**change)
    assert rc == _lib.EINVAL and (out == 7).all()


@pytest.mark.parametrize('change', [
    dict(size=3.4e38), dict(size=1e-45), dict(scaling=_lib.ROTARY_LINEAR, factor=1e-3), dict(scaling=_lib.ROTARY_LINEAR, factor=1e300),
    dict(scaling=_lib.ROTARY_YARN, factor=1e300), dict(theta=1e300), dict(theta=1.0000001)], ids=str)
def test_settings_at_the_ends_of_their_ranges_give_a_table(change):
    rc, out = table(**change)
    assert rc == _lib.OK and np.isfinite(out).all() and (out != 7).all()


@pytest.mark.parametrize('trained,slow', [(64, 16.0), (4, 1.0), (1, 0.5)])
def test_yarn_where_every_pair_turns_less_than_slow_times(trained, slow):
    """Pair 0 turns trained / (2 pi) times: below `slow` it is divided by the factor like all behind it."""
    assert trained / (2 * np.pi) < slow
    rc, out = table(scaling=_lib.ROTARY_YARN, trained=trained, slow=slow, factor=4.0, size=1.0)
    plain, exact = table(scaling=_lib.ROTARY_LINEAR, factor=4.0)
    assert rc == plain == _lib.OK and np.array_equal(out, exact)
