"""Sizes far from 1. Softmax scales: queries and scale are multiplied by powers of two
that cancel, so every score is what it is with neither. Values: up to the size that
the sums are documented to hold, and as far below."""
import numpy as np
import pytest

from gpu_util import Keep
from test_gpu_paged import DIMS, FORMATS, KV8, cache, check_decode, check_prefill

pytestmark = pytest.mark.gpu


@FORMATS
@DIMS
@pytest.mark.parametrize('log', [-80, -40, 40, 100, 107])
def test_a_scale_that_undoes_the_queries_size(fmt, dim, log):
    """Queries times 2^log, the scale times 2^-log: products of 2^107 * 4 * 127 * 128 stay below 2^127."""
    lens = [200, 77]
    c = cache(abs(log), fmt, dim, 16, lens)
    keep = Keep()
    kv = c.upload(keep)
    for sign in (1, -1):
        scale = sign * 2.0 ** (-3 - log)
        check_decode(c, kv, keep, c.rand(2, 14, dim) * np.float32(2.0 ** log), None, scale=scale)
        check_prefill(c, kv, keep, c.rand(277, 14, dim) * np.float32(2.0 ** log), None, [0, 200, 277], scale=scale)


@FORMATS
@DIMS
@pytest.mark.parametrize('log', [-80, 79])
@pytest.mark.parametrize('spread', [1, 4])
def test_values_of_any_documented_size(fmt, dim, log, spread):
    """Values of some 2^log (unit variance, so none above 2^80), with scores a few or some ten powers of two apart."""
    lens = [400, 77]
    c = cache(abs(log) + spread, fmt, dim, 16, lens)
    if fmt == KV8:
        c.vs *= np.float32(2.0 ** (log - 2))
    else:
        c.v = np.ldexp(c.v, log - 2)
    keep = Keep()
    kv = c.upload(keep)
    assert 0 < np.nanmax(np.abs(c.read(0, 0, np.arange(400))[1])) < 2.0 ** 80
    check_decode(c, kv, keep, c.rand(2, 14, dim) * spread, None)
    check_prefill(c, kv, keep, c.rand(477, 14, dim) * spread, None, [0, 400, 477])
