"""Softmax scales far from 1: queries and scale are multiplied by powers of two
that cancel, so every score is what it is with neither."""
import numpy as np
import pytest

from gpu_util import Keep
from test_gpu_paged import DIMS, FORMATS, cache, check_decode, check_prefill

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
