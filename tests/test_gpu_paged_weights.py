"""Decode attention holds a softmax weight in 16 bits (two bf16 halves). Seen
through values that cancel: the result is some 2^-10 of what is summed, so its
own rounding to bf16 does not hide the weights'.

Tolerance, relative to size = sum(p |v|) / sum(p): a weight as a bf16 and the
bf16 of what is left errs by half a step of half a step, (2^-8)^2 = 2^-16. A
query has one entry that is not zero, so a product q.k is one term and exact;
the factors of the score and the subtraction of the maximum err by 8 U times the
largest |score| at most, exp2 by 2^-21, the sums of n terms by n U each in
numerator and denominator (what the denominator errs by counts with |ctx| <=
size). The result is rounded to bf16 once."""
import numpy as np
import pytest

from gpu_util import Keep
from paged_ref import BF16_HALF, U, Cache, bf16
from qwen_b200 import _lib
from test_gpu_paged import DIMS, FORMATS, decode

W = 2.0 ** -16


def cancelling(fmt, dim, n, scale):
    """A cache of one sequence whose values nearly cancel under the query's weights, the query, the weights and the
    values in 64 bits."""
    c = Cache(n + dim, fmt, 2, dim, 16, -(-n // 16) + 2, 1, -(-n // 16)).give([n])
    q = np.zeros((1, 14, dim), np.float32)
    q[:, :7, 5], q[:, 7:, dim - 3] = 3.5, -2.75
    k, v = c.read(0, 0, np.arange(n))
    x = np.stack([k[:, 0, 5] * 3.5, k[:, 1, dim - 3] * -2.75], 1) * scale
    w = np.exp(x - x.max(0))
    w /= w.sum(0)
    # each value turned against the sum so far, the heaviest first and the last ones of the lightest key's size
    total = np.zeros((2, dim))
    page, offset = c.at(0, np.arange(n))
    for h in range(2):
        for t in np.argsort(-w[:, h]):
            sign = np.where(total[h] * v[t, h] > 0, -1, 1)
            if fmt == _lib.KV8:
                c.v[0, page[t], h, offset[t]] = np.maximum(c.v[0, page[t], h, offset[t]], -127) * sign
            else:
                c.v[0, page[t], h, offset[t]] = c.v[0, page[t], h, offset[t]] * sign
            total[h] += w[t, h] * v[t, h] * sign
    return c, q, w, c.read(0, 0, np.arange(n))[1], np.abs(x).max()


def expected(w, v, n, most):
    out, size = np.einsum('th,thd->hd', w, v), np.einsum('th,thd->hd', w, np.abs(v))
    bound = (W + 8 * U * most + 2.0 ** -21 + 2 * n * U) * 2 * size  # the error of a weight in numerator and denominator
    return out, size, bound + BF16_HALF * (np.abs(out) + bound)


CASES = pytest.mark.parametrize('n', [64, 200])


@FORMATS
@DIMS
@CASES
def test_the_bound_tells_16_bits_from_8(fmt, dim, n):
    """In 64 bits on the host: weights in two halves keep the bound, their first halves alone do not."""
    c, q, w, v, most = cancelling(fmt, dim, n, 0.5)
    out, size, bound = expected(w, v, n, most)
    assert np.median(np.abs(out) / size) < 2.0 ** -9
    scales = c.vs[0][c.at(0, np.arange(n))[0], :, c.at(0, np.arange(n))[1]] if fmt == _lib.KV8 else np.ones((n, 2))
    held = w / w.max(0) * scales
    high = bf16(held).astype(np.float64)
    both = high + bf16((held - high).astype(np.float32))
    for half, keeps in ((both, True), (high, False)):
        off = np.abs(np.einsum('th,thd->hd', half / scales * w.max(0), v) - out)
        assert (off <= bound).all() if keeps else (off > bound).mean() > 0.5


@pytest.mark.gpu
@FORMATS
@DIMS
@CASES
def test_decode_holds_weights_in_16_bits(fmt, dim, n):
    c, q, w, v, most = cancelling(fmt, dim, n, 0.5)
    out, size, bound = expected(w, v, n, most)
    keep = Keep()
    got = decode(c, c.upload(keep), keep, 0, q, None, scale=0.5)
    for h in range(14):
        assert (np.abs(got[0, h] - out[h // 7]) <= bound[h // 7]).all()
