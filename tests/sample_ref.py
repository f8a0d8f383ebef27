"""Sampling from a row of logits by its definition, in 64 bits: what the tests of
qwen_b200_op_sample compare with."""
import numpy as np

NO_TOKEN = 0xffffffff


def candidates(row):
    """Ids in the order of their logits, the lowest id first among equal ones; NaN and -infinity are none."""
    x = np.asarray(row, np.float64)
    ids = np.flatnonzero(x > -np.inf)
    return ids[np.argsort(-x[ids], kind='stable')]


def kept_weights(row, temperature, top_k, top_p, min_p):
    """(ids, weights) of the kept candidates; `near`: whether a border of theirs is too close to call in 64 bits."""
    row = np.asarray(row, np.float64)
    ids = candidates(row)
    if not ids.size:
        return ids, np.zeros(0), False
    x = row[ids]
    if not temperature > 0:
        n = int((x == x[0]).sum())
        return ids[n - 1:n], np.ones(1), False
    with np.errstate(invalid='ignore', over='ignore', divide='ignore'):
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / np.float64(np.float32(temperature))))
    if top_k:
        ids, w = ids[:top_k], w[:top_k]
    p, least = np.float64(np.float32(top_p)), np.float64(np.float32(min_p))
    before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
    share = max(p, 0.0) * w.sum() if not np.isnan(p) else 0.0
    keep = np.ones(w.size, bool) if p >= 1 else before < share
    near = not p >= 1 and bool((np.abs(before - share) < slack(row.size) + w.size * 2.0 ** -52 * share)[1:].any())
    keep &= w >= least
    keep[0] = True
    n = w.size if keep.all() else int(np.argmin(keep))
    return ids[:n], w[:n], near


def slack(vocab):
    """A weight is rounded to half of 2^-(63 - bits of vocab): a sum of at most vocab of them is off by vocab halves."""
    return vocab * 2.0 ** -(64 - int(vocab).bit_length())


def check(token, prob, row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token is the definition's, or one whose border u falls on within the weights' rounding; its probability to fp32."""
    ids, w, near = kept_weights(row, temperature, top_k, top_p, min_p)
    if not ids.size:
        assert token == NO_TOKEN and prob == 0
        return
    u = min(max(float(np.float32(u)), 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    upto = np.cumsum(w)
    target, tol = u * upto[-1], slack(len(row)) + w.size * 2.0 ** -52 * upto[-1]
    at = np.flatnonzero(ids == token)
    if near and not at.size:
        return
    assert at.size == 1, f'token {token} is not kept'
    i = int(at[0])
    if not near:
        assert upto[i] > target - tol and upto[i] - w[i] <= target + tol, (token, i, upto[i], w[i], target)
        assert w[i] > 0
        assert abs(prob - w[i] / upto[-1]) <= (2.0 ** -24 + 2.0 ** -30) * w[i] / upto[-1] + slack(len(row)), (prob, w[i] / upto[-1])
    expect = ids[min(int(np.searchsorted(upto, target, side='right')), int((w > 0).sum()) - 1)]
    return token == expect
