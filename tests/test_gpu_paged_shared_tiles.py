"""qwen_b200_op_paged_decode_shared on the ways that depend on how many rows and keys
a call has: tiles whose pieces the CTAs of a cluster join (few rows on a long prefix),
whole and ragged tiles of query rows, and the row kernel's softmax weights. Each test
makes sure that the call went the way that it is about."""
import ctypes

import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import Cache, bf16, bits, ref, unbits
from qwen_b200 import _lib
from test_gpu_paged import DIMS, FILL, FORMATS, PREFILL_W, assert_within, u32  # noqa: F401
from test_gpu_paged_shared import attention, shared_cache
from test_gpu_paged_weights import cancelling, expected

pytestmark = pytest.mark.gpu
L = qwen_b200.lib
KV8, BF16, NO_SEQ = _lib.KV8, _lib.KV_BF16, _lib.NO_SEQ
WORK = 3 << 24  # rows * shared keys * KV heads * dims from which a group goes to the tiles


def sms():
    return torch_cuda().cuda.get_device_properties(0).multi_processor_count


def call(c, kv, q, starts, prefix, seqs, scale, times=1):
    """ctx, and whether tiles were computed: their kernel is the only one that writes the workspace behind its first
    8 n + 512 bytes."""
    rows, heads, dim = q.shape
    n, keep = len(prefix), Keep()
    size = L().qwen_b200_paged_decode_shared_workspace(ref(kv), heads, n, rows)
    ws = dev(np.full(size, 0xA5, np.uint8))
    ws[:4] = 0
    out = dev(bits(np.full((rows, heads * dim), np.float32(FILL))).view(np.int16))
    args = (ref(kv), 0, keep(bits(q.reshape(rows, -1)).view(np.int16)), heads * dim, heads, n, keep(u32(starts)),
            keep(u32(prefix)), rows, keep(u32(seqs)) if seqs is not None else None, scale, vp(out), heads * dim, vp(ws), size, stream())
    first = None
    for _ in range(times):
        assert L().qwen_b200_op_paged_decode_shared(*args) == 0
        sync()
        assert first is None or np.array_equal(first, host(out))
        first = host(out)
    w = host(ws)
    assert not w[:4].any(), 'a wait ran out'
    return unbits(first).reshape(q.shape), bool((w[8 * n + 512:] != 0xA5).any())


def check(c, kv, q, starts, prefix, seqs=None, scale=None, tiles=True, times=1):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    got, ran = call(c, kv, q, starts, prefix, seqs, scale, times)
    assert ran == tiles
    exact, tol = attention(c, 0, q, np.arange(len(q)) if seqs is None else np.asarray(seqs, np.int64), scale)
    assert_within(got, exact, tol)
    return got


# few (row, KV head, block of 8 heads) items, so the CTAs of a cluster share a row: 16, 128 and 36 of them
FEW = pytest.mark.parametrize('dim,kv_heads,group,rows,prefix', [(128, 8, 4, 2, 24600), (64, 2, 7, 64, 8192), (64, 2, 7, 18, 24000)])


def few(fmt, dim, kv_heads, group, rows, prefix, page=128, lens=None):
    assert rows * prefix * kv_heads * dim >= WORK
    assert rows * kv_heads * ((group + 7) // 8) < sms()  # fewer items than SMs: more than one CTA each
    r = np.random.default_rng(rows + dim)
    lens = [prefix + int(x) for x in r.integers(0, 900, rows)] if lens is None else lens
    c = shared_cache(rows, fmt, dim, page, [(prefix, lens)], kv_heads)
    return c, bf16(c.rand(rows, kv_heads * group, dim) * 2)


@FORMATS
@FEW
def test_pieces_of_tiles_joined_by_a_cluster(fmt, dim, kv_heads, group, rows, prefix):
    c, q = few(fmt, dim, kv_heads, group, rows, prefix)
    keep = Keep()
    check(c, c.upload(keep), q, [0, rows], [prefix], times=3)


@FORMATS
@pytest.mark.parametrize('dim,kv_heads,group,rows,prefix', [(64, 2, 7, 64, 8192), (64, 2, 7, 18, 24000), (128, 1, 9, 20, 20000)])
def test_short_and_absent_rows_of_a_cluster(fmt, dim, kv_heads, group, rows, prefix):
    """Rows that end inside the prefix, at it, or have no key at all, beside rows that go on behind it."""
    lens = [prefix + 700] + [prefix + 3 * i for i in range(rows - 1)]
    lens[1:8] = [1, 0, 127, 128, prefix - 1, prefix, prefix // 2]
    c, q = few(fmt, dim, kv_heads, group, rows, prefix, 64, lens)
    seqs = np.arange(rows)
    seqs[[9, rows - 1]] = NO_SEQ
    keep = Keep()
    got = check(c, c.upload(keep), q, [0, rows], [prefix], seqs)
    assert not got[[2, 9, rows - 1]].any()


@FORMATS
@FEW
@pytest.mark.parametrize('where', ['prefix', 'own'])
def test_scores_far_apart_in_a_cluster(fmt, dim, kv_heads, group, rows, prefix, where):
    """A key that outweighs all others by hundreds of powers of two, in one of the pieces or behind them; rows of one query
    of different sizes, so that their references differ."""
    c, q = few(fmt, dim, kv_heads, group, rows, prefix, 128, [prefix + 1 + i % 5 for i in range(rows)])
    q = bf16(np.repeat(q[:1], rows, 0) * (0.5 + np.arange(rows) % 3)[:, None, None])
    k = bf16(q[0].reshape(kv_heads, group, dim)[:, 0][None] * 8)
    for s in range(1 if where == 'prefix' else rows):
        c.write(0, s, [prefix // 3 if where == 'prefix' else prefix], k, bf16(np.full((1, kv_heads, dim), 3.0)))
    keep = Keep()
    check(c, c.upload(keep), q, [0, rows], [prefix], scale=2.0)


@FORMATS
@pytest.mark.parametrize('dim,group,rows', [(64, 8, n) for n in (63, 64, 65, 128, 129)] + [(128, 8, n) for n in (31, 32, 33, 64, 65)] +
                         [(64, 7, 73), (64, 7, 74), (128, 7, 36), (128, 7, 37)])
def test_whole_and_ragged_tiles_of_query_rows(fmt, dim, group, rows):
    """512 (64 dims) or 256 query rows a tile: one less than a whole one, whole ones, one more."""
    prefix = -(-WORK // (rows * 8 * dim)) + 5
    r = np.random.default_rng(rows)
    c = shared_cache(rows, fmt, dim, 64, [(prefix, [prefix + int(x) for x in r.integers(0, 60, rows)])], 8)
    keep = Keep()
    check(c, c.upload(keep), bf16(c.rand(rows, 8 * group, dim) * 2), [0, rows], [prefix])


# ---------------------------------------------------------------- softmax weights
@FORMATS
@DIMS
@pytest.mark.parametrize('n', [64, 200])
@pytest.mark.parametrize('items', [1, 3, 6])
@pytest.mark.parametrize('wide', [False, True])
def test_rows_hold_weights_in_16_bits(fmt, dim, n, items, wide):
    """Where a row takes its whole context by itself, with 8, 4 and 2 warps (one, three and six items an SM), alone and
    behind a tile kernel that had nothing to do (a table wide enough for more)."""
    c, q, w, v, most = cancelling(fmt, dim, n, 0.5)
    rows = 1 if items == 1 else -(-items * sms() // 2)
    if wide:
        width = 1 + -(-WORK // (rows * 2 * dim * c.T))
        c.table = np.concatenate([c.table, np.full((1, width), 1 << 30, np.uint32)], 1)
        c.max_pages += width
    out, size, bound = expected(w, v, n, most)
    keep = Keep()
    got, ran = call(c, c.upload(keep), np.repeat(q, rows, 0), [0, rows], [n // 2], np.zeros(rows), 0.5)
    assert not ran and (got == got[:1]).all()
    for h in range(14):
        assert (np.abs(got[0, h] - out[h // 7]) <= bound[h // 7]).all()


@FORMATS
@DIMS
@pytest.mark.parametrize('n', [64, 200])
@pytest.mark.parametrize('few_rows', [True, False])
def test_own_keys_behind_tiles_hold_weights_in_16_bits(fmt, dim, n, few_rows):
    """All of the weight is on a row's own keys: those of its prefix score some 200 less (powers of e), so that their part is
    below 2^-200."""
    c, q, w, v, most = cancelling(fmt, dim, n, 0.5)
    rows = 2 if few_rows else 450
    prefix = -(-WORK // (rows * 2 * dim * 16)) * 16  # whole pages in front
    first = prefix // 16
    low = np.zeros((prefix, 2, dim), np.float32)
    low[:, 0, 5], low[:, 1, dim - 3] = -120.0, 150.0  # * 3.5 * 0.5 and * -2.75 * 0.5
    b = Cache(3, fmt, 2, dim, 16, c.pages + first, 1, c.max_pages + first)
    b.lengths[:] = prefix + n
    used = -(-n // 16)
    for name in ('k', 'v') + (('ks', 'vs') if fmt == KV8 else ()):
        getattr(b, name)[:, first:] = getattr(c, name)
    b.table[0, :first], b.table[0, first:first + used] = np.arange(first), c.table[0, :used] + first
    b.write(0, 0, np.arange(prefix), low, b.rand(prefix, 2, dim))
    out, size, bound = expected(w, v, n, most)
    keep = Keep()
    got, ran = call(b, b.upload(keep), np.repeat(q, rows, 0), [0, rows], [prefix], np.zeros(rows), 0.5)
    assert ran and (got == got[:1]).all()
    for h in range(14):
        assert (np.abs(got[0, h] - out[h // 7]) <= bound[h // 7]).all()


@FORMATS
@DIMS
@pytest.mark.parametrize('n', [64, 200])
@pytest.mark.parametrize('part', [1, 2])
def test_tiles_hold_weights_in_16_bits(fmt, dim, n, part):
    """All of a row's keys, or the first half of them, as its group's shared ones: a row's result has the precision of
    qwen_b200_op_paged_decode whatever the batch that it is in."""
    c, q, w, v, most = cancelling(fmt, dim, n, 0.5)
    rows = -(-WORK // (n // part * 2 * dim))
    out, size, bound = expected(w, v, n, most)
    keep = Keep()
    got, ran = call(c, c.upload(keep), np.repeat(q, rows, 0), [0, rows], [n // part], np.zeros(rows), 0.5)
    assert ran and (got == got[:1]).all()
    for h in range(14):
        assert (np.abs(got[0, h] - out[h // 7]) <= bound[h // 7]).all()


# ---------------------------------------------------------------- rows that see less than their group shares
@FORMATS
@pytest.mark.parametrize('dim,kv_heads,group,rows,prefix', [(64, 8, 2, 195, 520), (128, 8, 2, 150, 333), (64, 2, 7, 64, 8192)])
def test_values_that_a_row_does_not_see_do_not_reach_it(fmt, dim, kv_heads, group, rows, prefix):
    """NaN and infinities in shared keys and values behind a row's last token, and behind none at all, as in a group that
    has no tiles. Rows that do see them are not looked at."""
    lens = [prefix + 40] + [prefix + i % 30 for i in range(rows - 1)]
    short = np.arange(1, 12)
    lens[1:12] = [1, 0, 5, 63, 64, 65, 100, 127, 128, 129, 200]
    c = shared_cache(rows, fmt, dim, 64, [(prefix, lens)], kv_heads)
    q = bf16(c.rand(rows, kv_heads * group, dim) * 2)
    seqs = np.arange(rows)
    seqs[[20, rows - 1]] = NO_SEQ
    clean = np.concatenate([short, [20, rows - 1]])
    exact, tol = attention(c, 0, q[clean], seqs[clean], dim ** -0.5)
    bad = np.arange(200, prefix)  # (every short row ends in front of it)
    p, t = c.at(0, bad)
    for name, value in (('vs', np.nan), ('ks', np.inf)) if fmt == KV8 else (('v', np.nan), ('k', np.inf)):
        getattr(c, name)[0, p, :, t] = value
    keep = Keep()
    got, ran = call(c, c.upload(keep), q, [0, rows], [prefix], seqs, dim ** -0.5)
    assert ran
    assert_within(got[clean], exact, tol)
    assert not got[[2, 20, rows - 1]].any()


@FORMATS
@pytest.mark.parametrize('dim,kv_heads,group,rows,prefix', [(64, 8, 2, 195, 520), (128, 8, 2, 150, 333), (64, 2, 7, 64, 8200)])
def test_the_first_rows_own_values_do_not_reach_the_others(fmt, dim, kv_heads, group, rows, prefix):
    """The shared keys are read from the first row's pages, the last of which holds tokens of its own."""
    lens = [prefix + 40] + [prefix + i % 30 for i in range(rows - 1)]
    c = shared_cache(rows, fmt, dim, 64, [(prefix, lens)], kv_heads)
    q = bf16(c.rand(rows, kv_heads * group, dim) * 2)
    exact, tol = attention(c, 0, q, np.arange(rows), dim ** -0.5)
    p, t = c.at(0, np.arange(prefix, prefix + 40))
    for name, value in (('vs', np.nan), ('ks', np.inf)) if fmt == KV8 else (('v', np.nan), ('k', np.inf)):
        getattr(c, name)[0, p, :, t] = value
    keep = Keep()
    got, ran = call(c, c.upload(keep), q, [0, rows], [prefix], None, dim ** -0.5)
    assert ran and np.isnan(got[0]).all()
    assert_within(got[1:], exact[1:], tol[1:])


# ---------------------------------------------------------------- which calls go to the tiles
@FORMATS
@pytest.mark.parametrize('dim,group,groups', [(64, 64, [(4096, 64)]), (128, 32, [(2048, 120)]), (64, 16, [(40, 220), (2300, 4)])])
def test_many_heads_on_one_kv_head(fmt, dim, group, groups):
    """Three (row, block of 8 heads) items an SM, though rows x keys x KV heads x dims would be too few with the widest
    table: prefixes of 2048 keys go to the tiles."""
    r = np.random.default_rng(group)
    members = [(p, [p + int(x) for x in r.integers(0, 40, n)]) for p, n in groups]
    c = shared_cache(group, fmt, dim, 64, members, 1)
    rows = c.seqs
    assert rows * (group // 8) >= 3 * sms() and rows * c.max_pages * c.T * dim < WORK
    keep = Keep()
    check(c, c.upload(keep), bf16(c.rand(rows, group, dim) * 2), np.concatenate([[0], np.cumsum([n for _, n in groups])]),
          [p for p, _ in groups])


def test_one_row_has_no_tiles():
    c = shared_cache(1, KV8, 64, 256, [(30000, [30000])], 2)
    c.table = np.concatenate([c.table, np.full((1, 2000), 1 << 30, np.uint32)], 1)
    c.max_pages += 2000
    assert c.max_pages * c.T * 2 * 64 >= WORK
    keep = Keep()
    check(c, c.upload(keep), bf16(c.rand(1, 14, 64) * 2), [0, 1], [30000], tiles=False)
