"""The paged KV cache's operators (qwen_b200_op_paged_*, qwen_b200_op_pages_*)
against the host cache of paged_ref.py: appends bit for bit, attention within
the bound derived there, page management as whole numbers, and the operators
together as a server would run them."""
import ctypes

import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import BF16_HALF, U, Cache, bits, ref, unbits
from qwen_b200 import _lib

pytestmark = pytest.mark.gpu
L = qwen_b200.lib
KV8, BF16, NO_SEQ = _lib.KV8, _lib.KV_BF16, _lib.NO_SEQ
FORMATS = pytest.mark.parametrize('fmt', [KV8, BF16], ids=['kv8', 'bf16'])
DIMS = pytest.mark.parametrize('dim', [64, 128])
# the weights' rounding before the second product: fp16 (half a step 2^-11) or two bf16 halves at decode, bf16 in prompts
DECODE_W, PREFILL_W = 2.0 ** -11, 2.0 ** -8
FILL = 7.0  # what ctx holds before a call


def u32(a):
    return np.ascontiguousarray(a, np.uint32).view(np.int32)


def workspace(keep, nbytes):
    return keep(np.full(nbytes, 0xA5, np.uint8)), nbytes  # contents do not matter


def padded(a, extra):
    """Rows of a in a buffer with `extra` elements between them: (buffer, stride)."""
    n = a.shape[0]
    buf = np.full((n, a[0].size + extra), np.float32(FILL))
    buf[:, :a[0].size] = a.reshape(n, -1)
    return buf, buf.shape[1]


def decode(c, kv, keep, layer, q, seqs, window=0, sinks=0, scale=None, extra=0, st=None):
    rows, heads, dim = q.shape
    buf, stride = padded(q, extra)
    out = dev(bits(np.full((rows, stride), np.float32(FILL))).view(np.int16))
    ws, n = workspace(keep, L().qwen_b200_paged_decode_workspace(ref(kv), heads, rows))
    rc = L().qwen_b200_op_paged_decode(ref(kv), layer, keep(bits(buf).view(np.int16)), stride, heads, rows,
                                       keep(u32(seqs)) if seqs is not None else None, window, sinks,
                                       dim ** -0.5 if scale is None else scale, vp(out), stride, ws, n, st or stream())
    assert rc == 0
    sync()
    got = unbits(host(out))
    assert (got[:, heads * dim:] == FILL).all(), 'wrote between the rows'
    return got[:, :heads * dim].reshape(q.shape)


def prefill(c, kv, keep, layer, q, seqs, starts, window=0, sinks=0, scale=None, extra=0):
    rows, heads, dim = q.shape
    buf, stride = padded(q, extra)
    out = dev(bits(np.full((rows, stride), np.float32(FILL))).view(np.int16))
    n = len(starts) - 1
    ws, nb = workspace(keep, L().qwen_b200_paged_prefill_workspace(ref(kv), heads, n, rows))
    rc = L().qwen_b200_op_paged_prefill(ref(kv), layer, keep(bits(buf).view(np.int16)), stride, heads, n,
                                        keep(u32(seqs)) if seqs is not None else None, keep(u32(starts)), rows, window,
                                        sinks, dim ** -0.5 if scale is None else scale, vp(out), stride, ws, nb, stream())
    assert rc == 0
    sync()
    got = unbits(host(out))
    assert (got[:, heads * dim:] == FILL).all(), 'wrote between the rows'
    return got[:, :heads * dim].reshape(q.shape)


def assert_within(got, exact, tol, what=''):
    assert np.isfinite(got).all(), what
    off = np.abs(got - exact)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol + 1e-37).all(), f'{what}: at {worst} {got[worst]} for {exact[worst]}, bound {tol[worst]}'


def check_decode(c, kv, keep, q, seqs, window=0, sinks=0, scale=None, layer=0, extra=0):
    got = decode(c, kv, keep, layer, q, seqs, window, sinks, scale, extra)
    s = np.arange(len(q)) if seqs is None else np.asarray(seqs, np.int64)
    pos = [int(c.lengths[i]) - 1 if i < c.seqs else -1 for i in s]
    exact, tol = c.attention(layer, q, s, pos, window, sinks, q.shape[2] ** -0.5 if scale is None else scale, DECODE_W)
    assert_within(got, exact, tol, f'window {window} sinks {sinks}')
    return got


def check_prefill(c, kv, keep, q, seqs, starts, window=0, sinks=0, scale=None, layer=0, extra=0):
    got = prefill(c, kv, keep, layer, q, seqs, starts, window, sinks, scale, extra)
    n = len(starts) - 1
    s = np.arange(n) if seqs is None else np.asarray(seqs, np.int64)
    row_seq, pos = [], []
    for i in range(n):
        count = starts[i + 1] - starts[i]
        length = int(c.lengths[s[i]]) if s[i] < c.seqs else 0
        row_seq += [s[i]] * count
        pos += list(range(length - count, length))
    end = starts[-1]
    exact, tol = c.attention(layer, q[:end], row_seq, pos, window, sinks, q.shape[2] ** -0.5 if scale is None else scale,
                             PREFILL_W)
    assert_within(got[:end], exact, tol, f'window {window} sinks {sinks}')
    assert (got[end:] == FILL).all(), 'wrote rows behind the last sequence'
    return got


def cache(seed, fmt, dim, page, lens, kv_heads=2, layers=1, spare=3, **more):
    pages = sum(-(-n // page) for n in lens) + spare
    return Cache(seed, fmt, kv_heads, dim, page, pages, len(lens), max(1, -(-max(lens) // page)) + 1, layers, **more).give(lens)


# ---------------------------------------------------------------- append
@FORMATS
@DIMS
@pytest.mark.parametrize('page', [16, 256])
@pytest.mark.parametrize('pages_first', [False, True])
def test_append_writes_the_tokens_and_nothing_else(fmt, dim, page, pages_first):
    lens = [40, 1, 0, 300, 17]
    c = cache(dim + page, fmt, dim, page, lens, kv_heads=3, layers=2, pages_first=pages_first)
    keep = Keep()
    c.table[3, 0] = c.pages + 5  # a page that is not there
    kv = c.upload(keep)
    seqs = np.array([0, 3, 1, NO_SEQ, 4, 0, 3, 2, 5, 3, 0], np.uint32)
    pos = np.array([39, 299, 0, 3, 16, 7, 0, 0, 0, 300, 1 << 30], np.uint32)  # 0: no page, 300: beyond the length, ..
    rows = len(seqs)
    k, v = c.rand(rows, 3, dim), c.rand(rows, 3, dim)
    k[2, 1] = 0  # an all-zero row: scale 0
    v[4, 0, :5] = [64.0, -64.0, 32.0, 127.0, -127.0]
    qkv = np.concatenate([c.rand(rows, 1, dim), k, v], 1)
    buf = dev(bits(qkv).view(np.int16))
    base = buf.data_ptr()
    assert L().qwen_b200_op_paged_append(ref(kv), 1, base + 2 * dim, base + 2 * 4 * dim, 7 * dim, rows, keep(u32(seqs)),
                                         keep(u32(pos)), stream()) == 0
    sync()
    for r in range(rows):
        s = seqs[r]
        if s < c.seqs and pos[r] < c.lengths[s] and c.at(s, [pos[r]])[0][0] < c.pages:
            c.write(1, s, [int(pos[r])], k[r:r + 1], v[r:r + 1])
    c.assert_same()


@FORMATS
def test_append_a_prompt(fmt):
    lens = [1000, 257]
    c = cache(5, fmt, 64, 32, lens)
    keep = Keep()
    kv = c.upload(keep)
    seqs = np.repeat([0, 1], [900, 257])
    pos = np.concatenate([np.arange(100, 1000), np.arange(257)])
    k, v = unbits(bits(c.rand(len(seqs), 2, 64) * 3)), c.rand(len(seqs), 2, 64)
    assert L().qwen_b200_op_paged_append(ref(kv), 0, keep(bits(k).view(np.int16)), keep(bits(v).view(np.int16)), 128,
                                         len(seqs), keep(u32(seqs)), keep(u32(pos)), stream()) == 0
    sync()
    for s in (0, 1):
        c.write(0, s, pos[seqs == s], k[seqs == s], v[seqs == s])
    c.assert_same()


# ---------------------------------------------------------------- decode
LENS = [1, 0, 15, 16, 17, 31, 33, 64, 65, 127, 129, 255, 257, 600]


@FORMATS
@DIMS
@pytest.mark.parametrize('page', [16, 32, 64, 128, 256])
def test_decode_lengths_and_pages(fmt, dim, page):
    c = cache(dim + page, fmt, dim, page, LENS)
    keep = Keep()
    kv = c.upload(keep)
    check_decode(c, kv, keep, c.rand(len(LENS), 14, dim) * 2, None)


@FORMATS
@DIMS
@pytest.mark.parametrize('kv_heads,group', [(1, 1), (1, 7), (3, 2), (8, 1), (2, 8), (1, 9), (2, 16), (1, 17), (5, 3)])
def test_decode_head_layouts(fmt, dim, kv_heads, group):
    lens = [100, 0, 33, 515]
    c = cache(kv_heads * group, fmt, dim, 16, lens, kv_heads=kv_heads)
    keep = Keep()
    kv = c.upload(keep)
    check_decode(c, kv, keep, c.rand(4, kv_heads * group, dim), [3, 1, 0, 2], extra=8)


@FORMATS
@DIMS
@pytest.mark.parametrize('window,sinks', [(1, 0), (1, 1), (16, 0), (17, 4), (100, 64), (128, 16), (599, 1), (600, 3),
                                          (1000, 4), (1, 1 << 31), (0xffffffff, 7), (0, 9)])
def test_decode_windows_and_sinks(fmt, dim, window, sinks):
    c = cache(window % 1000 + sinks % 1000, fmt, dim, 32, LENS)
    keep = Keep()
    kv = c.upload(keep)
    check_decode(c, kv, keep, c.rand(len(LENS), 14, dim) * 2, None, window, sinks)


@FORMATS
def test_decode_does_not_read_what_a_window_hides(fmt):
    """Pages outside the window gone (ids out of range) or holding NaN: the result is that of the visible keys alone."""
    lens = [700, 700]
    c = cache(9, fmt, 64, 16, lens)
    for s in range(2):
        hidden = np.arange(4, 600)
        p, t = c.at(s, hidden)
        if fmt == KV8:
            c.ks[0, p, :, t] = np.inf
            c.vs[0, p, :, t] = np.nan
        else:
            c.k[0, p, :, t] = np.nan
            c.v[0, p, :, t] = np.inf
    c.table[1, 1:37] = c.pages + np.arange(36)
    keep = Keep()
    kv = c.upload(keep)
    check_decode(c, kv, keep, c.rand(2, 14, 64), None, window=100, sinks=4)


@FORMATS
@DIMS
def test_decode_long_contexts_split_and_joined(fmt, dim):
    """One sequence alone, and a few of very different lengths: pieces of one row end up on many CTAs."""
    for lens in ([20011], [9000, 3, 0, 1, 12345]):
        c = cache(len(lens), fmt, dim, 64, lens)
        keep = Keep()
        kv = c.upload(keep)
        check_decode(c, kv, keep, c.rand(len(lens), 14, dim), None)
        check_decode(c, kv, keep, c.rand(len(lens), 14, dim), None, window=5001, sinks=70)


@FORMATS
def test_decode_many_rows(fmt):
    r = np.random.default_rng(3)
    lens = [int(x) for x in r.integers(0, 150, 1500)]
    c = cache(4, fmt, 64, 16, lens, kv_heads=1)
    keep = Keep()
    kv = c.upload(keep)
    seqs = r.permutation(1500).astype(np.uint32)
    seqs[::97] = NO_SEQ
    check_decode(c, kv, keep, c.rand(1500, 2, 64), seqs)


@FORMATS
def test_decode_extreme_values(fmt):
    """Scores hundreds apart (one key takes the whole weight), scales over the fp32 range, a negative softmax scale."""
    lens = [200, 77]
    c = cache(11, fmt, 64, 16, lens)
    q = c.rand(2, 14, 64)
    p, t = c.at(0, np.arange(200))
    if fmt == KV8:
        c.ks[0, p, :, t] *= 40
        c.vs[0, p[::2], :, t[::2]] *= np.float32(1e-20)
        p, t = c.at(1, np.arange(77))
        c.vs[0, p, :, t] *= np.float32(1e20)
    else:
        c.k[0, p, :, t] = c.k[0, p, :, t] * 32
        c.v[0, p, :, t] = np.ldexp(c.v[0, p, :, t], 60)
    keep = Keep()
    kv = c.upload(keep)
    check_decode(c, kv, keep, q, None)
    check_decode(c, kv, keep, q, None, scale=-0.7)
    check_decode(c, kv, keep, q * np.float32(2.0 ** -30), None, scale=1.0)
    check_decode(c, kv, keep, q * np.float32(2.0 ** 20), None, scale=2.0 ** -18)
    check_decode(c, kv, keep, q, None, scale=0.0)


@FORMATS
def test_decode_pages_that_are_not_there_and_lengths_beyond_the_table(fmt):
    lens = [130, 64, 90]
    c = cache(12, fmt, 64, 16, lens)
    c.table[0, 2] = c.pages
    c.table[0, 8] = 0xffffffff
    c.table[2, :] = 1 << 30
    c.lengths[1] = 5000000  # cut to the table's max_pages, whose other entries are out of range
    keep = Keep()
    kv = c.upload(keep)
    q = c.rand(3, 14, 64)
    got = decode(c, kv, keep, 0, q, None)
    c.lengths[1] = c.max_pages * c.T
    exact, tol = c.attention(0, q, [0, 1, 2], [129, c.max_pages * c.T - 1, 89], 0, 0, 0.125, DECODE_W)
    assert_within(got, exact, tol)
    assert (got[2] == 0).all()


def test_rows_past_32_bit_offsets():
    """A pool of more than 4 GB: layer 1 of two, whose rows lie beyond 2^32 bytes."""
    torch = torch_cuda()
    lens, dim, page = [150, 70], 64, 64
    c = cache(13, KV8, dim, page, lens)
    keep = Keep()
    kv = c.upload(keep)
    block = c.hkv * page
    far = (1 << 26) + 4096 * 16  # rows: 4 GB of codes
    n = (c.pages - 1) * block + block
    for name in ('k', 'v'):
        big = torch.empty((far + n) * dim, dtype=torch.int8, device='cuda')
        big[far * dim:] = c.dev[name].flatten()
        keep.tensors.append(big)
        setattr(kv, name, big.data_ptr())
    for name, field in (('ks', 'kscales'), ('vs', 'vscales')):
        big = torch.empty(far + n, dtype=torch.float32, device='cuda')
        big[far:] = c.dev[name].flatten()
        keep.tensors.append(big)
        setattr(kv, field, big.data_ptr())
    kv.layers, kv.layer_stride = 2, far
    q = c.rand(2, 14, dim)
    got = decode(c, kv, keep, 1, q, None)
    exact, tol = c.attention(0, q, [0, 1], [149, 69], 0, 0, dim ** -0.5, DECODE_W)
    assert_within(got, exact, tol)
    q = c.rand(40, 14, dim)
    got = prefill(c, kv, keep, 1, q, [0], [0, 40])
    exact, tol = c.attention(0, q, [0] * 40, range(110, 150), 0, 0, dim ** -0.5, PREFILL_W)
    assert_within(got, exact, tol)


@FORMATS
@DIMS
@pytest.mark.parametrize('keys', [513, 1025, 1537, 2600, 3600, 4097, 4700, 6200, 7700, 8200])
def test_decode_clusters_of_every_size(fmt, dim, keys):
    """One row and KV head: the table's width lets 2 to 16 CTAs share it, some of them without a key."""
    c = cache(keys, fmt, dim, 64, [keys, 70], kv_heads=1)
    keep = Keep()
    kv = c.upload(keep)
    check_decode(c, kv, keep, c.rand(2, 7, dim), None)
    check_decode(c, kv, keep, c.rand(1, 3, dim), [1])
    check_decode(c, kv, keep, c.rand(1, 3, dim), [0], window=keys - 500, sinks=33)


def steep(c, s, q_dir, slope):
    """Keys of sequence s along one direction: token t scores slope[t] (before the softmax scale) with q_dir."""
    n = int(c.lengths[s])
    k = np.repeat((slope[:n, None] * q_dir / np.dot(q_dir, q_dir))[:, None], c.hkv, 1)
    c.write(0, s, np.arange(n), unbits(bits(k.astype(np.float32))), c.rand(n, c.hkv, c.dim))


@FORMATS
@DIMS
@pytest.mark.parametrize('shape', ['rising', 'falling', 'low', 'jumps', 'late'])
def test_scores_far_from_each_other(fmt, dim, shape):
    """The reference of the softmax has to move, up to hundreds of powers of two at a time, and the sums so far with it."""
    n = 700
    c = cache(ord(shape[0]), fmt, dim, 32, [n, 300])
    r = np.random.default_rng(2)
    slope = {'rising': np.linspace(-400, 400, n), 'falling': np.linspace(400, -400, n), 'low': -500 + r.standard_normal(n),
             'jumps': 300 * r.standard_normal(n), 'late': np.where(np.arange(n) < 650, -200.0, 90.0)}[shape]
    u = np.ones(dim)
    for s in range(2):
        steep(c, s, u, slope)
    keep = Keep()
    kv = c.upload(keep)
    # scores are slope * scale * the query's factor, which differs by row and head
    q = unbits(bits((u * r.uniform(0.2, 1.5, (2, 14, 1))).astype(np.float32)))
    check_decode(c, kv, keep, q, None, scale=1.0)
    p = unbits(bits((u * r.uniform(0.2, 1.5, (500, 14, 1))).astype(np.float32)))
    check_prefill(c, kv, keep, p, None, [0, 400, 500], scale=1.0)
    check_prefill(c, kv, keep, p, None, [0, 400, 500], 200, 5, scale=1.0)


@FORMATS
@DIMS
@pytest.mark.parametrize('log', [20, 27, 34, 66])
@pytest.mark.parametrize('sign', [1, -1])
def test_equal_scores_of_any_size_weigh_the_same(fmt, dim, log, sign):
    """All keys are alike, so every score of a row is the same number, of a size whose fp32 steps pass 1 by far: the
    result is the mean of the visible values.

    Tolerance: a weight is 1 (times the value's scale) rounded by half a step of its type at most, W; the sum of n
    products and n weights in fp32 errs by n U each; the result is rounded to bf16."""
    n = 300
    c = cache(log, fmt, dim, 32, [n, n])
    k = np.full((n, c.hkv, dim), 1.34375, np.float32)
    v = c.rand(n, c.hkv, dim)
    for s in range(2):
        c.write(0, s, np.arange(n), k, v)
    keep = Keep()
    kv = c.upload(keep)
    heads = 7 * c.hkv
    # scores of log2 size `log` or a little above, and no power of two
    q = unbits(bits((sign * 2.0 ** log / dim * np.linspace(1, 1.9, heads)[:, None] * np.ones(dim)).astype(np.float32)))
    values = c.read(0, 0, np.arange(n))[1].astype(np.float64).repeat(7, axis=1)
    count = np.arange(1, n + 1)[:, None, None]
    mean, size = values.cumsum(0) / count, abs(values).cumsum(0) / count

    def check(got, at, w):
        bound = (2 * w + 4 * n * U) * size[at]
        bound = bound + BF16_HALF * (abs(mean[at]) + bound)
        assert (abs(got - mean[at]) <= bound).all()

    check(decode(c, kv, keep, 0, np.stack([q, q]), None, scale=1.0), [n - 1, n - 1], DECODE_W)
    got = prefill(c, kv, keep, 0, np.stack([q] * (n + 20)), None, [0, n, n + 20], scale=1.0)
    check(got, list(range(n)) + list(range(n - 20, n)), PREFILL_W)


# ---------------------------------------------------------------- prefill
def runs(c, rows):
    return np.concatenate([[0], np.cumsum(rows)]).tolist()


@FORMATS
@DIMS
@pytest.mark.parametrize('page', [16, 64, 256])
def test_prefill_ragged_prompts(fmt, dim, page):
    lens = [1, 0, 130, 129, 40, 300, 17]
    rows = [1, 0, 130, 1, 39, 57, 16]
    c = cache(dim + page, fmt, dim, page, lens)
    keep = Keep()
    kv = c.upload(keep)
    starts = runs(c, rows)
    check_prefill(c, kv, keep, c.rand(starts[-1] + 5, 14, dim) * 2, None, starts)


@FORMATS
@DIMS
@pytest.mark.parametrize('kv_heads,group', [(1, 1), (3, 2), (8, 1), (2, 8), (1, 9), (1, 33), (5, 3)])
def test_prefill_head_layouts(fmt, dim, kv_heads, group):
    lens, rows = [140, 33, 70], [140, 2, 50]
    c = cache(kv_heads * group, fmt, dim, 32, lens, kv_heads=kv_heads)
    keep = Keep()
    kv = c.upload(keep)
    starts = runs(c, [rows[i] for i in (2, 0, 1)])
    check_prefill(c, kv, keep, c.rand(starts[-1], kv_heads * group, dim), [2, 0, 1], starts, extra=16)


@FORMATS
@DIMS
@pytest.mark.parametrize('window,sinks', [(1, 0), (1, 2), (16, 0), (100, 4), (128, 130), (257, 1), (500, 64), (700, 5),
                                          (1, 1 << 31), (0xffffffff, 7), (0, 9)])
def test_prefill_windows_and_sinks(fmt, dim, window, sinks):
    lens, rows = [600, 333], [450, 333]
    c = cache(window % 1000 + sinks % 1000, fmt, dim, 64, lens)
    keep = Keep()
    kv = c.upload(keep)
    check_prefill(c, kv, keep, c.rand(783, 4, dim) * 2, None, runs(c, rows), window, sinks)


@FORMATS
@DIMS
def test_prefill_short_chunks_of_long_contexts(fmt, dim):
    """Few rows over many keys: the keys of a tile are split and joined."""
    lens, rows = [9001, 5, 7777], [16, 5, 1]
    c = cache(2, fmt, dim, 128, lens)
    keep = Keep()
    kv = c.upload(keep)
    check_prefill(c, kv, keep, c.rand(22, 14, dim), None, runs(c, rows))
    check_prefill(c, kv, keep, c.rand(22, 14, dim), None, runs(c, rows), window=4000, sinks=300)


@FORMATS
def test_prefill_does_not_read_what_no_row_sees(fmt):
    lens, rows = [900, 900], [40, 300]
    c = cache(21, fmt, 64, 16, lens)
    for s in range(2):
        hidden = np.arange(4, 900 - rows[s] - 99)  # with a window of 100
        p, t = c.at(s, hidden)
        if fmt == KV8:
            c.ks[0, p, :, t] = np.inf
            c.vs[0, p, :, t] = np.nan
        else:
            c.k[0, p, :, t] = np.nan
            c.v[0, p, :, t] = np.inf
    c.table[0, 1:(900 - 139) // 16] = c.pages + 7
    keep = Keep()
    kv = c.upload(keep)
    check_prefill(c, kv, keep, c.rand(340, 14, 64), None, runs(c, rows), window=100, sinks=4)


@FORMATS
def test_prefill_more_rows_than_tokens_no_sequence_and_missing_pages(fmt):
    lens = [20, 300, 64]
    c = cache(22, fmt, 64, 16, lens)
    c.table[1, 3] = c.pages
    c.table[1, 18] = 0xffffffff
    keep = Keep()
    kv = c.upload(keep)
    check_prefill(c, kv, keep, c.rand(150, 14, 64), [0, NO_SEQ, 1, 2], [0, 33, 40, 140, 144])


@FORMATS
def test_prefill_starts_that_do_not_fit_the_buffer(fmt):
    """starts beyond `rows` or decreasing: nothing outside the q and ctx rows is touched."""
    c = cache(23, fmt, 64, 16, [64, 64, 64])
    keep = Keep()
    kv = c.upload(keep)
    q = c.rand(30, 14, 64)
    prefill(c, kv, keep, 0, q, None, [0, 20, 10, 1000])
    prefill(c, kv, keep, 0, q, None, [40, 50, 60, 4000000000])


@FORMATS
def test_prefill_extreme_values(fmt):
    lens = [200, 77]
    c = cache(24, fmt, 64, 16, lens)
    q = c.rand(277, 14, 64)
    p, t = c.at(0, np.arange(200))
    if fmt == KV8:
        c.ks[0, p, :, t] *= 40
        c.vs[0, p[::2], :, t[::2]] *= np.float32(1e-20)
    else:
        c.k[0, p, :, t] = c.k[0, p, :, t] * 32
        c.v[0, p, :, t] = np.ldexp(c.v[0, p, :, t], 60)
    keep = Keep()
    kv = c.upload(keep)
    for scale, f in ((0.125, 1), (-0.7, 1), (1.0, 2.0 ** -30), (2.0 ** -18, 2.0 ** 20), (0.0, 1)):
        check_prefill(c, kv, keep, q * np.float32(f), None, [0, 200, 277], scale=scale)


@FORMATS
def test_a_decode_row_equals_a_prompt_of_one_row(fmt):
    lens = [333, 1, 128]
    c = cache(25, fmt, 64, 64, lens)
    keep = Keep()
    kv = c.upload(keep)
    q = c.rand(3, 14, 64)
    check_decode(c, kv, keep, q, None, 90, 3)
    check_prefill(c, kv, keep, q, None, [0, 1, 2, 3], 90, 3)


@DIMS
@pytest.mark.parametrize('bad', [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize('what', ['ks', 'vs'])
def test_prefill_rows_before_a_broken_scale_do_not_see_it(dim, bad, what):
    """KV8: a key's or value's scale that is no number reaches the rows that see the token, and no other."""
    n, at = 300, 170
    c = cache(88, KV8, dim, 64, [n])
    q = c.rand(n, 14, dim)
    exact, tol = c.attention(0, q, [0] * n, range(n), 60, 3, dim ** -0.5, PREFILL_W)
    p, t = c.at(0, at)
    getattr(c, what)[0, p, :, t] = bad
    keep = Keep()
    kv = c.upload(keep)
    got = prefill(c, kv, keep, 0, q, None, [0, n], 60, 3)
    sees = (np.arange(n) >= at) & (np.arange(n) - at < 60)
    assert_within(got[~sees], exact[~sees], tol[~sees])
    if what == 'vs':
        assert not np.isfinite(got[sees]).any()


@FORMATS
@DIMS
@pytest.mark.parametrize('n', [1, 3, 26])
def test_prefill_tiles_in_several_pieces(fmt, dim, n):
    """Chunks of a few rows over hundreds of keys: every tile is split over CTAs, for few tiles and for many."""
    lens = [1500 - 370 * (i % 4) + i for i in range(n)]
    rows = [9 - i % 3 for i in range(n)]
    c = cache(60 + n, fmt, dim, 64, lens)
    keep = Keep()
    kv = c.upload(keep)
    check_prefill(c, kv, keep, c.rand(sum(rows), 14, dim) * 2, None, runs(c, rows))


@FORMATS
@DIMS
def test_prefill_of_many_tiles(fmt, dim):
    """More tiles than CTAs, so that a CTA walks several segments; against 64 bits on the GPU, with the host's bound."""
    torch = torch_cuda()
    lens, rows, heads, hkv, window, sinks = [2500, 1800], [2500, 900], 32, 8, 700, 130
    c = cache(77, fmt, dim, 64, lens, kv_heads=hkv)
    keep = Keep()
    kv = c.upload(keep)
    starts = runs(c, rows)
    q = c.rand(starts[-1], heads, dim) * 2
    got = prefill(c, kv, keep, 0, q, None, starts, window, sinks)
    scale = dim ** -0.5
    for i in range(2):
        k, v = (torch.from_numpy(x).cuda() for x in c.read(0, i, np.arange(lens[i])))
        pos = torch.arange(lens[i] - rows[i], lens[i], device='cuda')[:, None]
        t = torch.arange(lens[i], device='cuda')[None]
        seen = (t <= pos) & ((pos - t < window) | (t < sinks))
        qi = torch.from_numpy(q[starts[i]:starts[i + 1]].astype(np.float64)).cuda()
        for h in range(heads):
            kh, vh = k[:, h // (heads // hkv)], v[:, h // (heads // hkv)]
            x = (qi[:, h] @ kh.T * scale).masked_fill(~seen, -np.inf)
            mag = (qi[:, h].abs() @ kh.abs().T * scale).masked_fill(~seen, 0).amax(1)
            w = torch.softmax(x, 1)
            out = w @ vh
            size = w @ vh.abs() + out.abs()
            e = PREFILL_W + 2 * (dim + 4) * U * mag + 2.0 ** -21 + 2 * lens[i] * U
            tol = BF16_HALF * (out.abs() + e[:, None] * size) + e[:, None] * size
            assert_within(got[starts[i]:starts[i + 1], h], out.cpu().numpy(), tol.cpu().numpy(), f'sequence {i} head {h}')


@FORMATS
@DIMS
def test_prefill_waits_do_not_expire(fmt, dim):
    """The workspace's first word stays zero; two calls on two streams, a workspace each, at the same time."""
    torch = torch_cuda()
    lens = [900, 300, 5]
    c = cache(78, fmt, dim, 16, lens)
    keep = Keep()
    kv = c.upload(keep)
    starts = [0, 500, 800, 805]
    q = c.rand(805, 14, dim)
    want = prefill(c, kv, keep, 0, q, None, starts)
    qd, sd = keep(bits(q).view(np.int16)), keep(u32(starts))
    n = L().qwen_b200_paged_prefill_workspace(ref(kv), 14, 3, 805)
    ws = [torch.zeros(n, dtype=torch.uint8, device='cuda') for _ in range(2)]
    out = [dev(np.zeros((805, 14, dim), np.int16)) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    sync()
    for _ in range(5):
        for w, o, st in zip(ws, out, streams):
            assert L().qwen_b200_op_paged_prefill(ref(kv), 0, qd, 14 * dim, 14, 3, None, sd, 805, 0, 0, dim ** -0.5, vp(o),
                                                  14 * dim, vp(w), n, st.cuda_stream) == 0
    sync()
    for w, o in zip(ws, out):
        assert int(host(w)[:4].view(np.uint32)[0]) == 0, 'a bounded wait expired'
        assert np.array_equal(unbits(host(o)), want)


# ---------------------------------------------------------------- pages
class Book:
    """Page management in plain Python over a Cache's arrays."""

    def __init__(self, c):
        self.c = c

    def held(self, n):
        return -(-int(n) // self.c.T)

    def spare(self):
        return [int(p) for p in np.nonzero(self.c.refs == 0)[0]]

    def status(self, code):
        return [code, int((self.c.refs == 0).sum())]

    def reserve(self, seqs, tokens):
        c = self.c
        cap = c.max_pages * c.T
        if len(set(seqs)) < len(seqs) or any(s >= c.seqs for s in seqs):
            return self.status(_lib.PAGES_BAD)
        if any(int(c.lengths[s]) + t > cap for s, t in zip(seqs, tokens)):
            return self.status(_lib.PAGES_BAD)
        need = [self.held(int(c.lengths[s]) + t) - self.held(c.lengths[s]) for s, t in zip(seqs, tokens)]
        spare = self.spare()
        if sum(need) > len(spare):
            return self.status(_lib.PAGES_FULL)
        for s, t, n in zip(seqs, tokens, need):
            h = self.held(c.lengths[s])
            for j in range(n):
                p = spare.pop(0)
                c.table[s, h + j], c.refs[p] = p, 1
            c.lengths[s] += t
        return self.status(_lib.PAGES_OK)

    def fork(self, parents, children, prefix):
        c = self.c
        if len(set(children)) < len(children) or any(x >= c.seqs for x in list(parents) + list(children)):
            return self.status(_lib.PAGES_BAD)
        if any(c.lengths[x] for x in children) or any(t > c.lengths[p] for p, t in zip(parents, prefix)):
            return self.status(_lib.PAGES_BAD)
        spare = self.spare()
        if sum(t % c.T > 0 for t in prefix) > len(spare):
            return self.status(_lib.PAGES_FULL)
        for p, x, t in zip(parents, children, prefix):
            full = t // c.T
            c.table[x, :full] = c.table[p, :full]
            np.add.at(c.refs, c.table[p, :full], 1)
            if t % c.T:
                f, src = spare.pop(0), c.table[p, full]
                c.table[x, full], c.refs[f] = f, 1
                self.copy_tokens(src, f, t % c.T)
            c.lengths[x] = t
        return self.status(_lib.PAGES_OK)

    def copy_tokens(self, src, dst, n):
        c = self.c
        for a in (c.k, c.v, c.ks, c.vs):
            if a is not None:
                a[:, dst, :, :n] = a[:, src, :, :n]

    def free(self, seqs):
        c = self.c
        if len(set(seqs)) < len(seqs) or any(s >= c.seqs for s in seqs):
            return self.status(_lib.PAGES_BAD)
        for s in seqs:
            np.subtract.at(c.refs, c.table[s, :self.held(c.lengths[s])], 1)
            c.lengths[s] = 0
        return self.status(_lib.PAGES_OK)

    def compact(self):
        c = self.c
        n = int((c.refs > 0).sum())
        holes = [p for p in range(n) if not c.refs[p]]
        movers = [p for p in range(n, c.pages) if c.refs[p]]
        to = dict(zip(movers, holes))
        for src, dst in to.items():
            self.copy_tokens(src, dst, c.T)
            c.refs[dst], c.refs[src] = c.refs[src], 0
        for s in range(c.seqs):
            for j in range(self.held(c.lengths[s])):
                c.table[s, j] = to.get(int(c.table[s, j]), c.table[s, j])
        return self.status(_lib.PAGES_OK)


class DevicePages:
    def __init__(self, c, kv, keep):
        self.kv, self.keep, self.c = kv, keep, c
        self.ws, self.n = workspace(keep, L().qwen_b200_pages_workspace(ref(kv)))
        self.status = dev(u32([9, 9]))

    def __call__(self, name, *lists):
        fn = getattr(L(), f'qwen_b200_op_pages_{name}')
        args = [self.keep(u32(x)) for x in lists]
        count = [len(lists[0])] if lists else []
        assert fn(ref(self.kv), *args, *count, vp(self.status), self.ws, self.n, stream()) == 0
        sync()
        return host(self.status).view(np.uint32).tolist()


@FORMATS
@pytest.mark.parametrize('page,dim,layers,pages_first', [(16, 64, 3, False), (64, 128, 1, False), (256, 64, 2, True),
                                                         (32, 128, 4, True)])
def test_page_management_against_a_plain_one(fmt, page, dim, layers, pages_first):
    """Random calls, among them ones that are refused on the device, against lists in Python."""
    r = np.random.default_rng(page + dim)
    c = Cache(7, fmt, 3, dim, page, 90, 24, 12, layers, pages_first=pages_first)
    c.give([page * 3 + 1, page, 5, page * 6, 0, 1] + [0] * 18)
    keep = Keep()
    d, b = DevicePages(c, c.upload(keep), keep), Book(c)
    for step in range(60):
        live, empty = np.nonzero(c.lengths)[0], np.nonzero(c.lengths == 0)[0]
        what = r.choice(['reserve', 'reserve', 'fork', 'fork', 'free', 'compact', 'bad'])
        if what == 'reserve':
            s = r.choice(24, r.integers(1, 6), replace=False)
            t = [int(min(r.integers(0, 4 * page), 12 * page - c.lengths[x])) for x in s]
            args = (s.tolist(), t)
        elif what == 'fork' and len(live) and len(empty):
            x = r.choice(empty, r.integers(1, min(4, len(empty)) + 1), replace=False)
            p = r.choice(live, len(x))
            args = (p.tolist(), x.tolist(), [int(r.integers(0, c.lengths[i] + 1)) for i in p])
        elif what == 'free' and len(live):
            args = (r.choice(live, r.integers(1, min(4, len(live)) + 1), replace=False).tolist(),)
        elif what == 'compact':
            args = ()
        else:
            what, args = [('reserve', ([0, 0], [1, 1])), ('reserve', ([24], [1])), ('reserve', ([1], [12 * page + 1])),
                          ('reserve', ([2], [0xffffffff])), ('free', ([3, 3],)), ('free', ([NO_SEQ],)),
                          ('fork', ([0], [24], [0])), ('fork', ([24], [1], [0])),
                          ('fork', ([0, 0], [empty[0]] * 2, [0, 0]) if len(empty) else ([0], [0], [1])),
                          ('fork', ([0], [0], [0]) if c.lengths[0] else ([0], [0], [1]))][r.integers(10)]
        got = d(what, *args)
        want = getattr(b, what)(*args)
        assert got == want, (step, what, args)
        c.assert_same()
    for what, args in (('free', (list(range(24)),)), ('reserve', (list(range(8)), [12 * page] * 8)),  # 96 pages of 90
                       ('reserve', (list(range(7)), [12 * page - 1] * 7)), ('fork', ([0] * 7, list(range(7, 14)), [1] * 7)),
                       ('fork', ([0] * 6, list(range(7, 13)), [1] * 6)), ('reserve', ([6, 7], [1, page]))):
        got = d(what, *args)
        assert got == getattr(b, what)(*args)
        assert (got[0] == _lib.PAGES_FULL) == (what == 'reserve' and len(args[0]) in (8, 2) or len(args[0]) == 7
                                               and what == 'fork'), (what, args)
        c.assert_same()


def test_large_reserve_and_compact_of_many_pages():
    """More pages and sequences than one pass of the planning CTA takes."""
    c = Cache(8, BF16, 1, 64, 16, 9001, 3000, 200)
    c.k[:], c.v[:] = 0, 0
    keep = Keep()
    d, b = DevicePages(c, c.upload(keep), keep), Book(c)
    r = np.random.default_rng(1)
    steps = [('reserve', (list(range(2999, -1, -1)), r.integers(0, 60, 3000).tolist())), ('reserve', ([5], [2500])),
             ('free', (r.permutation(3000)[:2000].tolist(),)), ('compact', ()), ('compact', ())]
    for what, args in steps:
        assert d(what, *args) == getattr(b, what)(*args)
        c.assert_same()


@FORMATS
def test_copy_of_whole_pages(fmt):
    c = cache(31, fmt, 128, 32, [200, 100], kv_heads=5, layers=3)
    keep = Keep()
    kv = c.upload(keep)
    src, dst = [0, 0, 3, c.pages, 4], [5, 6, 7, 8, 0xffffffff]
    assert L().qwen_b200_op_pages_copy(ref(kv), keep(u32(src)), keep(u32(dst)), 5, stream()) == 0
    sync()
    for a, b in ((0, 5), (0, 6), (3, 7)):
        Book(c).copy_tokens(a, b, c.T)
    c.assert_same()


# ---------------------------------------------------------------- together
@FORMATS
def test_a_server_step_by_step(fmt):
    """Prompts reserved, appended and attended to, samples forked off them, decode steps, sequences freed, the pool
    compacted, and decoding on: each result against the cache as it should be by then, in both layers."""
    r = np.random.default_rng(6)
    c = Cache(6, fmt, 2, 64, 16, 64, 8, 20, layers=2)
    keep = Keep()
    kv = c.upload(keep)
    d, b = DevicePages(c, kv, keep), Book(c)

    def both(what, *args):
        assert d(what, *args) == getattr(b, what)(*args)

    def add(seqs, counts):
        """The last counts[i] tokens of each sequence get keys and values in both layers."""
        row_seq = np.repeat(seqs, counts)
        pos = np.concatenate([np.arange(int(c.lengths[s]) - n, int(c.lengths[s])) for s, n in zip(seqs, counts)])
        for layer in range(2):
            k, v = c.rand(len(pos), 2, 64), c.rand(len(pos), 2, 64)
            assert L().qwen_b200_op_paged_append(ref(kv), layer, keep(bits(k).view(np.int16)),
                                                 keep(bits(v).view(np.int16)), 128, len(pos), keep(u32(row_seq)),
                                                 keep(u32(pos)), stream()) == 0
            for s, x, y, z in zip(row_seq, pos, k, v):
                c.write(layer, s, [int(x)], y[None], z[None])
        sync()

    both('reserve', [1, 4], [100, 37])
    add([1, 4], [100, 37])
    for layer in range(2):
        check_prefill(c, kv, keep, c.rand(137, 14, 64), [1, 4], [0, 100, 137], 50, 4, layer=layer)
    both('fork', [1, 1, 4], [0, 2, 6], [100, 64, 37])
    for step in range(5):
        seqs = [0, 1, 2, 4, 6]
        both('reserve', seqs, [1] * 5)
        add(seqs, [1] * 5)
        check_decode(c, kv, keep, c.rand(6, 14, 64), seqs + [7], layer=step % 2)
    both('free', [1, 4])
    both('compact')
    for layer in range(2):
        check_decode(c, kv, keep, c.rand(3, 14, 64), [6, 2, 0], 40, 2, layer=layer)
    both('reserve', [1, 0], [30, 9])
    add([1, 0], [30, 9])
    check_prefill(c, kv, keep, c.rand(39, 14, 64), [1, 0], [0, 30, 39])
    c.assert_same()


@FORMATS
def test_a_captured_step_follows_the_tables(fmt):
    """A CUDA graph of reserve, append, decode and prefill, replayed on another stream while lengths, tables and inputs
    change in place: two graphs share one workspace."""
    torch = torch_cuda()
    c = Cache(16, fmt, 2, 64, 16, 40, 3, 10)
    c.give([20, 100, 0])
    keep = Keep()
    kv = c.upload(keep)
    d, b = DevicePages(c, kv, keep), Book(c)
    k, v, q = (dev(np.zeros((3, n, 64), np.int16)) for n in (2, 2, 14))
    pos, seqs, one, starts = dev(u32([0, 0, 0])), dev(u32([0, 1, 2])), dev(u32([1, 1, 1])), dev(u32([0, 1, 2, 3]))
    out = [dev(np.zeros((3, 14, 64), np.int16)) for _ in range(2)]
    n = max(L().qwen_b200_paged_decode_workspace(ref(kv), 14, 3), L().qwen_b200_paged_prefill_workspace(ref(kv), 14, 3, 3))
    ws, _ = workspace(keep, n)
    side = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]

    def step(which):
        st = torch.cuda.current_stream().cuda_stream
        if which == 0:
            assert L().qwen_b200_op_pages_reserve(ref(kv), vp(seqs), vp(one), 3, vp(d.status), d.ws, d.n, st) == 0
            assert L().qwen_b200_op_paged_append(ref(kv), 0, vp(k), vp(v), 128, 3, vp(seqs), vp(pos), st) == 0
            assert L().qwen_b200_op_paged_decode(ref(kv), 0, vp(q), 896, 14, 3, vp(seqs), 60, 2, 0.125, vp(out[0]), 896, ws,
                                                 n, st) == 0
        else:
            assert L().qwen_b200_op_paged_prefill(ref(kv), 0, vp(q), 896, 14, 3, vp(seqs), vp(starts), 3, 60, 2, 0.125,
                                                  vp(out[1]), 896, ws, n, st) == 0

    sync()
    for which, g in enumerate(graphs):
        with torch.cuda.graph(g, stream=side):
            step(which)
    for _ in range(20):
        at = c.lengths.copy()
        nk, nv, nq = c.rand(3, 2, 64), c.rand(3, 2, 64), c.rand(3, 14, 64)
        for t, x in ((k, nk), (v, nv), (q, nq)):
            t.copy_(torch.from_numpy(bits(x).view(np.int16)))
        pos.copy_(torch.from_numpy(u32(at)))
        sync()
        with torch.cuda.stream(side):
            graphs[0].replay()
            graphs[1].replay()
        sync()
        want = b.reserve([0, 1, 2], [1, 1, 1])
        assert host(d.status).view(np.uint32).tolist() == want
        for s in range(3):
            c.write(0, s, [int(at[s])], nk[s:s + 1], nv[s:s + 1])
        for got, w in zip(out, (DECODE_W, PREFILL_W)):
            exact, tol = c.attention(0, nq, [0, 1, 2], [int(x) - 1 for x in c.lengths], 60, 2, 0.125, w)
            assert_within(unbits(host(got)), exact, tol)
    c.assert_same()


@FORMATS
def test_same_inputs_same_bits(fmt):
    lens = [3000, 10, 777, 0, 4096]
    c = cache(41, fmt, 128, 64, lens)
    keep = Keep()
    kv = c.upload(keep)
    q = c.rand(5, 8, 128)
    first = decode(c, kv, keep, 0, q, None)
    p = c.rand(300, 8, 128)
    pfirst = prefill(c, kv, keep, 0, p, [2, 0], [0, 200, 300])
    for _ in range(3):
        assert np.array_equal(first, decode(c, kv, keep, 0, q, None))
        assert np.array_equal(pfirst, prefill(c, kv, keep, 0, p, [2, 0], [0, 200, 300]))


def test_host_memory_is_refused():
    """A host pointer in any place of a call that the host can look at."""
    c = cache(43, KV8, 64, 64, [300])
    keep = Keep()
    kv = c.upload(keep)
    q, i = keep(np.zeros((4, 896), np.int16)), keep(u32([0, 4]))
    bad = (ctypes.c_uint8 * 8192)()
    at = ctypes.c_void_p((ctypes.addressof(bad) + 255) & ~255)
    ws, n = workspace(keep, L().qwen_b200_paged_prefill_workspace(ref(kv), 14, 1, 4))
    for x in range(4):
        a, b, w, s = (at if x == y else z for y, z in enumerate((q, q, ws, i)))
        assert L().qwen_b200_op_paged_decode(ref(kv), 0, a, 896, 14, 1, s, 0, 0, 0.125, b, 896, w, n, stream()) == _lib.EINVAL
        assert L().qwen_b200_op_paged_prefill(ref(kv), 0, a, 896, 14, 1, None, s, 4, 0, 0, 0.125, b, 896, w, n,
                                              stream()) == _lib.EINVAL
        assert L().qwen_b200_op_paged_append(ref(kv), 0, a, b, 896, 1, s if x != 2 else at, i, stream()) == _lib.EINVAL


def test_a_workspace_too_small_is_refused():
    c = cache(42, KV8, 64, 64, [300])
    keep = Keep()
    kv = c.upload(keep)
    q = keep(np.zeros((4, 896), np.int16))
    n = L().qwen_b200_paged_decode_workspace(ref(kv), 14, 1)
    assert L().qwen_b200_op_paged_decode(ref(kv), 0, q, 896, 14, 1, None, 0, 0, 0.125, q, 896, keep(np.zeros(16, np.uint8)),
                                         n - 1, stream()) == _lib.EINVAL
    n = L().qwen_b200_paged_prefill_workspace(ref(kv), 14, 1, 4)
    assert L().qwen_b200_op_paged_prefill(ref(kv), 0, q, 896, 14, 1, None, keep(u32([0, 4])), 4, 0, 0, 0.125, q, 896,
                                          keep(np.zeros(16, np.uint8)), n - 1, stream()) == _lib.EINVAL


@pytest.mark.parametrize('field', ['k', 'v', 'kscales', 'vscales', 'table', 'lengths', 'refs'])
def test_a_cache_in_host_memory_is_refused(field):
    c = cache(44, KV8, 64, 64, [300])
    keep = Keep()
    kv = c.upload(keep)
    bad = (ctypes.c_uint8 * 8192)()
    setattr(kv, field, (ctypes.addressof(bad) + 255) & ~255)
    x, i = keep(np.zeros((4, 896), np.int16)), keep(u32([0, 4]))
    ws, n = keep(np.zeros(1 << 22, np.uint8)), 1 << 22
    if field != 'refs':
        assert L().qwen_b200_op_paged_decode(ref(kv), 0, x, 896, 14, 1, None, 0, 0, 0.125, x, 896, ws, n, stream()) == _lib.EINVAL
        assert L().qwen_b200_op_paged_append(ref(kv), 0, x, x, 896, 1, i, i, stream()) == _lib.EINVAL
    assert L().qwen_b200_op_pages_free(ref(kv), i, 1, i, ws, n, stream()) == _lib.EINVAL
    assert L().qwen_b200_op_pages_compact(ref(kv), i, ws, n, stream()) == _lib.EINVAL


def test_lists_in_host_memory_are_refused():
    c = cache(45, KV8, 64, 64, [300, 20])
    keep = Keep()
    kv = c.upload(keep)
    bad = (ctypes.c_uint8 * 8192)()
    at = (ctypes.addressof(bad) + 255) & ~255
    i, ws, n, st = keep(u32([0, 4])), keep(np.zeros(1 << 16, np.uint8)), 1 << 16, keep(u32([0, 0]))
    for x in range(3):
        a, b, d = (at if x == y else i for y in range(3))
        assert L().qwen_b200_op_pages_fork(ref(kv), a, b, d, 1, st, ws, n, stream()) == _lib.EINVAL
        if x < 2:
            assert L().qwen_b200_op_pages_reserve(ref(kv), a, b, 1, st, ws, n, stream()) == _lib.EINVAL
            assert L().qwen_b200_op_pages_copy(ref(kv), a, b, 1, stream()) == _lib.EINVAL
    assert L().qwen_b200_op_pages_free(ref(kv), at, 1, st, ws, n, stream()) == _lib.EINVAL
