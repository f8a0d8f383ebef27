"""Page management of the paged KV cache where sizes, tables and counts are at
their worst: requests beyond any pool, and caches whose tables, lengths and
reference counts do not belong together. A call that is refused changes
nothing but its status."""
import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import Cache, ref
from qwen_b200 import _lib
from test_gpu_paged import Book, DevicePages, u32, workspace

pytestmark = pytest.mark.gpu
L = qwen_b200.lib


@pytest.mark.parametrize('more', [0, 16, 64], ids=lambda n: f'and {n} tokens')
def test_a_request_of_more_than_32_bits_of_pages_is_full(more):
    """64 sequences that ask for 2^26 pages each want 2^32 of them, a 65th some more: in 32 bits that is 0 pages and the
    few of the 65th, of which the pool has enough. (Nothing reads the 16 GB of tables: no sequence holds a page.)"""
    torch = torch_cuda()
    seqs, pages, page = 65, 8, 16
    keep = Keep()
    pool = keep(np.zeros((2, pages, 1, page, 64), np.int16))
    table = torch.empty(seqs << 26, dtype=torch.int32, device='cuda')
    lengths, refs, status = dev(u32(np.zeros(seqs))), dev(u32(np.zeros(pages))), dev(u32([9, 9]))
    kv = qwen_b200.PagedKV(k=pool.value, v=pool.value + pages * page * 128, table=table.data_ptr(),
                           lengths=lengths.data_ptr(), refs=refs.data_ptr(), layer_stride=pages * page, page_stride=page,
                           format=_lib.KV_BF16, layers=1, pages=pages, kv_heads=1, page_tokens=page, head_dim=64, seqs=seqs,
                           max_pages=1 << 26)
    ws, n = workspace(keep, L().qwen_b200_pages_workspace(ref(kv)))
    tokens = [1 << 30] * 64 + [more]
    assert L().qwen_b200_op_pages_reserve(ref(kv), keep(u32(np.arange(seqs))), keep(u32(tokens)), seqs if more else 64,
                                          vp(status), ws, n, stream()) == 0
    sync()
    assert host(status).tolist() == [_lib.PAGES_FULL, pages]
    assert not host(lengths).any() and not host(refs).any()


FORMATS = pytest.mark.parametrize('fmt', [_lib.KV8, _lib.KV_BF16], ids=['kv8', 'bf16'])


def broken_caches(c):
    """(what, the arrays changed) of caches whose tables, lengths and counts do not belong together, one at a time; c is
    put back after each."""
    last = c.seqs - 1
    n = -(-int(c.lengths[last]) // c.T)
    for what, array, at, value in (('a length beyond the table', c.lengths, 2, c.max_pages * c.T + 1),
                                   ('the largest length', c.lengths, last, 0xffffffff),
                                   ('a page id behind the pool', c.table, (1, 1), c.pages),
                                   ('an id of no page', c.table, (last, n - 1), 0xffffffff),
                                   ('a held page that counts as free', c.refs, int(c.table[last, n - 1]), 0)):
        was = array[at].copy()
        array[at] = value
        yield what
        array[at] = was


@FORMATS
@pytest.mark.parametrize('seqs', [3, 70, 1100])
def test_compaction_of_a_broken_cache_is_refused(fmt, seqs):
    lens = [40 + (7 * i) % 60 for i in range(seqs)]
    c = Cache(seqs, fmt, 2, 64, 16, sum(-(-n // 16) for n in lens) + 200, seqs, 40).give(lens)
    for what in broken_caches(c):
        keep = Keep()
        d = DevicePages(c, c.upload(keep), keep)
        assert d('compact') == [_lib.PAGES_BAD, int((c.refs == 0).sum())], what
        c.assert_same()
    keep = Keep()
    d, b = DevicePages(c, c.upload(keep), keep), Book(c)
    for _ in range(2):  # the second finds nothing to move
        assert d('compact') == b.compact()
        c.assert_same()


def refused(c, what, *lists):
    """Runs a call on a fresh copy of c that has to change nothing."""
    keep = Keep()
    d = DevicePages(c, c.upload(keep), keep)
    assert d(what, *lists) == [_lib.PAGES_BAD, int((c.refs == 0).sum())], (what, lists)
    c.assert_same()


@FORMATS
@pytest.mark.parametrize('seqs', [3, 70])
def test_sequences_of_a_broken_cache_are_not_freed_or_forked(fmt, seqs):
    lens = [0] + [40 + (7 * i) % 60 for i in range(1, seqs)]
    c = Cache(seqs, fmt, 2, 64, 16, sum(-(-n // 16) for n in lens) + 20, seqs, 40).give(lens)
    last = seqs - 1
    c.table[0, 1] = c.pages  # (not held: sequence 0 is empty)
    for what in broken_caches(c):
        refused(c, 'free', list(range(seqs)))
        if what.startswith('a held page'):
            refused(c, 'free', [last])
            refused(c, 'fork', [last], [0], [int(c.lengths[last])])  # the page in question ends the prefix
            c.lengths[last] = 16 * (int(c.lengths[last]) // 16)
            keep = Keep()
            d, b = DevicePages(c, c.upload(keep), keep), Book(c)
            assert d('fork', [last], [0], [int(c.lengths[last])]) == b.fork([last], [0], [int(c.lengths[last])])
            c.assert_same()


@FORMATS
def test_a_page_of_more_holders_than_its_count_is_not_freed(fmt):
    """Two sequences on the same pages, counted once: freed together they would take a count below 0; one of them alone
    is freed, and the other is then refused."""
    c = Cache(4, fmt, 2, 64, 16, 80, 40, 12).give([100, 0, 35] + [16] * 37)
    c.table[1], c.lengths[1] = c.table[0], 100
    refused(c, 'free', [2, 0, 3, 1])
    refused(c, 'free', list(range(40)))
    keep = Keep()
    d, b = DevicePages(c, c.upload(keep), keep), Book(c)
    assert d('free', [2, 0]) == b.free([2, 0])
    c.assert_same()
    refused(c, 'free', [1])
    refused(c, 'compact')
