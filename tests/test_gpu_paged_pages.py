"""Page management of the paged KV cache where sizes, tables and counts are at
their worst: requests beyond any pool, and caches whose tables, lengths and
reference counts do not belong together. A call that is refused changes
nothing but its status."""
import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import ref
from qwen_b200 import _lib
from test_gpu_paged import u32, workspace

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
