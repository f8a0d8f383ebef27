"""Prompt attention of padded batches: rows of no sequence and rows in front of
a sequence's first token are zero however many there are, and cost less than
rows that attend to something."""
import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import bits, ref
from qwen_b200 import _lib
from test_gpu_paged import FORMATS, DIMS, NO_SEQ, cache, check_prefill, runs, u32, workspace

pytestmark = pytest.mark.gpu
L = qwen_b200.lib


@FORMATS
@DIMS
def test_padded_prompts_are_zero(fmt, dim):
    """Slots of no sequence, empty sequences and prompts of more rows than tokens, from a few rows (zeroed by one CTA)
    to a thousand (by all of them), between sequences that attend."""
    lens = [40, 0, 100, 7, 0, 130]
    c = cache(dim, fmt, dim, 16, lens, kv_heads=1)
    keep = Keep()
    kv = c.upload(keep)
    seqs, rows = [0, NO_SEQ, 2, 1, 3, NO_SEQ, 5], [40, 1000, 333, 31, 40, 3, 130]
    check_prefill(c, kv, keep, c.rand(sum(rows) + 9, 3, dim), seqs, runs(c, rows), 30, 2, extra=8)
    check_prefill(c, kv, keep, c.rand(1200, 3, dim), [NO_SEQ], [0, 1177])  # nothing attends


@FORMATS
def test_many_padded_prompts_are_zero(fmt):
    """More sequences than a CTA has warps, so that each warp numbers several; those of more rows than there are
    sequences are zeroed by all CTAs."""
    r = np.random.default_rng(3)
    n = 90
    lens = [int(x) for x in r.integers(0, 20, n)]
    c = cache(5, fmt, 64, 16, lens, kv_heads=1)
    rows = [int(min(x, r.integers(1, 20))) for x in lens]
    seqs = np.arange(n, dtype=np.uint32)
    for i, k in ((0, 91), (3, 90), (4, 200), (44, 300), (45, 12), (89, 150)):
        rows[i] = k
        if i % 2 == 0:
            seqs[i] = NO_SEQ
    keep = Keep()
    kv = c.upload(keep)
    check_prefill(c, kv, keep, c.rand(sum(rows), 2, 64), seqs, runs(c, rows))


def test_a_padded_prompt_costs_less_than_one_that_attends():
    """The smallest of ten timings of one prompt of 8192 rows, of no sequence and of one with its tokens."""
    torch = torch_cuda()
    n = 8192
    c = cache(1, _lib.KV8, 64, 256, [n])
    keep = Keep()
    kv = c.upload(keep)
    q, out, starts = keep(bits(c.rand(n, 14, 64)).view(np.int16)), dev(np.zeros((n, 14, 64), np.int16)), keep(u32([0, n]))
    ws, nb = workspace(keep, L().qwen_b200_paged_prefill_workspace(ref(kv), 14, 1, n))

    def smallest(seq):
        times, seqs = [], keep(u32([seq]))
        for _ in range(10):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            assert L().qwen_b200_op_paged_prefill(ref(kv), 0, q, 896, 14, 1, seqs, starts, n, 256, 4, 0.125, vp(out), 896, ws,
                                                  nb, stream()) == 0
            b.record()
            sync()
            times.append(a.elapsed_time(b))
        return min(times)

    assert smallest(0) > smallest(NO_SEQ)
    assert not host(out).any()
