"""Argument checks of the rotary, rotated append, shared-prefix and sampling entry
points: everything the host can see is refused before anything is launched. Runs
without a GPU: the addresses are made up and no call here gets as far as using one."""
import ctypes

import pytest

import qwen_b200
from qwen_b200 import _lib
from test_paged_refusals import A, kv

NAN, INF = float('nan'), float('inf')


def rotary(**change):
    return qwen_b200.Rotary(**(dict(table=A, positions=4096, rotated=64, layout=_lib.ROTARY_HALVES) | change))


def calls(c=None, rot=None, **change):
    d = dict(layer=0, x=A, stride=1024, heads=14, dim=64, rows=2, idx=A, out=A + 65536, out_stride=1024, k=A, row_stride=256,
             n=1, scale=0.125, ws=A, ws_bytes=1 << 40, logits=A, vocab=1000, param=A, u=A, tokens=A, probs=A, starts=A,
             prefix=A) | change
    L, p = qwen_b200.lib(), ctypes.byref(c if c is not None else kv())
    r = ctypes.byref(rot if rot is not None else rotary())
    return {
        'rotary': lambda: L.qwen_b200_op_rotary(r, d['x'], d['stride'], d['heads'], d['dim'], d['rows'], d['idx'], d['out'],
                                                d['out_stride'], None),
        'append': lambda: L.qwen_b200_op_paged_append_rotary(p, d['layer'], r, d['x'], d['stride'], d['heads'], d['out'],
                                                             d['out_stride'], d['k'], d['k'], d['row_stride'], d['rows'],
                                                             d['idx'], d['idx'], None),
        'shared': lambda: L.qwen_b200_op_paged_decode_shared(p, d['layer'], d['x'], d['stride'], d['heads'], d['n'],
                                                             d['starts'], d['prefix'], d['rows'], d['idx'], d['scale'],
                                                             d['out'], d['out_stride'], d['ws'], d['ws_bytes'], None),
        'sample': lambda: L.qwen_b200_op_sample(d['logits'], d['stride'], d['rows'], d['vocab'], d['param'], d['param'],
                                                d['param'], d['param'], d['u'], d['tokens'], d['probs'], None),
    }


@pytest.mark.parametrize('op,args', [
    ('rotary', dict(x=None)), ('rotary', dict(out=None)), ('rotary', dict(idx=None)), ('rotary', dict(idx=A + 2)),
    ('rotary', dict(x=A + 8)), ('rotary', dict(out=A + 8)), ('rotary', dict(stride=14 * 64 - 8)), ('rotary', dict(stride=1028)),
    ('rotary', dict(out_stride=14 * 64 - 8)), ('rotary', dict(out_stride=1028)), ('rotary', dict(rows=0)),
    ('rotary', dict(rows=1 << 31)), ('rotary', dict(heads=0)), ('rotary', dict(heads=65537, stride=1 << 30, out_stride=1 << 30)),
    ('rotary', dict(dim=0)), ('rotary', dict(dim=72)), ('rotary', dict(dim=528)), ('rotary', dict(dim=48)),
    ('rotary', dict(out=A, out_stride=2048)), ('rotary', dict(stride=1 << 33)),
    ('append', dict(layer=4)), ('append', dict(k=None)), ('append', dict(k=A + 8)), ('append', dict(rows=0)),
    ('append', dict(rows=1 << 31)), ('append', dict(idx=None)), ('append', dict(idx=A + 1)), ('append', dict(row_stride=120)),
    ('append', dict(row_stride=132)), ('append', dict(x=None)), ('append', dict(out=None)), ('append', dict(x=A + 8)),
    ('append', dict(stride=14 * 64 - 8)), ('append', dict(out_stride=1028)), ('append', dict(heads=65537)),
    ('append', dict(out=A, out_stride=2048)),
    ('shared', dict(layer=4)), ('shared', dict(x=None)), ('shared', dict(out=None)), ('shared', dict(x=A + 8)),
    ('shared', dict(rows=0)), ('shared', dict(rows=65537)), ('shared', dict(heads=13)), ('shared', dict(heads=0)),
    ('shared', dict(stride=14 * 64 - 8)), ('shared', dict(n=0)), ('shared', dict(n=65537)), ('shared', dict(starts=None)),
    ('shared', dict(prefix=None)), ('shared', dict(starts=A + 2)), ('shared', dict(prefix=A + 2)), ('shared', dict(idx=A + 2)),
    ('shared', dict(ws=None)), ('shared', dict(ws=A + 8)), ('shared', dict(scale=NAN)), ('shared', dict(scale=INF)),
    ('sample', dict(logits=None)), ('sample', dict(u=None)), ('sample', dict(tokens=None)), ('sample', dict(rows=0)),
    ('sample', dict(rows=65537)), ('sample', dict(vocab=0)), ('sample', dict(vocab=524217, stride=1 << 20)),
    ('sample', dict(stride=999)), ('sample', dict(stride=1 << 33)), ('sample', dict(logits=A + 1)), ('sample', dict(param=A + 2)), ('sample', dict(u=A + 2)),
    ('sample', dict(tokens=A + 2)), ('sample', dict(probs=A + 2)),
], ids=str)
def test_arguments_that_cannot_be_used_are_refused(op, args):
    assert calls(**args)[op]() == _lib.EINVAL


@pytest.mark.parametrize('change', [
    dict(table=None), dict(table=A + 8), dict(positions=0), dict(positions=(1 << 24) + 1), dict(rotated=0), dict(rotated=8),
    dict(rotated=80), dict(layout=2)], ids=str)
@pytest.mark.parametrize('op', ['rotary', 'append'])
def test_a_rotation_that_cannot_be_used_is_refused(op, change):
    assert calls(rot=rotary(**change))[op]() == _lib.EINVAL


@pytest.mark.parametrize('change', [dict(k=None), dict(format=2), dict(head_dim=96), dict(page_tokens=48), dict(seqs=0),
                                    dict(page_stride=64), dict(table=None), dict(vscales=None)], ids=str)
@pytest.mark.parametrize('op', ['append', 'shared'])
def test_a_descriptor_that_cannot_be_used_is_refused(op, change):
    assert calls(kv(**change))[op]() == _lib.EINVAL


@pytest.mark.parametrize('op', ['append', 'shared'])
def test_no_descriptor_no_rotation(op):
    L = qwen_b200.lib()
    r, p = ctypes.byref(rotary()), ctypes.byref(kv())
    assert L.qwen_b200_op_paged_append_rotary(None, 0, r, A, 896, 14, A, 896, A, A, 256, 1, A, A, None) == _lib.EINVAL
    assert L.qwen_b200_op_paged_append_rotary(p, 0, None, A, 896, 14, A, 896, A, A, 256, 1, A, A, None) == _lib.EINVAL
    assert L.qwen_b200_op_rotary(None, A, 896, 14, 64, 1, A, A, 896, None) == _lib.EINVAL
    assert L.qwen_b200_op_paged_decode_shared(None, 0, A, 896, 14, 1, A, A, 1, A, 0.125, A, 896, A, 1 << 40, None) == _lib.EINVAL


def test_workspace_sizes():
    L, good, bad = qwen_b200.lib(), ctypes.byref(kv()), ctypes.byref(kv(head_dim=80))
    size = L.qwen_b200_paged_decode_shared_workspace
    assert size(bad, 14, 1, 4) == 0 and size(None, 14, 1, 4) == 0
    assert size(good, 13, 1, 4) == 0 and size(good, 0, 1, 4) == 0 and size(good, 14, 1, 65537) == 0
    n = size(good, 14, 1, 4)
    assert n > 0 and size(good, 14, 4, 64) >= n
    assert calls(ws_bytes=n - 1, rows=4)['shared']() in (_lib.EINVAL, _lib.EDEVICE)


@pytest.mark.parametrize('change,rows,heads,n', [
    (dict(kv_heads=1, page_stride=64, layer_stride=32 * 64), 65536, 65536, 1),  # rows * (q_heads / kv_heads) of 2^32
    (dict(max_pages=1 << 24), 65536, 14, 65536),                                # blocks of tiles
    (dict(max_pages=1 << 24), 4096, 14, 1),                                     # keys of rows
], ids=['rows', 'blocks', 'keys'])
def test_shared_calls_of_more_than_32_bits_count_are_refused(change, rows, heads, n):
    assert calls(kv(**change), rows=rows, heads=heads, n=n, stride=1 << 22, out_stride=1 << 22)['shared']() == _lib.EINVAL


def test_memory_that_is_not_the_current_devices_is_refused():
    """Host memory: EINVAL where there is a GPU, EDEVICE where there is none; nothing is launched either way."""
    buf = (ctypes.c_uint8 * 4096)()
    at = (ctypes.addressof(buf) + 255) & ~255
    c = kv(k=at, v=at, kscales=at, vscales=at, table=at, lengths=at, refs=at)
    where = dict(x=at, idx=at, out=at + 1024, k=at, ws=at, logits=at, param=at, u=at, tokens=at, probs=at, starts=at, prefix=at)
    for op, call in calls(c, rotary(table=at), **where).items():
        assert call() in (_lib.EINVAL, _lib.EDEVICE), op
