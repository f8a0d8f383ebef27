"""Argument checks of the paged KV cache's entry points: everything the host can
see is refused before anything is launched. Runs without a GPU: the addresses
are made up and no call here gets as far as using one."""
import ctypes

import pytest

import qwen_b200
from qwen_b200 import _lib

A = 1 << 20  # an aligned address that nothing dereferences


def kv(**change):
    d = dict(k=A, v=A, kscales=A, vscales=A, table=A, lengths=A, refs=A, layer_stride=32 * 2 * 64, page_stride=2 * 64,
             format=_lib.KV8, layers=4, pages=32, kv_heads=2, page_tokens=64, head_dim=64, seqs=8, max_pages=8)
    d.update(change)
    return qwen_b200.PagedKV(**d)


def calls(c, layer=0, q_heads=14, rows=2, q_stride=14 * 128, ws=A, ws_bytes=1 << 40, x=A, idx=A, row_stride=256, scale=0.125,
          status=A, n=2):
    L, p = qwen_b200.lib(), ctypes.byref(c) if c is not None else None
    return {
        'append': lambda: L.qwen_b200_op_paged_append(p, layer, x, x, row_stride, rows, idx, idx, None),
        'decode': lambda: L.qwen_b200_op_paged_decode(p, layer, x, q_stride, q_heads, rows, None, 0, 0, scale, x, q_stride,
                                                      ws, ws_bytes, None),
        'prefill': lambda: L.qwen_b200_op_paged_prefill(p, layer, x, q_stride, q_heads, n, None, idx, rows, 0, 0, scale, x,
                                                        q_stride, ws, ws_bytes, None),
        'reserve': lambda: L.qwen_b200_op_pages_reserve(p, idx, idx, n, status, ws, ws_bytes, None),
        'fork': lambda: L.qwen_b200_op_pages_fork(p, idx, idx, idx, n, status, ws, ws_bytes, None),
        'free': lambda: L.qwen_b200_op_pages_free(p, idx, n, status, ws, ws_bytes, None),
        'compact': lambda: L.qwen_b200_op_pages_compact(p, status, ws, ws_bytes, None),
        'copy': lambda: L.qwen_b200_op_pages_copy(p, idx, idx, n, None),
    }


ALL = sorted(calls(kv()))


@pytest.mark.parametrize('change', [
    dict(k=None), dict(v=None), dict(table=None), dict(lengths=None), dict(kscales=None), dict(vscales=None),
    dict(format=2), dict(head_dim=32), dict(head_dim=96), dict(head_dim=0), dict(page_tokens=8), dict(page_tokens=48),
    dict(page_tokens=512), dict(page_tokens=0), dict(layers=0), dict(pages=0), dict(kv_heads=0), dict(seqs=0),
    dict(max_pages=0), dict(seqs=65537), dict(pages=1 << 31), dict(max_pages=1 << 25), dict(k=A + 8), dict(v=A + 4),
    dict(kscales=A + 4), dict(vscales=A + 8), dict(table=A + 2), dict(lengths=A + 1), dict(page_stride=2 * 64 + 8),
    dict(page_stride=64), dict(layer_stride=64), dict(layer_stride=32 * 2 * 64 - 16), dict(layer_stride=1 << 50),
], ids=str)
@pytest.mark.parametrize('op', ALL)
def test_a_descriptor_that_cannot_be_used_is_refused(op, change):
    assert calls(kv(**change))[op]() == _lib.EINVAL


@pytest.mark.parametrize('op', ALL)
def test_no_descriptor(op):
    assert calls(None)[op]() == _lib.EINVAL


def test_workspace_sizes_of_a_bad_descriptor_are_zero():
    L, bad = qwen_b200.lib(), ctypes.byref(kv(head_dim=80))
    assert L.qwen_b200_paged_decode_workspace(bad, 14, 4) == 0
    assert L.qwen_b200_paged_prefill_workspace(bad, 14, 1, 4) == 0
    assert L.qwen_b200_pages_workspace(bad) == 0
    good = ctypes.byref(kv())
    assert L.qwen_b200_paged_decode_workspace(good, 13, 4) == 0
    assert L.qwen_b200_pages_workspace(good) >= 24 * 32


@pytest.mark.parametrize('op,args', [
    ('append', dict(layer=4)), ('append', dict(x=None)), ('append', dict(x=A + 2)), ('append', dict(rows=0)),
    ('append', dict(idx=None)), ('append', dict(row_stride=120)), ('append', dict(row_stride=132)),
    ('decode', dict(layer=4)), ('decode', dict(x=None)), ('decode', dict(x=A + 8)), ('decode', dict(rows=0)),
    ('decode', dict(rows=65537)), ('decode', dict(q_heads=13)), ('decode', dict(q_heads=0)),
    ('decode', dict(q_stride=14 * 64 - 8)), ('decode', dict(q_stride=14 * 64 + 4)), ('decode', dict(ws=None)),
    ('decode', dict(ws=A + 8)), ('decode', dict(scale=float('nan'))), ('decode', dict(scale=float('inf'))),
    ('prefill', dict(layer=4)), ('prefill', dict(x=None)), ('prefill', dict(x=A + 8)), ('prefill', dict(rows=0)),
    ('prefill', dict(rows=(1 << 24) + 1)), ('prefill', dict(n=0)), ('prefill', dict(n=65537)), ('prefill', dict(idx=None)),
    ('prefill', dict(q_heads=15)), ('prefill', dict(q_stride=14 * 64 - 8)), ('prefill', dict(ws=None)),
    ('prefill', dict(scale=float('inf'))),
    ('reserve', dict(n=0)), ('reserve', dict(idx=None)), ('reserve', dict(status=None)), ('reserve', dict(ws=None)),
    ('reserve', dict(ws_bytes=24 * 32)), ('reserve', dict(status=A + 2)), ('fork', dict(n=0)), ('fork', dict(idx=None)),
    ('fork', dict(ws=A + 4)), ('fork', dict(status=None)), ('free', dict(n=0)), ('free', dict(idx=None)),
    ('free', dict(status=None)), ('compact', dict(status=None)), ('compact', dict(ws=None)),
    ('compact', dict(ws_bytes=0)), ('copy', dict(n=0)), ('copy', dict(idx=None)),
], ids=str)
def test_arguments_that_cannot_be_used_are_refused(op, args):
    assert calls(kv(), **args)[op]() == _lib.EINVAL


@pytest.mark.parametrize('op', ['reserve', 'fork', 'free', 'compact'])
def test_page_management_needs_reference_counts(op):
    assert calls(kv(refs=None))[op]() == _lib.EINVAL


def test_memory_that_is_not_the_current_devices_is_refused():
    """Host memory: EINVAL where there is a GPU, EDEVICE where there is none; nothing is launched either way."""
    buf = (ctypes.c_uint8 * 4096)()
    at = (ctypes.addressof(buf) + 255) & ~255
    c = kv(k=at, v=at, kscales=at, vscales=at, table=at, lengths=at, refs=at)
    for op, call in calls(c).items():
        assert call() in (_lib.EINVAL, _lib.EDEVICE), op


def test_both_pool_orders_pass_the_stride_check():
    """[layers][pages] and [pages][layers] descriptors get as far as the device check (made-up memory is refused there)."""
    L = qwen_b200.lib()
    for c in (kv(), kv(layer_stride=2 * 64, page_stride=4 * 2 * 64), kv(layers=1, layer_stride=0), kv(format=_lib.KV_BF16,
                                                                                                      kscales=None)):
        assert L.qwen_b200_pages_workspace(ctypes.byref(c)) > 0


@pytest.mark.parametrize('op', ['append', 'prefill', 'reserve', 'fork', 'free', 'copy'])
def test_index_lists_are_aligned(op):
    assert calls(kv(), idx=A + 2)[op]() == _lib.EINVAL


def test_index_lists_of_decode_are_aligned():
    L = qwen_b200.lib()
    assert L.qwen_b200_op_paged_decode(ctypes.byref(kv()), 0, A, 896, 14, 2, A + 1, 0, 0, 0.125, A, 896, A, 1 << 40,
                                       None) == _lib.EINVAL
    assert L.qwen_b200_op_paged_prefill(ctypes.byref(kv()), 0, A, 896, 14, 2, A + 3, A, 2, 0, 0, 0.125, A, 896, A, 1 << 40,
                                        None) == _lib.EINVAL


@pytest.mark.parametrize('op', ['reserve', 'fork', 'free', 'copy'])
def test_lists_too_long_for_31_bits_are_refused(op):
    assert calls(kv(), n=1 << 31)[op]() == _lib.EINVAL
    assert calls(kv(), n=(1 << 32) - 1)[op]() == _lib.EINVAL
