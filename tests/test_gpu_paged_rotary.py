"""Rotary positions (qwen_b200_op_rotary) and the rotated append of the paged cache
(qwen_b200_op_paged_append_rotary): bit for bit against fp32 products and sums
rounded one by one on the host, and within their bound of the rotation in 64 bits."""
import ctypes

import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import BF16_HALF, U, bf16, bits, ref, unbits
from qwen_b200 import _lib
from test_gpu_paged import cache, u32

pytestmark = pytest.mark.gpu
L = qwen_b200.lib
HALVES, PAIRS = _lib.ROTARY_HALVES, _lib.ROTARY_PAIRS
LAYOUTS = pytest.mark.parametrize('layout', [HALVES, PAIRS], ids=['halves', 'pairs'])
FILL = 7.0


def make_table(positions, rotated, **more):
    d = dict(theta=1e6, factor=4.0, fast=32.0, slow=1.0, size=0.0, rotated=rotated, scaling=_lib.ROTARY_YARN, trained=256) | more
    out = np.zeros((positions, rotated), np.float32)
    assert L().qwen_b200_rotary_table(ctypes.byref(qwen_b200.RotaryAngles(**d)), positions, _lib.ptr(out, ctypes.c_float)) == 0
    return out


def rotation(keep, table, layout):
    return qwen_b200.Rotary(table=keep(table), positions=table.shape[0], rotated=table.shape[1], layout=layout)


def pairs_of(rotated, layout):
    i = np.arange(rotated // 2)
    return (2 * i, 2 * i + 1) if layout == PAIRS else (i, i + rotated // 2)


def turned(x, table, positions, layout):
    """x [rows][heads][dim] in bf16 values: every product and sum one fp32 operation, then bf16."""
    rot = table.shape[1]
    a, b = pairs_of(rot, layout)
    c, s = (t[:, None] for t in np.split(table[positions], 2, 1))
    x = np.asarray(x, np.float32)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return bf16(y)


def assert_near(y, x, table, positions, layout):
    """In 64 bits: half a bf16 step of the result, and three fp32 roundings of products of at most (|a| + |b|) size."""
    rot = table.shape[1]
    a, b = pairs_of(rot, layout)
    c, s = (t[:, None].astype(np.float64) for t in np.split(table[positions], 2, 1))
    x = x.astype(np.float64)
    for i, exact in ((a, x[..., a] * c - x[..., b] * s), (b, x[..., b] * c + x[..., a] * s)):
        size = (np.abs(x[..., a]) + np.abs(x[..., b])) * max(1.0, np.abs(table).max())
        assert (np.abs(y[..., i] - exact) <= BF16_HALF * np.abs(exact) + (1 + BF16_HALF) * 3 * U * size + 1e-38).all()
    assert np.array_equal(y[..., rot:], x[..., rot:])


@LAYOUTS
@pytest.mark.parametrize('dim,rotated', [(16, 16), (32, 16), (64, 64), (64, 16), (64, 48), (80, 32), (96, 96), (128, 128),
                                         (128, 112), (256, 64), (512, 512)])
@pytest.mark.parametrize('rows,heads', [(1, 1), (3, 5), (70, 16)])
def test_rotation(dim, rotated, layout, rows, heads):
    r, keep = np.random.default_rng(dim + rotated + rows), Keep()
    table = make_table(333, rotated)
    positions = r.integers(0, 333, rows)
    x = bf16(r.standard_normal((rows, heads, dim)))
    buf = np.full((rows, heads * dim + 24), np.float32(FILL))
    buf[:, 8:8 + heads * dim] = x.reshape(rows, -1)
    xin = dev(bits(buf).view(np.int16))
    out = dev(bits(np.full((rows, heads * dim + 16), np.float32(FILL))).view(np.int16))
    rot = rotation(keep, table, layout)
    assert L().qwen_b200_op_rotary(ref(rot), xin.data_ptr() + 16, heads * dim + 24, heads, dim, rows, keep(u32(positions)),
                                   vp(out), heads * dim + 16, stream()) == 0
    sync()
    got = unbits(host(out))
    assert (got[:, heads * dim:] == FILL).all()
    y = got[:, :heads * dim].reshape(x.shape)
    assert np.array_equal(bits(y), bits(turned(x, table, positions, layout)))
    assert_near(y, x, table, positions, layout)
    # in place
    assert L().qwen_b200_op_rotary(ref(rot), xin.data_ptr() + 16, heads * dim + 24, heads, dim, rows, keep(u32(positions)),
                                   xin.data_ptr() + 16, heads * dim + 24, stream()) == 0
    sync()
    buf[:, 8:8 + heads * dim] = y.reshape(rows, -1)
    assert np.array_equal(host(xin).view(np.uint16), bits(buf))


def test_positions_outside_the_table_and_values_that_are_no_numbers():
    keep, table = Keep(), make_table(10, 64)
    positions = np.array([9, 10, 0, 0xffffffff, 1 << 31, 3], np.uint32)
    x = bf16(np.random.default_rng(1).standard_normal((6, 2, 64)))
    x[5, 0, 0], x[5, 1, 5], x[2, 0, 63] = np.nan, np.inf, -np.inf
    out = dev(bits(np.full((6, 128), np.float32(FILL))).view(np.int16))
    rot = rotation(keep, table, HALVES)
    assert L().qwen_b200_op_rotary(ref(rot), keep(bits(x).view(np.int16)), 128, 2, 64, 6, keep(u32(positions)), vp(out), 128,
                                   stream()) == 0
    sync()
    got = unbits(host(out)).reshape(6, 2, 64)
    assert (got[[1, 3, 4]] == FILL).all()
    with np.errstate(invalid='ignore'):
        y = x[[0, 2, 5]].copy()
        c, s = (t[:, None] for t in np.split(table[[9, 0, 3]], 2, 1))
        y[..., :32], y[..., 32:] = y[..., :32] * c - y[..., 32:] * s, y[..., 32:] * c + y[..., :32] * s
    live = got[[0, 2, 5]]
    assert np.array_equal(np.isnan(live), np.isnan(y))
    fine = np.isfinite(y)
    assert np.array_equal(bits(live[fine]), bits(bf16(y[fine]))) and np.array_equal(np.isposinf(live), np.isposinf(y))


def test_position_zero_of_a_plain_table_changes_nothing():
    keep, table = Keep(), make_table(1, 128, scaling=_lib.ROTARY_PLAIN)
    x = bf16(np.random.default_rng(2).standard_normal((9, 3, 128)))
    out = dev(np.zeros((9, 384), np.int16))
    rot = rotation(keep, table, PAIRS)
    assert L().qwen_b200_op_rotary(ref(rot), keep(bits(x).view(np.int16)), 384, 3, 128, 9, keep(u32(np.zeros(9))), vp(out), 384,
                                   stream()) == 0
    sync()
    assert np.array_equal(unbits(host(out)).reshape(x.shape), x)


def test_many_rows_and_heads():
    r, keep = np.random.default_rng(3), Keep()
    table = make_table(5000, 64, theta=1e4, scaling=_lib.ROTARY_NTK)
    x, positions = bf16(r.standard_normal((4111, 9, 128))), r.integers(0, 5000, 4111)
    out = dev(np.zeros((4111, 9 * 128), np.int16))
    rot = rotation(keep, table, PAIRS)
    assert L().qwen_b200_op_rotary(ref(rot), keep(bits(x).view(np.int16)), 9 * 128, 9, 128, 4111, keep(u32(positions)), vp(out),
                                   9 * 128, stream()) == 0
    sync()
    assert np.array_equal(host(out).view(np.uint16).reshape(x.shape), bits(turned(x, table, positions, PAIRS)))


# ---------------------------------------------------------------- rotated append
def append(c, kv, keep, layer, table, layout, q, k, v, seqs, pos, in_place=False, extra=8, call=None):
    """q | k | v rows through the entry point; what q_out holds then."""
    rows, heads, dim = q.shape
    qkv = np.concatenate([q, k, v], 1).reshape(rows, -1)
    stride = qkv.shape[1] + extra
    buf = np.full((rows, stride), np.float32(FILL))
    buf[:, :qkv.shape[1]] = qkv
    fused = dev(bits(buf).view(np.int16))
    out = fused if in_place else dev(bits(np.full((rows, heads * dim + 8), np.float32(FILL))).view(np.int16))
    base, width = fused.data_ptr(), stride if in_place else heads * dim + 8
    rot = rotation(keep, table, layout)
    keep.tensors += [fused, out]
    args = (ref(kv), layer, ref(rot), base, stride, heads, out.data_ptr(), width, base + 2 * heads * dim,
            base + 2 * (heads + c.hkv) * dim, stride, rows, keep(u32(seqs)), keep(u32(pos)), stream())
    assert L().qwen_b200_op_paged_append_rotary(*args) == 0
    sync()
    got = unbits(host(out))
    if in_place:
        assert np.array_equal(bits(got[:, heads * dim:]), bits(buf[:, heads * dim:]))
    else:
        assert (got[:, heads * dim:] == FILL).all()
    return got[:, :heads * dim].reshape(q.shape)


@LAYOUTS
@pytest.mark.parametrize('fmt', [_lib.KV8, _lib.KV_BF16], ids=['kv8', 'bf16'])
@pytest.mark.parametrize('dim,rotated', [(64, 64), (64, 16), (64, 48), (128, 128), (128, 80)])
@pytest.mark.parametrize('kv_heads,heads,page', [(1, 1, 16), (3, 9, 64), (2, 14, 256)])
def test_append(fmt, dim, rotated, layout, kv_heads, heads, page):
    lens = [40, 1, 0, 300, 17]
    c = cache(dim + page, fmt, dim, page, lens, kv_heads=kv_heads, layers=2, pages_first=rotated == dim)
    keep, table = Keep(), make_table(290, rotated)
    c.table[3, 0] = c.pages + 5  # a page that is not there
    kv = c.upload(keep)
    seqs = np.array([0, 3, 1, _lib.NO_SEQ, 4, 0, 3, 2, 5, 3, 0, 3, 3], np.uint32)
    # 0: no page, 299 and 290: behind the table, 300: behind the length
    pos = np.array([39, 289, 0, 3, 16, 7, 0, 0, 0, 300, 1 << 30, 299, 290], np.uint32)
    rows = len(seqs)
    q, k, v = c.rand(rows, heads, dim), c.rand(rows, kv_heads, dim), c.rand(rows, kv_heads, dim)
    k[2] = 0  # an all-zero row: scale 0
    v[4, 0, :5] = [64.0, -64.0, 32.0, 127.0, -127.0]
    got = append(c, kv, keep, 1, table, layout, q, k, v, seqs, pos, in_place=heads == 9)
    live = [r for r in range(rows) if seqs[r] < c.seqs and pos[r] < min(c.lengths[seqs[r]], 290) and
            c.at(seqs[r], [pos[r]])[0][0] < c.pages]
    assert len(live) == 5
    for r in live:
        c.write(1, seqs[r], [int(pos[r])], turned(k[r:r + 1], table, pos[r:r + 1], layout), v[r:r + 1])
    c.assert_same()
    want = q.copy() if heads == 9 else np.full(q.shape, np.float32(FILL))
    want[live] = turned(q[live], table, pos[live], layout)
    assert np.array_equal(bits(got), bits(want))


@pytest.mark.parametrize('fmt', [_lib.KV8, _lib.KV_BF16], ids=['kv8', 'bf16'])
def test_a_prompt_equals_the_rotation_and_the_append(fmt):
    """The bits of qwen_b200_op_rotary followed by qwen_b200_op_paged_append, and without queries the same cache."""
    lens = [1000, 257]
    c = cache(5, fmt, 128, 32, lens)
    keep, table = Keep(), make_table(1000, 96)
    kv = c.upload(keep)
    seqs = np.repeat([0, 1], [900, 257])
    pos = np.concatenate([np.arange(100, 1000), np.arange(257)])
    rows = len(seqs)
    q, k, v = c.rand(rows, 6, 128) * 3, c.rand(rows, 2, 128) * 3, c.rand(rows, 2, 128)
    got = append(c, kv, keep, 0, table, PAIRS, q, k, v, seqs, pos)
    qk = dev(bits(np.concatenate([q, k], 1)).view(np.int16))
    rot = rotation(keep, table, PAIRS)
    assert L().qwen_b200_op_rotary(ref(rot), vp(qk), 1024, 8, 128, rows, keep(u32(pos)), vp(qk), 1024, stream()) == 0
    sync()
    y = unbits(host(qk)).reshape(rows, 8, 128)
    assert np.array_equal(bits(got), bits(y[:, :6]))
    for s in (0, 1):
        c.write(0, s, pos[seqs == s], y[seqs == s, 6:], v[seqs == s])
    c.assert_same()
    c2 = cache(5, fmt, 128, 32, lens)
    kv2 = c2.upload(keep)
    kvbuf = keep(bits(np.concatenate([k, v], 1)).view(np.int16))
    assert L().qwen_b200_op_paged_append_rotary(ref(kv2), 0, ref(rot), None, 0, 0, None, 0, kvbuf, kvbuf.value + 512, 512, rows,
                                                keep(u32(seqs)), keep(u32(pos)), stream()) == 0
    sync()
    for name in ('k', 'v', 'table', 'lengths', 'refs') + (('ks', 'vs') if fmt == _lib.KV8 else ()):
        a, b = host(c.dev[name]), host(c2.dev[name])
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), name


def test_captured_and_replayed_as_positions_move():
    torch = torch_cuda()
    c = cache(11, _lib.KV8, 64, 16, [50, 50])
    keep, table = Keep(), make_table(64, 64)
    kv = c.upload(keep)
    q, k, v = c.rand(2, 14, 64), c.rand(2, 2, 64), c.rand(2, 2, 64)
    fused = dev(bits(np.concatenate([q, k, v], 1).reshape(2, -1)).view(np.int16))
    out, pos, seqs = dev(np.zeros((2, 896), np.int16)), dev(u32([48, 10])), dev(u32([0, 1]))
    rot = rotation(keep, table, HALVES)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def call():
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        base = fused.data_ptr()
        assert L().qwen_b200_op_paged_append_rotary(ref(kv), 0, ref(rot), base, 1152, 14, out.data_ptr(), 896, base + 1792,
                                                    base + 2048, 1152, 2, seqs.data_ptr(), pos.data_ptr(), st) == 0
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            call()
    for p in ([48, 10], [49, 11]):
        pos.copy_(torch.from_numpy(u32(p)))
        sync()
        graph.replay()
        sync()
        for r in range(2):
            c.write(0, r, [p[r]], turned(k[r:r + 1], table, [p[r]], HALVES), v[r:r + 1])
        c.assert_same()
        assert np.array_equal(host(out).view(np.uint16).reshape(q.shape), bits(turned(q, table, p, HALVES)))
