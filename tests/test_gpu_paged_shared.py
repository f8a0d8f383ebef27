"""Attention of sequences that share their first tokens
(qwen_b200_op_paged_decode_shared) against the host cache of paged_ref.py, and the
operators of sampling from a shared prompt together, as a server would run them."""
import ctypes

import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import BF16_HALF, U, Cache, bf16, bits, ref, unbits
from qwen_b200 import _lib
from test_gpu_paged import DIMS, FILL, FORMATS, PREFILL_W, assert_within, padded, u32, workspace

pytestmark = pytest.mark.gpu
L = qwen_b200.lib
KV8, BF16, NO_SEQ = _lib.KV8, _lib.KV_BF16, _lib.NO_SEQ


def shared_cache(seed, fmt, dim, page, groups, kv_heads=2, layers=1, copies=False, **more):
    """groups: [(tokens shared, lengths of the group's sequences)]. Full shared pages are one page in every table (or,
    with copies, pages of their own with the same contents); the page that a prefix ends in is always a copy."""
    lens = [t for _, members in groups for t in members]
    agree = [min(prefix, t, members[0]) for prefix, members in groups for t in members]  # tokens that a sequence has of the first
    first = [sum(len(m) for _, m in groups[:g]) for g, (_, members) in enumerate(groups) for _ in members]
    own = [0 if copies or first[i] == i else agree[i] // page for i in range(len(lens))]  # pages that are the first's
    c = Cache(seed, fmt, kv_heads, dim, page, sum(-(-t // page) for t in lens) - sum(own) + 3, len(lens),
              max(1, -(-max(lens) // page)) + 1, layers, **more)
    ids = iter(c.r.permutation(c.pages))
    c.lengths[:] = lens
    for i, t in enumerate(lens):
        c.table[i, :own[i]] = c.table[first[i], :own[i]]
        held = [next(ids) for _ in range(own[i], -(-t // page))]
        c.table[i, own[i]:own[i] + len(held)] = held
        c.refs[c.table[i, :-(-t // page)]] += 1
        n = agree[i] if first[i] != i else 0
        for a in [c.k, c.v] + ([c.ks, c.vs] if fmt == KV8 else []):
            for j in range(own[i], -(-n // page)):
                m = min(page, n - j * page)
                a[:, c.table[i, j], :, :m] = a[:, c.table[first[i], j], :, :m]
        for layer in range(layers):
            if t > n:
                c.write(layer, i, np.arange(n, t), c.rand(t - n, kv_heads, dim), c.rand(t - n, kv_heads, dim))
    return c


def shared(c, kv, keep, q, starts, prefix, seqs=None, scale=None, layer=0, extra=0, st=None):
    rows, heads, dim = q.shape
    buf, stride = padded(q, extra)
    out = dev(bits(np.full((rows, stride), np.float32(FILL))).view(np.int16))
    n = len(prefix)
    ws, nb = workspace(keep, L().qwen_b200_paged_decode_shared_workspace(ref(kv), heads, n, rows))
    rc = L().qwen_b200_op_paged_decode_shared(ref(kv), layer, keep(bits(buf).view(np.int16)), stride, heads, n,
                                              keep(u32(starts)), keep(u32(prefix)), rows,
                                              keep(u32(seqs)) if seqs is not None else None,
                                              dim ** -0.5 if scale is None else scale, vp(out), stride, ws, nb, st or stream())
    assert rc == 0
    sync()
    got = unbits(host(out))
    assert (got[:, heads * dim:] == FILL).all(), 'wrote between the rows'
    return got[:, :heads * dim].reshape(q.shape)


def attention(c, layer, q, seqs, scale):
    """Cache.attention without a window, with weights rounded as in prompts: the same values and the same bound (which
    its docstring derives), by matrix products of a row's heads."""
    rows, heads, dim = q.shape
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for r in range(rows):
        s = seqs[r]
        t = np.arange(int(c.lengths[s])) if s < c.seqs else np.arange(0)
        t = t[c.at(s, t)[0] < c.pages] if t.size else t
        if not t.size:
            continue
        k, v = (x.transpose(1, 0, 2) for x in c.read(layer, s, t))  # [kv head][key][dim]
        p = q[r].astype(np.float64).reshape(c.hkv, -1, dim)
        x = p @ k.transpose(0, 2, 1) * scale
        mag = (np.abs(p) @ np.abs(k).transpose(0, 2, 1) * abs(scale)).max(2)
        w = np.exp(x - x.max(2, keepdims=True))
        w /= w.sum(2, keepdims=True)
        y = w @ v
        size = w @ np.abs(v) + np.abs(y)
        e = (PREFILL_W + 2 * (dim + 4) * U * mag + 2.0 ** -21 + 2 * t.size * U)[..., None]
        out[r] = y.reshape(heads, dim)
        tol[r] = (BF16_HALF * (np.abs(y) + e * size) + e * size).reshape(heads, dim)
    return out, tol


def test_the_bound_is_that_of_the_cache():
    c = shared_cache(1, KV8, 64, 16, [(60, [70, 65, 0])])
    q = bf16(c.rand(3, 4, 64))
    for a, b in zip(attention(c, 0, q, np.arange(3), 0.3), c.attention(0, q, np.arange(3), [69, 64, -1], 0, 0, 0.3, PREFILL_W)):
        assert np.allclose(a, b, rtol=1e-12, atol=1e-300)


def check(c, kv, keep, q, starts, prefix, seqs=None, scale=None, layer=0, extra=0):
    got = shared(c, kv, keep, q, starts, prefix, seqs, scale, layer, extra)
    s = np.arange(len(q)) if seqs is None else np.asarray(seqs, np.int64)
    exact, tol = attention(c, layer, q, s, q.shape[2] ** -0.5 if scale is None else scale)
    a, b = min(starts[0], len(q)), min(starts[-1], len(q))
    if a < b:
        assert_within(got[a:b], exact[a:b], tol[a:b])
    assert (got[:a] == FILL).all() and (got[b:] == FILL).all(), 'wrote rows of no group'
    return got


def starts_of(groups):
    return np.concatenate([[0], np.cumsum([len(m) for _, m in groups])])


def run(seed, fmt, dim, page, groups, kv_heads=2, group=7, spread=2, **more):
    c = shared_cache(seed, fmt, dim, page, groups, kv_heads, **more)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(c.seqs, kv_heads * group, dim) * spread)
    return check(c, kv, keep, q, starts_of(groups), [p for p, _ in groups])


@FORMATS
@DIMS
@pytest.mark.parametrize('page', [16, 64, 256])
@pytest.mark.parametrize('copies', [False, True])
def test_prefixes_and_lengths(fmt, dim, page, copies):
    groups = [(300, [301, 310, 500, 300]), (128, [700, 129, 128, 0, 144]), (1, [1, 2, 65]), (511, [512])]
    run(dim + page, fmt, dim, page, groups, copies=copies)


@FORMATS
@DIMS
@pytest.mark.parametrize('prefix', [0, 1, 15, 16, 17, 63, 64, 127, 128, 129, 255, 256, 257, 1000])
def test_prefix_edges(fmt, dim, prefix):
    run(prefix, fmt, dim, 32, [(prefix, [prefix + 1, prefix + 16, prefix + 33, prefix])])


@FORMATS
@DIMS
@pytest.mark.parametrize('kv_heads,group', [(1, 1), (1, 7), (3, 2), (8, 1), (2, 8), (1, 9), (2, 16), (1, 17), (5, 3), (1, 64)])
def test_head_layouts(fmt, dim, kv_heads, group):
    run(kv_heads * group, fmt, dim, 16, [(270, [300, 271, 290]), (40, [41, 50])], kv_heads, group)


@FORMATS
@DIMS
@pytest.mark.parametrize('rows', [1, 2, 18, 19, 37, 73, 74, 75, 150])
def test_group_sizes(fmt, dim, rows):
    """Below, at and above whole tiles of query rows."""
    r = np.random.default_rng(rows)
    run(rows, fmt, dim, 64, [(400, [400 + int(x) for x in r.integers(0, 60, rows)])])


@FORMATS
def test_many_groups(fmt):
    r = np.random.default_rng(6)
    groups = [(int(p), [int(p) + int(x) for x in r.integers(1, 40, int(n))]) for p, n in zip(r.integers(0, 500, 70), r.integers(1, 5, 70))]
    run(70, fmt, 64, 32, groups, layers=1)


@FORMATS
def test_more_rows_and_heads_than_fit_the_gpu(fmt):
    """Some 70 blocks of the row kernel for each SM."""
    r = np.random.default_rng(2)
    groups = [(20, [20 + int(x) for x in r.integers(0, 9, 1300)])]
    run(1300, fmt, 64, 16, groups, kv_heads=8, group=1)


@FORMATS
@DIMS
def test_sequences_shorter_than_the_prefix(fmt, dim):
    """The prefix is a claim about the tokens that two sequences both have."""
    groups = [(600, [700, 100, 599, 600, 1, 650])]
    run(3, fmt, dim, 32, groups)


@FORMATS
@DIMS
def test_a_prefix_longer_than_the_first_sequence(fmt, dim):
    """It is cut to the first sequence; what the others hold behind it is their own."""
    groups = [(500, [200, 450, 700])]
    c = shared_cache(4, fmt, dim, 32, groups)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(3, 14, dim) * 2)
    check(c, kv, keep, q, [0, 3], [500])
    check(c, kv, keep, q, [0, 3], [0xffffffff])


@FORMATS
@DIMS
def test_rows_of_no_sequence_no_group_and_no_key(fmt, dim):
    groups = [(200, [210, 0, 220, 230]), (100, [150, 160])]
    c = shared_cache(5, fmt, dim, 16, groups)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(9, 14, dim) * 2)
    seqs = [4, 0, 1, NO_SEQ, 2, 3, 4, 5, c.seqs]
    got = check(c, kv, keep, q, [1, 6, 6, 8], [200, 7, 100], seqs, extra=16)
    assert not got[2:4].any()
    # a group whose first row is no sequence, or has no token, shares nothing
    check(c, kv, keep, q, [2, 6, 9], [200, 100], seqs)
    check(c, kv, keep, q, [3, 6, 6], [200, 100], seqs)
    # starts beyond the rows count as their end
    check(c, kv, keep, q, [0, 1, 50], [200, 0], seqs)
    # no group at all
    check(c, kv, keep, q, [4, 4], [200], seqs)


@FORMATS
def test_rows_in_another_order_and_one_sequence_in_two_rows(fmt):
    groups = [(333, [400, 350, 360, 340])]
    c = shared_cache(8, fmt, 64, 16, groups)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(6, 14, 64) * 2)
    check(c, kv, keep, q, [0, 6], [333], [2, 0, 3, 3, 1, 2])


@FORMATS
@DIMS
@pytest.mark.parametrize('scale', [-0.2, 0.0, 1e-30, 3.0])
def test_scales(fmt, dim, scale):
    groups = [(260, [300, 280, 270])]
    c = shared_cache(9, fmt, dim, 32, groups)
    keep = Keep()
    kv = c.upload(keep)
    check(c, kv, keep, bf16(c.rand(3, 14, dim)), [0, 3], [260], scale=scale)


@FORMATS
@DIMS
def test_pages_that_are_not_there(fmt, dim):
    """Tokens on a page id out of range are left out, in the prefix (the first sequence's table counts) and behind it."""
    groups = [(256, [300, 310])]
    c = shared_cache(10, fmt, dim, 32, groups)
    c.table[:, 2] = c.pages + 9
    c.table[0, 9] = c.pages
    keep = Keep()
    kv = c.upload(keep)
    check(c, kv, keep, bf16(c.rand(2, 14, dim) * 2), [0, 2], [256])
    c.table[:] = c.pages
    keep2 = Keep()
    kv = c.upload(keep2)
    got = shared(c, kv, keep2, bf16(c.rand(2, 14, dim)), [0, 2], [256])
    assert not got.any()


@FORMATS
@DIMS
@pytest.mark.parametrize('where', ['prefix', 'own', 'neither'])
def test_scores_far_apart(fmt, dim, where):
    """One key outweighs all others by hundreds of powers of two, before or behind the border; or all scores are far from 0."""
    groups = [(200, [260, 270, 280])]
    c = shared_cache(12, fmt, dim, 16, groups)
    q = bf16(c.rand(3, 4, dim))
    for s in range(3):
        at = {'prefix': 77, 'own': 205 + s, 'neither': None}[where]
        if at is not None:
            k = np.repeat(q[s].reshape(2, 2, dim)[:, :1], 1, 1)[:, 0][None] * 8
            if where == 'prefix':
                if s == 0:
                    for i in range(3):
                        c.write(0, i, [at], bf16(k), c.rand(1, 2, dim))
            else:
                c.write(0, s, [at], bf16(k), c.rand(1, 2, dim))
    if where == 'prefix':  # the same token in every copy
        for a in [c.k, c.v] + ([c.ks, c.vs] if fmt == KV8 else []):
            p, t = c.at(0, [77])
            for i in (1, 2):
                pi, ti = c.at(i, [77])
                a[:, pi, :, ti] = a[:, p, :, t]
    keep = Keep()
    kv = c.upload(keep)
    check(c, kv, keep, q, [0, 3], [200], scale=20.0 if where == 'neither' else 4.0)


@FORMATS
def test_long_prefix_few_rows_and_layers(fmt):
    """More pieces of a tile than fit a CTA; the second layer of a cache in the other order."""
    groups = [(9000, [9100, 9001])]
    c = shared_cache(13, fmt, 64, 256, groups, layers=2, pages_first=True)
    keep = Keep()
    kv = c.upload(keep)
    check(c, kv, keep, bf16(c.rand(2, 14, 64) * 2), [0, 2], [9000], layer=1)


@FORMATS
@DIMS
def test_equals_decode_attention(fmt, dim):
    """The same rows through qwen_b200_op_paged_decode, both within their bounds of 64 bits and so of one another."""
    groups = [(700, [730, 701, 1000]), (64, [65, 200])]
    c = shared_cache(14, fmt, dim, 64, groups)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(5, 14, dim) * 2)
    got = check(c, kv, keep, q, [0, 3, 5], [700, 64])
    from test_gpu_paged import DECODE_W, decode
    other = decode(c, kv, keep, 0, q, None)
    exact, tol = c.attention(0, q, np.arange(5), [int(n) - 1 for n in c.lengths], 0, 0, dim ** -0.5, PREFILL_W)
    _, tol2 = c.attention(0, q, np.arange(5), [int(n) - 1 for n in c.lengths], 0, 0, dim ** -0.5, DECODE_W)
    assert (np.abs(got - other) <= tol + tol2).all()


def test_the_same_call_gives_the_same_bits():
    groups = [(2000, [2000 + i for i in range(1, 40)])]
    c = shared_cache(15, KV8, 64, 64, groups)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(39, 14, 64))
    first = shared(c, kv, keep, q, [0, 39], [2000])
    for _ in range(3):
        assert np.array_equal(bits(first), bits(shared(c, kv, keep, q, [0, 39], [2000])))


@FORMATS
def test_captured_and_replayed_as_sequences_grow(fmt):
    torch = torch_cuda()
    groups = [(250, [260, 251, 270])]
    c = shared_cache(16, fmt, 64, 32, groups)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(3, 14, 64) * 2)
    qd, out = dev(bits(q).view(np.int16)), dev(np.zeros((3, 896), np.int16))
    starts, prefix = dev(u32([0, 3])), dev(u32([250]))
    ws = dev(np.zeros(L().qwen_b200_paged_decode_shared_workspace(ref(kv), 14, 1, 3), np.uint8))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def call():
        assert L().qwen_b200_op_paged_decode_shared(ref(kv), 0, vp(qd), 896, 14, 1, vp(starts), vp(prefix), 3, None, 0.125,
                                                    vp(out), 896, vp(ws), ws.numel(),
                                                    ctypes.c_void_p(side.cuda_stream)) == 0
    call()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call()
    for cut, p in (([260, 251, 270], 250), ([255, 100, 270], 250), ([12, 251, 0], 12), ([200, 199, 222], 190)):
        c.lengths[:] = cut
        c.dev['lengths'].copy_(torch.from_numpy(u32(cut)))
        prefix.copy_(torch.from_numpy(u32([p])))
        sync()
        graph.replay()
        sync()
        exact, tol = c.attention(0, q, np.arange(3), [n - 1 for n in cut], 0, 0, 0.125, PREFILL_W)
        assert_within(unbits(host(out)).reshape(q.shape), exact, tol, str(cut))


def test_two_streams_with_workspaces_of_their_own():
    torch = torch_cuda()
    groups = [(1500, [1500 + 7 * i for i in range(1, 30)])]
    caches = [shared_cache(20 + i, f, 64, 64, groups) for i, f in enumerate((KV8, BF16))]
    keep, jobs = Keep(), []
    for c in caches:
        kv = c.upload(keep)
        q = bf16(c.rand(29, 14, 64) * 2)
        out = dev(np.zeros((29, 896), np.int16))
        ws = dev(np.zeros(L().qwen_b200_paged_decode_shared_workspace(ref(kv), 14, 1, 29), np.uint8))
        jobs.append((c, kv, q, dev(bits(q).view(np.int16)), out, ws, torch.cuda.Stream()))
    starts, prefix = dev(u32([0, 29])), dev(u32([1500]))
    sync()
    for _ in range(20):
        for c, kv, q, qd, out, ws, st in jobs:
            assert L().qwen_b200_op_paged_decode_shared(ref(kv), 0, vp(qd), 896, 14, 1, vp(starts), vp(prefix), 29, None, 0.125,
                                                        vp(out), 896, vp(ws), ws.numel(), ctypes.c_void_p(st.cuda_stream)) == 0
    sync()
    for c, kv, q, qd, out, ws, st in jobs:
        exact, tol = c.attention(0, q, np.arange(29), [int(n) - 1 for n in c.lengths], 0, 0, 0.125, PREFILL_W)
        assert_within(unbits(host(out)).reshape(q.shape), exact, tol)


@FORMATS
def test_samples_of_one_prompt(fmt):
    """A prompt forked into samples that each go on with tokens of their own: fork, reserve, rotated append, shared
    attention, sampling, step after step, against the host cache."""
    from sample_ref import check as check_token
    from test_gpu_paged_rotary import append, make_table, rotation, turned  # noqa: F401
    heads, hkv, dim, T, samples, prompt = 6, 2, 64, 16, 5, 75
    c = Cache(30, fmt, hkv, dim, T, 40, samples + 1, 10, 1).give([prompt] + [0] * samples)
    keep, table = Keep(), make_table(200, dim)
    c.table[:] = np.where(np.arange(10) * T < c.lengths[:, None], c.table, 0)
    kv = c.upload(keep)
    ws = dev(np.zeros(L().qwen_b200_pages_workspace(ref(kv)), np.uint8))
    status, wsn = dev(np.zeros(2, np.int32)), ws.numel()
    kids = np.arange(1, samples + 1)
    assert L().qwen_b200_op_pages_fork(ref(kv), keep(u32(np.zeros(samples))), keep(u32(kids)), keep(u32(np.full(samples, prompt))),
                                       samples, vp(status), vp(ws), wsn, stream()) == 0
    r = np.random.default_rng(31)
    head = bf16(r.standard_normal((heads * dim, 500)) * 0.2)
    for step in range(4):
        assert L().qwen_b200_op_pages_reserve(ref(kv), keep(u32(kids)), keep(u32(np.ones(samples))), samples, vp(status), vp(ws),
                                              wsn, stream()) == 0
        sync()
        assert host(status)[0] == _lib.PAGES_OK
        # the device's books are the server's: the host cache follows them
        c.table[:] = host(c.dev['table']).view(np.uint32)
        c.lengths[:] = host(c.dev['lengths']).view(np.uint32)
        c.refs[:] = host(c.dev['refs']).view(np.uint32)
        if step == 0:  # the page that the prompt ends in was copied to each sample
            n = prompt % T
            for a in [c.k, c.v] + ([c.ks, c.vs] if fmt == KV8 else []):
                for s in kids:
                    # (the rest of that page is as it was)
                    a[:, c.table[s, prompt // T], :, :n] = a[:, c.table[0, prompt // T], :, :n]
        pos = np.full(samples, prompt + step)
        assert (c.lengths[1:] == prompt + step + 1).all()
        q, k, v = c.rand(samples, heads, dim), c.rand(samples, hkv, dim), c.rand(samples, hkv, dim)
        got_q = append(c, kv, keep, 0, table, _lib.ROTARY_HALVES, q, k, v, kids, pos)
        for s in kids:
            c.write(0, s, [prompt + step], turned(k[s - 1:s], table, pos[:1], _lib.ROTARY_HALVES), v[s - 1:s])
        c.assert_same()
        assert np.array_equal(bits(got_q), bits(turned(q, table, pos, _lib.ROTARY_HALVES)))
        ctx = check(c, kv, keep, got_q, [0, samples], [prompt], kids)
        logits = bf16(ctx.reshape(samples, -1) @ head)
        u = r.random(samples, np.float32)
        tokens, probs = dev(np.zeros(samples, np.int32)), dev(np.zeros(samples, np.float32))
        assert L().qwen_b200_op_sample(keep(bits(logits).view(np.int16)), 500, samples, 500,
                                       keep(np.full(samples, 0.8, np.float32)), keep(u32(np.full(samples, 50))),
                                       keep(np.full(samples, 0.95, np.float32)), None, keep(u), vp(tokens), vp(probs),
                                       stream()) == 0
        sync()
        for i in range(samples):
            check_token(int(host(tokens)[i]), host(probs)[i], logits[i], u[i], 0.8, 50, 0.95)


# ---------------------------------------------------------------- groups large enough for tiles of query rows
# (rows * shared keys * KV heads * dims of 3 * 2^24 and more)
BIG = pytest.mark.parametrize('dim,rows,prefix', [(64, 195, 520), (128, 150, 333)])


def big(seed, fmt, dim, rows, prefix, page=64, kv_heads=8, group=2, own=40, **more):
    assert rows * prefix * kv_heads * dim >= 3 << 24
    r = np.random.default_rng(seed)
    return [(prefix, [prefix + int(x) for x in r.integers(0, own, rows)])], dict(kv_heads=kv_heads, group=group, **more)


@FORMATS
@BIG
@pytest.mark.parametrize('page', [16, 64, 256])
@pytest.mark.parametrize('copies', [False, True])
def test_tiles_pages(fmt, dim, rows, prefix, page, copies):
    groups, more = big(page, fmt, dim, rows, prefix, copies=copies)
    run(page, fmt, dim, page, groups, **more)


@FORMATS
@DIMS
@pytest.mark.parametrize('prefix', [513, 575, 576, 577, 639, 640, 641, 767, 768, 1024])
def test_tiles_prefix_edges(fmt, dim, prefix):
    groups, more = big(prefix, fmt, dim, 200, prefix)
    run(prefix, fmt, dim, 32, groups, **more)


@FORMATS
@pytest.mark.parametrize('dim,kv_heads,group,rows,prefix', [
    (64, 1, 1, 780, 1024), (64, 2, 7, 384, 1030), (64, 8, 1, 380, 260), (128, 4, 3, 247, 400), (128, 2, 8, 180, 1100),
    (128, 1, 17, 385, 1025), (64, 3, 9, 585, 450), (128, 1, 70, 358, 1100), (64, 32, 5, 82, 300)])
def test_tiles_head_layouts(fmt, dim, kv_heads, group, rows, prefix):
    """Tiles that end inside a row's heads, at them, and rows over several tiles."""
    groups, more = big(rows, fmt, dim, rows, prefix, kv_heads=kv_heads, group=group)
    run(rows, fmt, dim, 128, groups, **more)


@FORMATS
@BIG
def test_tiles_many_groups(fmt, dim, rows, prefix):
    """Groups with and without tiles between one another, one of them empty, rows of no group around them."""
    r = np.random.default_rng(dim)
    sizes = [(0, 3), (prefix, rows), (prefix, 5), (prefix + 200, rows + 31), (90, 8), (2 * prefix, rows // 2 + 1), (0, 2)]
    groups = [(p, [p + int(x) for x in r.integers(1, 30, n)]) for p, n in sizes]
    c = shared_cache(dim, fmt, dim, 32, groups, kv_heads=8)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(c.seqs, 16, dim) * 2)
    starts = np.cumsum([n for _, n in sizes])[:-1]
    prefixes = [p for p, _ in sizes[1:-1]]
    # an empty group in the middle, with a prefix of its own
    starts, prefixes = np.insert(starts, 2, starts[2]), prefixes[:2] + [777] + prefixes[2:]
    check(c, kv, keep, q, starts, prefixes, extra=16)


@FORMATS
@BIG
def test_tiles_short_rows_no_sequences_and_missing_pages(fmt, dim, rows, prefix):
    """Rows that end inside the prefix, rows of no sequence, a prefix cut to its first sequence, pages that are not there."""
    groups, more = big(3, fmt, dim, rows, prefix)
    lens = groups[0][1]
    lens[0] = prefix + 9
    lens[1:8] = [1, 0, 63, 64, 65, prefix - 1, 127]
    c = shared_cache(4, fmt, dim, 32, groups, kv_heads=8)
    seqs = np.arange(rows)
    seqs[[9, 50]] = NO_SEQ
    c.table[:, 3] = c.pages + 1
    c.table[20, prefix // 32 + 1:] = c.pages
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(rows, 16, dim) * 2)
    got = check(c, kv, keep, q, [0, rows], [prefix], seqs)
    assert not got[[2, 9, 50]].any() and got[1].any()
    c.table[:] = c.pages
    keep2 = Keep()
    kv = c.upload(keep2)
    assert not shared(c, kv, keep2, q, [0, rows], [prefix]).any()


@FORMATS
@BIG
def test_tiles_a_prefix_longer_than_the_first_sequence(fmt, dim, rows, prefix):
    """It is cut to the first sequence, in whose tokens the others agree; what they hold behind it is their own."""
    groups, more = big(31, fmt, dim, rows, prefix)
    groups[0][1][0] = prefix
    c = shared_cache(31, fmt, dim, 32, [(prefix, groups[0][1])], kv_heads=8)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(rows, 16, dim) * 2)
    for claim in (prefix + 1, 2 * prefix, 0xffffffff):
        check(c, kv, keep, q, [0, rows], [claim])


@FORMATS
@BIG
@pytest.mark.parametrize('scale', [-0.2, 0.0, 1e-30, 4.0])
def test_tiles_scales(fmt, dim, rows, prefix, scale):
    groups, more = big(9, fmt, dim, rows, prefix)
    c = shared_cache(9, fmt, dim, 64, groups, kv_heads=8)
    keep = Keep()
    kv = c.upload(keep)
    check(c, kv, keep, bf16(c.rand(rows, 16, dim)), [0, rows], [prefix], scale=scale)


@FORMATS
@BIG
@pytest.mark.parametrize('where', ['prefix', 'own'])
def test_tiles_one_key_outweighs_the_rest(fmt, dim, rows, prefix, where):
    groups, more = big(12, fmt, dim, rows, prefix, own=2)
    groups[0][1][:] = [prefix + 1 + i % 3 for i in range(rows)]
    c = shared_cache(12, fmt, dim, 64, groups, kv_heads=8)
    q = bf16(np.repeat(c.rand(1, 16, dim), rows, 0) * (1 + np.arange(rows) % 3)[:, None, None])
    k = bf16(q[0].reshape(8, 2, dim)[:, 0][None] * 8)
    for s in range(rows):
        if where == 'own' or s == 0 or prefix % 64 > 0 and prefix - 5 >= prefix // 64 * 64:
            c.write(0, s, [prefix - 5 if where == 'prefix' else prefix], k, bf16(np.ones((1, 8, dim)) * 3))
    keep = Keep()
    kv = c.upload(keep)
    check(c, kv, keep, q, [0, rows], [prefix], scale=4.0)


@FORMATS
@DIMS
def test_tiles_of_values_that_nobody_sees(fmt, dim):
    """What the pages hold behind the prefix of the first sequence and behind each length does not matter (NaN there)."""
    groups = [(577, [577] + [577 + i % 7 for i in range(179)])]
    run(17, fmt, dim, 256, groups, kv_heads=8, group=1)


def test_tiles_give_the_same_bits_again_and_with_two_streams():
    torch = torch_cuda()
    jobs, keep = [], Keep()
    for fmt in (KV8, BF16):
        groups, _ = big(21, fmt, 64, 300, 600)
        c = shared_cache(21, fmt, 64, 64, groups, kv_heads=8)
        kv = c.upload(keep)
        q = bf16(c.rand(300, 16, 64) * 2)
        first = check(c, kv, keep, q, [0, 300], [600])
        ws = dev(np.zeros(L().qwen_b200_paged_decode_shared_workspace(ref(kv), 16, 1, 300), np.uint8))
        jobs.append((kv, dev(bits(q).view(np.int16)), dev(np.zeros((300, 1024), np.int16)), ws, torch.cuda.Stream(), first, c))
    starts, prefix = dev(u32([0, 300])), dev(u32([600]))
    sync()
    for _ in range(10):
        for kv, qd, out, ws, st, _, _ in jobs:
            assert L().qwen_b200_op_paged_decode_shared(ref(kv), 0, vp(qd), 1024, 16, 1, vp(starts), vp(prefix), 300, None, 0.125,
                                                        vp(out), 1024, vp(ws), ws.numel(), ctypes.c_void_p(st.cuda_stream)) == 0
    sync()
    for kv, qd, out, ws, st, first, _ in jobs:
        assert np.array_equal(host(out).view(np.uint16).reshape(first.shape), bits(first))
        assert not host(ws)[:4].any()  # no wait ran out


def test_tiles_captured_and_replayed_as_the_prefix_changes():
    """A graph of the call answers for groups that are worth tiles and for those that are not."""
    torch = torch_cuda()
    groups, _ = big(22, KV8, 128, 130, 400)
    c = shared_cache(22, KV8, 128, 64, groups, kv_heads=8)
    keep = Keep()
    kv = c.upload(keep)
    q = bf16(c.rand(130, 16, 128) * 2)
    qd, out = dev(bits(q).view(np.int16)), dev(np.zeros((130, 2048), np.int16))
    starts, prefix = dev(u32([0, 130])), dev(u32([400]))
    ws = dev(np.zeros(L().qwen_b200_paged_decode_shared_workspace(ref(kv), 16, 1, 130), np.uint8))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def call():
        assert L().qwen_b200_op_paged_decode_shared(ref(kv), 0, vp(qd), 2048, 16, 1, vp(starts), vp(prefix), 130, None, 0.088,
                                                    vp(out), 2048, vp(ws), ws.numel(), ctypes.c_void_p(side.cuda_stream)) == 0
    call()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call()
    exact, tol = attention(c, 0, q, np.arange(130), 0.088)
    for p in (400, 20, 399, 0, 350):
        prefix.copy_(torch.from_numpy(u32([p])))
        out.zero_()
        sync()
        graph.replay()
        sync()
        assert_within(unbits(host(out)).reshape(q.shape), exact, tol, str(p))


@FORMATS
@DIMS
def test_tiles_for_few_rows_with_a_long_prefix_among_many(fmt, dim):
    """From three items an SM on, prefixes of 2048 keys go to the tiles whatever their rows; others of the call do not."""
    r = np.random.default_rng(dim)
    groups = [(70, [70 + int(x) for x in r.integers(0, 50, 40)]), (2048, [2100, 2048]), (2047, [2050, 2060]), (2300, [2301, 2500, 100]),
              (64, [64 + int(x) for x in r.integers(0, 50, 30)])]
    run(dim, fmt, dim, 64, groups, kv_heads=8, group=3)


def test_two_host_threads_with_calls_of_other_sizes():
    """Each call's blocks ask for shared memory by the call's size: one thread's call does not get in another's way."""
    import threading
    torch = torch_cuda()
    keep, jobs = Keep(), []
    for seed, (rows, prefix) in enumerate(((120, 900), (450, 300))):
        groups, _ = big(seed, KV8, 64, rows, prefix)
        c = shared_cache(seed, KV8, 64, 64, groups, kv_heads=8)
        kv = c.upload(keep)
        q = bf16(c.rand(rows, 16, 64) * 2)
        n = L().qwen_b200_paged_decode_shared_workspace(ref(kv), 16, 1, rows)
        jobs.append((c, kv, q, dev(bits(q).view(np.int16)), dev(np.zeros((rows, 1024), np.int16)), dev(np.zeros(n, np.uint8)),
                     dev(u32([0, rows])), dev(u32([prefix])), torch.cuda.Stream(), []))
    sync()

    def work(job):
        c, kv, q, qd, out, ws, starts, prefix, st, codes = job
        for _ in range(300):
            codes.append(L().qwen_b200_op_paged_decode_shared(ref(kv), 0, vp(qd), 1024, 16, 1, vp(starts), vp(prefix), len(q), None,
                                                              0.125, vp(out), 1024, vp(ws), ws.numel(),
                                                              ctypes.c_void_p(st.cuda_stream)))
    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    sync()
    for c, kv, q, qd, out, ws, starts, prefix, st, codes in jobs:
        assert not any(codes)
        exact, tol = attention(c, 0, q, np.arange(len(q)), 0.125)
        assert_within(unbits(host(out)).reshape(q.shape), exact, tol)
