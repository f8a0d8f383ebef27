"""qwen_b200_op_sample against the definition in 64 bits (sample_ref.py): filters
alone and together, ties, masks, rows without candidates, sizes and alignments."""
import ctypes

import numpy as np
import pytest

import qwen_b200
from gpu_util import Keep, dev, host, stream, sync, torch_cuda, vp
from paged_ref import bf16, bits
from qwen_b200 import _lib
from sample_ref import NO_TOKEN, check

pytestmark = pytest.mark.gpu
L = qwen_b200.lib
INF, NAN = np.inf, np.nan
LOWEST = -3.3895313892515355e38


def to_bits(x):
    """bf16 bits; NaN, infinities and both zeros as they are."""
    x = np.asarray(x, np.float32)
    return np.where(np.isnan(x), np.uint16(0x7fc0), bits(bf16(np.nan_to_num(x, nan=0.0, posinf=INF, neginf=-INF)))).astype(np.uint16)


def values(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, skew=0, gap=0, probs=True):
    """tokens, probabilities; every parameter None (not given) or one value per row."""
    rows, vocab = logits.shape
    buf = np.full((rows, vocab + gap), 0x4680, np.uint16)  # 16384 between the rows: it would win
    buf[:, :vocab] = to_bits(logits)
    flat = dev(np.concatenate([np.full(skew + 8, 0x4680, np.uint16), buf.ravel(), np.full(16, 0x4680, np.uint16)]).view(np.int16))
    keep = Keep()
    f32 = lambda v: None if v is None else keep(np.broadcast_to(np.asarray(v, np.float32), (rows,)).copy())  # noqa: E731
    ki = None if top_k is None else keep(np.broadcast_to(np.asarray(top_k, np.uint32), (rows,)).view(np.int32).copy())
    tokens, out = dev(np.full(rows + 1, 77, np.int32)), dev(np.full(rows + 1, 7, np.float32))
    assert L().qwen_b200_op_sample(flat.data_ptr() + 2 * (skew + 8), vocab + gap, rows, vocab, f32(temperature), ki, f32(top_p),
                                   f32(min_p), f32(u), vp(tokens), vp(out) if probs else None, stream()) == 0
    sync()
    assert host(tokens)[rows] == 77 and host(out)[rows] == 7
    return host(tokens)[:rows].view(np.uint32), host(out)[:rows]


def check_all(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, **more):
    tokens, probs = sample(logits, u, temperature, top_k, top_p, min_p, **more)
    rows = logits.shape[0]
    of = lambda v, d: np.broadcast_to(np.asarray(d if v is None else v), (rows,))  # noqa: E731
    same = 0
    x = values(to_bits(logits))
    for r in range(rows):
        same += check(int(tokens[r]), probs[r], x[r], of(u, 0)[r], of(temperature, 1.0)[r], int(of(top_k, 0)[r]),
                      of(top_p, 1.0)[r], of(min_p, 0.0)[r]) is not False
    assert same >= rows - 1  # a border within the weights' rounding of u is met once in thousands of rows
    return tokens, probs


def rows_of(seed, rows, vocab, spread=2.5):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, vocab)) * spread
    for i in range(rows):
        x[i, r.integers(0, vocab, 5)] += r.random(5) * 10
    return x, r.random(rows, np.float32)


@pytest.mark.parametrize('vocab', [1, 2, 7, 8, 9, 31, 100, 1023, 4097, 50257, 65528, 65529, 151936, 524216])
@pytest.mark.parametrize('rows', [1, 5])
def test_vocabularies(vocab, rows):
    x, u = rows_of(vocab, rows, vocab)
    check_all(x, u)
    check_all(x, u, 0.7, 40, 0.9, 0.01)


@pytest.mark.parametrize('rows', [1, 2, 9, 10, 18, 19, 37, 74, 75, 150, 300])
def test_row_counts(rows):
    """Every split of a row over CTAs."""
    x, u = rows_of(rows, rows, 3001)
    check_all(x, u, np.linspace(0.2, 2, rows), np.arange(rows) % 7 * 11, np.linspace(0.3, 1.1, rows), np.linspace(0, 0.2, rows))


@pytest.mark.parametrize('skew', range(9))
@pytest.mark.parametrize('gap', [0, 1, 5, 8])
def test_alignments(skew, gap):
    x, u = rows_of(skew + 10 * gap, 4, 1000 + skew)
    check_all(x, u, 1.0, 0, 0.95, 0.0, skew=skew, gap=gap)


@pytest.mark.parametrize('top_k', [1, 2, 3, 50, 999, 1000, 1001, 0xffffffff])
def test_top_k(top_k):
    x, u = rows_of(top_k % 1000, 20, 1000)
    check_all(x, u, 1.3, top_k)


@pytest.mark.parametrize('top_p', [-1.0, 0.0, 1e-30, 0.1, 0.5, 0.9, 0.999, 1.0, 2.0, NAN])
@pytest.mark.parametrize('min_p', [-1.0, 0.0, 0.3, 1.0, 1.5, NAN])
def test_top_p_and_min_p(top_p, min_p):
    x, u = rows_of(7, 20, 1000)
    check_all(x, u, 1.0, None, top_p, min_p)
    check_all(x, u, 2.0, 30, top_p, min_p)


@pytest.mark.parametrize('temperature', [1e-40, 1e-3, 0.1, 1.0, 10.0, 1e6, INF])
def test_temperatures(temperature):
    x, u = rows_of(8, 20, 3000)
    check_all(x, u, temperature)
    check_all(x, u, temperature, 100, 0.8, 0.05)


def test_random_numbers():
    x, _ = rows_of(9, 1, 2000)
    u = np.array([0, 2.0 ** -149, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 3.0, -1.0, NAN, INF], np.float32)
    x = np.repeat(x, len(u), 0)
    tokens, _ = check_all(x, u)
    assert tokens[0] == tokens[7] == tokens[8] == np.argmax(values(to_bits(x[0])))
    assert tokens[4] == tokens[5] == tokens[6] == tokens[9]


def test_equal_logits_come_in_the_order_of_their_ids():
    x = np.zeros((8, 4096))
    x[:, ::2] = -0.0  # both zeros are equal
    u = np.arange(8, dtype=np.float32) / 8
    tokens, probs = sample(x, u)
    assert tokens.tolist() == [512 * i for i in range(8)] and (probs == 2.0 ** -12).all()
    tokens, probs = sample(x, u, top_k=np.full(8, 16))
    assert tokens.tolist() == [2 * i for i in range(8)] and (probs == 0.0625).all()
    tokens, _ = sample(x, u, top_p=np.full(8, 0.25))
    assert tokens.tolist() == [128 * i for i in range(8)]
    tokens, probs = sample(x, u, temperature=np.zeros(8))
    assert (tokens == 4095).all() and (probs == 1).all()


@pytest.mark.parametrize('vocab', [5000, 151936])
def test_greedy_is_the_highest_id_of_the_largest(vocab):
    r = np.random.default_rng(vocab)
    x = np.round(r.standard_normal((6, vocab)) * 2)
    for t in (0.0, -1.0, NAN):
        tokens, probs = sample(x, r.random(6), np.full(6, t), np.full(6, 1), np.full(6, 0.1), np.full(6, 2.0))
        assert tokens.tolist() == [int(np.flatnonzero(row == row.max())[-1]) for row in x] and (probs == 1).all()


@pytest.mark.parametrize('hidden', [-INF, LOWEST, -1e4, NAN])
@pytest.mark.parametrize('allowed', [0, 1, 2, 300])
@pytest.mark.parametrize('vocab', [3000, 151936])
def test_masks(hidden, allowed, vocab):
    r = np.random.default_rng(allowed)
    x = np.full((6, vocab), hidden)
    for i in range(6):
        x[i, r.choice(vocab, allowed, replace=False)] = r.standard_normal(allowed) * 3
    tokens, probs = check_all(x, r.random(6, np.float32), 0.9, [0, 0, 10, 500, 0, 1], [1, 0.9, 1, 0.9, 1, 1], [0, 0, 0, 0, 0.1, 0])
    if allowed == 0 and not np.isfinite(hidden):
        assert (tokens == NO_TOKEN).all() and (probs == 0).all()
        tokens, probs = sample(x, r.random(6), np.zeros(6))
        assert (tokens == NO_TOKEN).all() and (probs == 0).all()


def test_infinities_and_extremes():
    r = np.random.default_rng(4)
    x = r.standard_normal((5, 700))
    x[0, [3, 600]] = INF
    x[1, :] = LOWEST
    x[1, 5] = -LOWEST
    x[2] *= 1e-39  # denormals
    x[3] *= 1e30
    x[4, ::3] = NAN
    for u in (0.0, 0.3, 0.7, 0.99):
        tokens, _ = check_all(x, np.full(5, u, np.float32))
        assert tokens[0] == (3 if u < 0.5 else 600) and tokens[1] == 5


def test_a_long_row_of_one_value():
    """Counters of one value as large as they get."""
    x = np.full((2, 524216), 1.5)
    tokens, probs = sample(x, np.array([0.25, 1 - 2.0 ** -24], np.float32))
    assert tokens[0] == 524216 // 4 and tokens[1] == int(np.floor((1 - 2.0 ** -24) * 524216))
    assert (probs == np.float32(1 / 524216)).all()


def test_without_probabilities_and_every_default():
    x, u = rows_of(12, 3, 500)
    tokens, probs = sample(x, u, probs=False)
    assert (probs == 7).all()
    assert np.array_equal(tokens, sample(x, u)[0])
    assert np.array_equal(tokens, sample(x, u, np.ones(3), np.zeros(3), np.ones(3), np.zeros(3))[0])


def test_how_often_each_token_comes():
    """4096 evenly spaced u: each token as often as its probability says, to one."""
    x = np.repeat(np.random.default_rng(5).standard_normal((1, 40)), 4096, 0)
    u = ((np.arange(4096) + 0.5) / 4096).astype(np.float32)
    tokens, _ = sample(x, u)
    v = values(to_bits(x[0])).astype(np.float64)
    p = np.exp(v - v.max())
    assert np.abs(np.bincount(tokens, minlength=40) - 4096 * p / p.sum()).max() <= 1 + 1e-6


def test_captured_replayed_and_on_another_stream():
    torch = torch_cuda()
    x, u = rows_of(13, 6, 2000)
    logits, keep = dev(to_bits(x).view(np.int16)), Keep()
    un, tokens, t = dev(u), dev(np.zeros(6, np.int32)), dev(np.full(6, 0.8, np.float32))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def call(st):
        assert L().qwen_b200_op_sample(vp(logits), 2000, 6, 2000, vp(t), None, None, None, vp(un), vp(tokens), None,
                                       ctypes.c_void_p(st.cuda_stream)) == 0
    call(side)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call(side)
    for seed in (1, 2):
        nu = np.random.default_rng(seed).random(6, np.float32)
        un.copy_(torch.from_numpy(nu))
        sync()
        graph.replay()
        sync()
        assert np.array_equal(host(tokens).view(np.uint32), sample(x, nu, np.full(6, 0.8))[0])
    del keep


SPECIAL = [2.0 ** 8, -2.0 ** 8, 255.0, -255.0, 254.0, 2.0 ** -39, -2.0 ** -39, 2.0 ** -40, -2.0 ** -40, 0.0, -0.0, 1e-38, -1e-39, 9.2e-41,
           300.0, -300.0, 1.0, -1.0, 1.0078125, LOWEST, -INF, NAN, -1e4]


@pytest.mark.parametrize('temperature', [0.05, 1.0, 60.0, 1e5])
@pytest.mark.parametrize('upto', [1e9, 255.5, 1.5])
@pytest.mark.parametrize('vocab', [37, 1000, 40000])
def test_values_at_the_edges_of_what_is_counted(temperature, upto, vocab):
    """Zeros, the smallest and largest values, masks and ordinary logits side by side, in every order."""
    r = np.random.default_rng(vocab)
    some = np.array([v for v in SPECIAL if not v > upto])
    x = r.standard_normal((24, vocab)) * 0.7
    for i in range(24):
        special = r.random(vocab) < (0.02, 0.3, 0.95)[i % 3]
        x[i, special] = r.choice(some, special.sum())
    check_all(x, r.random(24, np.float32), np.full(24, temperature), np.where(np.arange(24) % 4 == 0, 20, 0),
              np.where(np.arange(24) % 4 == 1, 0.9, 1.0), np.where(np.arange(24) % 4 == 2, 0.05, 0.0))


@pytest.mark.parametrize('k', range(12))
def test_a_mask_with_a_value_at_each_place_of_a_load(k):
    """One allowed token among masked ones: 16-byte loads with one counted element each."""
    for hidden in (-INF, LOWEST, NAN, -1000.0):
        x = np.full((3, 4096), hidden)
        x[0, k::16] = np.linspace(-3, 3, len(range(k, 4096, 16)))
        x[1, 100 + k] = 0.0
        x[2, 4095 - k] = -20.0
        tokens, _ = check_all(x, np.array([0.37, 0.5, 0.9], np.float32), np.full(3, 0.7))
        assert tokens[1] == 100 + k and tokens[2] == 4095 - k


def test_more_rows_than_the_gpu_holds_at_once():
    x, u = rows_of(77, 700, 300)
    check_all(x, u, np.linspace(0.2, 2, 700), np.arange(700) % 5 * 9, np.linspace(0.3, 1.1, 700))


def test_two_streams_at_once():
    torch = torch_cuda()
    jobs = []
    for seed, (rows, vocab) in enumerate(((3, 151936), (40, 20000), (200, 5000))):
        x, u = rows_of(seed, rows, vocab)
        jobs.append((x, u, dev(to_bits(x).view(np.int16)), dev(u), dev(np.zeros(rows, np.int32)), torch.cuda.Stream()))
    sync()
    for _ in range(10):
        for x, u, logits, ud, tokens, st in jobs:
            assert L().qwen_b200_op_sample(vp(logits), x.shape[1], x.shape[0], x.shape[1], None, None, None, None, vp(ud), vp(tokens),
                                           None, ctypes.c_void_p(st.cuda_stream)) == 0
    sync()
    for x, u, logits, ud, tokens, st in jobs:
        assert np.array_equal(host(tokens).view(np.uint32), sample(x, u)[0])


def test_as_many_rows_as_a_call_takes():
    u = np.random.default_rng(3).random(65536, np.float32)
    tokens, probs = sample(np.zeros((65536, 4)), u)
    assert np.array_equal(tokens, np.floor(u * 4).astype(np.uint32)) and (probs == 0.25).all()
