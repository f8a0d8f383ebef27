"""qwen_b200_op_sample where a row is split over 8, 4, 2 CTAs or none, against the
definition in 64 bits (sample_ref.py): what decides a row (its largest logit, a
value that is not counted in the usual window, the tokens that a mask leaves) lies
in the part of one CTA, each in turn, and every CTA has to learn of it."""
import ctypes

import numpy as np
import pytest

from gpu_util import dev, host, sync, torch_cuda, vp
from sample_ref import check
from test_gpu_lm_sample import INF, L, LOWEST, check_all, rows_of, to_bits, values

pytestmark = pytest.mark.gpu
VOCAB = 33000  # 4125 groups of 8: every one of 8 CTAs has work


def rows_at(ctas, edge):
    """Few and many rows that are split over `ctas` each: two CTAs an SM in all, clusters not quite as many."""
    slots = 2 * torch_cuda().cuda.get_device_properties(0).multi_processor_count
    least = 1 if ctas == 8 else slots // (2 * ctas) + 1
    return least if edge == 'least' else slots // 2 + 40 if ctas == 1 else slots // ctas * 7 // 8


def deciding(seed, rows, vocab):
    """Rows whose deciding values lie in the part of CTA r % 8 (of fewer CTAs: in its half or quarter)."""
    x, u = rows_of(seed, rows, vocab)
    r = np.random.default_rng(seed + 1)
    for i in range(rows):
        part = np.arange(vocab * (i % 8) // 8, vocab * (i % 8 + 1) // 8)
        some = r.choice(part, 12, replace=False)
        kind = i % 5
        if kind == 0:    # the largest alone
            x[i, some[0]] = 14.0
        elif kind == 1:  # a mask leaves tokens of one part
            hidden = (-INF, LOWEST, -1e4)[i % 3]
            keep = x[i, some]
            x[i] = hidden
            x[i, some] = keep
        elif kind == 2:  # a value that the usual window does not hold
            x[i, some[0]] = 300.0
            x[i, some[1:]] = 299.0
        elif kind == 3:
            x[i, some[0]] = 2.0 ** -41
        else:            # the lowest values still have weight
            x[i, some[:3]] = -257.0
    return x, u


@pytest.mark.parametrize('ctas', [8, 4, 2, 1])
@pytest.mark.parametrize('edge', ['least', 'most'])
def test_every_part_of_a_row_counts(ctas, edge):
    rows = rows_at(ctas, edge)
    x, u = deciding(ctas, rows, VOCAB)
    i = np.arange(rows)
    check_all(x, u, np.where(i % 5 == 4, 60.0, 0.9))
    check_all(x, u, np.linspace(0.3, 1.5, rows), i % 7 * 11, np.linspace(0.4, 1.1, rows), np.linspace(0, 0.1, rows))


@pytest.mark.parametrize('rows', [1, 32, 40, 64, 100, 190])
def test_vocabularies_that_take_several_loads_of_a_thread(rows):
    """151936 logits: 3 to 38 groups of a thread, by the number of CTAs."""
    x, u = deciding(rows, rows, 151936)
    check_all(x, u, 0.8, np.where(np.arange(rows) % 3 == 0, 50, 0), 0.95, np.where(np.arange(rows) % 3 == 1, 0.05, 0.0))


def test_many_launches_of_clusters_agree():
    """CTAs of a cluster start in any order: the same rows over and over, the SMs busy with another stream's rows."""
    torch = torch_cuda()
    jobs = []
    for seed, rows in enumerate((3, 32, 37, 70, 148, 200)):
        x, u = deciding(seed, rows, VOCAB)
        logits, ud = dev(to_bits(x).view(np.int16)), dev(u)
        tokens, probs = dev(np.zeros((20, rows), np.int32)), dev(np.zeros((20, rows), np.float32))
        jobs.append((values(to_bits(x)), u, logits, ud, tokens, probs, torch.cuda.Stream()))
    sync()
    for i in range(20):
        for x, u, logits, ud, tokens, probs, st in jobs:
            assert L().qwen_b200_op_sample(vp(logits), VOCAB, len(u), VOCAB, None, None, None, None, vp(ud), vp(tokens[i]),
                                           vp(probs[i]), ctypes.c_void_p(st.cuda_stream)) == 0
    sync()
    for x, u, logits, ud, tokens, probs, st in jobs:
        t, p = host(tokens).view(np.uint32), host(probs)
        assert (t == t[0]).all() and (p == p[0]).all()
        assert sum(check(int(t[0, r]), p[0, r], x[r], u[r]) is not False for r in range(len(u))) >= len(u) - 1
