"""Sizes that the paged prompt attention can count in 32 bits are taken, larger
ones are refused; so are softmax scales whose product with log2(e) is not finite. Runs without a GPU: a call that passes the checks of its
numbers goes on to look at its (made-up) pointers, which EDEVICE shows there;
on a machine with a GPU those are refused with EINVAL too, so only the refusals
are told apart there."""
import ctypes

import pytest

import qwen_b200
from qwen_b200 import _lib
from test_paged_refusals import A, calls, kv


def has_gpu():
    import torch
    return torch.cuda.is_available()


def prefill(max_tokens, rows, q_heads, kv_heads=1, dim=64, n=1, window=0, sinks=0):
    c = kv(layers=1, pages=1 << 20, kv_heads=kv_heads, page_tokens=256, head_dim=dim, max_pages=max_tokens // 256,
           page_stride=kv_heads * 256, layer_stride=0)
    return qwen_b200.lib().qwen_b200_op_paged_prefill(ctypes.byref(c), 0, A, q_heads * dim, q_heads, n, None, A, rows, window,
                                                      sinks, 0.125, A, q_heads * dim, A, 1 << 40, None)


@pytest.mark.parametrize('args', [
    # one prompt of 2^22 tokens, 32 heads on one: 2^18 tiles and 2^15 blocks of the table, 2^32 + 2^17 blocks to visit
    dict(max_tokens=1 << 22, rows=1 << 22, q_heads=32),
    dict(max_tokens=1 << 22, rows=1 << 22, q_heads=16, dim=128),
    # a chunk of 2^20 rows on a context of 64 million tokens, 1.7e10 blocks
    dict(max_tokens=1 << 26, rows=1 << 20, q_heads=8, dim=128),
    dict(max_tokens=1 << 26, rows=1 << 20, q_heads=64, kv_heads=8, dim=128),
    dict(max_tokens=1 << 30, rows=65536, q_heads=8, n=65536),
    # a window does not help where its first tokens or its width are as long
    dict(max_tokens=1 << 26, rows=1 << 20, q_heads=8, dim=128, window=64, sinks=0xffffffff),
    dict(max_tokens=1 << 26, rows=1 << 20, q_heads=8, dim=128, window=0xffffffff),
], ids=str)
def test_prompts_of_more_blocks_than_32_bits_count_are_refused(args):
    assert prefill(**args) == _lib.EINVAL


@pytest.mark.skipif('has_gpu()')
@pytest.mark.parametrize('args', [
    dict(max_tokens=1 << 20, rows=1 << 20, q_heads=32),
    dict(max_tokens=1 << 22, rows=1 << 22, q_heads=15),  # (2^22 * 15 / 512 + 1) * 2^15 is 4.03e9
    dict(max_tokens=1 << 30, rows=1 << 15, q_heads=7),
    dict(max_tokens=1 << 26, rows=1 << 20, q_heads=8, dim=128, window=4096, sinks=64),
    dict(max_tokens=1 << 30, rows=65536, q_heads=8, n=65536, window=1024),
], ids=str)
def test_prompts_that_can_be_counted_pass_the_checks_of_their_sizes(args):
    assert prefill(**args) == _lib.EDEVICE


def test_the_bound_holds_every_block_that_a_tile_visits():
    """The host's bound against the device's rule, in Python, over tiles at every place of a context."""
    def span(pos, window, sinks):
        low = pos + 1 - window if window and pos >= window else 0
        return min(sinks, low), low

    for tile in (512, 256):
        for group in (1, 3, 7, 8, 33, 600):
            for window, sinks in ((1, 0), (100, 4), (128, 130), (1000, 64), (5, 700)):
                bound = (window + tile // group + 1) // 128 + 2 + (sinks + 127) // 128
                for pos0 in list(range(-3, 140, 7)) + list(range(1000, 1300, 13)):
                    for k in range(4):
                        first, last = max(pos0 + k * tile // group, 0), pos0 + (k * tile + tile - 1) // group
                        if last < 0:
                            continue
                        low = span(first, window, sinks)[1]
                        lead = min((span(last, window, sinks)[0] + 127) >> 7, low >> 7)
                        assert lead + (last >> 7) + 1 - (low >> 7) <= bound


@pytest.mark.parametrize('op', ['decode', 'prefill'])
@pytest.mark.parametrize('scale', [2.4e38, -2.4e38, 2.99e38])
def test_scales_whose_factor_would_be_infinite_are_refused(op, scale):
    assert calls(kv(), scale=scale)[op]() == _lib.EINVAL


@pytest.mark.skipif('has_gpu()')
@pytest.mark.parametrize('op', ['decode', 'prefill'])
@pytest.mark.parametrize('scale', [2.0e38, -2.0e38, 0.0, 1e-44])
def test_scales_that_can_be_used_pass(op, scale):
    assert calls(kv(), scale=scale)[op]() == _lib.EDEVICE
