"""A process whose first call of an entry point is captured into a graph: what a call
looks up or sets once (sizes of clusters, limits of shared memory) has to work there.
Each runs in a process of its own and compares a replay with a call behind it."""
import os
import subprocess
import sys

import pytest

from conftest import PKG, REPO

pytestmark = pytest.mark.gpu

SETUP = '''
import ctypes
import torch
import qwen_b200
from qwen_b200 import _lib
L = qwen_b200.lib()
dev = dict(device='cuda')
g = torch.Generator('cuda').manual_seed(1)
bf = lambda *s: torch.randn(*s, generator=g, dtype=torch.bfloat16, **dev)
ints = lambda v: torch.tensor(v, dtype=torch.int32, **dev)
stream = lambda: torch.cuda.current_stream().cuda_stream
ROWS, DIM, HKV, HEADS, T, PAGES = 200, 64, 8, 16, 64, 640
table = torch.randn(1000, DIM, generator=g, **dev)
rotation = qwen_b200.Rotary(table=table.data_ptr(), positions=1000, rotated=DIM, layout=0)
def cache(fmt, rows=ROWS, width=16):
    shape = (PAGES, HKV, T, DIM)
    if fmt == 0:
        k, v = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, **dev) for _ in range(2))
        scales = torch.rand(shape[:3], generator=g, **dev) * 0.02
    else:
        k, v, scales = bf(*shape), bf(*shape), torch.zeros(4, **dev)
    tab = (torch.arange(rows * width, **dev) % PAGES).to(torch.int32).view(rows, width)
    tab[:, :10] = torch.arange(10, dtype=torch.int32, **dev)
    lengths = ints([600 + i % 40 for i in range(rows)])
    kv = qwen_b200.PagedKV(k=k.data_ptr(), v=v.data_ptr(), kscales=scales.data_ptr(), vscales=scales.data_ptr(), table=tab.data_ptr(),
                           lengths=lengths.data_ptr(), refs=None, layer_stride=PAGES * HKV * T, page_stride=HKV * T, format=fmt,
                           layers=1, pages=PAGES, kv_heads=HKV, page_tokens=T, head_dim=DIM, seqs=rows, max_pages=width)
    return kv, (k, v, scales, tab, lengths)
def shared(fmt, rows, width):
    kv, held = cache(fmt, rows, width)
    q, out = bf(rows, HEADS * DIM), torch.zeros(rows, HEADS * DIM, dtype=torch.bfloat16, **dev)
    starts, prefix = ints([0, rows]), ints([600])
    n = L.qwen_b200_paged_decode_shared_workspace(ctypes.byref(kv), HEADS, 1, rows)
    ws = torch.zeros(n, dtype=torch.uint8, **dev)
    def call():
        _ = held
        return L.qwen_b200_op_paged_decode_shared(ctypes.byref(kv), 0, q.data_ptr(), HEADS * DIM, HEADS, 1, starts.data_ptr(), prefix.data_ptr(),
                                                  rows, None, 0.125, out.data_ptr(), HEADS * DIM, ws.data_ptr(), n, stream())
    return call, out
def sample(rows):
    x, u, tokens = bf(rows, 40000), torch.rand(rows, generator=g, **dev), ints([7] * rows)
    return lambda: L.qwen_b200_op_sample(x.data_ptr(), 40000, rows, 40000, None, None, None, None, u.data_ptr(), tokens.data_ptr(), None,
                                         stream()), tokens
def rotary():
    x, out, pos = bf(ROWS, 1024), torch.zeros(ROWS, 1024, dtype=torch.bfloat16, **dev), ints([i % 1000 for i in range(ROWS)])
    return lambda: L.qwen_b200_op_rotary(ctypes.byref(rotation), x.data_ptr(), 1024, 16, 64, ROWS, pos.data_ptr(), out.data_ptr(), 1024,
                                         stream()), out
def append(fmt):
    kv, held = cache(fmt)
    x, out = bf(ROWS, 2048), torch.zeros(ROWS, 1024, dtype=torch.bfloat16, **dev)
    seqs, pos = ints(list(range(ROWS))), ints([599] * ROWS)
    def call():
        _ = held
        return L.qwen_b200_op_paged_append_rotary(ctypes.byref(kv), 0, ctypes.byref(rotation), x.data_ptr(), 2048, 16, out.data_ptr(), 1024,
                                                  x.data_ptr() + 2048, x.data_ptr() + 3072, 2048, ROWS, seqs.data_ptr(), pos.data_ptr(), stream())
    return call, out
call, out = {make}
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    assert call() == 0
graph.replay()
torch.cuda.synchronize()
first = out.clone()
assert first.float().abs().sum() > 0
out.zero_()
assert call() == 0
torch.cuda.synchronize()
assert torch.equal(first, out)
print('same')
'''


@pytest.mark.parametrize('make', ['sample(3)', 'sample(300)', 'rotary()', 'append(0)',
                                  'shared(0, 200, 16)', 'shared(1, 3, 200)',
                                  'shared(0, 70, 2000)'])
def test_first_call(make):
    env = os.environ | {'PYTHONPATH': f'{PKG}{os.pathsep}{REPO}'}
    p = subprocess.run([sys.executable, '-c', SETUP.replace('{make}', make)], env=env, capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.split() == ['same'], p.stderr[-2000:]
