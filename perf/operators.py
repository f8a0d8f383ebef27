"""The operators of the paged key-value cache: their workloads, their plain forms
in elementary torch operations, and their values in 64 bits.

  append   keys and values of new tokens written into the cache's pages, as
           bf16 or quantised to 8 bits per (token, head)
  decode   attention of one new token per sequence over its pages, with an
           optional sliding window and first tokens that stay visible
  prefill  attention of the newest rows of several sequences over their pages,
           causal, with the same window and first tokens
  pages    finished sequences freed, prefixes forked, sequences grown by new
           tokens, and the pages in use compacted to the front of the pool

`own` selects the library's kernels (libqwen_b200's paged entry points); without
it every operator runs in its plain form.
"""
import ctypes
import math
import random
import sys
from pathlib import Path

import torch

own = False

PACKAGE = 'fpga2026-40999-llm-accelerator-for-qwen2.5-0.5b-on-fpga_b200'
# the model's geometry (14 query heads on 2 KV heads of 64) and a generic larger one
SMALL = {'q_heads': 14, 'kv_heads': 2, 'dim': 64}
LARGE = {'q_heads': 32, 'kv_heads': 8, 'dim': 128}


def listed():
    return [
        # one new token of each of 64 sequences: the append of a batched decode step
        {'name': 'append step', 'op': 'append', 'format': 'kv8', **SMALL, 'page': 64, 'seqs': 64, 'ctx': 2048,
         'rows': 1, 'ragged': False, 'idle': 0, 'lens': 1},
        # eight prompts of up to 4096 tokens written at once after their prefill
        {'name': 'append prompts', 'op': 'append', 'format': 'bf16', **LARGE, 'page': 128, 'seqs': 8, 'ctx': 4096,
         'rows': 4096, 'ragged': True, 'idle': 0, 'lens': 2},
        # the same prompts in the model's own cache
        {'name': 'append prompts kv8', 'op': 'append', 'format': 'kv8', **SMALL, 'page': 64, 'seqs': 8, 'ctx': 4096,
         'rows': 4096, 'ragged': True, 'idle': 1, 'lens': 3},
        # a single short chat: nothing but latency
        {'name': 'decode short', 'op': 'decode', 'format': 'kv8', **SMALL, 'page': 16, 'seqs': 1, 'ctx': 96,
         'window': 0, 'sinks': 0, 'ragged': False, 'idle': 0, 'lens': 4},
        # batched serving: 64 sequences at context 2048
        {'name': 'decode batch', 'op': 'decode', 'format': 'kv8', **SMALL, 'page': 64, 'seqs': 64, 'ctx': 2048,
         'window': 0, 'sinks': 0, 'ragged': False, 'idle': 0, 'lens': 5},
        # one long document: the only parallelism is along the context
        {'name': 'decode long', 'op': 'decode', 'format': 'bf16', **LARGE, 'page': 128, 'seqs': 1, 'ctx': 32768,
         'window': 0, 'sinks': 0, 'ragged': False, 'idle': 0, 'lens': 6},
        # a batch of very different contexts with empty slots, each row limited to a window behind 4 first tokens
        {'name': 'decode window ragged', 'op': 'decode', 'format': 'kv8', **SMALL, 'page': 16, 'seqs': 256,
         'ctx': 8192, 'window': 1024, 'sinks': 4, 'ragged': True, 'idle': 16, 'lens': 7},
        # the last 16 rows of one prompt over a cached prefix
        {'name': 'prefill chunk', 'op': 'prefill', 'format': 'kv8', **SMALL, 'page': 64, 'seqs': 1, 'ctx': 1000,
         'rows': 16, 'window': 256, 'sinks': 4, 'ragged': False, 'idle': 0, 'lens': 8},
        # eight whole prompts of 4096 tokens, sliding window of 1024
        {'name': 'prefill prompts window', 'op': 'prefill', 'format': 'kv8', **SMALL, 'page': 64, 'seqs': 8,
         'ctx': 4096, 'rows': 4096, 'window': 1024, 'sinks': 4, 'ragged': False, 'idle': 0, 'lens': 9},
        # prompts of up to 8192 tokens, bf16 cache, window of 4096: the longest products
        {'name': 'prefill long', 'op': 'prefill', 'format': 'bf16', **LARGE, 'page': 128, 'seqs': 3, 'ctx': 8192,
         'rows': 8192, 'window': 4096, 'sinks': 16, 'ragged': True, 'idle': 0, 'lens': 10},
        # parallel sampling in a small server: one finished sequence freed, its prompt's other samples forked
        {'name': 'pages fork', 'op': 'pages', 'format': 'kv8', **SMALL, 'page': 64, 'layers': 24, 'pool': 128,
         'seqs': 8, 'ctx': 256, 'free': 1, 'fork': 3, 'compact': False, 'lens': 11},
        # a busy pool: some sequences end, others fork, all grow by a token, and the pool is compacted
        {'name': 'pages turnover', 'op': 'pages', 'format': 'bf16', **SMALL, 'page': 64, 'layers': 24, 'pool': 2048,
         'seqs': 128, 'ctx': 2048, 'free': 16, 'fork': 32, 'compact': True, 'lens': 12},
    ]


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c['op'] == op) for op in ('append', 'decode', 'prefill', 'pages')}

    def span(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))

    while True:
        op = rng.choice(('append', 'decode', 'prefill', 'pages'))
        dim = rng.choice((64, 128))
        kv_heads = span(1, 8)
        case = {'op': op, 'format': rng.choice(('kv8', 'bf16')), 'q_heads': kv_heads * rng.choice((1, 2, 4, 7, 8)),
                'kv_heads': kv_heads, 'dim': dim, 'page': rng.choice((16, 32, 64, 128)), 'lens': rng.randrange(1 << 30)}
        if op == 'pages':
            seqs = span(6, 128)
            case |= {'layers': span(1, 24), 'seqs': seqs, 'ctx': span(16, 2048), 'free': rng.randint(0, seqs // 6),
                     'fork': rng.randint(1, seqs // 3), 'compact': rng.random() < 0.5}
            case['pool'] = sum(-(-t // case['page']) for t in _lengths(case)) + 3 * seqs + span(1, 64)
        else:
            case |= {'seqs': span(1, 256 if op == 'decode' else 64), 'ctx': span(1, 32768 if op == 'decode' else 8192),
                     'ragged': rng.random() < 0.7}
            case['idle'] = rng.randint(0, case['seqs'] // 4)
            if op != 'decode':
                case['rows'] = span(1, case['ctx'])
            if op != 'append':
                window = rng.choice((0, span(1, max(2, case['ctx']))))
                case |= {'window': window, 'sinks': rng.choice((0, 1, 4, 64)) if window else 0}
        if _cost(case) > most[op]:
            continue
        # what the plain forms hold at once: padded scores and gathered pages in 64 bits
        longest, heads = max(_lengths(case)), case['q_heads']
        pad = case['seqs'] * longest * (heads * max(_rows(case)) + 4 * kv_heads * dim) if op in ('decode', 'prefill') else 0
        if pad < 2.5e9:
            return case


# ---------------------------------------------------------------- sizes of a case


def _lengths(case):
    """Tokens of each sequence in the cache, the new ones included; idle sequences have none."""
    rng = random.Random(case['lens'])
    n, top = case['seqs'], case['ctx']
    if case['op'] == 'pages':
        # of the slots, a third is empty: forks go there
        return [0 if i < case['seqs'] // 3 else rng.randint(1, top) for i in range(n)]
    lens = [top if i == 0 or not case['ragged'] else
            max(1, round(math.exp(rng.uniform(math.log(max(1, top // 16)), math.log(top))))) for i in range(n)]
    idle = rng.sample(range(1, n), min(case['idle'], n - 1)) if n > 1 else []
    return [0 if i in set(idle) else t for i, t in enumerate(lens)]


def _rows(case):
    """New rows of each sequence: its last tokens."""
    if case['op'] == 'decode':
        return [1] * case['seqs']
    rng = random.Random(case['lens'] + 1)
    most = case['rows']
    return [min(t, most if not case['ragged'] else max(1, round(most * rng.uniform(0.25, 1)))) for t in _lengths(case)]


def _seen(position, window, sinks):
    """Keys visible to the token at `position`."""
    low = max(0, position + 1 - window) if window else 0
    return position + 1 - low + min(sinks, low)


def _row_bytes(case):
    """Bytes of one head's key of one token in the cache."""
    return case['dim'] + 4 if case['format'] == 'kv8' else 2 * case['dim']


def _page_plan(case):
    """Which sequences are freed, forked and grown, and the pages that they hold, drawn from the case."""
    rng = random.Random(case['lens'] + 2)
    lens, T = _lengths(case), case['page']
    live = [i for i, t in enumerate(lens) if t]
    empty = [i for i, t in enumerate(lens) if not t]
    rng.shuffle(live)
    freed = live[:min(case['free'], len(live) - 1)]
    parents = [rng.choice(live[len(freed):]) for _ in range(min(case['fork'], len(empty)))]
    children = rng.sample(empty, len(parents))
    prefix = [rng.randint(1, lens[p]) for p in parents]
    grown = [i for i in live if i not in set(freed)] + children
    ids = rng.sample(range(case['pool']), sum(-(-t // T) for t in lens))
    return freed, parents, children, prefix, grown, ids


def _moves(case):
    """Pages whose data moves: (tokens copied at forks, whole pages at compaction)."""
    T, lens = case['page'], _lengths(case)
    freed, parents, children, prefix, grown, ids = _page_plan(case)
    tails = sum(t % T for t in prefix)
    if not case['compact']:
        return tails, 0
    held, at = set(), 0
    own_pages = {}
    for i, t in enumerate(lens):
        n = -(-t // T)
        own_pages[i] = ids[at:at + n]
        at += n
        if i not in set(freed):
            held.update(own_pages[i])
    now = dict(enumerate(lens))
    spare = iter([p for p in range(case['pool']) if p not in held])
    for p, c, t in zip(parents, children, prefix):
        now[c] = t
        if t % T:
            held.add(next(spare))
    for i in grown:
        if now[i] % T == 0:
            held.add(next(spare))
    return tails, sum(p >= len(held) for p in held)


def work(case):
    hkv, hq, dim, each = case['kv_heads'], case['q_heads'], case['dim'], _row_bytes(case)
    if case['op'] == 'append':
        rows = sum(_rows(case))
        return {'bytes': rows * hkv * 2 * (2 * dim + each), 'flops': 0}
    if case['op'] == 'pages':
        tails, pages = _moves(case)
        tables = 4 * (case['pool'] + sum(-(-t // case['page']) for t in _lengths(case)))
        return {'bytes': 2 * (2 * case['layers'] * hkv * each * (tails + pages * case['page']) + tables), 'flops': 0}
    read = pairs = rows = 0
    for t, r in zip(_lengths(case), _rows(case)):
        if not t:
            continue
        first = _seen(t - r, case['window'], case['sinks'])
        read += first + r - 1  # each later row sees one key that no earlier one does
        rows += r
        if case['window'] and r > 1:
            pairs += sum(_seen(p, case['window'], case['sinks']) for p in range(t - r, t))
        elif r > 1:
            pairs += r * (t - r) + r * (r + 1) // 2
        else:
            pairs += first
    return {'bytes': read * hkv * 2 * each + rows * hq * dim * 4, 'flops': 4 * pairs * hq * dim}


def _cost(case):
    w = work(case)
    return max(w['bytes'], w['flops'] / 50)


# ---------------------------------------------------------------- inputs


def _quantised(x):
    """8-bit codes and the scale of each row: scale = amax / 127, code = the nearest whole number to x / scale, all in fp32."""
    amax = x.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    codes = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-127, 127)
    return codes.to(torch.int8), scale.squeeze(-1)


def _pool(case, layers, pages, gen):
    """K and V pools [layers][pages][kv_heads][page][dim] (and scales without the last axis) of unit-variance entries."""
    shape = (layers, pages, case['kv_heads'], case['page'], case['dim'])
    out = []
    for _ in range(2):
        if case['format'] == 'bf16':
            out.append((torch.randn(shape, generator=gen, device='cuda', dtype=torch.bfloat16), None))
        else:
            codes = torch.empty(shape, device='cuda', dtype=torch.int8)
            scales = torch.empty(shape[:-1], device='cuda', dtype=torch.float32)
            for l in range(layers):
                codes[l], scales[l] = _quantised(torch.randn(shape[1:], generator=gen, device='cuda'))
            out.append((codes, scales))
    return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    rng = random.Random(seed)
    lens, T = _lengths(case), case['page']
    counts = [-(-t // T) for t in lens]
    s = {'case': case, 'width': max(1, max(counts))}
    if case['op'] == 'pages':
        freed, parents, children, prefix, grown, ids = _page_plan(case)
        pages, layers = case['pool'], case['layers']
        s['width'] = max(counts) + 2
        s |= {'freed': _ints(freed), 'parents': _ints(parents), 'children': _ints(children), 'prefix': _ints(prefix),
              'grown': _ints(grown), 'ones': _ints([1] * len(grown)), 'status': _ints([0, 0])}
    else:
        pages, layers = sum(counts) + 3, 1
        ids = rng.sample(range(pages), sum(counts))
    table = torch.zeros(case['seqs'], s['width'], dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    refs[torch.tensor(ids, dtype=torch.int64)] = 1
    # the page table, the lengths and the reference counts lie in one allocation
    book = torch.cat([table.flatten(), torch.tensor(lens, dtype=torch.int32), refs]).cuda()
    n = table.numel()
    s |= {'book': book, 'table': book[:n].view_as(table), 'lengths': book[n:n + len(lens)], 'refs': book[n + len(lens):]}
    (s['k'], s['kscales']), (s['v'], s['vscales']) = _pool(case, layers, pages, gen)
    if case['op'] == 'pages':
        s['before'] = book.clone()
        s['workspace'] = torch.zeros(4096 + 64 * pages, dtype=torch.uint8, device='cuda')
        return s
    hq, hkv, dim, rows = case['q_heads'], case['kv_heads'], case['dim'], _rows(case)
    total = sum(rows)
    # a fused projection's output: query, key and value heads of a token side by side
    qkv = torch.randn(total, hq + 2 * hkv, dim, generator=gen, device='cuda', dtype=torch.bfloat16)
    # sharper than uniform attention: the logits' standard deviation is 2
    qkv[:, :hq] *= 2
    s |= {'q': qkv[:, :hq], 'new_k': qkv[:, hq:hq + hkv], 'new_v': qkv[:, hq + hkv:],
          'scale': dim ** -0.5, 'ctx': torch.empty(total, hq, dim, device='cuda', dtype=torch.bfloat16)}
    order = list(range(case['seqs']))
    rng.shuffle(order)
    starts = [0]
    for i in order:
        starts.append(starts[-1] + rows[i])
    s |= {'seqs': _ints(order), 'starts': _ints(starts), 'most': max(rows)}
    if case['op'] == 'append':
        s['row_seqs'] = _ints([i for i in order for _ in range(rows[i])])
        s['positions'] = _ints([p for i in order for p in range(lens[i] - rows[i], lens[i])])
        row = torch.arange(total, device='cuda')
        page = s['table'][s['row_seqs'].long(), (s['positions'] // T).long()].long()
        # the cache rows (per head) that the new tokens fall on
        s['where'] = ((page * hkv)[:, None] + torch.arange(hkv, device='cuda')) * T + (s['positions'] % T).long()[:, None]
        del row
    else:
        s['workspace'] = torch.zeros(96 << 20, dtype=torch.uint8, device='cuda')
    return s


# ---------------------------------------------------------------- one pass


def run(s):
    if own:
        return _own_run(s)
    return {'append': _append, 'decode': _attention, 'prefill': _attention, 'pages': _turnover}[s['case']['op']](s)


def _read_back(s):
    """The values that the cache holds for the new rows."""
    dim = s['case']['dim']
    out = []
    for pool, scales in ((s['k'], s['kscales']), (s['v'], s['vscales'])):
        if scales is None:
            out.append(pool)
        else:
            out.append(pool.view(-1, dim)[s['where']] * scales.view(-1)[s['where']].unsqueeze(-1))
    return out


def _append(s):
    dim = s['case']['dim']
    for x, pool, scales in ((s['new_k'], s['k'], s['kscales']), (s['new_v'], s['v'], s['vscales'])):
        if scales is None:
            pool.view(-1, dim)[s['where']] = x
        else:
            pool.view(-1, dim)[s['where']], scales.view(-1)[s['where']] = _quantised(x.float())
    return _read_back(s)


def _gathered(s, name):
    """[sequence][kv head][position][dim] in 32 bits, in the order of s['seqs']."""
    pool, scales = s[name][0], s[name + 'scales']
    pages = s['table'][s['seqs'].long()].long()
    x = pool[pages].float()
    if scales is not None:
        x = x * scales[0][pages].unsqueeze(-1)
    n, p, h, t, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, h, p * t, d)


def _attention(s):
    case = s['case']
    hkv, group, window, sinks = case['kv_heads'], case['q_heads'] // case['kv_heads'], case['window'], case['sinks']
    lens, starts = s['lengths'][s['seqs'].long()].long(), s['starts'].long()
    rows = starts[1:] - starts[:-1]
    k, v = _gathered(s, 'k'), _gathered(s, 'v')
    n, _, keys, dim = k.shape
    # each sequence's rows side by side, padded to the longest
    r = torch.arange(s['most'], device='cuda')
    there = r < rows[:, None]
    q = torch.zeros(n, s['most'], hkv, group, dim, device='cuda')
    q[there] = s['q'].float().unflatten(1, (hkv, group))
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, dim), k.transpose(2, 3)) * s['scale']
    scores = scores.view(n, hkv, group, s['most'], keys)
    position = (lens - rows)[:, None] + r
    j = torch.arange(keys, device='cuda')
    seen = (j <= position[..., None]) & (j < lens[:, None, None]) & there[..., None]
    if window:
        seen &= (position[..., None] - j < window) | (j < sinks)
    seen = seen[:, None, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = v.masked_fill((j >= lens[:, None])[:, None, :, None], 0)
    out = torch.matmul(scores.view(n, hkv, -1, keys), v).view(n, hkv, group, s['most'], dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    s['ctx'].copy_(out.permute(0, 3, 1, 2, 4)[there].flatten(1, 2))
    return s['ctx']


def _fresh(refs, count):
    return torch.nonzero(refs == 0).flatten()[:count]


def _turnover(s):
    case, T = s['case'], s['case']['page']
    s['book'].copy_(s['before'])
    table, lengths, refs = s['table'], s['lengths'], s['refs']
    column = torch.arange(table.shape[1], device='cuda')
    one = torch.ones((), dtype=torch.int32, device='cuda')

    def held(rows):
        return column < ((lengths[rows] + T - 1) // T)[:, None]

    # free
    f = s['freed'].long()
    ids = table[f][held(f)].long()
    refs.index_add_(0, ids, -one.expand(ids.numel()))
    lengths[f] = 0
    # fork: full pages are shared, the tail of a prefix is copied to a page of its own
    p, c, prefix = s['parents'].long(), s['children'].long(), s['prefix']
    full, tail = prefix // T, prefix % T
    shared = column < full[:, None]
    ids = table[p][shared].long()
    refs.index_add_(0, ids, one.expand(ids.numel()))
    table[c] = torch.where(shared, table[p], table[c])
    cut = torch.nonzero(tail > 0).flatten()
    src = table[p[cut], full[cut].long()].long()
    dst = _fresh(refs, cut.numel())
    table[c[cut], full[cut].long()] = dst.int()
    refs[dst] = 1
    lengths[c] = prefix
    copied = torch.arange(T, device='cuda') < tail[cut][:, None, None]
    for x in _pools(s):
        w = copied[..., None] if x.dim() == 5 else copied
        x[:, dst] = torch.where(w, x[:, src], x[:, dst])
    # grow by one token each
    g = s['grown'].long()
    old = lengths[g]
    new = old + s['ones']
    need = torch.nonzero((new + T - 1) // T > (old + T - 1) // T).flatten()
    dst = _fresh(refs, need.numel())
    table[g[need], (old[need] // T).long()] = dst.int()
    refs[dst] = 1
    lengths[g] = new
    # compact: the i-th free page of the front takes the i-th page in use behind it
    if case['compact']:
        live = refs > 0
        count = live.sum()
        index = torch.arange(refs.numel(), device='cuda')
        holes, movers = torch.nonzero(~live & (index < count)).flatten(), torch.nonzero(live & (index >= count)).flatten()
        for x in _pools(s):
            x[:, holes] = x[:, movers]
        refs[holes] = refs[movers]
        refs[movers] = 0
        index[movers] = holes
        inside = column < ((lengths + T - 1) // T)[:, None]
        table[inside] = index[table[inside].long()].int()
    s['status'][0] = 0
    s['status'][1] = (refs == 0).sum()
    return _page_outputs(s)


def _pools(s):
    return [x for x in (s['k'], s['v'], s['kscales'], s['vscales']) if x is not None]


def _page_outputs(s):
    # pages move as they are: codes of 8 bits have to be the same codes
    return [s['table'], s['lengths'], s['refs'], s['status'], *_pools(s)]


# ---------------------------------------------------------------- the library's calls


def _library():
    root = str(Path(__file__).resolve().parents[1] / PACKAGE)
    if root not in sys.path:
        sys.path.insert(0, root)
    import qwen_b200
    return qwen_b200


def _descriptor(q, s):
    """What the library's calls know a cache by: addresses and sizes, kept by a program as long as the cache."""
    layers, pages, hkv, T, dim = s['k'].shape
    kv8 = s['kscales'] is not None
    return q.PagedKV(k=s['k'].data_ptr(), v=s['v'].data_ptr(), kscales=s['kscales'].data_ptr() if kv8 else None,
                     vscales=s['vscales'].data_ptr() if kv8 else None, table=s['table'].data_ptr(),
                     lengths=s['lengths'].data_ptr(), refs=s['refs'].data_ptr(), layer_stride=pages * hkv * T,
                     page_stride=hkv * T, format=q.KV8 if kv8 else q.KV_BF16, layers=layers, pages=pages, kv_heads=hkv,
                     page_tokens=T, head_dim=dim, seqs=s['case']['seqs'], max_pages=s['width'])


def _own_run(s):
    if 'library' not in s:
        s['library'] = _library()
        s['descriptor'] = _descriptor(s['library'], s)
    q, kv, case = s['library'], ctypes.byref(s['descriptor']), s['case']
    lib, op = q.lib(), case['op']
    st = torch.cuda.current_stream().cuda_stream
    if op == 'append':
        q.check(lib.qwen_b200_op_paged_append(kv, 0, s['new_k'].data_ptr(), s['new_v'].data_ptr(),
                                              s['new_k'].stride(0), s['row_seqs'].numel(), s['row_seqs'].data_ptr(),
                                              s['positions'].data_ptr(), st))
        return _read_back(s)
    ws, ws_bytes = s['workspace'].data_ptr(), s['workspace'].numel()
    if op == 'decode':
        q.check(lib.qwen_b200_op_paged_decode(kv, 0, s['q'].data_ptr(), s['q'].stride(0), case['q_heads'],
                                              case['seqs'], s['seqs'].data_ptr(), case['window'], case['sinks'],
                                              s['scale'], s['ctx'].data_ptr(), s['ctx'].stride(0), ws, ws_bytes, st))
        return s['ctx']
    if op == 'prefill':
        q.check(lib.qwen_b200_op_paged_prefill(kv, 0, s['q'].data_ptr(), s['q'].stride(0), case['q_heads'],
                                               case['seqs'], s['seqs'].data_ptr(), s['starts'].data_ptr(),
                                               s['q'].shape[0], case['window'], case['sinks'], s['scale'],
                                               s['ctx'].data_ptr(), s['ctx'].stride(0), ws, ws_bytes, st))
        return s['ctx']
    status = s['status'].data_ptr()
    s['book'].copy_(s['before'])
    if s['freed'].numel():
        q.check(lib.qwen_b200_op_pages_free(kv, s['freed'].data_ptr(), s['freed'].numel(), status, ws, ws_bytes, st))
    q.check(lib.qwen_b200_op_pages_fork(kv, s['parents'].data_ptr(), s['children'].data_ptr(), s['prefix'].data_ptr(),
                                        s['parents'].numel(), status, ws, ws_bytes, st))
    q.check(lib.qwen_b200_op_pages_reserve(kv, s['grown'].data_ptr(), s['ones'].data_ptr(), s['grown'].numel(), status,
                                           ws, ws_bytes, st))
    if case['compact']:
        q.check(lib.qwen_b200_op_pages_compact(kv, status, ws, ws_bytes, st))
    return _page_outputs(s)


# ---------------------------------------------------------------- in 64 bits


def exact(case, seed):
    if case['op'] == 'pages':
        return None  # nothing is computed: the outputs are copies and whole numbers
    s = prepare(case, seed)
    if case['op'] == 'append':
        return _exact_append(s)
    lens, table, T, dim = s['lengths'].tolist(), s['table'].long(), case['page'], case['dim']
    starts, hkv, group = s['starts'].tolist(), case['kv_heads'], case['q_heads'] // case['kv_heads']
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda')
    for i, seq in enumerate(s['seqs'].tolist()):
        t, a, b = lens[seq], starts[i], starts[i + 1]
        if not t or a == b:
            continue
        token = torch.arange(t, device='cuda')
        page, offset = table[seq][token // T], token % T
        first = t - (b - a)
        for h in range(hkv):
            k, v = s['k'][0, page, h, offset].double(), s['v'][0, page, h, offset].double()
            if s['kscales'] is not None:
                k *= s['kscales'][0, page, h, offset].double()[:, None]
                v *= s['vscales'][0, page, h, offset].double()[:, None]
            for lo in range(a, b, 1024):
                hi = min(b, lo + 1024)
                at = torch.arange(first + lo - a, first + hi - a, device='cuda')
                hidden = token[None] > at[:, None]
                if case['window']:
                    hidden |= (token[None] <= at[:, None] - case['window']) & (token[None] >= case['sinks'])
                x = torch.einsum('rgd,td->grt', s['q'][lo:hi, h * group:(h + 1) * group].double(), k) * s['scale']
                w = torch.softmax(x.masked_fill(hidden[None], -math.inf), -1)
                out[lo:hi, h * group:(h + 1) * group] = torch.einsum('grt,td->rgd', w, v)
    return out


def _exact_append(s):
    out = []
    for x, pool, scales in ((s['new_k'], s['k'], s['kscales']), (s['new_v'], s['v'], s['vscales'])):
        x = x.double()
        if scales is None:
            y = pool.double()
            y.view(-1, x.shape[-1])[s['where'].flatten()] = x.flatten(0, 1)
            out.append(y)
            continue
        # the cache's rule: the scale and the quotient are values of 32 bits (a quotient in 64 bits rounds to
        # the same 32-bit value), the code is the nearest whole number, the even one of two
        top = x.abs().max(-1, keepdim=True).values
        step = (top / torch.tensor(127.0, dtype=torch.float64, device='cuda')).float().double()
        ratio = torch.nan_to_num(x / step).float().double()
        out.append(torch.clamp(torch.round(ratio), -127, 127) * step)
    return out
