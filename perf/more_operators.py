"""The operators of sampling continuations of shared prompts: their workloads, their
plain forms in elementary torch operations, and their values in 64 bits.

  rotary   rotary positions on query and key heads: pairs in halves or interleaved,
           whole heads or their first dims, angles scaled for long contexts
  append   new tokens into the paged cache with the rotation on the way: queries
           rotated beside it, keys rotated, keys and values as bf16 or 8-bit codes
  shared   attention of one token per sequence where groups of sequences share
           their first tokens, which are read once for a group
  sample   one token per row of logits from a given random number, under a
           temperature, the k largest, a share of the probability and a least
           probability relative to the largest

`own` selects the library's kernels (libqwen_b200's entry points); without it
every operator runs in its plain form.
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
VOCAB = 151936


def listed():
    return [
        # query and key heads of a batched decode step, contexts up to the model's 32768 positions
        {'name': 'rotary step', 'op': 'rotary', **SMALL, 'seqs': 64, 'ctx': 32768, 'rows': 1, 'ragged': True,
         'rotated': 64, 'interleaved': False, 'scaling': 'none', 'factor': 1.0, 'lens': 1},
        # eight prompts of 4096 tokens behind long contexts: half of each head in interleaved pairs
        {'name': 'rotary prompts part', 'op': 'rotary', **LARGE, 'seqs': 8, 'ctx': 65536, 'rows': 4096, 'ragged': False,
         'rotated': 64, 'interleaved': True, 'scaling': 'yarn', 'factor': 4.0, 'lens': 2},
        # one new token of each of 64 sequences: the append of a batched decode step, with its empty slots
        {'name': 'append step', 'op': 'append', 'format': 'kv8', **SMALL, 'page': 64, 'seqs': 64, 'ctx': 2048,
         'rows': 1, 'ragged': False, 'idle': 3, 'rotated': 64, 'interleaved': False, 'scaling': 'none', 'factor': 1.0,
         'lens': 3},
        # eight prompts of up to 4096 tokens after their prefill's projections, the model's own cache
        {'name': 'append prompts kv8', 'op': 'append', 'format': 'kv8', **SMALL, 'page': 64, 'seqs': 8, 'ctx': 4096,
         'rows': 4096, 'ragged': True, 'idle': 1, 'rotated': 64, 'interleaved': False, 'scaling': 'ntk', 'factor': 2.0,
         'lens': 4},
        # the same with larger heads, interleaved pairs and a bf16 cache
        {'name': 'append prompts', 'op': 'append', 'format': 'bf16', **LARGE, 'page': 128, 'seqs': 8, 'ctx': 4096,
         'rows': 4096, 'ragged': True, 'idle': 0, 'rotated': 128, 'interleaved': True, 'scaling': 'linear',
         'factor': 4.0, 'lens': 5},
        # eight samples of one prompt: little but latency
        {'name': 'shared samples', 'op': 'shared', 'format': 'kv8', **SMALL, 'page': 64, 'groups': 1, 'seqs': 8,
         'prefix': 2048, 'own': 64, 'ragged': False, 'idle': 0, 'lens': 6},
        # a server whose requests all begin with one long system prompt
        {'name': 'shared system prompt', 'op': 'shared', 'format': 'kv8', **SMALL, 'page': 64, 'groups': 1, 'seqs': 256,
         'prefix': 4096, 'own': 512, 'ragged': True, 'idle': 5, 'lens': 7},
        # several long documents, each with questions of its own
        {'name': 'shared documents', 'op': 'shared', 'format': 'bf16', **LARGE, 'page': 128, 'groups': 4, 'seqs': 128,
         'prefix': 8192, 'own': 512, 'ragged': True, 'idle': 0, 'lens': 8},
        # one request's token, every filter on
        {'name': 'sample one', 'op': 'sample', 'rows': 1, 'vocab': VOCAB, 'top_k': 50, 'top_p': 0.95, 'min_p': 0.05,
         'mixed': False, 'masked': 0, 'peaked': True, 'lens': 9},
        # a batch of requests with settings of their own, some under a grammar that forbids most tokens
        {'name': 'sample batch', 'op': 'sample', 'rows': 64, 'vocab': VOCAB, 'top_k': 1000, 'top_p': 0.9, 'min_p': 0.02,
         'mixed': True, 'masked': 8, 'peaked': True, 'lens': 10},
        # many rows, a share of the probability alone: every logit counts
        {'name': 'sample many', 'op': 'sample', 'rows': 256, 'vocab': VOCAB, 'top_k': 0, 'top_p': 0.95, 'min_p': 0.0,
         'mixed': False, 'masked': 0, 'peaked': False, 'lens': 11},
    ]


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c['op'] == op) for op in ('rotary', 'append', 'shared', 'sample')}

    def span(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))

    while True:
        op = rng.choice(('rotary', 'append', 'shared', 'sample'))
        case = {'op': op, 'lens': rng.randrange(1 << 30)}
        if op == 'sample':
            case |= {'rows': span(1, 256), 'vocab': span(50, VOCAB), 'top_k': rng.choice((0, 1, span(2, 2000))),
                     'top_p': rng.choice((1.0, rng.uniform(0.05, 0.999))), 'min_p': rng.choice((0.0, rng.uniform(0.001, 0.5))),
                     'mixed': rng.random() < 0.6, 'peaked': rng.random() < 0.6}
            case['masked'] = rng.choice((0, rng.randint(0, case['rows'])))
        else:
            dim, kv_heads = rng.choice((64, 128)), span(1, 8)
            case |= {'q_heads': kv_heads * rng.choice((1, 2, 4, 7, 8)), 'kv_heads': kv_heads, 'dim': dim,
                     'seqs': span(1, 256 if op == 'shared' else 64), 'ragged': rng.random() < 0.7}
            case['idle'] = rng.randint(0, case['seqs'] // 4)
            if op != 'rotary':
                case |= {'format': rng.choice(('kv8', 'bf16')), 'page': rng.choice((16, 32, 64, 128))}
            if op == 'shared':
                case |= {'groups': span(1, min(8, case['seqs'])), 'prefix': span(1, 16384), 'own': span(1, 2048)}
            else:
                case['ctx'] = span(1, 65536 if op == 'rotary' else 8192)
                case['rows'] = span(1, min(case['ctx'], 8192))
                scaling = rng.choice(('none', 'linear', 'ntk', 'yarn'))
                case |= {'rotated': 16 * rng.randint(1, dim // 16), 'interleaved': rng.random() < 0.5, 'scaling': scaling,
                         'factor': 1.0 if scaling == 'none' else rng.uniform(1.5, 8)}
        if _cost(case) <= most[op]:
            return case


# ---------------------------------------------------------------- sizes of a case


def _lengths(case):
    """Tokens of each sequence, the new ones included; idle sequences have none."""
    rng = random.Random(case['lens'])
    n, idle = case['seqs'], set()
    if case.get('idle') and n > 1:
        idle = set(rng.sample(range(1, n), min(case['idle'], n - 1)))
    if case['op'] == 'shared':
        # a sequence has its group's prefix and at least one token of its own
        lens = []
        for members, prefix in _groups(case):
            idle -= {members[0]}  # the prefix is read from the first
            lens += [prefix + (case['own'] if not case['ragged'] else rng.randint(1, case['own'])) for _ in members]
    else:
        top = case['ctx']
        lens = [top if i == 0 or not case['ragged'] else
                max(1, round(math.exp(rng.uniform(math.log(max(1, top // 16)), math.log(top))))) for i in range(n)]
    return [0 if i in idle else t for i, t in enumerate(lens)]


def _groups(case):
    """(sequences, tokens that they share) of each group."""
    rng = random.Random(case['lens'] + 1)
    n, seqs = case['groups'], case['seqs']
    cuts = [0] + (sorted(rng.sample(range(1, seqs), n - 1)) if case['ragged'] else [seqs * i // n for i in range(1, n)]) + [seqs]
    return [(list(range(a, b)), case['prefix'] if i == 0 or not case['ragged'] else
             max(1, round(case['prefix'] * rng.uniform(0.25, 1)))) for i, (a, b) in enumerate(zip(cuts, cuts[1:]))]


def _rows(case):
    """New rows of each sequence: its last tokens."""
    rng = random.Random(case['lens'] + 2)
    most = case['rows']
    return [min(t, most if not case['ragged'] else max(1, round(most * rng.uniform(0.25, 1)))) for t in _lengths(case)]


def _row_bytes(case):
    """Bytes of one head's key of one token in the cache."""
    return case['dim'] + 4 if case['format'] == 'kv8' else 2 * case['dim']


def work(case):
    if case['op'] == 'sample':
        return {'bytes': case['rows'] * (2 * case['vocab'] + 28), 'flops': 0}
    hkv, hq, dim = case['kv_heads'], case['q_heads'], case['dim']
    if case['op'] == 'shared':
        lens = _lengths(case)
        keys = sum(lens)
        for members, prefix in _groups(case):
            keys -= prefix * (sum(lens[i] > 0 for i in members) - 1)
        rows = sum(t > 0 for t in lens)
        return {'bytes': keys * hkv * 2 * _row_bytes(case) + rows * hq * dim * 4, 'flops': 4 * sum(lens) * hq * dim}
    lens, rows = _lengths(case), _rows(case)
    total = sum(rows)
    # each position's row of the table once
    spans, seen, end = sorted((t - r, t) for t, r in zip(lens, rows)), 0, 0
    for a, b in spans:
        seen += max(0, b - max(a, end))
        end = max(end, b)
    table = seen * case['rotated'] * 4
    if case['op'] == 'rotary':
        return {'bytes': total * (hq + hkv) * dim * 4 + table, 'flops': 3 * total * (hq + hkv) * case['rotated']}
    return {'bytes': total * (hq * dim * 4 + hkv * 2 * (2 * dim + _row_bytes(case))) + table,
            'flops': 3 * total * (hq + hkv) * case['rotated']}


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


def _pool(case, pages, gen):
    """K and V pools [1][pages][kv_heads][page][dim] (and scales without the last axis) of unit-variance entries."""
    shape = (1, pages, case['kv_heads'], case['page'], case['dim'])
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen, device='cuda', dtype=torch.bfloat16)
        out.append((x, None) if case['format'] == 'bf16' else _quantised(x.float()))
    return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _table(case, positions):
    """cos | sin of each position's angles, in 64 bits, rounded to 32: [positions][rotated]. A program makes it once."""
    rot, theta, factor = case['rotated'], 1e6, case['factor']
    i = torch.arange(0, rot, 2, dtype=torch.float64, device='cuda')
    size = 1.0
    if case['scaling'] == 'ntk' and rot > 2:
        theta *= factor ** (rot / (rot - 2))
    freq = theta ** (-i / rot)
    if case['scaling'] == 'linear':
        freq /= factor
    if case['scaling'] == 'yarn':
        # frequencies that turn more than 32 times in the 32768 positions of training stay, those that turn less than
        # once are divided by the factor, and a ramp over the dims joins them
        def dim_of(turns):
            return rot * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(dim_of(32)), 0), min(math.ceil(dim_of(1)), rot - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        size = 0.1 * math.log(factor) + 1
    angle = torch.arange(positions, dtype=torch.float64, device='cuda')[:, None] * freq
    return torch.cat([angle.cos() * size, angle.sin() * size], 1).float()


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    rng = random.Random(seed)
    s = {'case': case}
    if case['op'] == 'sample':
        return _prepare_sample(case, s, gen, rng)
    lens, hq, hkv, dim = _lengths(case), case['q_heads'], case['kv_heads'], case['dim']
    if case['op'] != 'shared':
        rows = _rows(case)
        total = sum(rows)
        order = list(range(case['seqs']))
        rng.shuffle(order)
        # a fused projection's output: query, key and value heads of a token side by side
        qkv = torch.randn(total, hq + 2 * hkv, dim, generator=gen, device='cuda', dtype=torch.bfloat16)
        s |= {'table': _table(case, max(lens)), 'q': qkv[:, :hq], 'qk': qkv[:, :hq + hkv], 'new_k': qkv[:, hq:hq + hkv],
              'new_v': qkv[:, hq + hkv:], 'positions': _ints([p for i in order for p in range(lens[i] - rows[i], lens[i])])}
        if case['op'] == 'rotary':
            s['out'] = torch.empty(total, hq + hkv, dim, device='cuda', dtype=torch.bfloat16)
            return s
        s['q_out'] = torch.empty(total, hq, dim, device='cuda', dtype=torch.bfloat16)
        s['row_seqs'] = _ints([i for i in order for _ in range(rows[i])])
    T = case['page']
    counts = [-(-t // T) for t in lens]
    # full pages of a prefix are one page in all its sequences' tables
    owner = list(range(case['seqs']))
    full = [0] * case['seqs']
    if case['op'] == 'shared':
        for members, prefix in _groups(case):
            for i in members[1:]:
                if lens[i]:
                    owner[i], full[i] = members[0], prefix // T
    pages = sum(counts) - sum(full) + 3
    ids = rng.sample(range(pages), pages - 3)
    book = torch.zeros(case['seqs'], max(1, max(counts)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        book[i, :full[i]] = book[owner[i], :full[i]]
        book[i, full[i]:n] = torch.tensor(ids[at:at + n - full[i]], dtype=torch.int32)
        at += n - full[i]
    s |= {'book': book.cuda(), 'lengths': _ints(lens)}
    (s['k'], s['kscales']), (s['v'], s['vscales']) = _pool(case, pages, gen)
    if case['op'] == 'append':
        row = s['book'].long()[s['row_seqs'].long(), (s['positions'] // T).long()]
        # the cache rows (per head) that the new tokens fall on
        s['where'] = ((row * hkv)[:, None] + torch.arange(hkv, device='cuda')) * T + (s['positions'] % T).long()[:, None]
        return s
    # the page that a prefix ends in is a copy in each sequence but the first
    src, dst, count = [], [], []
    for members, prefix in _groups(case):
        for i in members[1:]:
            if lens[i] and prefix % T:
                src.append(int(book[members[0], prefix // T]))
                dst.append(int(book[i, prefix // T]))
                count.append(prefix % T)
    if src:
        src, dst = torch.tensor(src, device='cuda'), torch.tensor(dst, device='cuda')
        kept = torch.arange(T, device='cuda') < torch.tensor(count, device='cuda')[:, None, None]
        for x in (s['k'], s['v'], s['kscales'], s['vscales']):
            if x is not None:
                w = kept[..., None] if x.dim() == 5 else kept
                x[0, dst] = torch.where(w, x[0, src], x[0, dst])
    groups = _groups(case)
    starts = [0]
    for members, _ in groups:
        starts.append(starts[-1] + len(members))
    q = torch.randn(case['seqs'], hq, dim, generator=gen, device='cuda')
    # sharper than uniform attention: the logits' standard deviation is 2
    s |= {'q': (2 * q).bfloat16(), 'scale': dim ** -0.5, 'starts': _ints(starts), 'prefix': _ints([p for _, p in groups]),
          'seqs': _ints(list(range(case['seqs']))), 'most': max(len(m) for m, _ in groups),
          'longest': max(p for _, p in groups),
          'ctx': torch.empty(case['seqs'], hq, dim, device='cuda', dtype=torch.bfloat16),
          'workspace': torch.zeros(256 << 20, dtype=torch.uint8, device='cuda')}
    s['own'] = max(1, max(lens[i] - p for m, p in groups for i in m))
    return s


def _prepare_sample(case, s, gen, rng):
    rows, vocab = case['rows'], case['vocab']
    x = torch.randn(rows, vocab, generator=gen, device='cuda') * 2.5
    if case['peaked']:
        # a few dozen likely tokens in each row
        at = torch.randint(vocab, (rows, 40), generator=gen, device='cuda')
        x.scatter_add_(1, at, torch.rand(rows, 40, generator=gen, device='cuda') * 10 + 4)
    masked = rng.sample(range(rows), min(case['masked'], rows))
    for n, r in enumerate(masked):
        # a grammar allows from one token to a tenth of them; the others are at -infinity or the type's lowest value
        allowed = rng.choice((1, 2, max(1, vocab // 1000), max(1, vocab // 10)))
        keep = torch.randperm(vocab, generator=gen, device='cuda')[:allowed]
        row = torch.full((vocab,), -math.inf if n % 2 else torch.finfo(torch.bfloat16).min, device='cuda')
        row[keep] = x[r, keep]
        x[r] = row
    on = [[not case['mixed'] or rng.random() < 0.6 for _ in range(3)] for _ in range(rows)]
    k = [case['top_k'] if not case['mixed'] else rng.randint(1, max(1, case['top_k'])) for _ in range(rows)]

    def floats(values):
        return torch.tensor(values, dtype=torch.float32, device='cuda')
    return s | {
        'logits': x.bfloat16(), 'u': torch.rand(rows, generator=gen, device='cuda'),
        'temperature': floats([0.8 if not case['mixed'] else rng.uniform(0.3, 1.5) for _ in range(rows)]),
        'top_k': _ints([v if o[0] else 0 for v, o in zip(k, on)]),
        'top_p': floats([case['top_p'] if o[1] else 1.0 for o in on]),
        'min_p': floats([case['min_p'] if o[2] else 0.0 for o in on]),
        'tokens': torch.empty(rows, dtype=torch.int32, device='cuda'),
        'probs': torch.empty(rows, dtype=torch.float32, device='cuda')}


# ---------------------------------------------------------------- one pass


def run(s):
    if own:
        return _own_run(s)
    return {'rotary': _rotary, 'append': _append, 'shared': _shared, 'sample': _sample}[s['case']['op']](s)


def _rotated(s, x):
    """x [rows][heads][dim] with the pairs of its first `rotated` dims turned, in bf16. Products and sums are values of 32 bits."""
    case, rot = s['case'], s['case']['rotated']
    c, n = s['table'][s['positions'].long()].view(-1, 1, 2, rot // 2).unbind(2)
    x = x.float()
    if case['interleaved']:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([turned, x[..., rot:]], -1).bfloat16()


def _rotary(s):
    s['out'].copy_(_rotated(s, s['qk']))
    return s['out']


def _read_back(s):
    """The rotated queries and the values that the cache holds for the new rows."""
    dim = s['case']['dim']
    out = [s['q_out']]
    for pool, scales in ((s['k'], s['kscales']), (s['v'], s['vscales'])):
        if scales is None:
            out.append(pool)
        else:
            at = s['where'].view(-1)
            values = pool.view(-1, dim).index_select(0, at) * scales.view(-1, 1).index_select(0, at)
            out.append(values.view(*s['where'].shape, dim))
    return out


def _append(s):
    dim = s['case']['dim']
    s['q_out'].copy_(_rotated(s, s['q']))
    for x, pool, scales in ((_rotated(s, s['new_k']), s['k'], s['kscales']), (s['new_v'], s['v'], s['vscales'])):
        if scales is None:
            pool.view(-1, dim)[s['where']] = x
        else:
            pool.view(-1, dim)[s['where']], scales.view(-1)[s['where']] = _quantised(x.float())
    return _read_back(s)


def _gathered(s, name, seqs, position):
    """[sequence][kv head][position][dim] in 32 bits: the tokens at position[sequence], cut to the sequence's pages."""
    T, book = s['case']['page'], s['book']
    page = book[seqs[:, None], (position // T).clamp(max=book.shape[1] - 1)].long()
    x = s[name][0][page, :, position % T].float()
    if s[name + 'scales'] is not None:
        x = x * s[name + 'scales'][0][page, :, position % T].unsqueeze(-1)
    return x.transpose(1, 2)


def _shared(s):
    case = s['case']
    hkv, G, dim = case['kv_heads'], case['q_heads'] // case['kv_heads'], case['dim']
    starts, seqs = s['starts'].long(), s['seqs'].long()
    rows, n = case['seqs'], starts.numel() - 1
    lens = s['lengths'].long()[seqs]
    row = torch.arange(rows, device='cuda')
    group = torch.bucketize(row, starts[1:], right=True)
    slot = row - starts[group]
    prefix = torch.minimum(s['prefix'].long(), lens[starts[:-1]])
    minus = torch.tensor(-math.inf, device='cuda')
    # a group's rows side by side, padded to the most, against its prefix
    q = s['q'].float().view(rows, hkv, G, dim)
    side = torch.zeros(n, s['most'], hkv, G, dim, device='cuda')
    side[group, slot] = q
    reach = torch.zeros(n, s['most'], dtype=torch.long, device='cuda')
    reach[group, slot] = torch.minimum(prefix[group], lens)
    j = torch.arange(s['longest'], device='cuda').expand(n, -1)
    first = seqs[starts[:-1]]
    k, v = _gathered(s, 'k', first, j), _gathered(s, 'v', first, j)
    x = torch.matmul(side.permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, dim), k.transpose(2, 3)) * s['scale']
    x = x.view(n, hkv, s['most'], G, -1)
    x = torch.where(j[:, None, None, None] < reach[:, None, :, None, None], x, minus)
    # each row against its own tokens
    mine = prefix[group][:, None] + torch.arange(s['own'], device='cuda')
    there = (mine < lens[:, None])[:, None, None]
    mk, mv = _gathered(s, 'k', seqs, mine), _gathered(s, 'v', seqs, mine)
    y = torch.where(there, torch.matmul(q, mk.transpose(2, 3)) * s['scale'], minus)
    # one softmax over both
    top = torch.maximum(x.amax(-1).transpose(1, 2)[group, slot], y.amax(-1))
    top = torch.where(top == minus, 0, top)
    side_top = torch.zeros(n, s['most'], hkv, G, device='cuda')
    side_top[group, slot] = top
    x = (x - side_top.transpose(1, 2).unsqueeze(-1)).exp()
    y = (y - top.unsqueeze(-1)).exp()
    total = x.sum(-1).transpose(1, 2)[group, slot] + y.sum(-1)
    out = torch.matmul(x.view(n, hkv, -1, x.shape[-1]), v).view(n, hkv, s['most'], G, dim).transpose(1, 2)[group, slot]
    out = (out + torch.matmul(y, mv)) / total.unsqueeze(-1)
    out = torch.where(total.unsqueeze(-1) > 0, out, 0)
    s['ctx'].copy_(out.view(rows, -1, dim))
    return s['ctx']


def _sample(s):
    # in 64 bits: a token's border is a sum over up to the whole vocabulary
    x = torch.nan_to_num(s['logits'].double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    place = torch.arange(x.shape[1], device='cuda')
    w = ((x - x[:, :1]) / s['temperature'].double()[:, None]).exp()
    k = s['top_k'].long()[:, None]
    w = torch.where((place < k) | (k == 0), w, 0)
    share = s['top_p'].double()[:, None] * w.sum(1, keepdim=True)
    before = w.cumsum(1) - w
    kept = ((before < share) | (s['top_p'][:, None] >= 1)) & (w >= s['min_p'].double()[:, None])
    kept[:, 0] = True
    w = torch.where(kept, w, 0)
    upto = w.cumsum(1)
    total = upto[:, -1:]
    at = (upto <= s['u'].double()[:, None] * total).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    s['tokens'].copy_(order.gather(1, at).squeeze(1))
    s['probs'].copy_((w.gather(1, at) / total).squeeze(1))
    return [s['tokens'], s['probs']]


# ---------------------------------------------------------------- the library's calls


def _library():
    root = str(Path(__file__).resolve().parents[1] / PACKAGE)
    if root not in sys.path:
        sys.path.insert(0, root)
    import qwen_b200
    return qwen_b200


def _descriptors(q, s):
    """What the library's calls know a cache and a rotation by: addresses and sizes, kept by a program as long as those."""
    case = s['case']
    if 'table' in s:
        s['rotation'] = q.Rotary(table=s['table'].data_ptr(), positions=s['table'].shape[0], rotated=case['rotated'],
                                 layout=q.ROTARY_PAIRS if case['interleaved'] else q.ROTARY_HALVES)
    if 'k' not in s:
        return
    layers, pages, hkv, T, dim = s['k'].shape
    kv8 = s['kscales'] is not None
    s['descriptor'] = q.PagedKV(k=s['k'].data_ptr(), v=s['v'].data_ptr(), kscales=s['kscales'].data_ptr() if kv8 else None,
                                vscales=s['vscales'].data_ptr() if kv8 else None, table=s['book'].data_ptr(),
                                lengths=s['lengths'].data_ptr(), refs=None, layer_stride=pages * hkv * T,
                                page_stride=hkv * T, format=q.KV8 if kv8 else q.KV_BF16, layers=layers, pages=pages,
                                kv_heads=hkv, page_tokens=T, head_dim=dim, seqs=case['seqs'], max_pages=s['book'].shape[1])


def _own_run(s):
    if 'library' not in s:
        s['library'] = _library()
        _descriptors(s['library'], s)
    q, case = s['library'], s['case']
    lib, op = q.lib(), case['op']
    st = torch.cuda.current_stream().cuda_stream
    if op == 'sample':
        x = s['logits']
        q.check(lib.qwen_b200_op_sample(x.data_ptr(), x.stride(0), case['rows'], case['vocab'],
                                        s['temperature'].data_ptr(), s['top_k'].data_ptr(), s['top_p'].data_ptr(),
                                        s['min_p'].data_ptr(), s['u'].data_ptr(), s['tokens'].data_ptr(),
                                        s['probs'].data_ptr(), st))
        return [s['tokens'], s['probs']]
    if op == 'rotary':
        x, out = s['qk'], s['out']
        q.check(lib.qwen_b200_op_rotary(ctypes.byref(s['rotation']), x.data_ptr(), x.stride(0), x.shape[1], x.shape[2],
                                        x.shape[0], s['positions'].data_ptr(), out.data_ptr(), out.stride(0), st))
        return out
    kv = ctypes.byref(s['descriptor'])
    if op == 'append':
        q.check(lib.qwen_b200_op_paged_append_rotary(
            kv, 0, ctypes.byref(s['rotation']), s['q'].data_ptr(), s['q'].stride(0), case['q_heads'], s['q_out'].data_ptr(),
            s['q_out'].stride(0), s['new_k'].data_ptr(), s['new_v'].data_ptr(), s['new_k'].stride(0), s['q'].shape[0],
            s['row_seqs'].data_ptr(), s['positions'].data_ptr(), st))
        return _read_back(s)
    q.check(lib.qwen_b200_op_paged_decode_shared(
        kv, 0, s['q'].data_ptr(), s['q'].stride(0), case['q_heads'], case['groups'], s['starts'].data_ptr(),
        s['prefix'].data_ptr(), case['seqs'], s['seqs'].data_ptr(), s['scale'], s['ctx'].data_ptr(), s['ctx'].stride(0),
        s['workspace'].data_ptr(), s['workspace'].numel(), st))
    return s['ctx']


# ---------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {'rotary': _exact_rotary, 'append': _exact_append, 'shared': _exact_shared, 'sample': _exact_sample}[case['op']](s)


def _exact_turned(s, x):
    """Each pair as a complex number times cos + i sin."""
    case = s['case']
    rot, half = case['rotated'], case['rotated'] // 2
    angle = s['table'].double()[s['positions'].long()]
    unit = torch.complex(angle[:, :half], angle[:, half:])[:, None]
    y = x.double()
    if case['interleaved']:
        z = torch.view_as_complex(y[..., :rot].unflatten(-1, (half, 2)).contiguous()) * unit
        y[..., :rot] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., :half], y[..., half:rot]) * unit
        y[..., :half], y[..., half:rot] = z.real, z.imag
    return y


def _exact_rotary(s):
    return _exact_turned(s, s['qk'])


def _exact_append(s):
    q, k, v = _exact_turned(s, s['q']), _exact_turned(s, s['new_k']), s['new_v'].double()
    out = [q]
    for x, pool, scales in ((k, s['k'], s['kscales']), (v, s['v'], s['vscales'])):
        if scales is None:
            y = pool.double()
            y.view(-1, x.shape[-1])[s['where'].flatten()] = x.flatten(0, 1)
            out.append(y)
        else:
            # the cache's rule: what is stored are the codes of bf16 values; the products and sums of the rotation, the
            # scale and the quotient are values of 32 bits, the code is the nearest whole number, the even one of two
            if x is k:
                x = _key_rule(s)
            top = x.abs().max(-1, keepdim=True).values
            step = (top / 127).float().double()
            ratio = torch.nan_to_num(x / step).float().double()
            out.append(torch.clamp(torch.round(ratio), -127, 127) * step)
    return out


def _key_rule(s):
    """The rotated keys as bf16 values, each product and each sum rounded to 32 bits on the way."""
    case, x = s['case'], s['new_k'].double()
    rot = case['rotated']
    first = list(range(0, rot, 2)) if case['interleaved'] else list(range(rot // 2))
    second = [i + (1 if case['interleaved'] else rot // 2) for i in first]
    cos, sin = (t[:, None] for t in s['table'].double()[s['positions'].long()].split(rot // 2, 1))

    def product(i, by):
        return (x[..., i] * by).float().double()
    a, b = product(first, cos) - product(second, sin), product(second, cos) + product(first, sin)
    y = x.clone()
    y[..., first], y[..., second] = a.float().double(), b.float().double()
    return y.float().bfloat16().double()


def _exact_shared(s):
    case = s['case']
    T, dim, hkv, G = case['page'], case['dim'], case['kv_heads'], case['q_heads'] // case['kv_heads']
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda')
    book = s['book'].long()
    for r, t in enumerate(_lengths(case)):
        if not t:
            continue
        token = torch.arange(t, device='cuda')
        page, at = book[r][token // T], token % T
        k, v = s['k'][0][page, :, at].double(), s['v'][0][page, :, at].double()
        if s['kscales'] is not None:
            k *= s['kscales'][0][page, :, at].double()[..., None]
            v *= s['vscales'][0][page, :, at].double()[..., None]
        q = s['q'][r].double().view(hkv, G, dim)
        w = torch.softmax(torch.einsum('hgd,thd->hgt', q, k) * s['scale'], -1)
        out[r] = torch.einsum('hgt,thd->hgd', w, v).reshape(-1, dim)
    return out


def _exact_sample(s):
    """Row by row over the distinct logits and how often each occurs."""
    probs = []
    for r in range(s['case']['rows']):
        x = s['logits'][r].double()
        value, count = torch.unique(x[x > -math.inf], return_counts=True)
        value, count = value.flip(0), count.flip(0).double()
        w = torch.exp((value - value[0]) / s['temperature'][r].double())
        k, p, least = s['top_k'][r].double(), s['top_p'][r].double(), s['min_p'][r].double()
        before = count.cumsum(0) - count
        if k > 0:
            count = torch.minimum(count, (k - before).clamp(min=0))
        mass = count * w
        if p < 1:
            # of equal logits as many as begin below the share
            left = p * mass.sum() - (mass.cumsum(0) - mass)
            count = torch.minimum(count, torch.ceil(left / w).nan_to_num(0, 0, 0).clamp(min=0))
            count[0] = count[0].clamp(min=1)
        count = torch.where(w >= least, count, 0)
        count[0] = count[0].clamp(min=1)
        mass = count * w
        at = torch.searchsorted(mass.cumsum(0), (s['u'][r].double() * mass.sum())[None], right=True)
        probs.append(w[at.clamp(max=int((mass > 0).sum()) - 1)] / mass.sum())
    return [None, torch.cat(probs)]
