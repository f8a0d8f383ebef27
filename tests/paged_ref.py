"""A paged KV cache on the host and its operators in 64 bits: what the tests of
the paged entry points compare with. The cache holds NaN wherever nothing was
written, and page ids out of range in unused table entries, so a kernel that
reads what it should not shows it."""
import ctypes

import numpy as np

import qwen_b200
from qwen_b200 import _lib

U = 2.0 ** -24  # half a step of fp32 at 1
BF16_HALF = 2.0 ** -8


def bf16(a):
    a = np.ascontiguousarray(a, np.float32)
    u = a.view(np.uint32).astype(np.uint64)
    u = (u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000
    return u.astype(np.uint32).view(np.float32)


def bits(a):
    return (np.ascontiguousarray(a, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def unbits(b):
    return (np.asarray(b).view(np.uint16).astype(np.uint32) << 16).view(np.float32)


def quantise(x):
    """[..., dim] fp32 (bf16 values) -> int8 codes, fp32 scales: every step one fp32 operation."""
    x = np.asarray(x, np.float32)
    s = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide='ignore', invalid='ignore'):
        c = np.clip(np.rint((x / s[..., None]).astype(np.float32)), -127, 127)
    return np.where(s[..., None] > 0, c, 0).astype(np.int8), s


class Cache:
    """pool arrays indexed [layer, page, head, token(, dim)]; `pages_first` stores them as [page][layer]."""

    def __init__(self, seed, fmt, kv_heads, dim, page, pages, seqs, max_pages, layers=1, pages_first=False):
        self.r = np.random.default_rng(seed)
        self.fmt, self.hkv, self.dim, self.T = fmt, kv_heads, dim, page
        self.pages, self.seqs, self.max_pages, self.layers, self.pages_first = pages, seqs, max_pages, layers, pages_first
        shape = (layers, pages, kv_heads, page)
        self.kc = self.vc = self.ks = self.vs = None
        if fmt == _lib.KV8:
            self.k = self.r.integers(-128, 128, shape + (dim,)).astype(np.int8)
            self.v = self.r.integers(-128, 128, shape + (dim,)).astype(np.int8)
            self.ks = np.full(shape, np.nan, np.float32)
            self.vs = np.full(shape, np.nan, np.float32)
        else:
            self.k = np.full(shape + (dim,), np.nan, np.float32)
            self.v = np.full(shape + (dim,), np.nan, np.float32)
        self.table = self.r.integers(1 << 30, 1 << 31, (seqs, max_pages)).astype(np.uint32)
        self.lengths = np.zeros(seqs, np.uint32)
        self.refs = np.zeros(pages, np.uint32)

    def rand(self, *shape):
        return bf16(self.r.standard_normal(shape))

    def give(self, lens):
        """Random pages for the sequences, and their tokens filled with unit-variance keys and values."""
        ids = iter(self.r.permutation(self.pages))
        for s, n in enumerate(lens):
            self.lengths[s] = n
            for j in range(-(-n // self.T)):
                p = next(ids)
                self.table[s, j], self.refs[p] = p, 1
            for layer in range(self.layers):
                if n:
                    self.write(layer, s, np.arange(n), self.rand(n, self.hkv, self.dim), self.rand(n, self.hkv, self.dim))
        return self

    def at(self, s, tokens):
        tokens = np.asarray(tokens)
        return self.table[s][tokens // self.T].astype(np.int64), tokens % self.T

    def write(self, layer, s, tokens, k, v):
        p, t = self.at(s, tokens)
        if self.fmt == _lib.KV8:
            self.k[layer, p, :, t], self.ks[layer, p, :, t] = quantise(k)
            self.v[layer, p, :, t], self.vs[layer, p, :, t] = quantise(v)
        else:
            self.k[layer, p, :, t], self.v[layer, p, :, t] = k, v

    def read(self, layer, s, tokens):
        """float64 [tokens][heads][dim] keys and values."""
        p, t = self.at(s, tokens)
        k, v = self.k[layer, p, :, t].astype(np.float64), self.v[layer, p, :, t].astype(np.float64)
        if self.fmt == _lib.KV8:
            k, v = k * self.ks[layer, p, :, t][..., None], v * self.vs[layer, p, :, t][..., None]
        return k, v

    def seen(self, pos, window, sinks, length):
        t = np.arange(length)
        ok = t <= pos
        if window:
            ok &= (pos - t < window) | (t < sinks)
        return t[ok]

    def attention(self, layer, q, seqs, positions, window, sinks, scale, weight_rounding):
        """ctx in 64 bits [rows][heads][dim] and how far a kernel may be from it: q [rows][heads][dim]; row r is token
        positions[r] of sequence seqs[r].

        The bound: the result is rounded once (BF16_HALF of itself). A weight is off by the rounding it is held with
        (weight_rounding) and by its score: a dot product of dim fp32 terms is off by at most dim U times the sum
        S of their magnitudes, the scale and the subtraction of the maximum by 4 U S more (|score| <= S), and exp2 by
        2^-21. A relative weight error e changes sum(p v) / sum(p) by at most e (sum(p |v|) + |ctx|); the sums over n
        keys in fp32 add n U at most to each."""
        rows, heads, dim = q.shape
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        group = heads // self.hkv
        for r in range(rows):
            s = seqs[r]
            if s >= self.seqs or positions[r] < 0 or not self.lengths[s]:
                continue
            t = self.seen(positions[r], window, sinks, int(self.lengths[s]))
            t = t[self.at(s, t)[0] < self.pages]
            if not t.size:
                continue
            k, v = self.read(layer, s, t)
            k, v = np.repeat(k, group, 1), np.repeat(v, group, 1)
            x = np.einsum('hd,thd->ht', q[r].astype(np.float64), k) * scale
            mag = (np.einsum('hd,thd->ht', np.abs(q[r]).astype(np.float64), np.abs(k)) * abs(scale)).max(1)
            w = np.exp(x - x.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            out[r] = np.einsum('ht,thd->hd', w, v)
            size = np.einsum('ht,thd->hd', w, np.abs(v)) + np.abs(out[r])
            e = weight_rounding + 2 * (dim + 4) * U * mag + 2.0 ** -21 + 2 * t.size * U
            tol[r] = BF16_HALF * (np.abs(out[r]) + e[:, None] * size) + e[:, None] * size
        return out, tol

    # -------------------------------------------------------- on the GPU
    def _order(self, a):
        return np.ascontiguousarray(a.swapaxes(0, 1)) if self.pages_first else np.ascontiguousarray(a)

    def upload(self, keep):
        """PagedKV of device copies (held by `keep`)."""
        import torch
        self.dev = {}
        for name in ('k', 'v', 'ks', 'vs', 'table', 'lengths', 'refs'):
            a = getattr(self, name)
            if a is None:
                continue
            if name in ('k', 'v', 'ks', 'vs'):
                a = self._order(a)
                if name in ('k', 'v') and self.fmt != _lib.KV8:
                    a = bits(a).view(np.int16)
            else:
                a = a.view(np.int32)
            self.dev[name] = torch.from_numpy(np.array(a)).cuda()
            keep.tensors.append(self.dev[name])
        block = self.hkv * self.T
        strides = (block, self.layers * block) if self.pages_first else (self.pages * block, block)
        return self.descriptor({n: t.data_ptr() for n, t in self.dev.items()}, strides)

    def descriptor(self, ptr, strides):
        return qwen_b200.PagedKV(k=ptr['k'], v=ptr['v'], kscales=ptr.get('ks'), vscales=ptr.get('vs'), table=ptr['table'],
                                 lengths=ptr['lengths'], refs=ptr['refs'], layer_stride=strides[0],
                                 page_stride=strides[1], format=self.fmt, layers=self.layers, pages=self.pages,
                                 kv_heads=self.hkv, page_tokens=self.T, head_dim=self.dim, seqs=self.seqs,
                                 max_pages=self.max_pages)

    def assert_same(self):
        """The device's pools, tables, lengths and reference counts are this object's, bit for bit (NaN included)."""
        for name, t in self.dev.items():
            a = getattr(self, name)
            if name in ('k', 'v', 'ks', 'vs'):
                a = self._order(a)
                if name in ('k', 'v') and self.fmt != _lib.KV8:
                    a = bits(a)
            got = t.cpu().numpy()
            assert np.array_equal(got.view(np.uint8), np.ascontiguousarray(a).view(np.uint8)), name


def ref(kv):
    return ctypes.byref(kv)
