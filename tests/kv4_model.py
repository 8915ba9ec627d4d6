"""The 4-bit cache in numpy, in 64 bits: the quantisation, the byte layout of a
page and attention over it (include/holo_forward.h), and device buffers for
them.  Test infrastructure."""
from __future__ import annotations

import ctypes as C

import numpy as np


def bf16(x):
    """float32 values rounded to bfloat16 (ties to even), as float32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def quantise(x):
    """Codes 0 .. 15 [..., hd] and f16 scales [..., hd / 32] of float32 x [..., hd]."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], np.float32(0), b)
    low, high = b.min(-1), b.max(-1)
    d = np.minimum(bf16(np.maximum(-low, high) * np.float32(0.125)), np.float32(2720))
    d = np.where(-low >= high, d, -d).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.clip(np.rint(b.astype(np.float64) / d.astype(np.float64)[..., None]), -8, 7)
    c = np.where((d == 0)[..., None] | bad[..., None], 0, c) + 8
    d = np.where(bad, np.float16(np.nan), d)
    return c.astype(np.uint8).reshape(x.shape), d


def values(codes, d):
    c = codes.reshape(*codes.shape[:-1], -1, 32).astype(np.float64) - 8
    return (c * d.astype(np.float64)[..., None]).reshape(codes.shape)


class Cache:
    """The pool of a cache as bytes, written position by position."""

    def __init__(self, hd, page_len, n_layers, n_kv, n_pages, n_seqs, max_pages, fill=None):
        self.hd, self.page_len, self.n_layers, self.n_kv = hd, page_len, n_layers, n_kv
        self.n_pages, self.n_seqs, self.max_pages = n_pages, n_seqs, max_pages
        self.tiles = page_len // 32
        self.tile_bytes = 36 * hd
        shape = (n_pages, n_layers, n_kv, self.tiles, self.tile_bytes)
        rng = np.random.default_rng(99)
        self.pool = (rng.integers(0, 256, shape, dtype=np.uint8) if fill is None else np.full(shape, fill, np.uint8))
        self.table = np.full((n_seqs, max_pages), -1, np.int32)
        self.len = np.zeros(n_seqs, np.int32)

    def where(self, p, which):
        """Byte and shift of the codes of a tile's position p, and the byte of its scales."""
        hd, nb = self.hd, self.hd // 32
        d, b = np.arange(hd), np.arange(nb)
        half, r = p // 16, p % 16
        if which == 0:
            w, slot = d // 8, d % 8
            word = ((half * 4 + w // nb) * 16 + r) * nb + w % nb
            scale = 32 * hd + 2 * (b * 32 + r * 2 + half)
        else:
            vw = 2 if nb % 2 else 4
            g, slot, m = r // 4, np.full(hd, half * 4 + r % 4), d // 16
            word = 4 * hd + ((m // vw * 4 + g) * 16 + d % 16) * vw + m % vw
            scale = 34 * hd + 2 * (b * 32 + g * 8 + half * 4 + r % 4)
        nib = slot // 2 + 4 * (slot % 2)
        return 4 * word + nib // 2, 4 * (nib % 2), scale

    def _tile(self, seq, layer, head, pos):
        page = self.table[seq, pos // self.page_len]
        if page < 0 or page >= self.n_pages:
            return None
        return self.pool[page, layer, head, pos % self.page_len // 32]

    def put(self, seq, layer, head, pos, k, v):
        """One position's fp32 key and value."""
        t = self._tile(seq, layer, head, pos)
        if t is None:
            return
        for which, x in ((0, k), (1, v)):
            c, d = quantise(x)
            at, sh, sc = self.where(pos % 32, which)
            for s in (0, 4):  # two dims can share a byte: low nibbles, then high ones
                i = sh == s
                t[at[i]] = (t[at[i]] & np.uint8(240 >> s)) | (c[i] << np.uint8(s))
            u = d.view(np.uint16)
            t[sc], t[sc + 1] = u & 255, u >> 8

    def get(self, seq, layer, head, pos, which):
        """The float64 value of one position [hd], or None where there is no page."""
        t = self._tile(seq, layer, head, pos)
        if t is None:
            return None
        at, sh, sc = self.where(pos % 32, which)
        d = (t[sc].astype(np.uint16) | (t[sc + 1].astype(np.uint16) << 8)).view(np.float16)
        return values((t[at] >> sh) & 15, d)

    def held(self, seq, layer, head, n):
        """k and v [n][hd] in 64 bits and which positions have a page."""
        k, v, there = np.zeros((n, self.hd)), np.zeros((n, self.hd)), np.zeros(n, bool)
        for p in range(n):
            x = self.get(seq, layer, head, p, 0)
            if x is not None:
                k[p], v[p], there[p] = x, self.get(seq, layer, head, p, 1), True
        return k, v, there


def attend(q, k, v, seen):
    """softmax(q k / sqrt(hd)) v over the positions where `seen`; zeros where there is none."""
    if not seen.any():
        return np.zeros(k.shape[1])
    k, v = k[seen], v[seen]
    with np.errstate(invalid="ignore", over="ignore"):
        s = k @ q.astype(np.float64) / np.sqrt(k.shape[1])
        p = np.exp(s - s.max())
        return (p / p.sum()) @ v


def want_attention(cache, layer, q, rows, lens, seqs, n_heads):
    """q [total][n_heads * hd] of rows[i] rows an entry."""
    hd, out, at = cache.hd, np.zeros((q.shape[0], n_heads * cache.hd)), 0
    group = n_heads // cache.n_kv
    for n, seq in zip(rows, seqs):
        ln = int(lens[seq]) if 0 <= seq < cache.n_seqs else 0
        for kvh in range(cache.n_kv):
            k, v, there = cache.held(seq, layer, kvh, ln) if ln else (np.zeros((0, hd)),) * 2 + (np.zeros(0, bool),)
            for i in range(n):
                seen = there & (np.arange(ln) <= ln - n + i)
                for h in range(kvh * group, (kvh + 1) * group):
                    out[at + i, h * hd:(h + 1) * hd] = attend(q[at + i, h * hd:(h + 1) * hd], k, v, seen)
        at += n
    return out


class OnDevice:
    """A Cache's arrays on the device, and its descriptor."""

    def __init__(self, holo, cache):
        self.holo, self.cache = holo, cache
        up = holo.DeviceBuffer.from_array
        self.pool, self.table, self.len = up(cache.pool), up(cache.table), up(cache.len)
        self.desc = holo.KV4(pool=self.pool.ptr, table=self.table.ptr, len=self.len.ptr, n_pages=cache.n_pages,
                             page_len=cache.page_len, n_layers=cache.n_layers, n_kv_heads=cache.n_kv,
                             head_dim=cache.hd, n_seqs=cache.n_seqs, max_pages=cache.max_pages)
        self.ref = C.byref(self.desc)

    def refresh(self):
        self.table.upload(self.cache.table)
        self.len.upload(self.cache.len)

    def bytes(self):
        return self.pool.download(np.uint8).reshape(self.cache.pool.shape)


class Batch:
    """holo_batch_t of rows[i] rows for entry i."""

    def __init__(self, holo, rows, seqs=None, max_rows=None, max_len=0):
        up = holo.DeviceBuffer.from_array
        cu = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
        self.cu, self.seqs = up(cu), None if seqs is None else up(np.asarray(seqs, np.int32))
        self.total = int(cu[-1])
        self.desc = holo.Batch(rows=self.total, n_seqs=len(rows), max_rows=max(rows) if max_rows is None else max_rows,
                               max_len=int(max_len), cu_rows=self.cu.ptr, seqs=None if seqs is None else self.seqs.ptr)
        self.ref = C.byref(self.desc)


def normwise(got, want):
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))
