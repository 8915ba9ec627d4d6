"""Drafted tokens on the GPU, operator by operator against numpy in 64 bits
(draft_model.py), and a whole step of them.

Tolerances.  Attention: 1e-5 normwise, as test_gpu_kv4.py derives it.  Rotation: a
value is rounded once, 2^-24 of it; the angle of a position below 2^17 (times a
frequency of 1 at most) is within four roundings, 2^17 * 4 * 2^-53 = 6e-11, and
sine and cosine with it: 2^-24 |value| + 1e-10 of the pair's magnitude.  Cached
keys are compared bit for bit at positions below 2^11: an angle's 1e-12 moves a
rotated value across the middle of two floats once in 10^4 or 10^5, and then a code
or a scale only if the float lies next to a border of theirs as well.  Softmax: in
32 bits, expf within 2 units of 2^-24 relative, its argument (a difference of two
floats times the scale, each rounded) within 2^-23 of itself, up to 104 where the
result is not 0: 1.3e-5 relative at the far end of a row, 2^-23 |argument| + 2^-22 on
average.  The sum: terms of one sign, 2^-24 for each of at most 40 additions in a row
(32 of a thread, the waves') up to 32768 values, one more for every 1024 above."""
import ctypes as C

import numpy as np
import pytest

import draft_model as dm
from kv4_model import Batch, Cache, OnDevice, attend, normwise, quantise, values

pytestmark = pytest.mark.gpu

TOL = 1e-5


def up(holo, a):
    return holo.DeviceBuffer.from_array(np.ascontiguousarray(a))


def pages(cache, lens, rng):
    """Pages in random order for sequences of these lengths."""
    order = list(rng.permutation(cache.n_pages))
    for s, n in enumerate(lens):
        k = -(-n // cache.page_len)
        cache.table[s, :k] = [order.pop() for _ in range(k)]
        cache.len[s] = n


def fill(cache, rng, layer, first=None):
    for s, n in enumerate(cache.len):
        for h in range(cache.n_kv):
            for p in range(0 if first is None else first[s], n):
                cache.put(s, layer, h, p, *rng.standard_normal((2, cache.hd)).astype(np.float32))


# ---- trees -----------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,words", [([1], 1), ([32, 1, 33, 0, 7], 2), ([64, 65, 200], 7), ([1024, 5], 32),
                                        ([40] * 70, 3)], ids=lambda x: str(x)[:20])
def test_plan(holo, rows, words):
    print(f"case plan {rows[:5]} {words}", flush=True)
    rng = np.random.default_rng(sum(rows))
    parents = [dm.tree(rng, n, 3) for n in rows]
    if rows[0] == 1024:
        parents[0] = list(range(-1, 1023))  # a chain through every word
    if len(rows) == 5:
        parents[2][5:9] = [5, 7, -9, 1 << 30]  # itself, a later row, none there
    b, total = Batch(holo, rows), sum(rows)
    dp = up(holo, np.int32([p for t in parents for p in t]))
    dd, dk = up(holo, np.full(total + 1, -7, np.int32)), up(holo, np.full((total + 1, words), 0xABCDEF01, np.uint32))
    assert holo.lib().holo_draft_plan(dp.ptr, dd.ptr, dk.ptr, words, b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("plan")
    depth, mask = dd.download(np.int32), dk.download(np.uint32).reshape(total + 1, words)
    seen = [dm.seen_rows(t) for t in parents]
    assert np.array_equal(depth[:-1], np.concatenate([s.sum(1) - 1 for s in seen if len(s)]))
    assert np.array_equal(mask[:-1], np.concatenate([dm.words(s, words) for s in seen if len(s)]))
    assert depth[-1] == -7 and (mask[-1] == 0xABCDEF01).all()


def test_plan_leaves_rows_past_max_rows(holo):
    print("case plan bound", flush=True)
    b = Batch(holo, [6, 3], max_rows=4)
    dp, dd, dk = up(holo, np.int32([-1, 0, 1, 2, 3, 4, -1, 0, 0])), up(holo, np.full(9, -7, np.int32)), up(
        holo, np.full(9, 99, np.uint32))
    assert holo.lib().holo_draft_plan(dp.ptr, dd.ptr, dk.ptr, 1, b.ref) == 0
    holo.lib().cuda_sync()
    assert dd.download(np.int32).tolist() == [0, 1, 2, 3, -7, -7, 0, 1, 1]
    assert dk.download(np.uint32).tolist() == [1, 3, 7, 15, 99, 99, 1, 3, 5]


# ---- rotation and append -------------------------------------------------------------------------

def freq_of(dims, stretch=1.0):
    return 10000.0 ** (-2 * np.arange(dims // 2) / dims) / stretch


def close(got, want, x, hd):
    """Rounded once, and the angle's error on the pair's magnitude (a head's at most)."""
    size = np.abs(x.astype(np.float64)).reshape(len(x), -1, hd).max(-1, keepdims=True).repeat(hd, -1).reshape(x.shape)
    return (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 3e-10 * size).all()


@pytest.mark.parametrize("hd,heads,n_kv,page_len,dims,interleaved", [
    (128, 8, 2, 64, 128, 0), (128, 3, 3, 32, 96, 1), (64, 12, 2, 32, 64, 1), (64, 2, 2, 128, 2, 0),
    (96, 6, 3, 32, 96, 0), (96, 10, 1, 32, 50, 0), (32, 4, 4, 64, 32, 0), (32, 5, 1, 32, 30, 1), (128, 0, 2, 32, 74, 0),
    (64, 9, 1, 32, 32, 0)], ids=str)
def test_rotated_rows_into_pages(holo, hd, heads, n_kv, page_len, dims, interleaved):
    """Prompts, then trees behind them, in strided rows: queries, rotated keys and the whole pool."""
    print(f"case rope hd {hd} heads {heads}/{n_kv} dims {dims} {interleaved}", flush=True)
    rng = np.random.default_rng(hd + dims)
    layer, scale = 1, float(np.float32(1.1386)) if interleaved else 1.0  # (what the descriptor holds)
    c = Cache(hd, page_len, 2, n_kv, 26, 5, 256 // page_len)
    pages(c, [150, 70, 1, 0, 97], rng)
    c.len[:] = 0
    dev, lib = OnDevice(holo, c), holo.lib()
    kd, qd = n_kv * hd, heads * hd
    freq = freq_of(dims)
    df = up(holo, freq)
    rope = holo.Rope(freq=df.ptr, dims=dims, interleaved=interleaved, scale=scale)
    for rows, seqs, trees in (([33, 40, 1, 60], [4, 0, 2, 1], False), ([9, 5, 1, 0], [0, 4, 1, 3], True),
                              ([70, 3], [0, -1], True), ([1], [4], False), ([100], [1], True)):
        for n, s in zip(rows, seqs):
            if s >= 0:
                c.len[s] = min(c.len[s] + n, 70 if s == 1 else 1000)  # sequence 1: later rows before position 0
        dev.refresh()
        total, ld = sum(rows), qd + 2 * kd + 12
        wide = rng.standard_normal((total, ld)).astype(np.float32)
        q, k, v = wide[:, :qd], wide[:, qd:qd + kd], wide[:, qd + kd:qd + 2 * kd]
        first = np.repeat([(c.len[s] if s >= 0 else 0) - n for n, s in zip(rows, seqs)], rows)
        depth = np.concatenate([dm.seen_rows(dm.tree(rng, n, 2)).sum(1) - 1 if trees else np.arange(n) for n in rows])
        pos = first + depth
        b, d, ddepth = Batch(holo, rows, seqs), up(holo, wide), up(holo, depth.astype(np.int32))
        ldqo, ldko = qd + 4, kd + 8
        dq, dk = up(holo, np.full((total, ldqo), 5.0, np.float32)), up(holo, np.full((total, ldko), 5.0, np.float32))
        assert lib.holo_kv4_append_rope(dev.ref, layer, C.byref(rope), d.ptr if heads else None, d.ptr + 4 * qd,
                                        d.ptr + 4 * (qd + kd), ld, ld, ld, dq.ptr if heads else None, dk.ptr, ldqo, ldko,
                                        heads, ddepth.ptr if trees else None, b.ref) == 0
        lib.cuda_sync()
        holo.check("append with rotation")
        got_q, got_k = dq.download(np.float32).reshape(total, ldqo), dk.download(np.float32).reshape(total, ldko)
        want_k = dm.turned(k, pos, freq, dims, interleaved, scale, hd)
        if heads:
            assert close(got_q[:, :qd], dm.turned(q, pos, freq, dims, interleaved, scale, hd), q, hd)
        assert close(got_k[:, :kd], want_k, k, hd)
        for x, got in ((q, got_q), (k, got_k)):  # dims that do not turn: bit for bit
            x, y = x.reshape(total, -1, hd)[..., dims:], got[:, :x.shape[1]].reshape(total, -1, hd)[..., dims:]
            assert np.array_equal(x, y)
        assert (got_q[:, qd:] == 5.0).all() and (got_k[:, kd:] == 5.0).all() and (heads or (got_q == 5.0).all())
        at = 0
        for n, s in zip(rows, seqs):
            for i in range(n):
                p = c.len[s] - n + i if s >= 0 else -1
                for h in range(n_kv):
                    if p >= 0:
                        x = slice(h * hd, (h + 1) * hd)
                        c.put(s, layer, h, p, want_k[at + i, x].astype(np.float32), v[at + i, x])
            at += n
        assert np.array_equal(dev.bytes(), c.pool)
        # in place, and without the keys: the same
        assert lib.holo_kv4_append_rope(dev.ref, layer, C.byref(rope), d.ptr if heads else None, d.ptr + 4 * qd,
                                        d.ptr + 4 * (qd + kd), ld, ld, ld, d.ptr if heads else None, None, ld, 0, heads,
                                        ddepth.ptr if trees else None, b.ref) == 0
        lib.cuda_sync()
        wide[:, :qd] = got_q[:, :qd]
        assert np.array_equal(d.download(np.float32).reshape(total, ld), wide)
        assert np.array_equal(dev.bytes(), c.pool)
        d.upload(np.concatenate([q, k, v, wide[:, qd + 2 * kd:]], 1))
        assert lib.holo_kv4_append_rope(dev.ref, layer, C.byref(rope), None, d.ptr + 4 * qd, d.ptr + 4 * (qd + kd), 0, ld,
                                        ld, None, d.ptr + 4 * qd, 0, ld, 0, ddepth.ptr if trees else None, b.ref) == 0
        lib.cuda_sync()
        assert np.array_equal(d.download(np.float32).reshape(total, ld)[:, qd:qd + kd], got_k[:, :kd])
        assert np.array_equal(dev.bytes(), c.pool)


def test_rotation_at_far_positions(holo):
    """A sequence of 0x7FFFF000 positions, whose last page is there, and depths of any size."""
    print("case rope far", flush=True)
    rng = np.random.default_rng(2)
    hd, rows, n = 32, 70, 0x7FFFF000
    c = Cache(hd, 1024, 1, 1, 2, 1, n // 1024)
    c.table[0, -1], c.len[0] = 1, n
    dev, lib = OnDevice(holo, c), holo.lib()
    q, k, v = rng.standard_normal((3, rows, hd)).astype(np.float32)
    freq = 2.0 ** -np.arange(hd // 2)  # angles that 64 bits hold exactly
    df = up(holo, freq)
    rope = holo.Rope(freq=df.ptr, dims=hd, interleaved=1, scale=1.0)
    b = Batch(holo, [rows])
    b.desc.max_rows = b.desc.rows = 0x7FFFF000
    dq, dk, dv, dko = up(holo, q), up(holo, k), up(holo, v), holo.DeviceBuffer(k.nbytes)
    depth = rng.integers(-(1 << 31), 1 << 31, rows).astype(np.int32)
    for d in (None, up(holo, depth)):
        dq.upload(q)
        assert lib.holo_kv4_append_rope(dev.ref, 0, C.byref(rope), dq.ptr, dk.ptr, dv.ptr, hd, hd, hd, dq.ptr, dko.ptr,
                                        hd, hd, 1, d.ptr if d else None, b.ref) == 0
        lib.cuda_sync()
        holo.check("far positions")
        pos = n - rows + (np.arange(rows) if d is None else depth.astype(np.int64))
        # 2^32 * 2 roundings of 2^-53 in the angle's half turns
        for x, got in ((q, dq), (k, dko)):
            want = dm.turned(x, pos, freq, hd, 1, 1.0, hd)
            got = got.download(np.float32).reshape(rows, hd)
            assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -18 * np.abs(x).max()).all()
        ok, ov = holo.DeviceBuffer(k.nbytes), holo.DeviceBuffer(k.nbytes)
        assert lib.holo_kv4_read(dev.ref, 0, ok.ptr, ov.ptr, hd, hd, b.ref) == 0
        lib.cuda_sync()
        assert np.array_equal(ok.download(np.float32), values(*quantise(dko.download(np.float32).reshape(rows, hd))).ravel())
        assert np.array_equal(ov.download(np.float32), values(*quantise(v)).ravel())


def test_rotation_leaves_rows_past_max_rows_and_passes_bad_values(holo):
    print("case rope bound", flush=True)
    rng = np.random.default_rng(3)
    hd, rows = 64, [9, 4]
    c = Cache(hd, 32, 1, 1, 4, 2, 1)
    pages(c, [20, 4], rng)
    dev, lib = OnDevice(holo, c), holo.lib()
    q, k, v = rng.standard_normal((3, 13, hd)).astype(np.float32)
    k[1, 3], k[10, 40], q[2, 5] = np.nan, np.inf, np.nan
    df = up(holo, freq_of(hd))
    rope = holo.Rope(freq=df.ptr, dims=hd, interleaved=0, scale=1.0)
    b = Batch(holo, rows, max_rows=6)
    dq, dk, dv = up(holo, q), up(holo, k), up(holo, v)
    do, dko = up(holo, np.full(q.shape, -9.0, np.float32)), up(holo, np.full(q.shape, -9.0, np.float32))
    assert lib.holo_kv4_append_rope(dev.ref, 0, C.byref(rope), dq.ptr, dk.ptr, dv.ptr, hd, hd, hd, do.ptr, dko.ptr, hd, hd,
                                    1, None, b.ref) == 0
    lib.cuda_sync()
    holo.check("bound")
    pos = np.r_[11:20, 0:4]
    kept = [0, 1, 2, 3, 4, 5, 9, 10, 11, 12]
    with np.errstate(invalid="ignore"):
        wq, wk = (dm.turned(x, pos, freq_of(hd), hd, 0, 1.0, hd) for x in (q, k))
    for got, want, x in ((do, wq, q), (dko, wk, k)):
        got = got.download(np.float32).reshape(13, hd)
        assert (got[6:9] == -9.0).all()
        assert np.array_equal(np.isfinite(got[kept]), np.isfinite(want[kept]))
        ok = np.isfinite(want[kept])
        assert (np.abs(got[kept][ok] - want[kept][ok]) <= 2.0 ** -24 * np.abs(want[kept][ok]) + 1e-9).all()
    for i in kept:
        s, p = (0, 11 + i) if i < 9 else (1, i - 9)
        with np.errstate(invalid="ignore"):
            c.put(s, 0, 0, p, wk[i].astype(np.float32), v[i])
    assert np.array_equal(dev.bytes(), c.pool)


# ---- attention ---------------------------------------------------------------------------------------

def attention(holo, dev, layer, q, rows, n_heads, mask, seqs=None, ldq=None, ldo=None, max_rows=None, max_len=None):
    cache = dev.cache
    dim = n_heads * cache.hd
    ldq, ldo = ldq or dim, ldo or dim
    total = sum(rows)
    b = Batch(holo, rows, seqs, max_rows, cache.len.max() if max_len is None else max_len)
    wide = np.full((total, ldq), 7.0, np.float32)
    wide[:, :dim] = q
    dq, do, dm_ = up(holo, wide), up(holo, np.full((total, ldo), -9.0, np.float32)), up(holo, mask)
    assert holo.lib().holo_attention_kv4_draft(dev.ref, layer, do.ptr, dq.ptr, ldo, ldq, n_heads, dm_.ptr,
                                               mask.shape[1], b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("holo_attention_kv4_draft")
    got = do.download(np.float32).reshape(total, ldo)
    assert (got[:, dim:] == -9.0).all()
    return got[:, :dim]


@pytest.mark.parametrize("hd,heads,n_kv,page_len,lens,rows,words", [
    (128, 8, 2, 32, [5, 33, 200], [5, 5, 5], 1),
    (128, 4, 4, 64, [64, 65], [1, 1], 1),
    (64, 12, 2, 32, [31, 32, 100, 45], [1, 5, 40, 33], 2),
    (96, 6, 3, 32, [70, 3], [17, 1], 3),
    (32, 16, 1, 64, [90, 130], [33, 2], 2),
    (64, 40, 2, 32, [75], [7], 1),
    (128, 2, 2, 256, [300, 0, 290], [3, 2, 1], 1),
    (64, 8, 1, 128, [1300, 900], [25, 40], 2),
    (96, 6, 2, 64, [1000], [150], 5),
    (32, 40, 40, 32, [200, 90], [70, 33], 3),
    (128, 16, 2, 32, [140], [9], 1),
    (128, 8, 2, 64, [150, 64], [64, 64], 2),
    (64, 4, 1, 32, [600], [260], 9),
    (32, 3, 1, 32, [1030], [1024], 32),
], ids=str)
def test_attention_of_trees(holo, hd, heads, n_kv, page_len, lens, rows, words):
    print(f"case draft attention hd {hd} heads {heads}/{n_kv} page {page_len} lens {lens} rows {rows}", flush=True)
    rng = np.random.default_rng(len(lens) * hd + heads)
    c = Cache(hd, page_len, 2, n_kv, sum(-(-n // page_len) for n in lens) + 2, len(lens) + 1, -(-max(lens) // page_len))
    pages(c, lens, rng)
    fill(c, rng, 1)
    dev = OnDevice(holo, c)
    seqs = list(range(len(lens)))
    seen = [dm.seen_rows(dm.tree(rng, n, 3)) for n in rows]
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    got = attention(holo, dev, 1, q, rows, heads, np.concatenate([dm.words(s, words) for s in seen]))
    want = dm.want_attention(c, 1, q, rows, seqs, heads, seen)
    assert normwise(got, want) <= TOL
    # the entries in another order, by their sequences; any mask; strides; a far bound on the lengths
    order = seqs[::-1]
    rows2 = [rows[s] for s in order]
    seen = [rng.random((n, n)) < 0.4 for n in rows2]
    mask = np.concatenate([dm.words(s, words) for s in seen])
    for i, n in enumerate(np.cumsum([0, *rows2])[:-1]):  # bits past the entry's rows mean nothing
        extra = dm.words(np.tile(np.arange(32 * words) >= rows2[i], (rows2[i], 1)), words)
        mask[n:n + rows2[i]] |= extra & rng.integers(0, 1 << 32, extra.shape, dtype=np.uint32)
    q2 = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    got = attention(holo, dev, 1, q2, rows2, heads, mask, seqs=order, ldq=heads * hd + 8, ldo=heads * hd + 4,
                    max_len=c.len.max() + 77)
    want = dm.want_attention(c, 1, q2, rows2, order, heads, seen)
    assert normwise(got, want) <= TOL


@pytest.mark.parametrize("rows,heads", [([1, 1, 1], 4), ([5, 5, 5], 4), ([20, 40, 7], 4)], ids=str)
def test_attention_of_long_sequences_is_joined_from_ranges(holo, rows, heads):
    """2,500 positions: many ranges, whose count depends on max_len; the same bits twice."""
    print(f"case draft attention 2500 {rows}", flush=True)
    rng = np.random.default_rng(8)
    hd, n_kv, lens = 64, 1, [2500, 130, 7]
    c = Cache(hd, 128, 1, n_kv, 24, 3, 20)
    pages(c, lens, rng)
    fill(c, rng, 0)
    dev = OnDevice(holo, c)
    seen = [dm.seen_rows(dm.tree(rng, n, 3)) for n in rows]
    mask = np.concatenate([dm.words(s, 2) for s in seen])
    q = (3 * rng.standard_normal((sum(rows), heads * hd))).astype(np.float32)
    want = dm.want_attention(c, 0, q, rows, [0, 1, 2], heads, seen)
    first = attention(holo, dev, 0, q, rows, heads, mask)
    for got in (first, attention(holo, dev, 0, q, rows, heads, mask, max_len=2560),
                attention(holo, dev, 0, q, rows, heads, mask, max_len=100000),
                attention(holo, dev, 0, q, rows, heads, mask, max_len=0x7FFFF000)):
        assert normwise(got, want) <= TOL
    assert np.array_equal(first, attention(holo, dev, 0, q, rows, heads, mask))
    # sharp rows, rows of zeros, tiny q
    at = np.cumsum([0, *rows])
    q[:at[1]] *= 1e3
    q[at[1]:at[2]] = 0
    q[at[2]:] *= 1e-30
    want = dm.want_attention(c, 0, q, rows, [0, 1, 2], heads, seen)
    got = attention(holo, dev, 0, q, rows, heads, mask)
    for i in range(3):
        # sequence 0: a score of about 3e3 is within 2^-21 of it, 1.5e-3, and so a probability
        assert normwise(got[at[i]:at[i + 1]], want[at[i]:at[i + 1]]) <= (2e-3 if i == 0 else TOL)


@pytest.mark.parametrize("heads", [4, 16])
def test_attention_where_nothing_is_seen(holo, heads):
    """Pages that are not there, rows before position 0, entries of no sequence, masks without a bit, on their own and in
    front of rows that see."""
    print(f"case draft attention empty {heads}", flush=True)
    rng = np.random.default_rng(4)
    hd, n_kv = 64, 2
    lens = [100, 3, 0, 96, 64, 33]
    c = Cache(hd, 32, 1, n_kv, 16, 6, 4)
    pages(c, lens, rng)
    fill(c, rng, 0)
    c.table[0, 1] = -1            # a page in the middle is gone
    c.table[3, :] = (-5, 16, 1 << 30, -(1 << 31))  # no page at all: outside the pool
    c.table[4, 0] = 99            # the first page is gone
    dev = OnDevice(holo, c)
    rows, seqs = [2, 5, 1, 3, 40, 1, 1, 33], [0, 1, 2, 3, 4, -1, 6, 5]
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    seen = [dm.seen_rows(dm.tree(rng, n, 2)) for n in rows]
    seen[-1][[0, 5, 17, 32]] = False  # the whole sequence is the entry: nothing before it
    seen[4][:20] = False              # its first 24 positions have no page
    got = attention(holo, dev, 0, q, rows, heads, np.concatenate([dm.words(s, 2) for s in seen]), seqs=seqs)
    want = dm.want_attention(c, 0, q, rows, seqs, heads, seen)
    assert normwise(got, want) <= TOL
    nothing = (want == 0).all(1)
    assert nothing.sum() >= 2 + 1 + 3 + 2 + 4 and (got[nothing] == 0).all()


def test_attention_bounds_of_the_batch(holo):
    """max_rows leaves the rows past it, which others may still see; a sequence past max_len gives NaN; rows past the words
    have no bit."""
    print("case draft attention bounds", flush=True)
    rng = np.random.default_rng(6)
    hd, heads, n_kv, lens = 32, 4, 2, [50, 60]
    c = Cache(hd, 32, 1, n_kv, 4, 2, 2)
    pages(c, lens, rng)
    fill(c, rng, 0)
    dev = OnDevice(holo, c)
    rows = [9, 40]
    q = rng.standard_normal((49, heads * hd)).astype(np.float32)
    seen = [rng.random((n, n)) < 0.5 for n in rows]
    mask = np.concatenate([dm.words(s, 2) for s in seen])
    want = dm.want_attention(c, 0, q, rows, [0, 1], heads, seen)
    kept = [*range(6), *range(9, 15)]
    got = attention(holo, dev, 0, q, rows, heads, mask, max_rows=6)
    assert (np.delete(got, kept, 0) == -9.0).all() and normwise(got[kept], want[kept]) <= TOL
    got = attention(holo, dev, 0, q, rows, heads, mask, max_len=59)
    assert np.isnan(got[9:]).all() and normwise(got[:9], want[:9]) <= TOL
    short = [s & (np.arange(s.shape[1]) < 32) for s in seen]
    got = attention(holo, dev, 0, q, rows, heads, np.ascontiguousarray(mask[:, :1]), max_rows=32)
    kept = [*range(9), *range(9, 41)]
    want = dm.want_attention(c, 0, q, rows, [0, 1], heads, short)
    assert (got[41:] == -9.0).all() and normwise(got[kept], want[kept]) <= TOL


@pytest.mark.parametrize("heads,rows", [(4, 40), (2, 3), (32, 40)])
def test_attention_is_not_touched_by_what_a_row_does_not_see(holo, heads, rows):
    """NaN behind a sequence's end, and NaN and infinite keys and values at drafted rows that only some rows see."""
    print(f"case draft attention poison {heads} {rows}", flush=True)
    rng = np.random.default_rng(7)
    hd, n_kv, n = 64, 2, 77
    seen = [dm.seen_rows(dm.tree(rng, rows, 2))]
    mask = dm.words(seen[0], 2)
    q = rng.standard_normal((rows, heads * hd)).astype(np.float32)
    for fill_byte in (0xFF, 0x7C):  # scales of NaN, of a large finite value
        c = Cache(hd, 32, 1, n_kv, 4, 1, 3, fill=fill_byte)
        pages(c, [n], rng)
        fill(c, rng, 0)
        got = attention(holo, OnDevice(holo, c), 0, q, [rows], heads, mask)
        assert normwise(got, dm.want_attention(c, 0, q, [rows], [0], heads, seen)) <= TOL
    k, v = rng.standard_normal((2, hd)).astype(np.float32)
    v[40] = np.nan
    c.put(0, 0, 1, n - rows + 1, k, v)      # head 1, row 1: dims 32 .. 63 of the value
    bad = rng.standard_normal(hd).astype(np.float32)
    bad[3] = np.inf
    c.put(0, 0, 0, n - rows + 2, bad, bad)  # head 0, row 2: key and value
    got = attention(holo, OnDevice(holo, c), 0, q, [rows], heads, mask).reshape(rows, heads, hd)
    want = dm.want_attention(c, 0, q, [rows], [0], heads, seen).reshape(rows, heads, hd)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    s, g = seen[0], heads // 2
    assert np.isnan(want[s[:, 1], g:, 32:]).all() and not np.isnan(want[~s[:, 1], g:]).any()
    assert np.isnan(want[s[:, 2], :g]).all() and not np.isnan(want[~s[:, 2], :g]).any()
    ok = ~np.isnan(want)
    assert normwise(got[ok], want[ok]) <= TOL
    # q: a NaN or an infinity makes its own row and head NaN
    q[0, 5], q[2, hd + 1] = np.nan, np.inf
    got = attention(holo, OnDevice(holo, c), 0, q, [rows], heads, mask).reshape(rows, heads, hd)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[2, 1]).all()
    got[0, 0], got[2, 1] = want[0, 0], want[2, 1]
    ok = ~np.isnan(want)
    assert normwise(got[ok], want[ok]) <= TOL
    # a NaN value before all rows reaches every one
    c.put(0, 0, 1, 3, k, v)
    got = attention(holo, OnDevice(holo, c), 0, q, [rows], heads, mask).reshape(rows, heads, hd)
    assert np.isnan(got[:, g:, 32:]).all() and not np.isnan(got[~s[:, 1], g:, :32]).any()


def test_attention_of_a_batch_of_many_entries(holo):
    """More workgroups than one row of the grid has: 60000 entries by 80 tiles of columns, a few of them with rows."""
    print("case draft attention 60000 entries", flush=True)
    rng = np.random.default_rng(16)
    hd, heads, n, lens = 32, 40, 60000, [40, 33, 3]
    c = Cache(hd, 32, 1, heads, 6, 3, 2)
    pages(c, lens, rng)
    fill(c, rng, 0)
    dev = OnDevice(holo, c)
    rows, seqs = np.zeros(n, int), np.full(n, -1)
    at = [7, 31234, n - 1]
    rows[at], seqs[at] = [17, 32, 2], [0, 1, 2]
    seen = [dm.seen_rows(dm.tree(rng, r, 2)) for r in (17, 32, 2)]
    q = rng.standard_normal((51, heads * hd)).astype(np.float32)
    got = attention(holo, dev, 0, q, rows.tolist(), heads, np.concatenate([dm.words(s, 1) for s in seen]), seqs=seqs)
    assert normwise(got, dm.want_attention(c, 0, q, [17, 32, 2], [0, 1, 2], heads, seen)) <= TOL


@pytest.mark.parametrize("n", [70, 300, 1024, 1025])
def test_attention_of_many_ragged_sequences_in_ranges(holo, n):
    """Ranges found from the lengths of more entries than a wave has lanes: entries without rows, empty sequences, one
    sequence past max_len, and long ones between short ones."""
    print(f"case draft attention ragged {n}", flush=True)
    rng = np.random.default_rng(n)
    hd, heads, n_kv = 32, 1, 1
    lens = np.minimum(rng.integers(0, 60, n), 50)
    long = rng.choice(n, 6, replace=False)
    lens[long] = [1700, 900, 1311, 257, 1500, 2000]
    c = Cache(hd, 64, 1, n_kv, int(sum(-(-x // 64) for x in lens)) + 1, n, 32)
    pages(c, lens.tolist(), rng)
    c.pool[:] = rng.integers(0, 256, c.pool.shape, dtype=np.uint8)
    f = c.pool[..., 32 * hd:].view(np.uint16)  # scales of 0.5 to 2, either sign, in the cache's 8 significant bits
    f[:] = (f & 0x83F8) | (0x3800 + (f & 0x0400))
    dev = OnDevice(holo, c)
    rows = rng.integers(0, 4, n)
    rows[long] = 3
    order = rng.permutation(n)
    seen = [dm.seen_rows(dm.tree(rng, int(r), 2)) for r in rows[order]]
    mask = np.concatenate([dm.words(s, 1) for s in seen if len(s)])
    q = rng.standard_normal((int(rows.sum()), heads * hd)).astype(np.float32)
    got = attention(holo, dev, 0, q, rows[order].tolist(), heads, mask, seqs=order, max_len=1700)
    want = dm.want_attention(c, 0, q, rows[order].tolist(), order.tolist(), heads, seen)
    first = np.cumsum([0, *rows[order]])[list(order).index(long[5])]
    assert np.isnan(got[first:first + 3]).all()  # 2000 positions
    keep = np.delete(np.arange(len(q)), range(first, first + 3))
    assert normwise(got[keep], want[keep]) <= TOL


# ---- softmax ---------------------------------------------------------------------------------------------

def softmax(holo, x, scale, ldx=None, ldd=None, in_place=False, shift=0):
    """shift: floats that the rows lie past a 16-byte border."""
    rows, n = x.shape
    ldx, ldd = ldx or n, ldd or n
    wide = np.full((rows * ldx + 4,), 3.0, np.float32)
    view = np.lib.stride_tricks.as_strided(wide[shift:], (rows, n), (4 * ldx, 4))
    view[:] = x
    dx = up(holo, wide)
    dd = dx if in_place else up(holo, np.full(rows * ldd + 4, -9.0, np.float32))
    assert holo.lib().holo_softmax_rows(dd.ptr + 4 * shift, dx.ptr + 4 * shift, rows, n, ldx if in_place else ldd, ldx,
                                        scale) == 0
    holo.lib().cuda_sync()
    holo.check("softmax")
    got = dd.download(np.float32)[shift:]
    ldd = ldx if in_place else ldd
    if ldd > n:
        rest = np.lib.stride_tricks.as_strided(got[n:], (rows - 1, ldd - n), (4 * ldd, 4))
        assert (rest == (3.0 if in_place else -9.0)).all()
    return np.lib.stride_tricks.as_strided(got, (rows, n), (4 * ldd, 4)).copy()


def check_softmax(got, x, scale):
    y = (x.astype(np.float64) - x.max(1, keepdims=True).astype(np.float64)) * np.float64(np.float32(scale))
    p = np.exp(y)
    total = p.sum(1, keepdims=True)
    want = p / total
    n = x.shape[1]
    adds = 40 + max(0, n - 32768) / 1024
    mean = (want * np.where(p > 0, -y, 0)).sum(1, keepdims=True)  # of |argument|, in the sum
    with np.errstate(invalid="ignore"):
        tol = np.where(p > 0, 2.0 ** -23 * -y, 0) + 2.0 ** -23 * mean + (8 + adds) * 2.0 ** -24
    assert (np.abs(got - want) <= tol * want + 2e-38 + 1e-38 / total).all()  # (and what lies below a float's normal range)


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 5), (2, 64), (70, 257), (5, 1000), (1, 4096), (7, 4099), (3, 32000),
                                    (2, 32768), (2, 32769), (1, 50257), (2, 131072), (1, 150001), (2000, 33)])
def test_softmax_rows(holo, rows, n):
    print(f"case softmax {rows} x {n}", flush=True)
    rng = np.random.default_rng(rows + n)
    x = (4 * rng.standard_normal((rows, n))).astype(np.float32)
    for scale in (1.0, 0.7, 30.0):
        check_softmax(softmax(holo, x, scale), x, scale)
    got = softmax(holo, x, 1.3)
    for kw in (dict(ldx=n + 3, ldd=n + 1), dict(shift=1), dict(in_place=True), dict(in_place=True, ldx=n + 5, shift=2),
               dict(ldx=n + 4, ldd=n + 8)):
        other = softmax(holo, x, 1.3, **kw)
        check_softmax(other, x, 1.3)
    assert np.array_equal(got, softmax(holo, x, 1.3))


def test_softmax_of_extreme_rows(holo):
    print("case softmax extreme", flush=True)
    inf, big = np.float32(np.inf), np.float32(3.4e38)
    for n in (8, 40000, 40001):
        x = np.zeros((9, n), np.float32)
        x[0] = -inf                                  # nothing: zeros
        x[1, 1:] = -inf                              # one value alone
        x[2] = -big
        x[2, 3] = big                                # a difference past a float's range
        x[3] = -big                                  # all of a type's lowest value: uniform
        x[4, 2] = np.nan
        x[5, 4] = inf
        x[6] = -inf
        x[6, 5:7] = -big                             # two lowest values beside nothing
        x[7, 7] = 1e-30                              # values that a float's step does not part
        x[8] = -inf
        x[8, 0] = np.nan
        with np.errstate(invalid="ignore", over="ignore"):
            got = softmax(holo, x, 2.0)
            one = softmax(holo, x, 3e38)             # as good as the largest alone
        for y in (got, one):
            assert (y[0] == 0).all() and np.isnan(y[[4, 5, 8]]).all()
            assert y[1, 0] == 1 and (y[1, 1:] == 0).all() and y[2, 3] == 1 and (np.delete(y[2], 3) == 0).all()
            assert (np.abs(y[3] - 1 / n) <= 2.0 ** -19 / n).all() and (y[6, 5:7] == 0.5).all() and y[6].sum() == 1
        assert (np.abs(got[7] - 1 / n) <= 2.0 ** -19 / n).all() and one[7, 7] > 0
        z = np.float32([[1, 5, 5, -inf, 4.999999]])
        assert np.array_equal(softmax(holo, z, 1e30), np.float32([[0, 0.5, 0.5, 0, 0]]))


# ---- verification ------------------------------------------------------------------------------------------

MODES = ["chosen", "drawn", "distinct"]


def verify(holo, rows, parents, tokens, u, target, draft, mode, ldt=None, ldd=None, max_rows=None):
    vocab, total = target.shape[1], sum(rows)
    ldt, ldd = ldt or vocab, ldd or vocab
    b = Batch(holo, rows, max_rows=max_rows)

    def wide(x, ld):
        w = np.full((total, ld), 9.0, np.float32)
        w[:, :vocab] = x
        return up(holo, w)

    dt, dd = wide(target, ldt), wide(draft, ldd)
    ins = [up(holo, np.int32(tokens)), up(holo, np.int32([p for t in parents for p in t])), up(holo, np.float32(u))]
    outs = [up(holo, np.full(total + 1, -7, np.int32)), up(holo, np.full(len(rows) + 1, -7, np.int32)),
            up(holo, np.full(len(rows) + 1, -7, np.int32))]
    assert holo.lib().holo_draft_verify(*[o.ptr for o in outs], dt.ptr, None if mode == "chosen" else dd.ptr, ldt, ldd,
                                        vocab, *[i.ptr for i in ins], MODES.index(mode), b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("verify")
    path, n_path, after = (o.download(np.int32) for o in outs)
    assert path[-1] == n_path[-1] == after[-1] == -7
    return path[:-1], n_path[:-1], after[:-1]


def check_verify(holo, rng, rows, width, vocab, mode, sharp=1.0, **kw):
    total = sum(rows)
    z = (2.5 * rng.standard_normal((total, vocab))).astype(np.float32)

    def soft(x):
        p = np.exp(x - x.max(1, keepdims=True), dtype=np.float32)
        return p / p.sum(1, keepdims=True, dtype=np.float32)

    target, draft = soft(z), soft(z + (sharp * rng.standard_normal(z.shape)).astype(np.float32))
    parents = [dm.tree(rng, n, width) for n in rows]
    tokens, at = [], 0
    for t in parents:  # what the mode is for: the most probable ones, draws, draws without repeats
        first, taken = at, {}
        for p in t:
            q = draft[first + max(p, 0)].astype(np.float64)
            mine = taken.setdefault(p, [])
            if mode == "chosen":
                x = int(np.argsort(-q, kind="stable")[min(len(mine), vocab - 1)])
            else:
                if mode == "distinct" and len(mine) < vocab:
                    q[mine] = 0
                x = int(rng.choice(vocab, p=q / q.sum()))
            mine.append(x)
            tokens.append(x)
        at += len(t)
    u = rng.random(total).astype(np.float32)
    path, n_path, after = verify(holo, rows, parents, tokens, u, target, draft, mode, **kw)
    at, long = 0, 0
    for i, t in enumerate(parents):
        n = len(t)
        if n == 0:
            assert n_path[i] == 0 and after[i] == -1
            continue
        want, token, margin = dm.verify(t, tokens[at:at + n], u[at:at + n], target[at:at + n], draft[at:at + n], mode)
        assert margin > 1e-12, "a comparison that 64 bits do not decide"
        assert path[at:at + n].tolist() == want + [-1] * (n - len(want)) and n_path[i] == len(want) and after[i] == token
        long += len(want) > 1
        at += n
    return long


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("rows,width,vocab", [
    ([5] * 40, 1, 1000), ([26, 1, 13, 0, 26, 7], 4, 3001), ([64, 65, 130], 3, 257), ([9] * 30, 8, 12), ([3, 2], 2, 32000),
    ([6] * 4, 5, 131072), ([4], 3, 600001), ([5, 5], 2, 1), ([8] * 6, 3, 2), ([1] * 9, 1, 300)],
                         ids=lambda x: str(x)[:20])
def test_verification(holo, mode, rows, width, vocab):
    print(f"case verify {mode} {rows[:6]} width {width} vocab {vocab}", flush=True)
    rng = np.random.default_rng(vocab + width)
    long = check_verify(holo, rng, rows, width, vocab, mode)
    if len(rows) >= 30:
        assert long > 3  # drafts do stand
    check_verify(holo, rng, rows, width, vocab, mode, sharp=4.0, ldt=vocab + 3, ldd=vocab + 1)


@pytest.mark.parametrize("mode", MODES)
def test_verification_of_a_thousand_rows(holo, mode):
    print(f"case verify {mode} 1024", flush=True)
    rng = np.random.default_rng(1)
    vocab, rows = 40, [1024, 900]
    # one row's target follows the draft: long chains stand
    check_verify(holo, rng, rows, 1, vocab, mode, sharp=0.01)
    check_verify(holo, rng, rows, 1000, vocab, mode, sharp=2.0)  # and many judged behind one row


@pytest.mark.parametrize("mode", MODES)
def test_verification_at_its_borders(holo, mode):
    print(f"case verify borders {mode}", flush=True)
    p = np.zeros((4, 600), np.float32)
    p[:, 3], p[:, 300], p[:, 599] = 0.25, 0.5, 0.25
    q = np.zeros_like(p)
    q[:, 300] = 1.0
    t = [[-1, 0, 0, 1]]
    rows = [4]
    just_below = np.nextafter(np.float32(1), np.float32(0))

    def call(tokens, u, p=p, q=q):
        path, n, after = verify(holo, rows, t, tokens, u, p, q, mode)
        want, token, _ = dm.verify(t[0], tokens, np.float32(u), p, q, mode)
        assert path.tolist() == want + [-1] * (4 - len(want)) and after[0] == token and n[0] == len(want)
        return want, token

    # u of 0 takes whatever has a weight, u below 1 the last of them at most
    assert call([0, 300, 3, 599], [0, 0, 0, 0]) == ([0, 1, 3], 3)
    assert call([0, 300, 300, 300], [just_below] * 4)[0] == [0]
    assert call([0, 300, 300, 300], [just_below] * 4)[1] == 599
    assert call([0, 300, 3, 300], [0.5, 0.5, 0, 0.6])[1] is not None
    # tokens outside the vocabulary, of no probability, the same one twice
    assert call([0, -1, 600, 300], [0.3, 0, 0, 0]) == ([0], 300)
    call([0, 1 << 30, 300, 300], [0.3, 0, 0.4, 0.6])
    call([0, 5, 5, 5], [0.2, 0, 0, 0])
    call([0, 300, 300, 3], [0.7, 0.9, 0.1, 0.2])
    # nothing is left: the most probable token, the lowest of equals
    one = np.zeros_like(p)
    one[:, 7] = 1.0
    if mode != "chosen":
        assert call([0, 9, 9, 9], [0.5, 0.5, 0.5, 0.5], one, one)[1] == 7
    half = np.zeros_like(p)
    half[:, 20] = half[:, 10] = 0.5
    w = call([0, 20, 10, 0], [0.5, 0.6, just_below, 0.5], half, half)
    assert w[1] in (10, 20)
    none = np.zeros_like(p)
    assert call([0, 1, 2, 3], [0.5, 0.5, 0.5, 0.5], none, q)[1] == 0
    # no numbers and negative values count as 0
    bad, worse = p.copy(), q.copy()
    bad[:, 100], bad[:, 101], bad[:, 102] = np.nan, -1.0, np.inf
    worse[:, 3], worse[:, 599], worse[:, 200] = np.nan, -5.0, np.inf
    for tokens in ([0, 300, 3, 599], [0, 100, 101, 102], [0, 102, 300, 3]):
        for u in ([0.1, 0.9, 0.9, 0.9], [0.6, 0.2, 0.5, 0.1], [0.99, 0.7, 0.9, 0.3]):
            call(tokens, u, bad, worse)


def test_verification_of_rows_out_of_place(holo):
    """Parents that are no earlier row, several without any, rows past max_rows, entries cut off by `rows`."""
    print("case verify places", flush=True)
    rng = np.random.default_rng(5)
    vocab = 50
    p = np.full((12, vocab), 1 / vocab, np.float32)
    parent = [-1, 0, 5, 2, -1, 4, 1, 0, 7, 8, -3, 10]
    tokens = rng.integers(0, vocab, 12)
    for mode in MODES:
        for u in (np.zeros(12), rng.random(12), np.full(12, 0.999)):
            path, n, after = verify(holo, [12], [parent], tokens, u, p, p, mode)
            want, token, _ = dm.verify([q if q < i else -1 for i, q in enumerate(parent)], tokens, np.float32(u), p, p, mode)
            assert path.tolist() == want + [-1] * (12 - len(want)) and after[0] == token
            path, n, after = verify(holo, [7, 5], [parent[:7], [-1, 0, 1, 2, 3]], tokens, u, p, p, mode, max_rows=3)
            want, token, _ = dm.verify(parent[:2] + [-1], tokens, np.float32(u), p, p, mode)
            assert path[:3].tolist() == want + [-1] * (3 - len(want)) and after[0] == token and (path[3:7] == -7).all()
            want, token, _ = dm.verify([-1, 0, 1], tokens[7:], np.float32(u[7:]), p, p, mode)
            assert path[7:10].tolist() == want + [-1] * (3 - len(want)) and after[1] == token and (path[10:] == -7).all()


@pytest.mark.parametrize("mode", MODES)
def test_verification_of_many_entries_keeps_the_targets_distribution(holo, mode):
    """60000 entries of the same distributions: the first token behind row 0 has the target's probabilities, within five
    standard deviations of a share; every entry as the model has it."""
    print(f"case verify law {mode}", flush=True)
    rng = np.random.default_rng(17)
    n, t = 60000, [-1, 0, 0, 1]
    p = np.float32([0.4, 0.3, 0.15, 0.1, 0.05, 0])
    q = np.float32([0.1, 0.2, 0.2, 0.25, 0.15, 0.1])
    tokens = rng.integers(0, 6, (n, 4))
    for i in range(n if mode != "chosen" else 0):
        tokens[i, 1:3] = rng.choice(6, 2, mode == "drawn", q.astype(np.float64) / q.sum(dtype=np.float64))
    if mode == "chosen":
        tokens[:, 1:3] = (3, 1)
    u = rng.random((n, 4)).astype(np.float32)
    path, n_path, after = verify(holo, [4] * n, [t] * n, tokens.ravel(), u.ravel(), np.tile(p, (4 * n, 1)),
                                 np.tile(q, (4 * n, 1)), mode)
    path = path.reshape(n, 4)
    first = np.where(n_path > 1, tokens[np.arange(n), path[:, 1]], after)
    share = np.bincount(first, minlength=6) / n
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-7).all()
    for i in range(0, n, 29):
        want, token, margin = dm.verify(t, tokens[i], u[i], np.tile(p, (4, 1)), np.tile(q, (4, 1)), mode)
        # (0.1 * 3 and the like lie on the borders of sums of 0.3: those are for either side)
        if margin > 1e-12:
            assert path[i].tolist() == want + [-1] * (4 - len(want)) and after[i] == token


# ---- the rows that stand ------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,n_kv,page_len,layers", [(128, 2, 32, 3), (64, 1, 64, 1), (96, 3, 32, 2), (32, 2, 128, 2)])
def test_kept_rows(holo, hd, n_kv, page_len, layers):
    """Short and long paths, across tiles and pages, onto themselves, without pages, before position 0; every byte."""
    print(f"case keep hd {hd} page {page_len}", flush=True)
    rng = np.random.default_rng(hd)
    lens = [90, 200, 64, 31, 20, 130, 0, 150]
    c = Cache(hd, page_len, layers, n_kv, 34, 9, 256 // page_len)
    pages(c, lens, rng)
    rows, seqs = [26, 150, 40, 31, 30, 64, 4, 60, 3, 2], [0, 1, 2, 3, 4, 5, 6, 7, -1, 8]
    c.table[5, 64 // page_len] = -1  # a place without a page, from or to which nothing moves
    c.pool[:] = rng.integers(0, 256, c.pool.shape, dtype=np.uint8)
    dev, path, n_path = OnDevice(holo, c), [], []
    for i, n in enumerate(rows):
        kept = {1: 70, 2: 40, 7: 33}.get(i, min(n, 7))
        p = [0] + sorted(rng.choice(np.arange(1, n), kept - 1, replace=False).tolist())
        if i == 2:
            p = list(range(n))        # all of it as it is
        path += p + [-1] * (n - len(p))
        n_path.append(len(p))
    n_path[8], n_path[3] = 99, 0      # more than there are; none
    b = Batch(holo, rows, seqs)
    dp, dn = up(holo, np.int32(path)), up(holo, np.int32(n_path))
    assert holo.lib().holo_kv4_keep(dev.ref, dp.ptr, dn.ptr, b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("keep")
    at = 0
    for n, s, m in zip(rows, seqs, n_path):
        if 0 <= s < 9:
            dm.keep(c, s, n, path[at:at + min(m, n)])
        at += n
    assert np.array_equal(dev.bytes(), c.pool)


def test_kept_rows_within_bounds(holo):
    """Rows that path names outside the entry move nothing, rows past max_rows are not written to."""
    print("case keep bounds", flush=True)
    rng = np.random.default_rng(1)
    c = Cache(64, 32, 2, 1, 4, 1, 3)
    pages(c, [80], rng)
    dev = OnDevice(holo, c)
    path, n = np.int32([0, 3, 8, 1 << 30, -5, -(1 << 31), 9, 0]), np.int32([7])
    b = Batch(holo, [8], max_rows=6)
    dp, dn = up(holo, path), up(holo, n)
    assert holo.lib().holo_kv4_keep(dev.ref, dp.ptr, dn.ptr, b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("keep bounds")
    dm.keep(c, 0, 8, [0, 3])
    assert np.array_equal(dev.bytes(), c.pool)


# ---- offsets that 32 bits do not hold -------------------------------------------------------------------------

def attend_held(q, hk, hv, heads, hd, seen):
    """Attention of q's rows over values [n][n_kv * hd]; seen [rows][n]."""
    out, group = np.zeros((len(q), heads, hd)), heads * hd // hk.shape[1]
    for i in range(len(q)):
        for h in range(heads):
            x = slice(h // group * hd, (h // group + 1) * hd)
            out[i, h] = attend(q[i, h * hd:(h + 1) * hd], hk[:, x], hv[:, x], seen[i])
    return out.reshape(len(q), -1)


def test_a_pool_past_four_gigabytes(holo):
    """Pages whose bytes lie past 2^32: rows rotated into them, a tree's attention, the rows that stand."""
    print("case draft large pool", flush=True)
    rng = np.random.default_rng(21)
    hd, heads, n_kv, n, rows, layer = 128, 8, 8, 1500, 26, 7
    c = Cache(hd, 1024, 1, n_kv, 1, 1, 2)  # the arrays around a pool that only the device holds
    dev, lib = OnDevice(holo, c), holo.lib()
    dev.desc.n_layers, dev.desc.n_pages = 8, 500
    size = lib.holo_kv4_page_bytes(dev.ref)
    assert 470 * size > 1 << 32
    dev.pool = holo.DeviceBuffer(500 * size)
    dev.desc.pool = dev.pool.ptr
    c.table[0], c.len[0] = (499, 470), n
    dev.refresh()
    dim = n_kv * hd
    k, v = rng.standard_normal((2, n, dim)).astype(np.float32)
    q = rng.standard_normal((n, heads * hd)).astype(np.float32)
    dk, dv, dq, do = up(holo, k), up(holo, v), up(holo, q), holo.DeviceBuffer(q.nbytes)
    df = up(holo, np.zeros(hd // 2))  # no angle: rows as they are
    rope = holo.Rope(freq=df.ptr, dims=hd, interleaved=0, scale=1.0)
    b, last = Batch(holo, [n], None, None, n), Batch(holo, [rows], None, None, n)
    parent = dm.tree(rng, rows, 3)
    seen = dm.seen_rows(parent)
    mask, path, n_path = up(holo, dm.words(seen, 1)), up(holo, np.int32([0, 3, 4, 11, 25] + [-1] * 21)), up(holo, np.int32([5]))
    for i in range(8):  # (every layer: the rows that stand are moved in all of them)
        assert lib.holo_kv4_append_rope(dev.ref, i, C.byref(rope), dq.ptr, dk.ptr, dv.ptr, dim, dim, dim, dq.ptr, None, dim, 0,
                                        heads, None, b.ref) == 0
    assert lib.holo_attention_kv4_draft(dev.ref, layer, do.ptr, dq.ptr + 4 * (n - rows) * dim, dim, dim, heads, mask.ptr, 1,
                                        last.ref) == 0
    lib.cuda_sync()
    holo.check("large pool")
    assert np.array_equal(dq.download(np.float32), q.ravel())
    hk, hv = values(*quantise(k)), values(*quantise(v))
    see = np.concatenate([np.ones((rows, n - rows), bool), seen], 1)
    got = do.download(np.float32)[:rows * dim].reshape(rows, dim)
    assert normwise(got, attend_held(q[n - rows:], hk, hv, heads, hd, see)) <= TOL
    assert lib.holo_kv4_keep(dev.ref, path.ptr, n_path.ptr, last.ref) == 0
    for x in (hk, hv):
        x[n - rows:n - rows + 5] = x[n - rows + np.array([0, 3, 4, 11, 25])]
    for i in (0, layer):
        assert lib.holo_kv4_read(dev.ref, i, dk.ptr, dv.ptr, dim, dim, b.ref) == 0
        lib.cuda_sync()
        holo.check("large pool, kept")
        assert np.array_equal(dk.download(np.float32), hk.ravel()) and np.array_equal(dv.download(np.float32), hv.ravel())


def test_the_last_positions_there_are(holo):
    """A sequence of 0x7FFFF000 positions, of which the last page is there: a tree's attention, the rows that stand."""
    print("case draft last positions", flush=True)
    rng = np.random.default_rng(22)
    hd, rows, n, held = 32, 20, 0x7FFFF000, 1024
    c = Cache(hd, 1024, 1, 1, 2, 1, n // 1024)
    c.table[0, -1], c.len[0] = 1, n
    dev, lib = OnDevice(holo, c), holo.lib()
    k, v, q = rng.standard_normal((3, held, hd)).astype(np.float32)
    dk, dv, dq, do = up(holo, k), up(holo, v), up(holo, q), holo.DeviceBuffer(4 * rows * hd)
    held_rows = Batch(holo, [held], None, None, n)
    assert lib.holo_kv4_append(dev.ref, 0, dk.ptr, dv.ptr, hd, hd, held_rows.ref) == 0
    hk, hv = values(*quantise(k)), values(*quantise(v))
    seen = dm.seen_rows(dm.tree(rng, rows, 2))
    see = np.concatenate([np.ones((rows, held - rows), bool), seen], 1)
    mask, b = up(holo, dm.words(seen, 1)), Batch(holo, [rows], None, None, n)
    path, n_path = up(holo, np.int32([0, 2, 3, 19] + [-1] * 16)), up(holo, np.int32([4]))
    assert lib.holo_attention_kv4_draft(dev.ref, 0, do.ptr, dq.ptr, hd, hd, 1, mask.ptr, 1, b.ref) == 0
    assert lib.holo_kv4_keep(dev.ref, path.ptr, n_path.ptr, b.ref) == 0
    assert lib.holo_kv4_read(dev.ref, 0, dk.ptr, dv.ptr, hd, hd, held_rows.ref) == 0
    lib.cuda_sync()
    holo.check("last positions")
    assert normwise(do.download(np.float32).reshape(rows, hd), attend_held(q[:rows], hk, hv, 1, hd, see)) <= TOL
    for x, got in ((hk, dk), (hv, dv)):
        x[held - rows:held - rows + 4] = x[held - rows + np.array([0, 2, 3, 19])]
        assert np.array_equal(got.download(np.float32), x.ravel())


# ---- all of it ---------------------------------------------------------------------------------------------------

class Step:
    """The device's side of a step of drafted rows: buffers for at most n_seqs entries of max_rows rows."""

    def __init__(self, holo, dev, heads, vocab, n_seqs, max_rows, max_len, freq, layers):
        self.holo, self.dev, self.heads, self.vocab, self.layers = holo, dev, heads, vocab, layers
        c = dev.cache
        self.qd, self.kd, n = heads * c.hd, c.n_kv * c.hd, n_seqs * max_rows
        self.ld = self.qd + 2 * self.kd
        new = holo.DeviceBuffer
        self.qkv = [new(4 * n * self.ld) for _ in range(layers)]
        self.out = [new(4 * n * self.qd) for _ in range(layers)]
        self.logits, self.draft = new(4 * n * vocab), new(4 * n * vocab)
        self.parent, self.depth, self.mask, self.tokens, self.u, self.path = (new(4 * n) for _ in range(6))
        self.n_path, self.next, self.cu, self.seqs = (new(4 * (n_seqs + 1)) for _ in range(4))
        self.freq = up(holo, freq)
        self.rope = holo.Rope(freq=self.freq.ptr, dims=2 * len(freq), interleaved=0, scale=1.0)
        self.b = holo.Batch(rows=n, n_seqs=n_seqs, max_rows=max_rows, max_len=max_len, cu_rows=self.cu.ptr,
                            seqs=self.seqs.ptr)
        self.ref = C.byref(self.b)

    def issue(self):
        """Every call of a step but the pages'."""
        lib, dev = self.holo.lib(), self.dev
        assert lib.holo_draft_plan(self.parent.ptr, self.depth.ptr, self.mask.ptr, 1, self.ref) == 0
        for layer in range(self.layers):
            q = self.qkv[layer].ptr
            k, v = q + 4 * self.qd, q + 4 * (self.qd + self.kd)
            assert lib.holo_kv4_append_rope(dev.ref, layer, C.byref(self.rope), q, k, v, self.ld, self.ld, self.ld, q,
                                            None, self.ld, 0, self.heads, self.depth.ptr, self.ref) == 0
            assert lib.holo_attention_kv4_draft(dev.ref, layer, self.out[layer].ptr, q, self.qd, self.ld, self.heads,
                                                self.mask.ptr, 1, self.ref) == 0
        assert lib.holo_softmax_rows(self.logits.ptr, self.logits.ptr, self.b.rows, self.vocab, self.vocab, self.vocab,
                                     0.8) == 0
        assert lib.holo_draft_verify(self.path.ptr, self.n_path.ptr, self.next.ptr, self.logits.ptr, self.draft.ptr,
                                     self.vocab, self.vocab, self.vocab, self.tokens.ptr, self.parent.ptr, self.u.ptr,
                                     self.holo.DRAFT_DRAWN, self.ref) == 0
        assert lib.holo_kv4_keep(dev.ref, self.path.ptr, self.n_path.ptr, self.ref) == 0


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,page_len", [(64, 8, 2, 32), (128, 4, 4, 64)])
def test_steps_of_drafted_rows(holo, hd, heads, n_kv, page_len, captured):
    """Prompts, then steps of drafted trees: after each the cache holds, bit for bit, what the rows that stand give when
    they are appended one after the other, and their outputs are those of a step per token.  Captured: one graph, replayed
    with the program's own work on the pages between the replays."""
    print(f"case drafted steps hd {hd} captured {captured}", flush=True)
    rng = np.random.default_rng(hd)
    lib, layers, n_seqs, most, vocab = holo.lib(), 2, 3, 9, 64
    c = Cache(hd, page_len, layers, n_kv, 30, n_seqs, 8)
    dev = OnDevice(holo, c)
    handle = lib.holo_kv4_pages_create(dev.ref)
    assert handle
    ints = lambda x: (C.c_int * max(len(x), 1))(*x)
    freq = freq_of(hd)
    step = Step(holo, dev, heads, vocab, n_seqs, most, 256, freq, layers)
    kept = {(s, l): [np.zeros((0, n_kv * hd), np.float32)] * 2 for s in range(n_seqs) for l in range(layers)}
    before, st = lib.holo_get_stream(), lib.holo_stream_create()
    lib.holo_set_stream(st)
    graph = None
    try:
        lens = [40, 95, 3]
        assert lib.holo_kv4_pages_reserve(handle, ints([0, 1, 2]), ints(lens), 3) == 0
        b = Batch(holo, lens)
        for l in range(layers):
            k, v = rng.standard_normal((2, sum(lens), n_kv * hd)).astype(np.float32)
            dk, dv = up(holo, k), up(holo, v)
            assert lib.holo_kv4_append_rope(dev.ref, l, C.byref(step.rope), None, dk.ptr, dv.ptr, 0, n_kv * hd, n_kv * hd,
                                            None, dk.ptr, 0, n_kv * hd, 0, None, b.ref) == 0
            lib.cuda_sync()
            k, at = dk.download(np.float32).reshape(k.shape), 0
            for s, n in enumerate(lens):
                kept[s, l] = [k[at:at + n], v[at:at + n]]
                at += n
        if captured:
            step.cu.upload(np.int32([0] * (n_seqs + 1)))
            assert lib.holo_graph_begin() == 0
            step.issue()
            graph = lib.holo_graph_end()
            assert graph
        for turn in range(4):
            seqs = [[0, 1, 2], [2, 0], [1, 2, 0], [1]][turn]
            rows = [[9, 5, 1], [9, 9], [4, 8, 9], [6]][turn]
            cu = np.concatenate(([0], np.cumsum(rows + [0] * (n_seqs - len(rows))))).astype(np.int32)
            total = int(cu[-1])
            assert lib.holo_kv4_pages_reserve(handle, ints(seqs), ints(rows), len(seqs)) == 0
            parents = [dm.tree(rng, n, 3) for n in rows]
            step.cu.upload(cu)
            step.seqs.upload(np.int32(seqs + [-1] * (n_seqs - len(seqs))))
            step.parent.upload(np.int32([p for t in parents for p in t]))
            qkv = rng.standard_normal((layers, total, step.ld)).astype(np.float32)
            for l in range(layers):
                step.qkv[l].upload(qkv[l])
            z = (2 * rng.standard_normal((n_seqs * most, vocab))).astype(np.float32)
            q = np.exp(z + 0.7 * rng.standard_normal(z.shape))
            q = (q / q.sum(1, keepdims=True)).astype(np.float32)
            tokens = np.int32([rng.choice(vocab, p=q[cu[i] + max(p, 0)].astype(np.float64) / q[cu[i] + max(p, 0)].sum(
                dtype=np.float64)) for i, t in enumerate(parents) for p in t])
            u = rng.random(total).astype(np.float32)
            step.logits.upload(z)
            step.draft.upload(q)
            step.tokens.upload(tokens)
            step.u.upload(u)
            lib.cuda_sync()
            if captured:
                assert lib.holo_graph_launch(graph) == 0
            else:
                step.issue()
            lib.cuda_sync()
            holo.check("step")
            p = step.logits.download(np.float32).reshape(z.shape)
            check_softmax(p[:total], z[:total], 0.8)
            path, n_path, after = (x.download(np.int32) for x in (step.path, step.n_path, step.next))
            trims = []
            for i, (s, n, t) in enumerate(zip(seqs, rows, parents)):
                at = cu[i]
                want, token, margin = dm.verify(t, tokens[at:at + n], u[at:at + n], p[at:at + n], q[at:at + n], "drawn")
                assert margin > 1e-12 and path[at:at + n].tolist() == want + [-1] * (n - len(want)) and after[i] == token
                trims.append(n - n_path[i])
                old = len(kept[s, 0][0])
                for l in range(layers):
                    rq = step.qkv[l].download(np.float32).reshape(-1, step.ld)[at:at + n, :step.qd]
                    out = step.out[l].download(np.float32).reshape(-1, step.qd)[at:at + n]
                    depth = dm.seen_rows(t).sum(1) - 1
                    kq, v = qkv[l, at:at + n, step.qd:step.qd + step.kd], qkv[l, at:at + n, step.qd + step.kd:]
                    k = dm.turned(kq, old + depth, freq, hd, 0, 1.0, hd).astype(np.float32)
                    k, v = (np.concatenate((a, x[want])) for a, x in zip(kept[s, l], (k, v)))
                    kept[s, l] = [k, v]
                    hk, hv = (values(*quantise(x)).reshape(-1, n_kv, hd) for x in (k, v))
                    for j, row in enumerate(want):  # a step per token
                        for h in range(heads):
                            y = attend(rq[row, h * hd:(h + 1) * hd], hk[:, h * n_kv // heads], hv[:, h * n_kv // heads],
                                       np.arange(len(k)) <= old + j)
                            assert normwise(out[row, h * hd:(h + 1) * hd], y) <= 3 * TOL  # (one row and head alone)
            assert lib.holo_kv4_pages_trim(handle, ints(seqs), ints(trims), len(seqs)) == 0
            for s in range(n_seqs):
                n = lib.holo_kv4_pages_len(handle, s)
                assert n == len(kept[s, 0][0])
                b = Batch(holo, [n], [s])
                for l in range(layers):
                    dk, dv = holo.DeviceBuffer(4 * n * n_kv * hd), holo.DeviceBuffer(4 * n * n_kv * hd)
                    assert lib.holo_kv4_read(dev.ref, l, dk.ptr, dv.ptr, n_kv * hd, n_kv * hd, b.ref) == 0
                    lib.cuda_sync()
                    for got, x in zip((dk, dv), kept[s, l]):
                        assert np.array_equal(got.download(np.float32).reshape(n, -1), values(*quantise(x)))
    finally:
        if graph:
            lib.holo_graph_destroy(graph)
        lib.holo_set_stream(before)
        lib.holo_stream_destroy(st)
        lib.holo_kv4_pages_destroy(handle)


@pytest.mark.parametrize("hd,heads,rows,vocab", [(64, 4, 5, 3000), (128, 32, 20, 40000)])
def test_two_graphs_at_once(holo, hd, heads, rows, vocab):
    """Attention in ranges and verification, captured on two streams and replayed together, after lengths, masks, random
    numbers and probabilities changed; eager calls between the replays.  The second size's partial sums are past 1 MiB."""
    print(f"case draft two graphs hd {hd} rows {rows}", flush=True)
    rng = np.random.default_rng(hd)
    lib, n_kv, n = holo.lib(), max(heads // 4, 1), 2500 if hd == 64 else 1700
    before, streams, sides = lib.holo_get_stream(), [lib.holo_stream_create() for _ in range(2)], []
    dim = heads * hd
    new = holo.DeviceBuffer
    try:
        for side in range(2):
            c = Cache(hd, 64, 1, n_kv, 60, 2, 50)
            pages(c, [n + 6, 100], rng)
            c.len[:] = (n, 90)
            c.pool[:] = rng.integers(0, 256, c.pool.shape, dtype=np.uint8)
            f = c.pool[..., 32 * hd:].view(np.uint16)  # scales of 1/16 to 1/4, in the cache's 8 significant bits
            f[:] = (f & 0x83F8) | (0x2C00 + (f & 0x0400))
            dev, b = OnDevice(holo, c), Batch(holo, [rows, 3], [0, 1], None, 3000)
            total = rows + 3
            d = dict(q=new(4 * total * dim), o=new(4 * total * dim), mask=new(4 * total), parent=new(4 * total),
                     depth=new(4 * total), p=new(4 * total * vocab), d=new(4 * total * vocab), tokens=new(4 * total),
                     u=new(4 * total), path=new(4 * total), count=new(8), next=new(8))

            def issue(dev=dev, b=b, d=d):
                assert lib.holo_draft_plan(d["parent"].ptr, d["depth"].ptr, d["mask"].ptr, 1, b.ref) == 0
                assert lib.holo_attention_kv4_draft(dev.ref, 0, d["o"].ptr, d["q"].ptr, dim, dim, heads, d["mask"].ptr, 1,
                                                    b.ref) == 0
                assert lib.holo_draft_verify(d["path"].ptr, d["count"].ptr, d["next"].ptr, d["p"].ptr, d["d"].ptr, vocab,
                                             vocab, vocab, d["tokens"].ptr, d["parent"].ptr, d["u"].ptr,
                                             holo.DRAFT_DISTINCT, b.ref) == 0

            lib.holo_set_stream(streams[side])
            assert lib.holo_graph_begin() == 0
            issue()
            graph = lib.holo_graph_end()
            assert graph
            holo.check("capture")
            sides.append((c, dev, b, d, issue, graph))
        for step in range(3):
            wants = []
            for side, (c, dev, b, d, issue, graph) in enumerate(sides):
                lib.holo_set_stream(streams[side])
                c.len += 1
                dev.refresh()
                parents = [dm.tree(rng, k, 3) for k in (rows, 3)]
                seen = [dm.seen_rows(t) for t in parents]
                total = rows + 3
                q = rng.standard_normal((total, dim)).astype(np.float32)
                z = (2 * rng.standard_normal((total, vocab))).astype(np.float32)
                p, r = np.exp(z), np.exp(z + rng.standard_normal(z.shape).astype(np.float32))
                p, r = (x / x.sum(1, keepdims=True) for x in (p, r))
                flat = [x for t in parents for x in t]
                first = [0] * rows + [rows] * 3
                tokens = np.int32([r[first[i] + max(x, 0)].argsort()[-1 - i % 3] for i, x in enumerate(flat)])
                u = rng.random(total).astype(np.float32)
                for name, x in (("q", q), ("parent", np.int32(flat)), ("p", p), ("d", r), ("tokens", tokens), ("u", u)):
                    d[name].upload(np.ascontiguousarray(x))
                paths = [dm.verify(parents[i], tokens[a:e], u[a:e], p[a:e], r[a:e], "distinct")
                         for i, (a, e) in enumerate(((0, rows), (rows, total)))]
                wants.append((dm.want_attention(c, 0, q, [rows, 3], [0, 1], heads, seen), paths))
            lib.cuda_sync()
            for side in range(2):  # both under way at once
                lib.holo_set_stream(streams[side])
                assert lib.holo_graph_launch(sides[side][5]) == 0
            for again in range(2):  # then the same calls eagerly
                lib.cuda_sync()
                holo.check("replay")
                for side, ((c, dev, b, d, issue, graph), (want, paths)) in enumerate(zip(sides, wants)):
                    assert normwise(d["o"].download(np.float32).reshape(want.shape), want) <= TOL
                    path, count, after = (d[x].download(np.int32) for x in ("path", "count", "next"))
                    for i, (rows_of, token, margin) in enumerate(paths):
                        a, e = ((0, rows), (rows, rows + 3))[i]
                        assert margin > 1e-12
                        assert path[a:e].tolist() == rows_of + [-1] * (e - a - len(rows_of))
                        assert count[i] == len(rows_of) and after[i] == token
                    if not again:
                        d["o"].upload(np.zeros(want.shape, np.float32))
                        lib.holo_set_stream(streams[side])
                        issue()
    finally:
        for *_, graph in sides:
            lib.holo_graph_destroy(graph)
        lib.holo_set_stream(before)
        for s in streams:
            lib.holo_stream_destroy(s)
