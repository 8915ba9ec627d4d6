"""The 4-bit cache on the GPU: rows in and out of its pages bit for bit, and
attention over them against float64 numpy on the values that the cache holds.

Tolerance of attention, 1e-5 normwise: the cached values are exact f16 numbers,
q and the probabilities two f16 halves (2^-22 of a value), sums of 32 to 128
products in fp32 (sqrt(2 * 128) * 2^-24 = 9.5e-7 of the sum of magnitudes,
about sqrt(hd) for normal q and k once divided by sqrt(hd)): a score is within
1.2e-5 at most and 2e-6 in the mean, and a probability within that relative;
the output averages them."""
import numpy as np
import pytest

from kv4_model import Batch, Cache, OnDevice, normwise, quantise, values, want_attention

pytestmark = pytest.mark.gpu

TOL = 1e-5


def up(holo, a):
    return holo.DeviceBuffer.from_array(np.ascontiguousarray(a))


def pages(cache, lens, rng, spare=0):
    """Pages in random order for sequences of these lengths."""
    order = list(rng.permutation(cache.n_pages))
    for s, n in enumerate(lens):
        k = -(-n // cache.page_len)
        cache.table[s, :k] = [order.pop() for _ in range(k)]
        cache.len[s] = n


def fill(cache, rng, lens, layer, scale=1.0):
    """Normal keys and values at every position of the sequences."""
    for s, n in enumerate(lens):
        for h in range(cache.n_kv):
            for p in range(n):
                k, v = rng.standard_normal((2, cache.hd)).astype(np.float32) * np.float32(scale)
                cache.put(s, layer, h, p, k, v)


def attention(holo, dev, layer, q, rows, n_heads, seqs=None, ldq=None, ldo=None, max_rows=None, max_len=None):
    cache = dev.cache
    dim = n_heads * cache.hd
    ldq, ldo = ldq or dim, ldo or dim
    total = sum(rows)
    b = Batch(holo, rows, seqs, max_rows, cache.len.max() if max_len is None else max_len)
    wide = np.full((total, ldq), 7.0, np.float32)
    wide[:, :dim] = q
    dq, do = up(holo, wide), up(holo, np.full((total, ldo), -9.0, np.float32))
    assert holo.lib().holo_attention_kv4(dev.ref, layer, do.ptr, dq.ptr, ldo, ldq, n_heads, b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("holo_attention_kv4")
    got = do.download(np.float32).reshape(total, ldo)
    assert (got[:, dim:] == -9.0).all()
    return got[:, :dim]


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("page_len", [32, 128])
def test_rows_into_pages_and_back(holo, hd, page_len):
    """Three appends of ragged rows, the whole pool checked byte by byte after each."""
    print(f"case kv4 append hd {hd} page {page_len}", flush=True)
    rng = np.random.default_rng(hd + page_len)
    n_kv, layers, layer = 3, 2, 1
    c = Cache(hd, page_len, layers, n_kv, 30, 5, 160 // page_len + 1)
    pages(c, [150, 40, 1, 0, 97], rng)
    c.len[:] = 0
    dev = OnDevice(holo, c)
    dim, lib = n_kv * hd, holo.lib()
    for rows, seqs in (([3, 40, 1, 60], [4, 0, 2, 1]), ([1, 1, 0], [4, 0, 3]), ([33, 109], [4, 0])):
        for n, s in zip(rows, seqs):
            c.len[s] = min(c.len[s] + n, 40 if s == 1 else 1000)  # sequence 1: 60 rows, 20 of them before position 0
        dev.refresh()
        total, ld = sum(rows), dim + 8
        k, v = rng.standard_normal((2, total, ld)).astype(np.float32)
        b = Batch(holo, rows, seqs)
        dk, dv = up(holo, k), up(holo, v)
        assert lib.holo_kv4_append(dev.ref, layer, dk.ptr, dv.ptr, ld, ld, b.ref) == 0
        at = 0
        for n, s in zip(rows, seqs):
            for i in range(n):
                p = c.len[s] - n + i
                for h in range(n_kv):
                    if p >= 0:
                        c.put(s, layer, h, p, k[at + i, h * hd:(h + 1) * hd], v[at + i, h * hd:(h + 1) * hd])
            at += n
        ok, ov = (up(holo, np.full((total, ld), 5.0, np.float32)) for _ in range(2))
        assert lib.holo_kv4_read(dev.ref, layer, ok.ptr, ov.ptr, ld, ld, b.ref) == 0
        lib.cuda_sync()
        holo.check("append and read")
        assert np.array_equal(dev.bytes(), c.pool)
        for x, out in ((k, ok), (v, ov)):
            got = out.download(np.float32).reshape(total, ld)
            want = values(*quantise(x[:, :dim]))
            at = 0
            for n, s in zip(rows, seqs):
                want[at:at + max(0, n - c.len[s])] = 0  # rows before position 0
                at += n
            assert np.array_equal(got[:, :dim], want) and (got[:, dim:] == 5.0).all()


def test_blocks_of_every_kind(holo):
    """Zeros, signed zeros, one value, values in the middle of two codes, equal
    magnitudes of both signs, the smallest and largest, infinities and NaN."""
    print("case kv4 blocks", flush=True)
    rng = np.random.default_rng(5)
    hd, rows = 64, []

    def block(*x):
        b = np.zeros(32, np.float32)
        b[:len(x)] = x
        rows.append(b)

    block()
    block(-0.0, 0.0)
    block(1.0)
    block(-1.0)
    block(-8.0, *[i + 0.5 for i in range(-8, 8)])  # d = 1: every middle, to the even code
    block(8.0, *[i + 0.5 for i in range(-8, 8)])   # d = -1
    block(-8.0, *np.nextafter(np.float32([i + 0.5 for i in range(-8, 8)]), np.float32(99)))
    block(-8.0, *np.nextafter(np.float32([i + 0.5 for i in range(-8, 8)]), np.float32(-99)))
    block(3.0, -3.0, 1.0)
    block(*[1e-9] * 32)
    block(2.0 ** -22, -2.0 ** -23)                 # d below f16's smallest step, and at it
    block(2.0 ** -21, 2.0 ** -20)
    block(*(3e-6 * rng.standard_normal(32)))
    block(1e-45, 1.0)
    block(21760.0, -21760.0, 5000.0)
    block(30000.0, -2e5, 3.4e38)
    block(np.inf, 1.0)
    block(1.0, -np.inf)
    block(np.nan)
    for e in range(-24, 15):
        block(*(2.0 ** e * rng.standard_normal(32)))
    if len(rows) % 2:
        block()
    x = np.stack(rows).reshape(-1, hd)
    # steps of an eighth of the scale: many values next to a border, many on it
    x = np.concatenate([x, (rng.integers(-64, 65, (200, hd)) / np.float32(8)).astype(np.float32)])
    n = len(x)
    c = Cache(hd, 32, 1, 1, -(-n // 32), 1, -(-n // 32))
    c.table[0] = np.arange(c.n_pages)
    c.len[0] = n
    dev, b, lib = OnDevice(holo, c), Batch(holo, [n]), holo.lib()
    dk, dv = up(holo, x), up(holo, x[::-1])
    ok, ov = holo.DeviceBuffer(x.nbytes), holo.DeviceBuffer(x.nbytes)
    assert lib.holo_kv4_append(dev.ref, 0, dk.ptr, dv.ptr, hd, hd, b.ref) == 0
    assert lib.holo_kv4_read(dev.ref, 0, ok.ptr, ov.ptr, hd, hd, b.ref) == 0
    lib.cuda_sync()
    holo.check("blocks")
    want = values(*quantise(x))
    assert np.array_equal(ok.download(np.float32).reshape(n, hd), want, equal_nan=True)
    assert np.array_equal(ov.download(np.float32).reshape(n, hd), values(*quantise(x[::-1])), equal_nan=True)
    finite = np.isfinite(x.reshape(-1, 32)).all(1)
    got = want.reshape(-1, 32)[finite]
    assert np.isfinite(got).all() and np.isnan(want.reshape(-1, 32)[~finite]).all()
    # within half a step, and a whole one for the far sign (codes -8 .. 7), of a scale
    # within 2^-9 and 2^-25 of an eighth of the largest value
    src = x.reshape(-1, 32)[finite].astype(np.float64)
    big = np.abs(src).max(1, keepdims=True)
    small = big[:, 0] <= 21760
    step = big / 8 * (1 + 2.0 ** -8) + 2.0 ** -24
    assert (np.abs(got - src) <= step + 8 * 2.0 ** -25 + big * 2.0 ** -8)[small].all()


@pytest.mark.parametrize("hd,heads,n_kv,page_len,lens,rows", [
    (128, 8, 2, 32, [1, 33, 200], [1, 1, 1]),
    (128, 4, 4, 64, [64, 65], [1, 1]),
    (64, 12, 2, 32, [31, 32, 100, 5], [1, 5, 40, 5]),
    (96, 6, 3, 32, [70, 3], [17, 1]),
    (32, 16, 1, 64, [90, 130], [33, 2]),
    (64, 40, 2, 32, [75], [7]),
    (128, 2, 2, 256, [300, 0, 290], [3, 2, 1]),
    (64, 8, 1, 128, [1300, 900], [25, 40]),
    (96, 6, 2, 64, [1000], [150]),
    (32, 40, 40, 32, [200, 90], [70, 33]),
    (128, 16, 2, 32, [140], [9]),
], ids=str)
def test_attention_over_pages(holo, hd, heads, n_kv, page_len, lens, rows):
    print(f"case kv4 attention hd {hd} heads {heads}/{n_kv} page {page_len} lens {lens} rows {rows}", flush=True)
    rng = np.random.default_rng(len(lens) * hd + heads)
    c = Cache(hd, page_len, 2, n_kv, sum(-(-n // page_len) for n in lens) + 2, len(lens) + 1,
              -(-max(lens) // page_len))
    pages(c, lens, rng)
    fill(c, rng, lens, 1)
    dev = OnDevice(holo, c)
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    seqs = list(range(len(lens)))
    got = attention(holo, dev, 1, q, rows, heads)
    want = want_attention(c, 1, q, rows, c.len, seqs, heads)
    assert normwise(got, want) <= TOL
    # the entries in another order, by their sequences; strides; a bound on the rows
    order = seqs[::-1]
    rows2 = [rows[s] for s in order]
    q2 = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    got = attention(holo, dev, 1, q2, rows2, heads, seqs=order, ldq=heads * hd + 8, ldo=heads * hd + 4,
                    max_len=c.len.max() + 77)
    want = want_attention(c, 1, q2, rows2, c.len, order, heads)
    assert normwise(got, want) <= TOL


def test_attention_of_a_long_sequence_is_joined_from_ranges(holo):
    """2,500 positions: many ranges, whose count depends on max_len; the same bits twice."""
    print("case kv4 attention 2500", flush=True)
    rng = np.random.default_rng(8)
    hd, heads, n_kv, lens = 64, 4, 1, [2500, 130, 7]
    c = Cache(hd, 128, 1, n_kv, 24, 3, 20)
    pages(c, lens, rng)
    fill(c, rng, lens, 0)
    dev = OnDevice(holo, c)
    q = (3 * rng.standard_normal((3, heads * hd))).astype(np.float32)
    want = want_attention(c, 0, q, [1, 1, 1], c.len, [0, 1, 2], heads)
    first = attention(holo, dev, 0, q, [1, 1, 1], heads)
    for got in (first, attention(holo, dev, 0, q, [1, 1, 1], heads, max_len=2560),
                attention(holo, dev, 0, q, [1, 1, 1], heads, max_len=100000)):
        assert normwise(got, want) <= TOL
    assert np.array_equal(first, attention(holo, dev, 0, q, [1, 1, 1], heads))
    # a wide range of scores: sharp rows, rows of zeros, tiny and huge q
    q[0] *= 1e3
    q[1] = 0
    q[2] *= 1e-30
    want = want_attention(c, 0, q, [1, 1, 1], c.len, [0, 1, 2], heads)
    got = attention(holo, dev, 0, q, [1, 1, 1], heads)
    for i in range(3):
        # row 0: a score of about 3e3 is within 2^-21 of it, 1.5e-3, and so a probability
        assert normwise(got[i], want[i]) <= (2e-3 if i == 0 else TOL)


def test_rows_that_see_nothing_and_pages_that_are_not_there(holo):
    print("case kv4 attention empty", flush=True)
    rng = np.random.default_rng(4)
    hd, heads, n_kv = 64, 4, 2
    lens = [100, 3, 0, 96, 64]
    c = Cache(hd, 32, 1, n_kv, 16, 5, 4)
    pages(c, lens, rng)
    fill(c, rng, lens, 0)
    c.table[0, 1] = -1            # a page in the middle is gone
    c.table[3, :] = (-5, 16, 1 << 30, -(1 << 31))  # no page at all: outside the pool
    c.table[4, 0] = 99            # the first page is gone
    dev = OnDevice(holo, c)
    # 5 rows of a sequence of 3: two of them before position 0; entries of no sequence
    rows, seqs = [2, 5, 1, 3, 40, 1, 1], [0, 1, 2, 3, 4, -1, 5]
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    got = attention(holo, dev, 0, q, rows, heads, seqs=seqs)
    want = want_attention(c, 0, q, rows, c.len, seqs, heads)
    assert normwise(got, want) <= TOL
    nothing = (want == 0).all(1)
    # two before position 0, one of an empty sequence, three without pages, positions 24 .. 31, two of no sequence
    assert nothing.sum() == 2 + 1 + 3 + 8 + 2 and (got[nothing] == 0).all()
    # nothing is stored where there is no page, and nothing else is touched
    k = rng.standard_normal((sum(rows), n_kv * hd)).astype(np.float32)
    b, lib = Batch(holo, rows, seqs), holo.lib()
    dk = up(holo, k)
    assert lib.holo_kv4_append(dev.ref, 0, dk.ptr, dk.ptr, n_kv * hd, n_kv * hd, b.ref) == 0
    ok, ov = (up(holo, np.full(k.shape, 5.0, np.float32)) for _ in range(2))
    assert lib.holo_kv4_read(dev.ref, 0, ok.ptr, ov.ptr, n_kv * hd, n_kv * hd, b.ref) == 0
    lib.cuda_sync()
    holo.check("no pages")
    at = 0
    for n, s in zip(rows, seqs):
        for i in range(n):
            if 0 <= s < 5:
                for h in range(n_kv):
                    if c.len[s] - n + i >= 0:
                        x = k[at + i, h * hd:(h + 1) * hd]
                        c.put(s, 0, h, c.len[s] - n + i, x, x)
        at += n
    assert np.array_equal(dev.bytes(), c.pool)
    held, at = ok.download(np.float32).reshape(k.shape), 0
    want = values(*quantise(k))
    for n, s in zip(rows, seqs):
        for i in range(n):
            p = c.len[s] - n + i if 0 <= s < 5 else -1
            if p < 0 or not 0 <= c.table[s, p // 32] < 16:
                want[at + i] = 0
        at += n
    assert np.array_equal(held, want)


def test_bounds_of_the_batch(holo):
    """max_rows leaves the rows past it; a sequence past max_len gives NaN; cu_rows past rows is cut."""
    print("case kv4 bounds", flush=True)
    rng = np.random.default_rng(6)
    hd, heads, n_kv, lens = 32, 4, 2, [50, 20]
    c = Cache(hd, 32, 1, n_kv, 4, 2, 2)
    pages(c, lens, rng)
    fill(c, rng, lens, 0)
    dev = OnDevice(holo, c)
    rows = [9, 4]
    q = rng.standard_normal((13, heads * hd)).astype(np.float32)
    want = want_attention(c, 0, q, rows, c.len, [0, 1], heads)
    got = attention(holo, dev, 0, q, rows, heads, max_rows=6)
    assert (got[6:9] == -9.0).all()
    keep = [0, 1, 2, 3, 4, 5, 9, 10, 11, 12]
    assert normwise(got[keep], want[keep]) <= TOL
    got = attention(holo, dev, 0, q, rows, heads, max_len=49)
    assert np.isnan(got[:9]).all() and normwise(got[9:], want[9:]) <= TOL
    got = attention(holo, dev, 0, q, rows, heads, max_len=0)
    assert np.isnan(got).all()
    # cu_rows: 0, 9, 500: the second entry has the 4 rows that are there
    b = Batch(holo, rows, None, None, 50)
    b.cu.upload(np.int32([0, 9, 500]))
    dq, do = up(holo, q), up(holo, np.full((14, heads * hd), -9.0, np.float32))
    assert holo.lib().holo_attention_kv4(dev.ref, 0, do.ptr, dq.ptr, heads * hd, heads * hd, heads, b.ref) == 0
    holo.lib().cuda_sync()
    got = do.download(np.float32).reshape(14, -1)
    assert (got[13] == -9.0).all() and normwise(got[:13], want) <= TOL


def test_what_lies_behind_a_row_does_not_reach_it(holo):
    """The cache past a sequence's end holds NaN scales; a NaN key or value is
    seen by the rows from its position on, and by those alone."""
    print("case kv4 poison", flush=True)
    rng = np.random.default_rng(7)
    hd, heads, n_kv, n = 64, 4, 2, 77
    for fill_byte in (0xFF, 0x7C):  # scales of NaN, of a large finite value
        c = Cache(hd, 32, 1, n_kv, 4, 1, 3, fill=fill_byte)
        pages(c, [n], rng)
        fill(c, rng, [n], 0)
        q = rng.standard_normal((40, heads * hd)).astype(np.float32)
        got = attention(holo, OnDevice(holo, c), 0, q, [40], heads)
        assert normwise(got, want_attention(c, 0, q, [40], c.len, [0], heads)) <= TOL
    k, v = rng.standard_normal((2, hd)).astype(np.float32)
    v[40] = np.nan
    c.put(0, 0, 1, 50, k, v)      # head 1, position 50: dims 32 .. 63 of the value
    bad = rng.standard_normal(hd).astype(np.float32)
    bad[3] = np.inf
    c.put(0, 0, 0, 70, bad, bad)  # head 0, position 70: key and value
    got = attention(holo, OnDevice(holo, c), 0, q, [40], heads)
    want = want_attention(c, 0, q, [40], c.len, [0], heads)
    got_, want_ = got.reshape(40, heads, hd), want.reshape(40, heads, hd)
    assert np.array_equal(np.isnan(got_), np.isnan(want_))
    assert np.isnan(want_[70 - 37:, :2]).all() and not np.isnan(want_[:70 - 37, :2]).any()
    assert np.isnan(want_[50 - 37:, 2:, 32:]).all() and not np.isnan(want_[:, 2:, :32]).any()
    ok = ~np.isnan(want)
    assert normwise(got[ok], want[ok]) <= TOL
    # q: a NaN or an infinity makes its own row and head NaN
    q[3, 5], q[4, hd + 1] = np.nan, np.inf
    got = attention(holo, OnDevice(holo, c), 0, q, [40], heads).reshape(40, heads, hd)
    assert np.isnan(got[3, 0]).all() and np.isnan(got[4, 1]).all()
    got[3, 0], got[4, 1] = want_[3, 0], want_[4, 1]
    ok = ~np.isnan(want_)
    assert normwise(got[ok], want_[ok]) <= TOL


def test_step_in_a_graph_follows_the_device_arrays(holo):
    """Append and attention captured once; replays after the lengths, the table,
    the rows and the entries changed, eager calls of other sizes between them;
    two graphs with partial sums of their own, replayed on two streams."""
    print("case kv4 graph", flush=True)
    rng = np.random.default_rng(9)
    lib = holo.lib()
    hd, heads, n_kv, n = 64, 4, 1, 900
    sides = []
    before = lib.holo_get_stream()
    streams = [lib.holo_stream_create(), lib.holo_stream_create()]
    try:
        for side in range(2):
            c = Cache(hd, 64, 1, n_kv, 40, 2, 16)
            pages(c, [n, 400], rng)
            fill(c, rng, [n, 400], 0)
            dev = OnDevice(holo, c)
            b = Batch(holo, [1, 1], [0, 1], None, 1000)
            bufs = [holo.DeviceBuffer(2 * heads * hd * 4) for _ in range(4)]
            dq, dk, dv, do = bufs
            lib.holo_set_stream(streams[side])
            assert lib.holo_graph_begin() == 0
            assert lib.holo_kv4_append(dev.ref, 0, dk.ptr, dv.ptr, n_kv * hd, n_kv * hd, b.ref) == 0
            assert lib.holo_attention_kv4(dev.ref, 0, do.ptr, dq.ptr, heads * hd, heads * hd, heads, b.ref) == 0
            graph = lib.holo_graph_end()
            assert graph
            holo.check("capture")
            sides.append((c, dev, b, bufs, graph))
        for step in range(3):
            wants = []
            for side, (c, dev, b, (dq, dk, dv, do), graph) in enumerate(sides):
                lib.holo_set_stream(streams[side])
                seqs = [0, 1] if step != 1 else [1, 0]
                c.len += 1
                dev.refresh()
                b.seqs.upload(np.int32(seqs))
                q = rng.standard_normal((2, heads * hd)).astype(np.float32)
                k, v = rng.standard_normal((2, 2, n_kv * hd)).astype(np.float32)
                dq.upload(q), dk.upload(k), dv.upload(v)
                for i, s in enumerate(seqs):
                    c.put(s, 0, 0, c.len[s] - 1, k[i], v[i])
                wants.append(want_attention(c, 0, q, [1, 1], c.len, seqs, heads))
            lib.cuda_sync()
            for side in range(2):  # both under way at once
                lib.holo_set_stream(streams[side])
                assert lib.holo_graph_launch(sides[side][4]) == 0
            lib.cuda_sync()
            holo.check("replay")
            for (c, dev, b, (dq, dk, dv, do), graph), want in zip(sides, wants):
                assert normwise(do.download(np.float32).reshape(2, -1), want) <= TOL
                assert np.array_equal(dev.bytes(), c.pool)
                q = rng.standard_normal((5, heads * hd)).astype(np.float32)  # eager, in between
                got = attention(holo, dev, 0, q, [4, 1], heads)
                assert normwise(got, want_attention(c, 0, q, [4, 1], c.len, [0, 1], heads)) <= TOL
    finally:
        for *_, graph in sides:
            lib.holo_graph_destroy(graph)
        lib.holo_set_stream(before)
        for s in streams:
            lib.holo_stream_destroy(s)


def test_copies_of_pages(holo):
    print("case kv4 copy", flush=True)
    rng = np.random.default_rng(10)
    for hd, layers, n_pages, n in ((32, 1, 700, 300), (96, 3, 9, 4)):
        c = Cache(hd, 32, layers, 1, n_pages, 1, 1)
        dev = OnDevice(holo, c)
        order = rng.permutation(n_pages).astype(np.int32)
        src, dst = order[:n].copy(), order[n:2 * n].copy()
        src[1] = src[0]  # a page may be copied twice
        assert holo.lib().holo_kv4_copy_pages(dev.ref, src.ctypes.data, dst.ctypes.data, n) == 0
        holo.lib().cuda_sync()
        holo.check("copy")
        c.pool[dst] = c.pool[src]
        assert np.array_equal(dev.bytes(), c.pool)


def test_pool_past_four_gigabytes(holo):
    """Pages whose bytes lie past 2^32, written, read, attended and copied from."""
    print("case kv4 large pool", flush=True)
    rng = np.random.default_rng(11)
    hd, heads, n_kv, n, layer = 128, 8, 8, 1500, 7
    c = Cache(hd, 1024, 1, n_kv, 1, 1, 2, fill=0)  # the arrays around a pool that only the device holds
    dev, lib = OnDevice(holo, c), holo.lib()
    dev.desc.n_layers, dev.desc.n_pages = 8, 500
    size = lib.holo_kv4_page_bytes(dev.ref)
    assert 470 * size > 1 << 32
    dev.pool = holo.DeviceBuffer(500 * size)
    dev.desc.pool = dev.pool.ptr
    c.table[0], c.len[0] = (499, 470), n
    dev.refresh()
    k, v = rng.standard_normal((2, n, n_kv * hd)).astype(np.float32)
    q = rng.standard_normal((3, heads * hd)).astype(np.float32)
    dk, dv, dq, do = up(holo, k), up(holo, v), up(holo, q), holo.DeviceBuffer(q.nbytes)
    b = Batch(holo, [n], None, None, n)
    assert lib.holo_kv4_append(dev.ref, layer, dk.ptr, dv.ptr, n_kv * hd, n_kv * hd, b.ref) == 0
    hk, hv = values(*quantise(k)), values(*quantise(v))
    last = Batch(holo, [3], None, None, n)
    for pages_ in ((499, 470), (3, 498)):
        c.table[0] = pages_
        dev.refresh()
        if pages_[0] == 3:
            src, dst = np.int32([470, 499]), np.int32([498, 3])
            assert lib.holo_kv4_copy_pages(dev.ref, src.ctypes.data, dst.ctypes.data, 2) == 0
        dk.upload(np.zeros_like(k))
        assert lib.holo_kv4_read(dev.ref, layer, dk.ptr, dv.ptr, n_kv * hd, n_kv * hd, b.ref) == 0
        assert lib.holo_attention_kv4(dev.ref, layer, do.ptr, dq.ptr, heads * hd, heads * hd, heads, last.ref) == 0
        lib.cuda_sync()
        holo.check("large pool")
        assert np.array_equal(dk.download(np.float32).reshape(n, -1), hk)
        assert np.array_equal(dv.download(np.float32).reshape(n, -1), hv)
        got, want = do.download(np.float32).reshape(3, heads, hd), np.zeros((3, heads, hd))
        for i in range(3):
            for h in range(heads):
                x = slice(h * hd, (h + 1) * hd)
                s = hk[:n - 2 + i, x] @ q[i, x].astype(np.float64) / np.sqrt(hd)
                p = np.exp(s - s.max())
                want[i, h] = p / p.sum() @ hv[:n - 2 + i, x]
        assert normwise(got, want) <= TOL


def test_the_last_positions_there_are(holo):
    """A sequence of 0x7FFFF000 positions, of which the last pages are there."""
    print("case kv4 last positions", flush=True)
    rng = np.random.default_rng(12)
    hd, rows, n = 32, 70, 0x7FFFF000
    c = Cache(hd, 1024, 1, 1, 2, 1, n // 1024, fill=0x30)  # scales of 0x3030: 7 significant bits
    c.table[0, -1], c.len[0] = 1, n
    dev, lib = OnDevice(holo, c), holo.lib()
    k, v, q = rng.standard_normal((3, rows, hd)).astype(np.float32)
    dk, dv, dq, do = up(holo, k), up(holo, v), up(holo, q), holo.DeviceBuffer(q.nbytes)
    b = Batch(holo, [rows], None, None, n)
    b.desc.max_rows = b.desc.rows = 0x7FFFF000  # bounds: the entry has 70
    assert lib.holo_kv4_append(dev.ref, 0, dk.ptr, dv.ptr, hd, hd, b.ref) == 0
    assert lib.holo_kv4_read(dev.ref, 0, dk.ptr, dv.ptr, hd, hd, b.ref) == 0
    b.desc.max_rows = 1  # and one of them here
    assert lib.holo_attention_kv4(dev.ref, 0, do.ptr, dq.ptr, hd, hd, 1, b.ref) == 0
    lib.cuda_sync()
    holo.check("last positions")
    assert np.array_equal(dk.download(np.float32).reshape(rows, hd), values(*quantise(k)))
    assert np.array_equal(dv.download(np.float32).reshape(rows, hd), values(*quantise(v)))
    held = [np.stack([c.get(0, 0, 0, p, w) for p in range(n - 1024, n - rows)]) for w in (0, 1)]
    hk, hv = (np.concatenate([x, values(*quantise(y))[:1]]) for x, y in zip(held, (k, v)))
    s = hk @ q[0].astype(np.float64) / np.sqrt(hd)
    p = np.exp(s - s.max())
    assert normwise(do.download(np.float32)[:hd], p / p.sum() @ hv) <= TOL


@pytest.mark.parametrize("scale", [1e12, 1e20, 1e30, -1e25])
def test_scores_far_past_the_exponential(holo, scale):
    """Scores so large that one position has all of the probability: its value comes back."""
    print(f"case kv4 scale {scale}", flush=True)
    rng = np.random.default_rng(13)
    hd, heads, n_kv, n = 64, 4, 2, 800
    c = Cache(hd, 64, 1, n_kv, 13, 1, 13)
    pages(c, [n], rng)
    fill(c, rng, [n], 0)
    q = (scale * rng.standard_normal((1, heads * hd))).astype(np.float32)
    got = attention(holo, OnDevice(holo, c), 0, q, [1], heads).reshape(heads, hd)
    for h in range(heads):
        k, v, _ = c.held(0, 0, h // 2, n)
        s = k @ q[0, h * hd:(h + 1) * hd].astype(np.float64)
        first, second = np.sort(s)[::-1][:2]
        # a score is within 9.5e-7 of the sum of magnitudes, about 4e-6 of the largest
        assert first - second > 1e-4 * first
        # p is 2^7.5 in two halves, and its sum the same number
        assert np.abs(got[h] - v[s.argmax()]).max() <= 2.0 ** -21 * np.abs(v[s.argmax()]).max()


@pytest.mark.parametrize("lens", [[1, 40, 255, 256, 257, 600], [3000, 2, 800]], ids=str)
def test_ranges_follow_the_lengths(holo, lens):
    """A bound on the lengths far above them: the sequences' own tiles are dealt out, one to many ranges."""
    print(f"case kv4 ranges {lens}", flush=True)
    rng = np.random.default_rng(14)
    hd, heads, n_kv = 32, 4, 1
    c = Cache(hd, 128, 1, n_kv, sum(-(-n // 128) for n in lens), len(lens), 24)
    pages(c, lens, rng)
    fill(c, rng, lens, 0)
    dev = OnDevice(holo, c)
    rows = [min(n, 5) for n in lens]
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    want = want_attention(c, 0, q, rows, c.len, list(range(len(lens))), heads)
    for bound in (c.len.max(), 3200, 40000, 1 << 20, 0x7FFFF000):
        if bound >= c.len.max():
            assert normwise(attention(holo, dev, 0, q, rows, heads, max_len=bound), want) <= TOL


def test_pages_on_the_device_follow_the_bookkeeping(holo):
    """More updates and copies than one launch takes: a long sequence, its fork, the pages compacted."""
    print("case kv4 bookkeeping", flush=True)
    rng = np.random.default_rng(15)
    lib = holo.lib()
    c = Cache(32, 32, 1, 1, 1500, 4, 700)
    dev = OnDevice(holo, c)
    p = lib.holo_kv4_pages_create(dev.ref)
    assert p
    ints = lambda *x: np.int32(x)

    def call(name, *arrays):
        assert getattr(lib, name)(p, *[a.ctypes.data for a in arrays], len(arrays[0])) == 0

    def device():
        lib.cuda_sync()
        holo.check("bookkeeping")
        return dev.table.download(np.int32).reshape(4, 700), dev.len.download(np.int32)

    def listed():
        table, lens = np.full((4, 700), -1, np.int32), np.zeros(4, np.int32)
        for s in range(4):
            n = lib.holo_kv4_pages_list(p, s, table[s].ctypes.data, 700)
            lens[s] = lib.holo_kv4_pages_len(p, s)
            assert n == -(-lens[s] // 32)
        return table, lens

    def same():
        (t, n), (t2, n2) = device(), listed()
        assert np.array_equal(t, t2) and np.array_equal(n, n2)
        return t, n

    try:
        same()
        call("holo_kv4_pages_reserve", ints(2, 0), ints(620 * 32, 650 * 32 - 5))
        same()
        call("holo_kv4_pages_fork", ints(0), ints(3))
        t, _ = same()
        before = dev.bytes()
        assert np.array_equal(t[0], t[3])
        call("holo_kv4_pages_reserve", ints(3), ints(40))  # a shared last page and new ones
        t, n = same()
        assert n[3] == 650 * 32 + 35 and np.array_equal(t[0, :649], t[3, :649]) and t[0, 649] != t[3, 649]
        assert np.array_equal(dev.bytes()[t[3, 649]], before[t[0, 649]])
        call("holo_kv4_pages_free", ints(2))
        held = dev.bytes()[same()[0][3, :650]]
        assert lib.holo_kv4_pages_compact(p) == 0  # more than 256 pages move
        t, n = same()
        used = set(t[t >= 0].tolist())
        assert used == set(range(len(used))) and np.array_equal(dev.bytes()[t[3, :650]], held)
        assert lib.holo_kv4_pages_available(p) == 1500 - len(used)
    finally:
        lib.holo_kv4_pages_destroy(p)
