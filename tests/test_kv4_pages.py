"""The 4-bit cache without a GPU: what its calls refuse, and the bookkeeping of
its pages (reserve, fork, free, compact) against a plain model."""
import ctypes as C
import random

import numpy as np
import pytest

import holo_mi355x as h


def ints(*x):
    return (C.c_int * max(len(x), 1))(*x)


def layout(**kw):
    d = dict(n_pages=8, page_len=64, n_layers=2, n_kv_heads=2, head_dim=64, n_seqs=4, max_pages=4)
    d.update(kw)
    return h.KV4(**d)


def rejected(rc):
    return rc == h.EINVAL and h.lib().holo_last_error() == h.EINVAL


def test_page_bytes():
    lib = h.lib()
    for hd, page, layers, kv in ((128, 64, 32, 8), (32, 32, 1, 1), (96, 1024, 3, 5)):
        c = layout(head_dim=hd, page_len=page, n_layers=layers, n_kv_heads=kv)
        # 4.5 bits a value, keys and values
        assert lib.holo_kv4_page_bytes(C.byref(c)) == layers * kv * page * 2 * hd * 9 // 16
    for bad in (dict(head_dim=80), dict(head_dim=0), dict(head_dim=256), dict(page_len=48), dict(page_len=16),
                dict(page_len=2048), dict(n_layers=0), dict(n_kv_heads=0), dict(n_pages=0), dict(n_kv_heads=65536)):
        assert lib.holo_kv4_page_bytes(C.byref(layout(**bad))) == 0
    assert lib.holo_kv4_page_bytes(None) == 0


def test_sizes_past_the_limits_are_refused():
    lib = h.lib()
    assert lib.holo_kv4_page_bytes(C.byref(layout(n_layers=65535))) > 0
    assert lib.holo_kv4_page_bytes(C.byref(layout(n_layers=65536))) == 0
    c = layout(**POINTERS)
    b = h.Batch(rows=0x7FFFF001, n_seqs=2, max_rows=1, max_len=64, cu_rows=16384)
    assert rejected(lib.holo_kv4_append(C.byref(c), 0, 4096, 8192, 128, 128, C.byref(b)))
    assert rejected(lib.holo_attention_kv4(C.byref(c), 0, 4096, 8192, 256, 256, 4, C.byref(b)))
    assert rejected(lib.holo_attention_packed(4096, 8192, 4096, 8192, 256, 256, 128, 128, 64, 4, 2, C.byref(b)))


POINTERS = dict(pool=4096, table=8192, len=12288)


@pytest.mark.parametrize("bad", [
    dict(head_dim=48), dict(page_len=33), dict(pool=None), dict(pool=4104), dict(table=None), dict(len=None),
    dict(n_seqs=0), dict(max_pages=0), dict(max_pages=1 << 30), dict(layer=2), dict(layer=-1), dict(rows=-1),
    dict(entries=-1), dict(entries=65536), dict(cu=None), dict(max_rows=0), dict(x=None), dict(x=4100), dict(ld=127),
    dict(ld=130), dict(ld=96), dict(heads=3), dict(heads=0), dict(max_len=-1), dict(null="cache"), dict(null="batch"),
    dict(rows=1 << 22, max_rows=1 << 22)], ids=str)
def test_calls_refuse(bad):
    """Every refusal comes before any device work (there is no device here)."""
    lib = h.lib()
    bad = dict(bad)
    c = layout(**{**POINTERS, **{k: bad[k] for k in bad if k in dict(h.KV4._fields_)}})
    b = h.Batch(rows=bad.get("rows", 4), n_seqs=bad.get("entries", 2), max_rows=bad.get("max_rows", 2),
                max_len=bad.get("max_len", 64), cu_rows=bad.get("cu", 16384))
    x, ld, layer = bad.get("x", 4096), bad.get("ld", 128), bad.get("layer", 0)
    cp, bp = C.byref(c), C.byref(b)
    if "null" in bad:
        cp, bp = (None, bp) if bad["null"] == "cache" else (cp, None)
    only_attention = {"heads", "max_len"} & set(bad) or bad.get("rows") == 1 << 22
    if not only_attention:
        assert rejected(lib.holo_kv4_append(cp, layer, x, 8192, ld, 128, bp))
        assert rejected(lib.holo_kv4_append(cp, layer, 8192, x, 128, ld, bp)) or not {"x", "ld"} & set(bad)
        assert rejected(lib.holo_kv4_read(cp, layer, x, 8192, ld, 128, bp))
    assert rejected(lib.holo_attention_kv4(cp, layer, x, 8192, ld, 128, bad.get("heads", 2), bp))


@pytest.mark.parametrize("bad", [
    dict(head_dim=80), dict(head_dim=256), dict(heads=3), dict(kv=0), dict(kv=65536), dict(rows=-1), dict(cu=None),
    dict(max_rows=0), dict(entries=65536), dict(out=None), dict(q=4100), dict(k=None), dict(v=8), dict(ldo=252),
    dict(ldq=258), dict(ldk=124), dict(ldv=130), dict(null=True)], ids=str)
def test_packed_attention_refuses(bad):
    g = bad.get
    b = h.Batch(rows=g("rows", 4), n_seqs=g("entries", 2), max_rows=g("max_rows", 2), cu_rows=g("cu", 16384))
    assert rejected(h.lib().holo_attention_packed(
        g("out", 4096), g("q", 4096), g("k", 4096), g("v", 4096), g("ldo", 256), g("ldq", 256), g("ldk", 128),
        g("ldv", 128), g("head_dim", 64), g("heads", 4), g("kv", 2), None if g("null") else C.byref(b)))


def test_nothing_to_do_is_no_error():
    lib = h.lib()
    c = layout(**POINTERS)
    for b in (h.Batch(rows=0, n_seqs=3, max_rows=1), h.Batch(rows=3, n_seqs=0)):
        assert lib.holo_kv4_append(C.byref(c), 0, None, None, 0, 0, C.byref(b)) == 0
        assert lib.holo_kv4_read(C.byref(c), 0, None, None, 0, 0, C.byref(b)) == 0
        assert lib.holo_attention_kv4(C.byref(c), 0, None, None, 0, 0, 2, C.byref(b)) == 0
        assert lib.holo_attention_packed(None, None, None, None, 0, 0, 0, 0, 64, 2, 2, C.byref(b)) == 0
    assert lib.holo_kv4_copy_pages(C.byref(c), None, None, 0) == 0
    assert lib.holo_last_error() == 0


@pytest.mark.parametrize("src,dst", [([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0]), ([8], [1]), ([1], [8]),
                                     ([-1], [1]), ([1], [-1])])
def test_copy_refuses(src, dst):
    c = layout(**POINTERS)
    assert rejected(h.lib().holo_kv4_copy_pages(C.byref(c), ints(*src), ints(*dst), len(src)))


def test_copy_refuses_arguments():
    lib = h.lib()
    assert rejected(lib.holo_kv4_copy_pages(None, ints(0), ints(1), 1))
    assert rejected(lib.holo_kv4_copy_pages(C.byref(layout()), ints(0), ints(1), 1))  # no pool
    assert rejected(lib.holo_kv4_copy_pages(C.byref(layout(**POINTERS)), None, ints(1), 1))
    assert rejected(lib.holo_kv4_copy_pages(C.byref(layout(**POINTERS)), ints(1), ints(2), -1))


# ---- the bookkeeping -----------------------------------------------------------------


class Pages:
    def __init__(self, **kw):
        self.c = layout(**kw)
        self.p = h.lib().holo_kv4_pages_create(C.byref(self.c))
        assert self.p

    def __getattr__(self, name):
        f = getattr(h.lib(), "holo_kv4_pages_" + name)
        return lambda *a: f(self.p, *a)

    def reserve_(self, seqs, rows):
        return self.reserve(ints(*seqs), ints(*rows), len(seqs))

    def fork_(self, src, dst):
        return self.fork(ints(*src), ints(*dst), len(src))

    def free_(self, *seqs):
        return self.free(ints(*seqs), len(seqs))

    def pages(self, seq):
        n = self.list(seq, None, 0)
        out = ints(*[-7] * n)
        assert self.list(seq, out, n) == n
        return list(out)[:n]


@pytest.mark.parametrize("bad", [dict(page_len=0), dict(n_seqs=0), dict(max_pages=0), dict(pool=4096),
                                 dict(table=4096, len=4096), dict(max_pages=1 << 29)], ids=str)
def test_create_refuses(bad):
    assert h.lib().holo_kv4_pages_create(C.byref(layout(**bad))) is None
    assert h.lib().holo_last_error() == h.EINVAL


def test_null_handle():
    lib = h.lib()
    assert rejected(lib.holo_kv4_pages_reserve(None, ints(0), ints(1), 1))
    assert rejected(lib.holo_kv4_pages_fork(None, ints(0), ints(1), 1))
    assert rejected(lib.holo_kv4_pages_free(None, ints(0), 1))
    assert rejected(lib.holo_kv4_pages_compact(None))
    assert lib.holo_kv4_pages_available(None) == 0
    assert lib.holo_kv4_pages_len(None, 0) == -1 and lib.holo_kv4_pages_list(None, 0, None, 0) == -1
    lib.holo_kv4_pages_destroy(None)


def test_reserve_takes_the_lowest_free_pages_and_all_or_nothing():
    p = Pages()
    assert p.reserve_([1, 0], [65, 1]) == 0
    assert p.pages(1) == [0, 1] and p.pages(0) == [2] and p.available() == 5
    assert p.reserve_([0], [63]) == 0 and p.pages(0) == [2]  # its page is full now
    assert p.reserve_([0], [1]) == 0 and p.pages(0) == [2, 3]
    # 4 pages are free: 3 and 2 are not there, and nothing changes
    assert p.reserve_([2, 3], [129, 65]) == h.ENOPAGES and h.lib().holo_last_error() == h.ENOPAGES
    assert p.len(2) == p.len(3) == 0 and p.available() == 4
    assert rejected(p.reserve_([2], [257]))  # past its row of the table
    assert rejected(p.reserve_([2, 2], [1, 1])) and rejected(p.reserve_([4], [1])) and rejected(p.reserve_([-1], [1]))
    assert rejected(p.reserve_([2], [-1])) and rejected(p.reserve(None, None, 1))
    assert p.reserve_([2], [0]) == 0 and p.len(2) == 0 and p.available() == 4
    assert p.free_(1) == 0 and p.reserve_([3], [1]) == 0 and p.pages(3) == [0]
    p.destroy()


def test_fork_shares_and_reserve_copies():
    p = Pages()
    assert p.reserve_([0], [100]) == 0 and p.pages(0) == [0, 1]
    assert p.fork_([0, 1], [1, 2]) == 0  # 2 from 1, which is forked in the same call
    assert p.pages(1) == p.pages(2) == [0, 1] and p.len(2) == 100 and p.available() == 6
    # three sequences share the last page: two take copies, the last keeps it
    assert p.reserve_([2, 0, 1], [1, 1, 1]) == 0
    assert p.pages(2) == [0, 2] and p.pages(0) == [0, 3] and p.pages(1) == [0, 1] and p.available() == 4
    assert p.free_(0, 0, 2) == 0 and p.len(0) == 0 and p.available() == 6  # page 0 is still 1's
    assert p.free_(1) == 0 and p.available() == 8
    # a full last page is shared, not copied
    assert p.reserve_([0], [64]) == 0 and p.fork_([0], [3]) == 0 and p.reserve_([3], [1]) == 0
    assert p.pages(3) == [0, 1] and p.pages(0) == [0]
    for src, dst in (([0], [0]), ([0], [3]), ([0, 0], [1, 1]), ([4], [1]), ([0], [4]), ([0], [-1])):
        assert rejected(p.fork_(src, dst))
    assert p.len(1) == 0
    p.destroy()


def test_compact_moves_the_last_pages_into_the_holes():
    p = Pages()
    assert p.reserve_([0, 1, 2], [128, 64, 100]) == 0  # pages 0 1 | 2 | 3 4
    assert p.fork_([2], [3]) == 0 and p.free_(0) == 0
    assert p.compact() == 0
    assert p.pages(1) == [2] and p.pages(2) == p.pages(3) == [0, 1] and p.available() == 5
    assert p.reserve_([0], [1]) == 0 and p.pages(0) == [3]
    assert p.compact() == 0 and p.pages(0) == [3]
    p.destroy()


@pytest.mark.parametrize("seed", range(6))
def test_random_calls_against_a_plain_model(seed):
    """Positions, sharing and the pages in use after random calls."""
    rng = random.Random(seed)
    n_seqs, page, n_pages, max_pages = 6, 32, 40, 12
    p = Pages(n_seqs=n_seqs, page_len=page, n_pages=n_pages, max_pages=max_pages)
    lens, own = [0] * n_seqs, [[] for _ in range(n_seqs)]
    for step in range(200):
        do = rng.choice(("reserve", "reserve", "fork", "free", "compact"))
        used = sorted({x for o in own for x in o})
        if do == "reserve":
            seqs = rng.sample(range(n_seqs), rng.randint(1, n_seqs))
            rows = [rng.choice((0, 1, 1, rng.randint(1, 90))) for _ in seqs]
            free = [x for x in range(n_pages) if x not in used]
            new, bad = [list(o) for o in own], any(lens[s] + r > max_pages * page for s, r in zip(seqs, rows))
            for s, r in zip(seqs, rows):
                if not r:
                    continue
                need = -(-(lens[s] + r) // page) - len(new[s])
                if lens[s] % page and sum(o.count(new[s][-1]) for o in new) > 1:
                    new[s][-1] = free.pop(0) if free else -1
                for _ in range(need):
                    new[s].append(free.pop(0) if free else -1)
            want = h.EINVAL if bad else h.ENOPAGES if any(-1 in o for o in new) else 0
            assert p.reserve_(seqs, rows) == want
            if want == 0:
                own = new
                for s, r in zip(seqs, rows):
                    lens[s] += r
        elif do == "fork":
            a, b = rng.sample(range(n_seqs), 2)
            assert p.fork_([a], [b]) == (h.EINVAL if lens[b] else 0)
            if not lens[b]:
                own[b], lens[b] = list(own[a]), lens[a]
        elif do == "free":
            s = rng.randrange(n_seqs)
            assert p.free_(s) == 0
            own[s], lens[s] = [], 0
        else:
            assert p.compact() == 0
            front = len(used)
            holes = [x for x in range(front) if x not in used]
            to = dict(zip([x for x in used if x >= front], holes))
            own = [[to.get(x, x) for x in o] for o in own]
        h.lib().holo_last_error()
        assert [p.len(s) for s in range(n_seqs)] == lens
        assert [p.pages(s) for s in range(n_seqs)] == own
        assert p.available() == n_pages - len({x for o in own for x in o})
    p.destroy()


def test_the_model_of_the_layout_is_consistent():
    """Every byte of a tile belongs to one nibble pair or scale of the numpy model."""
    from kv4_model import Cache
    for hd in (32, 64, 96, 128):
        c = Cache(hd, 32, 1, 1, 1, 1, 1, fill=0)
        seen = np.zeros(36 * hd, int)
        for which in (0, 1):
            for pos in range(32):
                at, sh, sc = c.where(pos, which)
                np.add.at(seen, at, 1)
                np.add.at(seen, np.concatenate((sc, sc + 1)), 2)
        assert (seen == 2).all()


def test_the_model_holds_what_is_put():
    from kv4_model import Cache, quantise, values
    rng = np.random.default_rng(1)
    for hd in (32, 96, 128):
        c = Cache(hd, 32, 1, 1, 2, 1, 2)
        c.table[0] = 1, 0
        x = rng.standard_normal((40, 2, hd)).astype(np.float32)
        for p in range(40):
            c.put(0, 0, 0, p, *x[p])
        k, v, there = c.held(0, 0, 0, 40)
        assert there.all() and np.array_equal(k, values(*quantise(x[:, 0]))) and np.array_equal(v, values(*quantise(x[:, 1])))
        # the far sign's largest value is held as 7 d, d within 2^-9 of an eighth of it
        step = np.abs(x.reshape(40, 2, -1, 32)).max(-1, keepdims=True) / 8 * (1 + 7 * 2.0 ** -9)
        assert (np.abs(np.stack((k, v), 1).reshape(40, 2, -1, 32) - x.reshape(40, 2, -1, 32)) <= step).all()
