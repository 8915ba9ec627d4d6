"""Drafted tokens and rotary positions without a GPU: what the calls refuse, the
frequencies, positions given back, and the verification's law in the model that
the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import draft_model as dm
import holo_mi355x as h
from test_kv4_pages import POINTERS, ints, layout, rejected


def batch(**kw):
    d = dict(rows=8, n_seqs=2, max_rows=4, max_len=64, cu_rows=16384)
    d.update(kw)
    return h.Batch(**d)


def rope(**kw):
    d = dict(freq=4096, dims=64, interleaved=0, scale=1.0)
    d.update(kw)
    return h.Rope(**d)


def append_rope(c=None, r=None, b=None, q=4096, k=8192, v=12288, qo=4096, ko=None, ld=256, ldk=128, ldv=128, ldqo=256,
                ldko=0, heads=4, depth=None, layer=0):
    c, r, b = (C.byref(x) if x is not None else None for x in (c, r, b))
    return h.lib().holo_kv4_append_rope(c, layer, r, q, k, v, ld, ldk, ldv, qo, ko, ldqo, ldko, heads, depth, b)


@pytest.mark.parametrize("bad", [
    dict(cache=dict(head_dim=48)), dict(cache=dict(pool=None)), dict(layer=2), dict(c=None), dict(r=None), dict(b=None),
    dict(rope=dict(freq=None)), dict(rope=dict(freq=4100)), dict(rope=dict(dims=0)), dict(rope=dict(dims=63)),
    dict(rope=dict(dims=66)), dict(rope=dict(dims=-2)), dict(rope=dict(scale=np.nan)), dict(rope=dict(scale=np.inf)),
    dict(batch=dict(rows=-1)), dict(batch=dict(cu_rows=None)), dict(batch=dict(n_seqs=65536)),
    dict(batch=dict(max_rows=0)), dict(k=None), dict(v=None), dict(k=8196), dict(v=8196), dict(ldk=96), dict(ldk=130),
    dict(ldv=124), dict(q=None), dict(qo=None), dict(q=4100), dict(qo=4100), dict(ld=252), dict(ldqo=257), dict(heads=3),
    dict(heads=-2), dict(ko=8192, ldko=96), dict(ko=8196, ldko=128), dict(depth=4098),
    dict(heads=1 << 20, ld=1 << 28, ldqo=1 << 28)], ids=str)
def test_append_with_rotation_refuses(bad):
    bad = dict(bad)
    kw = dict(c=layout(**{**POINTERS, **bad.pop("cache", {})}), r=rope(**bad.pop("rope", {})),
              b=batch(**bad.pop("batch", {})))
    assert rejected(append_rope(**{**kw, **bad}))


def test_empty_batches_do_nothing():
    c, r = layout(**POINTERS), rope()
    lib = h.lib()
    for kw in (dict(rows=0), dict(n_seqs=0)):
        b = batch(**kw)
        assert append_rope(c, r, b) == 0
        assert lib.holo_draft_plan(4096, 4096, 4096, 1, C.byref(b)) == 0
        assert lib.holo_attention_kv4_draft(C.byref(c), 0, 4096, 4096, 256, 256, 4, 4096, 1, C.byref(b)) == 0
        assert lib.holo_draft_verify(4096, 4096, 4096, 4096, 4096, 99, 99, 99, 4096, 4096, 4096, 1, C.byref(b)) == 0
        assert lib.holo_kv4_keep(C.byref(c), 4096, 4096, C.byref(b)) == 0
    assert lib.holo_softmax_rows(None, None, 0, 5, 5, 5, 1.0) == 0
    assert lib.holo_softmax_rows(None, None, 5, 0, 5, 5, 1.0) == 0
    assert lib.holo_last_error() == 0


@pytest.mark.parametrize("bad", [
    dict(cache=dict(head_dim=48)), dict(cache=dict(table=None)), dict(layer=-1), dict(heads=3), dict(heads=0),
    dict(q=None), dict(q=4100), dict(o=None), dict(ld=252), dict(ldo=257), dict(mask=None), dict(mask=4098),
    dict(words=0), dict(words=33), dict(words=-1), dict(batch=dict(max_rows=33, rows=40)),
    dict(batch=dict(max_rows=2000, rows=2000), words=32), dict(batch=dict(max_len=-1)),
    dict(batch=dict(max_len=0x7FFFF001)), dict(batch=dict(cu_rows=None))], ids=str)
def test_attention_refuses(bad):
    bad = dict(bad)
    c, b = layout(**{**POINTERS, **bad.pop("cache", {})}), batch(**bad.pop("batch", {}))
    a = dict(layer=0, o=4096, q=8192, ldo=256, ld=256, heads=4, mask=16384, words=1)
    a.update(bad)
    assert rejected(h.lib().holo_attention_kv4_draft(C.byref(c), a["layer"], a["o"], a["q"], a["ldo"], a["ld"],
                                                     a["heads"], a["mask"], a["words"], C.byref(b)))


def test_attention_refuses_more_columns_than_a_launch():
    c = layout(**POINTERS, n_kv_heads=65535)
    b = batch(rows=64, max_rows=32, max_len=100)
    n = 65535 * 64
    assert rejected(h.lib().holo_attention_kv4_draft(C.byref(c), 0, 4096, 8192, n, n, 65535, 4096, 1, C.byref(b)))


@pytest.mark.parametrize("bad", [
    dict(path=None), dict(n_path=None), dict(next=None), dict(target=None), dict(draft=None), dict(tokens=None),
    dict(parent=None), dict(u=None), dict(target=4098), dict(u=4097), dict(ldt=99), dict(ldd=99), dict(vocab=0),
    dict(vocab=-5), dict(vocab=(1 << 24) + 1, ldt=1 << 25, ldd=1 << 25), dict(mode=3), dict(mode=-1),
    dict(batch=dict(rows=2000, max_rows=1025)), dict(batch=dict(rows=-1)), dict(batch=dict(cu_rows=None))], ids=str)
def test_verification_refuses(bad):
    bad = dict(bad)
    b = batch(**bad.pop("batch", {}))
    a = dict(path=4096, n_path=4096, next=4096, target=4096, draft=4096, ldt=100, ldd=100, vocab=100, tokens=4096,
             parent=4096, u=4096, mode=1)
    a.update(bad)
    assert rejected(h.lib().holo_draft_verify(*a.values(), C.byref(b)))


def test_other_calls_refuse():
    lib, c = h.lib(), layout(**POINTERS)
    for args in ((None, 4096, 4096, 1), (4096, None, 4096, 1), (4096, 4096, None, 1), (4098, 4096, 4096, 1),
                 (4096, 4096, 4096, 0), (4096, 4096, 4096, 33)):
        assert rejected(lib.holo_draft_plan(*args, C.byref(batch())))
    assert rejected(lib.holo_draft_plan(4096, 4096, 4096, 1, C.byref(batch(rows=40, max_rows=33))))
    assert rejected(lib.holo_draft_plan(4096, 4096, 4096, 1, None))
    for args in ((None, 4096), (4096, None), (4098, 4096), (4096, 4097)):
        assert rejected(lib.holo_kv4_keep(C.byref(c), *args, C.byref(batch())))
    assert rejected(lib.holo_kv4_keep(C.byref(layout()), 4096, 4096, C.byref(batch())))
    assert rejected(lib.holo_kv4_keep(C.byref(c), 4096, 4096, C.byref(batch(rows=-1))))
    for dst, x, rows, n, ldd, ldx, scale in (
            (None, 4096, 2, 5, 5, 5, 1.0), (4096, None, 2, 5, 5, 5, 1.0), (4096, 4096, -1, 5, 5, 5, 1.0),
            (4096, 4096, 2, -1, 5, 5, 1.0), (4096, 4096, 2, 5, 4, 5, 1.0), (4096, 4096, 2, 5, 5, 4, 1.0),
            (4096, 4096, 2, 5, 5, 5, 0.0), (4096, 4096, 2, 5, 5, 5, -1.0), (4096, 4096, 2, 5, 5, 5, np.nan),
            (4096, 4096, 2, 5, 5, 5, np.inf)):
        assert rejected(lib.holo_softmax_rows(dst, x, rows, n, ldd, ldx, scale))


# ---- frequencies -----------------------------------------------------------------------------

def freqs(kind, dims=64, base=10000.0, factor=8.0, low=1.0, high=4.0, trained=8192, divisors=None):
    out, scale = np.full(dims // 2 + 1, -1.0), C.c_float(-1)
    d = None if divisors is None else np.ascontiguousarray(divisors, np.float32)
    s = h.RopeScaling(kind=kind, dims=dims, base=base, factor=factor, low=low, high=high, trained=trained,
                      divisors=None if d is None else d.ctypes.data)
    rc = h.lib().holo_rope_freqs(out.ctypes.data, C.byref(scale), C.byref(s))
    assert out[-1] == -1
    return rc, out[:-1], scale.value


@pytest.mark.parametrize("dims,base", [(64, 10000.0), (128, 500000.0), (2, 10000.0), (96, 1e6)])
def test_frequencies(dims, base):
    i = np.arange(dims // 2)
    plain = base ** (-2.0 * i / dims)
    close = dict(rtol=1e-14, atol=0)  # a few roundings of 2^-53 = 1.1e-16, pow's among them, some 15 of them relative

    def check(kind, want, scale=1.0, **kw):
        rc, got, s = freqs(kind, dims, base, **kw)
        assert rc == 0 and s == np.float32(scale)
        np.testing.assert_allclose(got, want, **close)

    check(h.ROPE_PLAIN, plain, factor=np.nan)  # not read
    check(h.ROPE_LINEAR, plain / 8)
    d = np.linspace(1, 3, dims // 2).astype(np.float32)
    check(h.ROPE_PLAIN, plain / d, divisors=d)
    check(h.ROPE_LINEAR, plain / d / 8, divisors=d)
    if dims > 2:
        check(h.ROPE_BASE, (base * 8 ** (dims / (dims - 2))) ** (-2.0 * i / dims))
    # by how often a pair turns over the trained positions, pair by pair
    want = []
    for w in plain:
        turns = 8192 * w / (2 * np.pi)
        if turns > 4:
            want.append(w)
        elif turns < 1:
            want.append(w / 8)
        else:
            t = (turns - 1) / 3
            want.append(t * w + (1 - t) * w / 8)
    check(h.ROPE_BANDS, want)
    # along the pairs' numbers: the pair whose wavelength is trained / turns
    first, last = (dims * np.log(8192 / (2 * np.pi * t)) / (2 * np.log(base)) for t in (32.0, 1.0))
    first, last = max(np.floor(first), 0), min(np.ceil(last), dims - 1)
    ramp = np.clip((i - first) / max(last - first, 0.001), 0, 1)
    check(h.ROPE_RAMP, plain * (1 - ramp) + plain / 8 * ramp, 0.1 * np.log(8) + 1, high=32.0)


def test_frequencies_refuse():
    for kw in (dict(kind=-1), dict(kind=5), dict(kind=0, dims=63), dict(kind=0, dims=0), dict(kind=0, dims=130),
               dict(kind=0, base=1.0), dict(kind=0, base=np.inf), dict(kind=0, base=np.nan), dict(kind=1, factor=0.5),
               dict(kind=1, factor=np.nan), dict(kind=1, factor=np.inf), dict(kind=2, dims=2), dict(kind=3, low=0.0),
               dict(kind=3, low=4.0), dict(kind=3, high=np.inf), dict(kind=4, trained=0),
               dict(kind=0, divisors=np.zeros(32)), dict(kind=0, divisors=np.full(32, np.nan))):
        assert rejected(freqs(**kw)[0])
    s = h.RopeScaling(kind=0, dims=4, base=10.0)
    out = np.zeros(2)
    assert rejected(h.lib().holo_rope_freqs(None, None, C.byref(s)))
    assert rejected(h.lib().holo_rope_freqs(out.ctypes.data, None, None))
    assert h.lib().holo_rope_freqs(out.ctypes.data, None, C.byref(s)) == 0 and out[0] == 1


# ---- positions given back ------------------------------------------------------------------------

def test_trim():
    lib = h.lib()
    p = lib.holo_kv4_pages_create(C.byref(layout(n_pages=8, page_len=32, max_pages=4)))
    try:
        def pages(s):
            a = ints(*[-1] * 4)
            n = lib.holo_kv4_pages_list(p, s, a, 4)
            return list(a)[:n]

        def trim(seqs, rows):
            return lib.holo_kv4_pages_trim(p, ints(*seqs), ints(*rows), len(seqs))

        assert lib.holo_kv4_pages_reserve(p, ints(0, 1), ints(70, 32), 2) == 0
        assert pages(0) == [0, 1, 2] and pages(1) == [3]
        assert trim([0], [5]) == 0 and lib.holo_kv4_pages_len(p, 0) == 65 and pages(0) == [0, 1, 2]
        assert trim([1, 0], [0, 1]) == 0 and lib.holo_kv4_pages_len(p, 0) == 64 and pages(0) == [0, 1]
        assert lib.holo_kv4_pages_len(p, 1) == 32 and lib.holo_kv4_pages_available(p) == 5
        for seqs, rows in (([0], [65]), ([0], [-1]), ([4], [0]), ([-1], [0]), ([0, 0], [1, 1]), ([1, 0], [1, 99])):
            assert rejected(trim(seqs, rows))
        assert rejected(lib.holo_kv4_pages_trim(p, None, ints(1), 1))
        assert rejected(lib.holo_kv4_pages_trim(None, ints(0), ints(1), 1))
        assert [lib.holo_kv4_pages_len(p, s) for s in (0, 1)] == [64, 32]
        # shared pages stay with the other sequence, and come back with the last
        assert lib.holo_kv4_pages_fork(p, ints(0), ints(2), 1) == 0
        assert trim([2], [40]) == 0 and pages(2) == [0] and lib.holo_kv4_pages_available(p) == 5
        assert lib.holo_kv4_pages_reserve(p, ints(2), ints(1), 1) == 0
        assert pages(2) == [2] and lib.holo_kv4_pages_len(p, 2) == 25  # its own copy of a shared, open page
        assert trim([0], [64]) == 0 and pages(0) == [] and lib.holo_kv4_pages_available(p) == 6
        assert trim([0], [0]) == 0 and lib.holo_kv4_pages_len(p, 0) == 0
        assert lib.holo_kv4_pages_trim(p, None, None, 0) == 0
    finally:
        lib.holo_kv4_pages_destroy(p)


# ---- the law of the verification ---------------------------------------------------------------------

@pytest.mark.parametrize("mode", ["chosen", "drawn", "distinct"])
def test_the_model_keeps_the_targets_distribution(mode):
    """The first token behind row 0, whichever way it came, has the target's probabilities."""
    rng = np.random.default_rng(3)
    p = np.float32([0.5, 0.25, 0.15, 0.1, 0])
    q = np.float32([0.1, 0.2, 0.3, 0.25, 0.15])
    n, parent = 30000, [-1, 0, 0, 0]
    target, draft = np.stack([p] * 4), np.stack([q] * 4)
    seen = np.zeros(5)
    for _ in range(n):
        if mode == "chosen":
            tokens = [9, 2, 0, 1]
        else:
            tokens = [9, *rng.choice(5, 3, mode == "drawn", q / q.sum(dtype=np.float64))]
        path, after, _ = dm.verify(parent, tokens, rng.random(4), target, draft, mode)
        seen[tokens[path[1]] if len(path) > 1 else after] += 1
    # five standard deviations of a share
    assert (np.abs(seen / n - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-7).all()
