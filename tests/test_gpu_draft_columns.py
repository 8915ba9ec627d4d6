"""Attention of drafted rows in 32 columns a workgroup, every head dim, with sequences in one range and cut into several:
what chooses the form is the batch's bounds, so small batches under far bounds run it."""
import numpy as np
import pytest

import draft_model as dm
from kv4_model import Cache, OnDevice, normwise
from test_gpu_draft import TOL, attention, fill, pages

pytestmark = pytest.mark.gpu

ENTRIES = 1025  # so many are never cut


def forms(holo, dev, q, rows, heads, mask, seqs):
    """The batch in one range and in several; entries without rows between its own do not count."""
    n_kv, G = dev.cache.n_kv, heads // dev.cache.n_kv
    cols, cus = max(rows) * G, 256
    assert cols > 16
    cut = attention(holo, dev, 0, q, rows, heads, mask, seqs=seqs, max_len=0x7FFFF000)
    groups = -(-cols // 32) * n_kv
    assert len(rows) * groups < 3 * cus // 2  # (otherwise nothing is cut)
    many, where = np.zeros(ENTRIES, int), np.linspace(0, ENTRIES - 1, len(rows)).astype(int)
    many[where] = rows
    at = np.full(ENTRIES, -1)
    at[where] = seqs
    assert ENTRIES * n_kv * -(-cols // 16) * 256 >= 2 * 256 * cus  # 8192 positions are 256 tiles
    return {"cut": cut, "whole": attention(holo, dev, 0, q, many.tolist(), heads, mask, seqs=at, max_len=8192)}


@pytest.mark.parametrize("heads,rows", [(8, [5, 9, 1]), (4, [12, 3, 40]), (24, [2, 1, 3]), (2, [20, 33, 64])], ids=str)
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_trees(holo, hd, heads, rows):
    """17 to 128 columns, the second half of the last 32 partly or wholly past them; lengths up to several ranges."""
    print(f"case columns trees {hd} {heads} {rows}", flush=True)
    rng = np.random.default_rng(hd + heads)
    n_kv, lens = 2, [rows[0] + 300, rows[1], 650]
    c = Cache(hd, 64, 1, n_kv, 20, 3, 12)
    pages(c, lens, rng)
    fill(c, rng, 0)
    dev, words = OnDevice(holo, c), 2
    seqs = [2, 0, 1]
    rows = [rows[2], rows[0], rows[1]]
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    for seen in ([dm.seen_rows(dm.tree(rng, n, 3)) for n in rows], [rng.random((n, n)) < 0.4 for n in rows]):
        want = dm.want_attention(c, 0, q, rows, seqs, heads, seen)
        mask = np.concatenate([dm.words(s, words) for s in seen])
        for form, got in forms(holo, dev, q, rows, heads, mask, seqs).items():
            assert normwise(got, want) <= TOL, form


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_where_nothing_is_seen(holo, hd):
    print(f"case columns empty {hd}", flush=True)
    rng = np.random.default_rng(hd)
    heads, n_kv, lens = 16, 2, [100, 3, 0, 96, 64, 33]
    c = Cache(hd, 32, 1, n_kv, 16, 6, 4)
    pages(c, lens, rng)
    fill(c, rng, 0)
    c.table[0, 1] = -1
    c.table[3, :] = (-5, 16, 1 << 30, -(1 << 31))
    c.table[4, 0] = 99
    dev = OnDevice(holo, c)
    rows, seqs = [2, 5, 1, 3, 40, 1, 1, 33], [0, 1, 2, 3, 4, -1, 6, 5]
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    seen = [dm.seen_rows(dm.tree(rng, n, 2)) for n in rows]
    seen[-1][[0, 5, 17, 32]] = False
    seen[4][:20] = False
    want = dm.want_attention(c, 0, q, rows, seqs, heads, seen)
    nothing = (want == 0).all(1)
    assert nothing.sum() >= 12
    for form, got in forms(holo, dev, q, rows, heads, np.concatenate([dm.words(s, 2) for s in seen]), seqs).items():
        assert normwise(got, want) <= TOL and (got[nothing] == 0).all(), form


@pytest.mark.parametrize("heads,rows", [(16, 3), (4, 40), (6, 9)])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_not_touched_by_what_a_row_does_not_see(holo, hd, heads, rows):
    """NaN behind the end, NaN and infinite keys and values at rows that only some see, in both halves of the columns."""
    print(f"case columns poison {hd} {heads} {rows}", flush=True)
    rng = np.random.default_rng(7)
    n_kv, n, g = 2, 290, heads // 2
    seen = dm.seen_rows(dm.tree(rng, rows, 2))
    mask = dm.words(seen, 2)
    q = rng.standard_normal((rows, heads * hd)).astype(np.float32)
    c = Cache(hd, 32, 1, n_kv, 11, 1, 10, fill=0xFF)  # scales of NaN where nothing is written
    pages(c, [n], rng)
    fill(c, rng, 0)
    k, v = rng.standard_normal((2, hd)).astype(np.float32)
    v[hd - 5] = np.nan
    c.put(0, 0, 1, n - rows + 1, k, v)      # head 1, row 1: the last 32 dims of the value
    bad = rng.standard_normal(hd).astype(np.float32)
    bad[3] = np.inf
    c.put(0, 0, 0, n - rows + 2, bad, bad)  # head 0, row 2: key and value
    want = dm.want_attention(c, 0, q, [rows], [0], heads, [seen]).reshape(rows, heads, hd)
    ok = ~np.isnan(want)
    assert np.isnan(want[seen[:, 1], g:, hd - 32:]).all() and not np.isnan(want[~seen[:, 1], g:]).any()
    for form, got in forms(holo, OnDevice(holo, c), q, [rows], heads, mask, [0]).items():
        got = got.reshape(rows, heads, hd)
        assert np.array_equal(np.isnan(got), ~ok) and normwise(got[ok], want[ok]) <= TOL, form
    # a NaN before all rows reaches every one, in its block of dims; NaN and infinities of q their own row and head
    c.put(0, 0, 1, 3, k, v)
    q[rows - 1, hd - 1], q[0, 2] = np.nan, np.inf
    want = dm.want_attention(c, 0, q, [rows], [0], heads, [seen]).reshape(rows, heads, hd)
    want[0, 0] = np.nan
    ok = ~np.isnan(want)
    assert not ok[:, g:, hd - 32:].any() and not ok[rows - 1, 0].any()
    for form, got in forms(holo, OnDevice(holo, c), q, [rows], heads, mask, [0]).items():
        got = got.reshape(rows, heads, hd)
        assert np.array_equal(np.isnan(got), ~ok) and normwise(got[ok], want[ok]) <= TOL, form


@pytest.mark.parametrize("hd,heads,n_kv", [(128, 2, 1), (32, 4, 2)])
def test_more_pages_than_lanes(holo, hd, heads, n_kv):
    """A wave holds 64 entries of the table at a time: ranges of up to 141 pages of 32 positions, some of them missing."""
    print(f"case columns pages {hd} {heads}/{n_kv}", flush=True)
    rng = np.random.default_rng(hd)
    lens, rows, seqs = [4500, 2080, 2047], [9, 20, 33], [0, 1, 2]
    c = Cache(hd, 32, 1, n_kv, 280, 3, 141)
    pages(c, lens, rng)
    c.table[0, [3, 64, 100]] = -1, 280, -7
    c.pool[:] = rng.integers(0, 256, c.pool.shape, dtype=np.uint8)
    f = c.pool[..., 32 * hd:].view(np.uint16)  # scales of 0.5 to 2, either sign, in the cache's 8 significant bits
    f[:] = (f & 0x83F8) | (0x3800 + (f & 0x0400))
    dev = OnDevice(holo, c)
    seen = [dm.seen_rows(dm.tree(rng, n, 2)) for n in rows]
    q = (0.1 * rng.standard_normal((sum(rows), heads * hd))).astype(np.float32)
    want = dm.want_attention(c, 0, q, rows, seqs, heads, seen)
    mask = np.concatenate([dm.words(s, 2) for s in seen])
    got = forms(holo, dev, q, rows, heads, mask, seqs)
    got["16 columns"] = attention(holo, dev, 0, q, rows, heads, mask, seqs=seqs)
    for form, x in got.items():
        assert normwise(x, want) <= TOL, form
