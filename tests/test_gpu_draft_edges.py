"""Drafted tokens on the GPU: calls at the edges of what they take."""
import ctypes as C

import numpy as np
import pytest

import draft_model as dm
from kv4_model import Batch, Cache, OnDevice, quantise, values
from test_gpu_draft import MODES, up, verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", MODES)
def test_verification_without_rows(holo, mode):
    """Entries without rows beside others get 0 and -1 over what was there; a batch without any writes nothing."""
    print(f"case verify no rows {mode}", flush=True)
    p = np.full((3, 40), 1 / 40, np.float32)
    u = np.full(3, 0.5)
    path, n_path, after = verify(holo, [0, 2, 0, 1, 0], [[], [-1, 0], [], [-1], []], np.int32([0, 50, 0]), u, p, p, mode)
    assert n_path.tolist() == [0, 1, 0, 1, 0] and after[[0, 2, 4]].tolist() == [-1] * 3 and path.tolist() == [0, -1, 0]
    outs = [up(holo, np.full(3, x, np.int32)) for x in (5, 6, 7)]
    ins = [up(holo, x) for x in (p, np.zeros(3, np.int32), np.full(3, -1, np.int32), np.float32(u))]
    b = Batch(holo, [0, 0, 0], max_rows=4)
    assert b.desc.rows == 0
    target, tokens, parent, us = (x.ptr for x in ins)
    assert holo.lib().holo_draft_verify(*[o.ptr for o in outs], target, target, 40, 40, 40, tokens, parent, us,
                                        MODES.index(mode), b.ref) == 0
    holo.lib().cuda_sync()
    holo.check("no rows")
    assert [o.download(np.int32).tolist() for o in outs] == [[5] * 3, [6] * 3, [7] * 3]


@pytest.mark.parametrize("mode", MODES)
def test_verification_at_its_borders_as_written_down(holo, mode):
    """Outcomes by the formulas, not by the model.  p: 0.25, 0.5, 0.25 at 3, 300, 599; q: all at 300."""
    print(f"case verify borders by hand {mode}", flush=True)
    p = np.zeros((4, 600), np.float32)
    p[:, 3], p[:, 300], p[:, 599] = 0.25, 0.5, 0.25
    q = np.zeros_like(p)
    q[:, 300] = 1.0
    t = [[-1, 0, 0, 1]]

    def call(tokens, u):
        path, n, after = verify(holo, [4], t, tokens, u, p, q, mode)
        assert (path[n[0]:] == -1).all()
        return path[:n[0]].tolist(), int(after[0])

    # row 1 (token 300, u 0.5): 0.5 < 0.5 does not hold, so it is refused; row 2 (token 3, u 0): 0 < 0.25 stands; nothing
    # follows row 2, and of 0.25, 0.5, 0.25 the second passes 0.5.  Without repeats all of q is gone with 300: 0 < 0.25 * 0
    # does not hold, and of p - q, 0.25 and 0.25, the second passes 0.25
    assert call([0, 300, 3, 300], [0.5, 0.5, 0, 0.6]) == (([0], 599) if mode == "distinct" else ([0, 2], 300))
    # row 1 stands (0.4 < 0.5), then row 3 behind it (0.3 < 0.5); 0.75 of the sum: the third
    assert call([0, 300, 3, 300], [0.75, 0.4, 0, 0.3]) == ([0, 1, 3], 599)
    # both refused.  Chosen: 300 again weighs nothing, 3 and 599 are left.  Otherwise p - q leaves the same two
    assert call([0, 300, 300, 9], [0.25, 0.9, 0.9, 0]) == ([0], 3)
    assert call([0, 300, 300, 9], [0.5, 0.9, 0.9, 0]) == ([0], 599)


@pytest.mark.parametrize("mode", MODES)
def test_every_entry_of_many_is_as_the_model_has_it(holo, mode):
    """Probabilities of odd numerators, whose sums meet no number drawn: every entry is compared."""
    print(f"case verify every entry {mode}", flush=True)
    rng = np.random.default_rng(18)
    n, t = 2000, [-1, 0, 0, 1]
    p, q = rng.dirichlet(np.ones(6), 2).astype(np.float32)
    tokens = rng.integers(0, 6, (n, 4))
    u = rng.random((n, 4)).astype(np.float32)
    p4, q4 = np.tile(p, (4, 1)), np.tile(q, (4, 1))
    path, n_path, after = verify(holo, [4] * n, [t] * n, tokens.ravel(), u.ravel(), np.tile(p, (4 * n, 1)),
                                 np.tile(q, (4 * n, 1)), mode)
    path, compared = path.reshape(n, 4), 0
    for i in range(n):
        want, token, margin = dm.verify(t, tokens[i], u[i], p4, q4, mode)
        if margin > 1e-12:
            compared += 1
            assert path[i].tolist() == want + [-1] * (4 - len(want)) and after[i] == token and n_path[i] == len(want)
    assert compared >= 0.95 * n


def test_softmax_of_more_rows_than_a_launch_has(holo):
    """2^24 rows of 256 threads each are 2^32 threads."""
    print("case softmax 2^24 rows", flush=True)
    rows, lib = (1 << 24) + 5, holo.lib()
    x = np.random.default_rng(0).random((rows, 2), dtype=np.float32)
    dx, dd = up(holo, x), up(holo, np.full(x.shape, -9.0, np.float32))
    assert lib.holo_softmax_rows(dd.ptr, dx.ptr, rows, 2, 2, 2, 1.0) == 0
    lib.cuda_sync()
    holo.check("softmax of many rows")
    got = dd.download(np.float32).reshape(rows, 2)
    e = np.exp(x.astype(np.float64))
    # an exponential, their sum, its reciprocal and a product: 2^-22 at most
    assert np.abs(got - e / e.sum(1, keepdims=True)).max() <= 2.0 ** -22


def test_small_exponentials_of_a_row(holo):
    """Rows of 0 and t below -17: their sum rounds to 1, so the second value is e^t itself, down to a float's least step."""
    print("case softmax exponentials", flush=True)
    rng, n, lib = np.random.default_rng(4), 1 << 18, holo.lib()
    x = np.zeros((2 * n, 2), np.float32)
    x[:n, 1], x[n:, 1] = rng.uniform(-87.3, -17, n), rng.uniform(-110, -87.3, n)
    x[-1, 1], x[-2, 1] = -np.inf, -3e38
    dx, dd = up(holo, x), up(holo, np.full(x.shape, -9.0, np.float32))
    assert lib.holo_softmax_rows(dd.ptr, dx.ptr, len(x), 2, 2, 2, 1.0) == 0
    lib.cuda_sync()
    holo.check("small exponentials")
    got = dd.download(np.float32).reshape(-1, 2).astype(np.float64)
    want = np.exp(x[:, 1].astype(np.float64))
    assert (got[:, 0] == 1).all()
    # the hardware's 2^f is within a unit of the last place, 2^-23 of itself; f within 2^-25, which counts times ln 2; below
    # the normal range half a step of 2^-149 for the last rounding
    off = np.abs(got[:, 1] - want)
    assert (off[:n] <= (2.0 ** -23 + 2.0 ** -25) * want[:n]).all()
    assert (off[n:] <= (2.0 ** -23 + 2.0 ** -25) * want[n:] + 2.0 ** -150).all()
    assert (got[-2:, 1] == 0).all()


@pytest.mark.parametrize("bound", [(1 << 29) - 63, (1 << 29) - 62, (1 << 29) - 30, 1 << 30, 0x7FFFF000])
def test_rows_under_far_bounds(holo, bound):
    """max_rows and rows are bounds: 70 rows go in and come back whatever they are, 2^32 threads and more among them."""
    print(f"case far bound {bound}", flush=True)
    hd, n, lib = 32, 70, holo.lib()
    rng = np.random.default_rng(2)
    k, v = rng.standard_normal((2, n, hd)).astype(np.float32)
    for rotated in (False, True):
        c = Cache(hd, 32, 1, 1, 3, 1, 3, fill=0)
        c.table[0], c.len[0] = (2, 0, 1), n
        dev = OnDevice(holo, c)
        dk, dv = up(holo, k), up(holo, v)
        b = Batch(holo, [n])
        b.desc.max_rows = b.desc.rows = bound
        if rotated:
            freq = up(holo, np.zeros(hd // 2))  # no angle: rows as they are
            rope = holo.Rope(freq=freq.ptr, dims=hd, interleaved=0, scale=1.0)
            assert lib.holo_kv4_append_rope(dev.ref, 0, C.byref(rope), None, dk.ptr, dv.ptr, 0, hd, hd, None, None, 0, 0, 0,
                                            None, b.ref) == 0
        else:
            assert lib.holo_kv4_append(dev.ref, 0, dk.ptr, dv.ptr, hd, hd, b.ref) == 0
        out = [up(holo, np.full((n, hd), -9.0, np.float32)) for _ in range(2)]
        assert lib.holo_kv4_read(dev.ref, 0, out[0].ptr, out[1].ptr, hd, hd, b.ref) == 0
        lib.cuda_sync()
        holo.check("far bounds")
        for got, x in zip(out, (k, v)):
            assert np.array_equal(got.download(np.float32).reshape(n, hd), values(*quantise(x)))
