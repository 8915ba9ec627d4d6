"""holo_attention_packed against float64 numpy: causal attention within packed
sequences, grouped heads, strides, ragged and odd lengths.

Tolerance 1e-5 normwise, as for attention over one sequence's fp32 rows: every
operand is two f16 halves (2^-22 of a value), products summed in fp32."""
import numpy as np
import pytest

from kv4_model import Batch, attend, normwise

pytestmark = pytest.mark.gpu

TOL = 1e-5


def want_packed(q, k, v, rows, hd, heads, n_kv):
    out, at = np.zeros((q.shape[0], heads * hd)), 0
    for n in rows:
        for h in range(heads):
            g = h * n_kv // heads
            kh, vh = (x[at:at + n, g * hd:(g + 1) * hd].astype(np.float64) for x in (k, v))
            for i in range(n):
                out[at + i, h * hd:(h + 1) * hd] = attend(q[at + i, h * hd:(h + 1) * hd], kh, vh, np.arange(n) <= i)
        at += n
    return out


def run(holo, q, k, v, rows, hd, heads, n_kv, lds=(0, 0, 0, 0), max_rows=None):
    total, lib = sum(rows), holo.lib()
    dims = (heads * hd, heads * hd, n_kv * hd, n_kv * hd)
    lds = [d + x for d, x in zip(dims, lds)]
    bufs = []
    for x, d, ld in zip((np.full((total, dims[0]), -9.0, np.float32), q, k, v), dims, lds):
        wide = np.full((total, ld), np.nan, np.float32)
        wide[:, :d] = x
        bufs.append(holo.DeviceBuffer.from_array(wide))
    b = Batch(holo, rows, None, max_rows)
    assert lib.holo_attention_packed(*[x.ptr for x in bufs], *lds, hd, heads, n_kv, b.ref) == 0
    lib.cuda_sync()
    holo.check("holo_attention_packed")
    got = bufs[0].download(np.float32).reshape(total, lds[0])
    assert np.isnan(got[:, dims[0]:]).all()
    return got[:, :dims[0]]


def inputs(seed, total, hd, heads, n_kv):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal((total, n * hd)).astype(np.float32) for n in (heads, n_kv, n_kv)]


@pytest.mark.parametrize("hd,heads,n_kv,rows,lds", [
    (128, 4, 2, [1, 2, 33, 64], (0, 0, 0, 0)),
    (64, 6, 6, [65, 0, 1, 31], (4, 8, 12, 16)),
    (96, 4, 1, [40, 100], (0, 4, 0, 4)),
    (32, 5, 5, [17, 129, 16, 15], (0, 0, 0, 0)),
    (128, 32, 8, [70], (0, 0, 0, 0)),
    (64, 12, 1, [1] * 40 + [90], (0, 0, 0, 0)),
    (64, 2, 1, [700], (0, 0, 0, 0)),
], ids=str)
def test_packed_attention(holo, hd, heads, n_kv, rows, lds):
    print(f"case packed hd {hd} heads {heads}/{n_kv} rows {rows[:5]}", flush=True)
    q, k, v = inputs(sum(rows) + hd, sum(rows), hd, heads, n_kv)
    got = run(holo, q, k, v, rows, hd, heads, n_kv, lds)
    want = want_packed(q, k, v, rows, hd, heads, n_kv)
    assert normwise(got, want) <= TOL
    assert np.array_equal(got, run(holo, q, k, v, rows, hd, heads, n_kv, lds))


@pytest.mark.parametrize("hd,heads,n_kv,rows", [
    (128, 64, 64, [1030]), (96, 32, 16, [1025, 300, 1000]), (128, 16, 4, [600, 33]), (96, 4, 4, [1500]),
    (32, 32, 32, [200] * 9), (128, 8, 8, [65] * 50),
], ids=str)
def test_larger_batches(holo, hd, heads, n_kv, rows):
    """Long prompts and many columns, on some of the rows and heads."""
    print(f"case packed larger hd {hd} heads {heads}/{n_kv} rows {rows[:3]}", flush=True)
    rng = np.random.default_rng(1)
    total = sum(rows)
    q, k, v = inputs(sum(rows), total, hd, heads, n_kv)
    got, at = run(holo, q, k, v, rows, hd, heads, n_kv), 0
    assert np.isfinite(got).all()
    for n in rows[:3]:
        for h in {0, heads - 1, int(rng.integers(heads))}:
            g = h * n_kv // heads
            kh, vh = (x[at:at + n, g * hd:(g + 1) * hd].astype(np.float64) for x in (k, v))
            s = q[at:at + n, h * hd:(h + 1) * hd].astype(np.float64) @ kh.T / np.sqrt(hd)
            s[np.arange(n)[None] > np.arange(n)[:, None]] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            want = (p / p.sum(1, keepdims=True)) @ vh
            assert normwise(got[at:at + n, h * hd:(h + 1) * hd], want) <= TOL
        at += n


def test_agrees_with_one_sequence_at_a_time(holo):
    """holo_attention_prefill of each sequence from position 0."""
    print("case packed against prefill", flush=True)
    hd, heads, n_kv, rows = 128, 8, 2, [150, 6, 300]
    q, k, v = inputs(3, sum(rows), hd, heads, n_kv)
    got, at = run(holo, q, k, v, rows, hd, heads, n_kv), 0
    for n in rows:
        d = [holo.DeviceBuffer.from_array(x[at:at + n]) for x in (q, k, v)]
        out = holo.DeviceBuffer(4 * n * heads * hd)
        holo.lib().holo_attention_prefill(out.ptr, d[0].ptr, d[1].ptr, d[2].ptr, n, 0, hd, heads, n_kv)
        holo.lib().cuda_sync()
        assert normwise(got[at:at + n], out.download(np.float32).reshape(n, -1).astype(np.float64)) <= 2 * TOL
        at += n


def test_rows_past_max_rows_are_left(holo):
    print("case packed max_rows", flush=True)
    hd, heads, n_kv, rows = 64, 4, 2, [50, 7]
    q, k, v = inputs(4, 57, hd, heads, n_kv)
    got = run(holo, q, k, v, rows, hd, heads, n_kv, max_rows=33)
    want = want_packed(q, k, v, rows, hd, heads, n_kv)
    assert (got[33:50] == -9.0).all()
    keep = list(range(33)) + list(range(50, 57))
    assert normwise(got[keep], want[keep]) <= TOL


@pytest.mark.parametrize("sq,sk,sv", [(1e-20, 1e15, 1e30), (1e20, 1e-20, 1e-30), (1, 1e-6, 1e-6), (1e5, 1e-5, 1e5),
                                      (1e-30, 1e-30, 1e38), (1, 1, 1e-38)])
def test_values_far_from_one(holo, sq, sk, sv):
    """Magnitudes that no f16 holds."""
    print(f"case packed scales {sq} {sk} {sv}", flush=True)
    hd, heads, n_kv, rows = 64, 2, 1, [70, 20]
    q, k, v = inputs(5, 90, hd, heads, n_kv)
    v = np.clip(v, -3, 3)
    q, k, v = (q * np.float32(sq)), (k * np.float32(sk)), (v * np.float32(sv))
    got = run(holo, q, k, v, rows, hd, heads, n_kv)
    want = want_packed(q, k, v, rows, hd, heads, n_kv)
    # the scores' error is 2e-6 of a score's magnitude of about sq sk
    assert normwise(got / sv, want / sv) <= max(TOL, 2e-6 * sq * sk)


def test_rows_behind_do_not_reach_a_row(holo):
    """Infinities, NaN and very large values in later rows: the rows before them
    are what they are without them; the rows from there on as in float64."""
    print("case packed poison", flush=True)
    hd, heads, n_kv, rows = 64, 4, 2, [100, 90]
    q, k, v = inputs(6, 190, hd, heads, n_kv)
    want = want_packed(q, k, v, rows, hd, heads, n_kv)
    for at, what in ((37, np.nan), (64, np.inf), (99, -np.inf), (5, np.nan)):
        k2, v2 = k.copy(), v.copy()
        k2[at, :hd] = what
        v2[at, hd + 3] = what  # one dim of the second KV head
        got = run(holo, q, k2, v2, rows, hd, heads, n_kv)
        want2 = want_packed(q, k2, v2, rows, hd, heads, n_kv)
        before = list(range(at)) + list(range(100, 190))
        assert normwise(got[before], want[before]) <= TOL
        assert np.isnan(got[at:100, :2 * hd]).all()
        second, w2 = got[at:100, 2 * hd:], want2[at:100, 2 * hd:]
        assert np.array_equal(np.isfinite(second), np.isfinite(w2))
        assert np.array_equal(second[np.isinf(w2)], w2[np.isinf(w2)])
        ok = np.isfinite(w2)
        assert normwise(second[ok], w2[ok]) <= TOL


def test_large_rows_behind_do_not_take_a_rows_precision(holo):
    print("case packed wide range", flush=True)
    hd, heads, n_kv, rows = 64, 4, 2, [100]
    q, k, v = inputs(7, 100, hd, heads, n_kv)
    want = want_packed(q, k, v, rows, hd, heads, n_kv)
    for at in (20, 45, 70):
        k2, v2 = k.copy(), v.copy()
        k2[at] *= np.float32(1e25)
        v2[at] *= np.float32(1e30)
        got = run(holo, q, k2, v2, rows, hd, heads, n_kv)
        assert normwise(got[:at], want[:at]) <= TOL
        want2 = want_packed(q, k2, v2, rows, hd, heads, n_kv)
        for i in range(at, 100):
            assert normwise(got[i], want2[i]) <= TOL


def test_captured(holo):
    """A captured call follows the device's cu_rows at each replay."""
    print("case packed graph", flush=True)
    lib = holo.lib()
    hd, heads, n_kv, total = 64, 4, 2, 120
    b = Batch(holo, [60, 60], None, 120)
    bufs = [holo.DeviceBuffer(4 * total * n * hd) for n in (heads, heads, n_kv, n_kv)]
    before, st = lib.holo_get_stream(), lib.holo_stream_create()
    lib.holo_set_stream(st)
    try:
        assert lib.holo_graph_begin() == 0
        assert lib.holo_attention_packed(*[x.ptr for x in bufs], heads * hd, heads * hd, n_kv * hd, n_kv * hd, hd,
                                         heads, n_kv, b.ref) == 0
        graph = lib.holo_graph_end()
        assert graph
        for i, rows in enumerate(([60, 60], [1, 119], [113, 7])):
            q, k, v = inputs(20 + i, total, hd, heads, n_kv)
            for x, y in zip(bufs[1:], (q, k, v)):
                x.upload(y)
            b.cu.upload(np.int32([0, rows[0], total]))
            assert lib.holo_graph_launch(graph) == 0
            lib.cuda_sync()
            got = bufs[0].download(np.float32).reshape(total, -1)
            assert normwise(got, want_packed(q, k, v, rows, hd, heads, n_kv)) <= TOL
            assert np.array_equal(got, run(holo, q, k, v, rows, hd, heads, n_kv))  # eager, on the same stream
        lib.holo_graph_destroy(graph)
    finally:
        lib.holo_set_stream(before)
        lib.holo_stream_destroy(st)


@pytest.mark.parametrize("hd,heads,n_kv,rows", [
    (64, 4, 2, [100]), (96, 4, 2, [20, 30]), (128, 64, 64, [1030]), (128, 16, 4, [600]), (32, 8, 8, [40] * 200),
], ids=str)
@pytest.mark.parametrize("low,sq", [(1e-5, 1), (1e-12, 1), (1e-5, 30)])
def test_low_rows_among_others(holo, hd, heads, n_kv, rows, low, sq):
    """Keys and values far smaller than their neighbours': a sequence's first rows
    (which rows see alone, and with others), and one in the middle that a head's rows look at
    alone.  Each row and head by itself, within what its scores allow."""
    print(f"case packed low rows hd {hd} heads {heads}/{n_kv} rows {rows[:3]} {low} {sq}", flush=True)
    total = sum(rows)
    q, k, v = inputs(8, total, hd, heads, n_kv)
    q *= np.float32(sq)
    at = 0
    for n in rows:
        k[at:at + 3] *= np.float32(low)
        v[at:at + 3] *= np.float32(low)
        v[at + n // 2] *= np.float32(low)
        k[at + n // 2, :hd] = np.sign(q[at + n - 1, :hd])  # the last row's first head
        at += n
    got, at = run(holo, q, k, v, rows, hd, heads, n_kv), 0
    for n in rows[:2]:
        for h in (0, heads - 1):
            g = h * n_kv // heads
            kh, vh = (x[at:at + n, g * hd:(g + 1) * hd].astype(np.float64) for x in (k, v))
            s = q[at:at + n, h * hd:(h + 1) * hd].astype(np.float64) @ kh.T / np.sqrt(hd)
            s[np.arange(n)[None] > np.arange(n)[:, None]] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            want = (p / p.sum(1, keepdims=True)) @ vh
            x = got[at:at + n, h * hd:(h + 1) * hd]
            err = np.linalg.norm(x - want, axis=1) / np.linalg.norm(want, axis=1)
            # a score is within 1.2e-5 of it at most for q of about 1, and a row's average within that of
            # the values that it averages, which cancel up to 1 / sqrt(n)
            assert err.max() <= 1.2e-5 * sq * np.sqrt(n)
            assert np.median(err) <= TOL * sq
        at += n
