"""holo_attention_packed at the magnitudes where its forms change, against
float64 numpy, in every form of the kernel.

Tolerance 1e-5 normwise, as for values of ordinary size: the planted products are
kept at an ordinary score's size (q is small where a key is large), and a
planted value's part is its probability, within 2e-6 in the mean, times it."""
import numpy as np
import pytest

from test_gpu_packed_attention import TOL, inputs, normwise, run

pytestmark = pytest.mark.gpu

# head_dim, heads, KV heads, rows: keys shared by eight waves, by four, 128 columns (two), 256 columns
FORMS = [(128, 4, 2, [100]), (128, 32, 32, [300]), (128, 8, 4, [30, 12]), (64, 64, 64, [600]), (96, 64, 64, [1030])]


def want_head(q, k, v, n, hd, h, g):
    """Rows 0 .. n - 1 of one sequence and head, in 64 bits."""
    kh, vh = (x[:n, g * hd:(g + 1) * hd].astype(np.float64) for x in (k, v))
    with np.errstate(invalid="ignore"):
        s = q[:n, h * hd:(h + 1) * hd].astype(np.float64) @ kh.T / np.sqrt(hd)
        s[np.arange(n)[None] > np.arange(n)[:, None]] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        return (p / p.sum(1, keepdims=True)) @ vh


@pytest.mark.parametrize("hd,heads,n_kv,rows", FORMS, ids=str)
@pytest.mark.parametrize("value", [False, True], ids=["key", "value"])
def test_around_the_largest_value_of_the_halves(holo, hd, heads, n_kv, rows, value):
    """Times 2^8, f16 rounds values from 255.9375 up to infinity: the rows that see a key or
    value just below, at and past that, and the rows before it."""
    total, n = sum(rows), rows[0]
    at, dim = n // 2, 5
    for x in (255.9374, 255.9375, -255.9375, -255.99, 256.0):
        print(f"case packed hd {hd} heads {heads}/{n_kv} rows {rows} {'value' if value else 'key'} {x}", flush=True)
        q, k, v = inputs(31, total, hd, heads, n_kv)
        q[:, dim::hd] /= 64
        (v if value else k)[at, dim::hd] = x
        got = run(holo, q, k, v, rows, hd, heads, n_kv)
        assert np.isfinite(got).all()
        for h in (0, heads - 1):
            want = want_head(q, k, v, n, hd, h, h * n_kv // heads)
            part = got[:n, h * hd:(h + 1) * hd]
            assert normwise(part[:at], want[:at]) <= TOL
            assert normwise(part[at:], want[at:]) <= TOL


@pytest.mark.parametrize("hd,heads,n_kv,rows", FORMS, ids=str)
@pytest.mark.parametrize("low", [-np.inf, -3e38], ids=["infinite", "finite"])
def test_first_keys_without_weight(holo, hd, heads, n_kv, rows, low):
    """Scores of -infinity (or of less than a float holds) at a sequence's first keys, one to
    five of them, and at one in its middle: those keys have no part in the rows that see others,
    and rows that see no others are NaN, as the formula's difference of two infinities."""
    total, n, dim = sum(rows), rows[0], 3
    for first in (1, 2, 4, 5):
        print(f"case packed hd {hd} heads {heads}/{n_kv} rows {rows} first {first} keys of {low}", flush=True)
        q, k, v = inputs(32, total, hd, heads, n_kv)
        q[:, dim::hd] = 4 + np.abs(q[:, dim::hd])
        # other keys: a dim's products of an ordinary score's size
        k[:, dim::hd] /= 8
        for at in (*range(first), n // 2):
            k[at, dim::hd] = low
        got = run(holo, q, k, v, rows, hd, heads, n_kv)
        for h in (0, heads - 1):
            want = want_head(q, k, v, n, hd, h, h * n_kv // heads)
            part = got[:n, h * hd:(h + 1) * hd]
            assert np.isnan(part[:first]).all()
            assert normwise(part[first:], want[first:]) <= TOL
