"""The token behind the last row that stands, without a GPU: the order in which the verification adds
(draft_model.choose) against exact sums, on distributions whose gaps its roundings fall into."""
from fractions import Fraction

import numpy as np
import pytest

import draft_model as dm

VOCAB = 32000


def gapped(seed, vocab=VOCAB):
    """Weights at the two ends of the row, the second half the mirror of the first: half of their sum is reached
    where a gap begins."""
    rng = np.random.default_rng(seed)
    n = vocab // 3
    w = np.zeros(vocab, np.float32)
    z = 5 * rng.standard_normal(n)
    w[:n] = np.exp(z - z.max())
    w[:n] /= 2 * w.sum(dtype=np.float64)
    w[vocab - n:] = w[:n][::-1]
    return w


def check(w, u, token):
    """w(token) > 0, and the exact sums up to it and before it lie about u times the sum of all.  The additions of n
    weights are off by at most 2^-53 of the sum each, here and in the product."""
    assert w[token] > 0
    slack = (len(w) + 2) * 2.0 ** -53
    s = np.cumsum(w.astype(np.longdouble))
    at, off = np.longdouble(dm.unit(u)) * s[-1], 2 * slack * s[-1]
    assert s[token] >= at - off and s[token] - w[token] <= at + off


def test_the_first_lane_that_passes_may_have_no_weight():
    """With u = 0.5 lanes without weight have sums above u times all, one rounding above their neighbours': a choice by
    those differences would take one of them.  The choice goes by the lanes' own sums."""
    met = 0
    for seed in range(40):
        w = gapped(seed).astype(np.float64)
        token, empty = dm.choose(w, 0.5)
        check(w, 0.5, token)
        met += empty.any()
    assert met >= 5


@pytest.mark.parametrize("u", [0.0, 1e-30, 0.3, 0.999, 1.0, 2.0, np.inf, -1.0, -np.inf, np.nan])
def test_numbers_outside_their_range(u):
    for seed in range(6):
        w = gapped(seed).astype(np.float64)
        token, _ = dm.choose(w, u)
        check(w, u, token)
        one = np.zeros(VOCAB)
        one[seed * 5000 + 7] = 1e-3
        assert dm.choose(one, u)[0] == seed * 5000 + 7


def test_small_rows_are_exact():
    """Against rational sums, where 64 bits hold every sum."""
    rng = np.random.default_rng(1)
    for vocab in (1, 2, 64, 65, 257, 3001):
        w = rng.integers(0, 3, vocab) / 4.0
        w[rng.integers(vocab)] = 1
        for u in (0.0, 0.25, 0.5, 0.75, 0.96875):
            at, s = Fraction(u) * Fraction(w.sum()), Fraction(0)
            for x in range(vocab):
                s += Fraction(w[x])
                if s > at and w[x] > 0:
                    break
            assert dm.choose(w, u)[0] == x
