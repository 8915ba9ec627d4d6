"""The token behind the last row that stands, on the GPU: rows with gaps whose sums round, and random numbers outside
their range (draft_model.choose has the kernel's order of additions, so tokens are compared exactly)."""
import numpy as np
import pytest

import draft_model as dm
from test_draft_choice import VOCAB, check, gapped
from test_gpu_draft import MODES, verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("vocab", [VOCAB, 128256, 600000])
def test_rows_with_gaps(holo, mode, vocab):
    print(f"case choice gaps {mode} {vocab}", flush=True)
    n = 40 if vocab == VOCAB else 6
    p = np.stack([gapped(seed, vocab) for seed in range(n)])
    path, n_path, after = verify(holo, [1] * n, [[-1]] * n, np.zeros(n), np.full(n, 0.5), p, p, mode)
    assert (path == 0).all() and (n_path == 1).all()
    met = 0
    for i in range(n):
        token, empty = dm.choose(p[i].astype(np.float64), 0.5)
        assert after[i] == token
        met += empty.any()
    assert met >= (5 if vocab == VOCAB else 0)


@pytest.mark.parametrize("mode", MODES)
def test_rows_with_gaps_behind_refusals(holo, mode):
    """Two rows behind row 0 are refused; the weights left are mirrored as well."""
    print(f"case choice refused {mode}", flush=True)
    n, parent = 40, [-1, 0, 0]
    rng = np.random.default_rng(3)
    p = np.repeat(np.stack([gapped(seed) for seed in range(n)]), 3, 0)
    q = p.copy()
    half = rng.random((3 * n, VOCAB // 2)).astype(np.float32)
    q *= np.concatenate([half, half[:, ::-1]], 1)  # (mirrored, and below p: some weight is left)
    q[:, VOCAB // 2 - 1:VOCAB // 2 + 1] = 0.1      # both tokens have no p
    tokens = np.tile([0, VOCAB // 2 - 1, VOCAB // 2], n)
    u = np.tile(np.float32([0.5, 0.5, 0.5]), n)
    path, n_path, after = verify(holo, [3] * n, [parent] * n, tokens, u, p, q, mode)
    assert (path.reshape(n, 3) == [0, -1, -1]).all() and (n_path == 1).all()
    for i in range(n):
        w, beta, gone, left = p[3 * i].astype(np.float64), 0.0, 0.0, 1.0
        if mode != "chosen":
            for _ in range(2):
                beta += left / (1 - gone)
                w = dm.weights(p[3 * i], q[3 * i], beta)
                left = w.sum()
                gone += float(np.float32(0.1)) if mode == "distinct" else 0.0
        # beta is off by the sums' roundings, 32000 * 2^-53 of it, and a weight by that and one more; the sum of all is
        # above 0.01, so the sums' share of it by less than 1e-9
        assert w[after[i]] > 0 and w.sum() > 0.01
        s = np.cumsum(w)
        assert s[after[i]] >= (0.5 - 1e-9) * s[-1] and s[after[i]] - w[after[i]] <= (0.5 + 1e-9) * s[-1]


@pytest.mark.parametrize("mode", MODES)
def test_numbers_outside_their_range(holo, mode):
    print(f"case choice numbers {mode}", flush=True)
    us = np.float32([1.0, 2.0, np.inf, -1.0, -np.inf, np.nan, 0.0, np.nextafter(np.float32(1), np.float32(0))])
    n = 12
    p = [gapped(seed) for seed in range(n)]
    for seed in range(n):  # a token alone, and three of very different weight
        w = np.zeros(VOCAB, np.float32)
        w[2500 * seed + 11] = 1
        if seed % 2:
            w[[3, 16000 + seed]] = 1e-20, 0.25
        p.append(w)
    p = np.repeat(np.stack(p), len(us), 0)
    u = np.tile(us, 2 * n)
    _, n_path, after = verify(holo, [1] * len(p), [[-1]] * len(p), np.zeros(len(p)), u, p, p, mode)
    assert (n_path == 1).all()
    for i in range(len(p)):
        w = p[i].astype(np.float64)
        assert after[i] == dm.choose(w, u[i])[0]
        check(w, u[i], after[i])
    # a drafted token that the target has with the draft's probability stands for every number; one of probability 0
    # for none
    half = np.zeros((2 * len(us), 300), np.float32)
    half[:, [20, 10]] = 0.5
    if mode == "chosen":
        half[:, [20, 10]] = 1, 0
    path, n_path, _ = verify(holo, [2] * len(us), [[-1, 0]] * len(us), np.tile([0, 20], len(us)), np.repeat(us, 2), half,
                             half, mode)
    assert (n_path == 2).all() and (path.reshape(-1, 2) == [0, 1]).all()
    _, n_path, after = verify(holo, [2] * len(us), [[-1, 0]] * len(us), np.tile([0, 30], len(us)), np.repeat(us, 2), half,
                              half, mode)
    assert (n_path == 1).all() and np.isin(after, [10, 20]).all()
