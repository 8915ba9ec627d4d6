"""Drafted tokens in numpy, in 64 bits (include/holo_forward.h): trees, rotation,
attention of their rows, verification, and the rows that stand moved together.
Test infrastructure."""
from __future__ import annotations

import numpy as np

from kv4_model import attend


def tree(rng, rows, width):
    """parent of each row: every row has up to `width` behind it."""
    parent, kids = [-1][:rows], [0]
    for j in range(1, rows):
        p = j - 1
        if rng.random() < 0.5 or kids[p] >= width:
            p = int(rng.choice([i for i in range(j) if kids[i] < width]))
        kids[p] += 1
        parent.append(p)
        kids.append(0)
    return parent


def seen_rows(parent):
    """[rows][rows]: row i sees itself and what it follows; parents that are no earlier row are none."""
    n = len(parent)
    out = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while True:
            out[i, j] = True
            if not 0 <= parent[j] < j:
                break
            j = parent[j]
    return out


def words(seen, n):
    """[rows][n] 32-bit words of the rows' bits."""
    out = np.zeros((len(seen), n), np.uint32)
    for j in range(min(seen.shape[1], 32 * n)):
        out[:, j // 32] |= seen[:, j].astype(np.uint32) << np.uint32(j % 32)
    return out


def turned(x, pos, freq, dims, interleaved, scale, hd):
    """x [rows][heads * hd] with the pairs of each head turned to the rows' positions, in 64 bits."""
    y = x.astype(np.float64).reshape(len(x), -1, hd)
    a, b = (y[..., 0:dims:2], y[..., 1:dims:2]) if interleaved else (y[..., :dims // 2], y[..., dims // 2:dims])
    t = np.asarray(pos, np.float64)[:, None] * np.asarray(freq, np.float64)
    c, s = (scale * np.cos(t))[:, None], (scale * np.sin(t))[:, None]
    a2, b2 = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0:dims:2], y[..., 1:dims:2] = a2, b2
    else:
        y[..., :dims // 2], y[..., dims // 2:dims] = a2, b2
    return y.reshape(len(x), -1)


def want_attention(cache, layer, q, rows, seqs, n_heads, seen, take=None):
    """q [total][n_heads * hd]; seen[i]: [rows][rows] of entry i.  Rows past `take` are not looked at."""
    hd, out, at = cache.hd, np.zeros((q.shape[0], n_heads * cache.hd)), 0
    group = n_heads // cache.n_kv
    for n, seq, bits in zip(rows, seqs, seen):
        ln = int(cache.len[seq]) if 0 <= seq < cache.n_seqs else 0
        for kvh in range(cache.n_kv):
            k, v, there = cache.held(seq, layer, kvh, ln) if ln else (np.zeros((0, hd)),) * 2 + (np.zeros(0, bool),)
            for i in range(n if take is None else min(n, take)):
                p = np.arange(ln) - (ln - n)  # positions as rows of the entry
                see = there & ((p < 0) | bits[i][np.clip(p, 0, n - 1)])
                for h in range(kvh * group, (kvh + 1) * group):
                    out[at + i, h * hd:(h + 1) * hd] = attend(q[at + i, h * hd:(h + 1) * hd], k, v, see)
        at += n
    return out


def probability(p):
    """In 64 bits; what is negative or no finite number is 0."""
    return np.where(np.isfinite(p) & (p > 0), p, 0).astype(np.float64)


def weights(p, q, beta):
    w = probability(p)
    return np.maximum(w - beta * probability(q), 0.0) if q is not None and beta else w


def verify(parent, tokens, u, target, draft, mode):
    """path, next token and the margin by which the nearest comparison was decided, of one entry."""
    node, path, n, beta, gone, refused, margin = 0, [0], 1.0, 0.0, 0.0, set(), 1.0
    vocab = target.shape[1]
    for j in range(1, len(parent)):
        if parent[j] != node:
            continue
        x, uj = int(tokens[j]), float(u[j])
        there = 0 <= x < vocab
        if mode == "chosen":
            px = float(weights(target[node, x:x + 1], None, 0)[0]) if there and x not in refused else 0.0
            left, right = uj * n, px
        else:
            q = float(probability(draft[node, x])) if there else 0.0
            px = float(weights(target[node, x:x + 1], draft[node, x:x + 1], beta)[0]) if there else 0.0
            left, right = uj * q * n, px * (1 - gone)
        if left or right:
            margin = min(margin, abs(left - right) / max(left, right))
        if left < right:
            node, n, beta, gone, refused = j, 1.0, 0.0, 0.0, set()
            path.append(j)
        elif mode == "chosen":
            refused.add(x)
            n -= px
        elif there and gone < 1:
            beta += n / (1 - gone)
            n = weights(target[node], draft[node], beta).sum()
            gone += q if mode == "distinct" else 0.0
    w = weights(target[node], draft[node] if mode != "chosen" else None, beta)
    for x in refused:
        if 0 <= x < vocab:
            w[x] = 0.0
    sums = np.cumsum(w)
    if sums[-1] == 0:
        return path, int(probability(target[node]).argmax()), margin
    at = float(u[0]) * sums[-1]
    x = int(np.searchsorted(sums, at, side="right"))
    margin = min(margin, np.abs(sums[w > 0] - at).min() / sums[-1])
    return path, min(x, int(np.flatnonzero(w)[-1])), margin


def keep(cache, seq, rows, path):
    """Rows path[i] of the last `rows` positions of a sequence to the places of rows i, every layer and head, as codes."""
    first = int(cache.len[seq]) - rows
    for layer in range(cache.n_layers):
        for head in range(cache.n_kv):
            for i, r in enumerate(path):
                if r == i or not 0 <= r < rows or first + i < 0:
                    continue
                src, dst = cache._tile(seq, layer, head, first + r), cache._tile(seq, layer, head, first + i)
                if src is None or dst is None:
                    continue
                for which in (0, 1):
                    at, sh, sc = cache.where((first + r) % 32, which)
                    to, th, tc = cache.where((first + i) % 32, which)
                    codes, scales = src[at] >> sh.astype(np.uint8) & np.uint8(15), (src[sc].copy(), src[sc + 1].copy())
                    for s in (0, 4):
                        m = th == s
                        dst[to[m]] = (dst[to[m]] & np.uint8(240 >> s)) | (codes[m] << np.uint8(s))
                    dst[tc], dst[tc + 1] = scales


def unit(u):
    """A random number as the verification takes it: the nearest one in [0, 1), NaN as 0."""
    below = np.nextafter(np.float32(1), np.float32(0))
    return np.float32(0) if np.isnan(u) else np.clip(np.float32(u), np.float32(0), below)


def lane_scan(v):
    """Sums of the lanes up to each, in the order of a wave's scan (64 values, 64 bits)."""
    v = v.copy()
    for off in (1, 2, 4, 8, 16, 32):
        v[off:] = v[off:] + v[:-off]
    return v


def choose(w, u):
    """The first x at which the sum of w(0 .. x) passes u times the sum of all, in the kernel's own order of additions (its
    weights w in 64 bits, some above 0), and which lanes' sums pass their neighbours' although the lanes have no weight."""
    vocab = len(w)
    block = -(-vocab // (256 * 2048)) * 256
    n = -(-vocab // block)
    w = np.concatenate([w, np.zeros(n * block - vocab)])
    lanes = np.zeros((n, 64))
    for o in range(0, block, 64):
        lanes += w.reshape(n, block)[:, o:o + 64]
    for off in (32, 16, 8, 4, 2, 1):
        lanes = lanes + lanes[:, np.arange(64) ^ off]
    sums, per = lanes[:, 0], -(-n // 64)
    own = np.zeros(64)
    of = [range(min(lane * per, n), min((lane + 1) * per, n)) for lane in range(64)]
    for lane in range(64):
        for i in of[lane]:
            own[lane] += sums[i]
    upto = lane_scan(own)
    at = float(unit(u)) * upto[63]
    some, steps = own > 0, np.diff(upto, prepend=0.0) > 0
    passes = np.flatnonzero((upto > at) & some)
    lane = int(passes[0]) if len(passes) else int(np.flatnonzero(some)[-1])
    run, e = upto[lane - 1] if lane else 0.0, -1
    for i in of[lane]:
        if sums[i] == 0:
            continue
        if e >= 0:
            run += sums[e]
        e = i
        if run + sums[i] > at:
            break
    assert e >= 0
    token = -1
    for o in range(e * block, (e + 1) * block, 64):
        v = w[o:o + 64]
        to = run + lane_scan(v)
        here = np.flatnonzero((to > at) & (v > 0))
        if len(here):
            return o + int(here[0]), steps & ~some & (upto > at)
        if (v > 0).any():
            token = o + int(np.flatnonzero(v)[-1])
        run = to[63]
    return token, steps & ~some & (upto > at)
