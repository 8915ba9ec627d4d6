"""The operators of decoding with drafted tokens, as measurable cases.

A program that serves several sequences from the 4-bit cache in pages lets a
small model draft the next tokens of each, a chain or a tree of them, and runs
the large one over all of them at once.  An entry's rows are then its last
token (row 0) and the drafted ones; parent[i] is the row that row i follows, -1
for row 0.  Row i stands at the position of row 0 plus its depth in the tree.

  turn     holo_draft_plan (depth of the rows, and which rows each follows, one
           bit a row) where there are trees, and holo_kv4_append_rope: queries
           and keys rotated to their positions, keys and values into the pages
  attend   holo_attention_kv4_draft: each row over the sequence's pages before
           the entry's rows and over those rows that its bits name
  softmax  holo_softmax_rows: the rows' logits to probabilities
  verify   holo_draft_verify: which drafted tokens stand, against the target's
           probabilities and given random numbers, and the token behind them
  keep     holo_kv4_keep: the rows that stand moved together in the pages, every
           layer

Rotation: pair i of the leading `dims` dims of a head turns by position * freq[i]
and is multiplied by `scale`; it is dims (2 i, 2 i + 1) where interleaved, else (i,
i + dims / 2).  In 64 bits, rounded once to 32.

Verification walks the rows in order with a node (row 0 at first), N = 1, beta =
0, Q = 0.  A row whose parent is the node is judged with its token x, its u and
the node's rows p of the target's and q of the draft's probabilities:
  drawn     u q(x) N < max(p(x) - beta q(x), 0) (1 - Q): it stands and becomes the node, N =
            1, beta = 0, Q = 0.  Else beta += N / (1 - Q), N = sum max(p - beta q, 0); and where the
            tokens behind a node were drawn without repeats, Q += q(x)
  chosen    u N < p(x), p(x) = 0 for the tokens refused at this node; else N -= p(x)
The next token is the first x where the sum of w(0 .. x) passes u of row 0 times
the sum of all: w = max(p - beta q, 0), or p less the refused tokens.

The pages are those of holo_kv4_t (4.5 bits a value): a page holds, for every
layer and KV head, tiles of 32 positions of 36 * hd bytes.  With nb = hd / 32
blocks of 32 dims and lane = 16 g + r, g < 4, r < 16:

  K codes   [half][lane][nb] 32-bit words: position 16 half + r, dims 8 w .. 8 w + 7,
            w = nb g + j of the lane's word j
  V codes   [chunk][lane][VW] words (VW = 4 where nb is even, else 2): dim 16 m + r,
            m = VW chunk + j, positions 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3
  K scales  f16 [block][r][half]
  V scales  f16 [block][g][8], the positions in the words' order

Value i of a word is its nibble i / 2 + 4 (i % 2), less 8, times the scale of
the position's block.  A block's scale: with m its value of largest magnitude
(the negative one of two), -m / 8 rounded to bfloat16, at most 2720, held in
f16; a value's code is the nearest to its quotient in -8 .. 7.
"""
from __future__ import annotations

import ctypes
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_MODES = ("chosen", "drawn", "distinct")


def _holo():
    path = os.path.join(_ROOT, "google-classic_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import holo_mi355x as holo
    holo.init()
    return holo


def listed():
    return [
        # a step of four conversations with short drafts: where latency counts
        {"name": "turn_4x8", "kind": "turn", "seqs": 4, "rows": 8, "width": 2, "spread": 0.0, "before": 701,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "dims": 128, "pairs": "half", "stretch": 1.0,
         "keys_out": False, "page": 64},
        # the prompts of a batch far into their contexts, on positions stretched for them; the packed attention
        # reads the rotated keys too
        {"name": "turn_4x1000", "kind": "turn", "seqs": 4, "rows": 1000, "width": 0, "spread": 0.8, "before": 90077,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "dims": 96, "pairs": "interleaved", "stretch": 4.0,
         "keys_out": True, "page": 128},
        # one short conversation, a chain of four tokens, every query head with keys of its own
        {"name": "attend_1x5_at_512", "kind": "attend", "seqs": 1, "rows": 5, "width": 1, "len": 517, "spread": 0.0,
         "heads": 32, "kv_heads": 32, "head_dim": 128, "page": 64},
        # trees over conversations of all lengths
        {"name": "attend_16x26_to_4096", "kind": "attend", "seqs": 16, "rows": 26, "width": 4, "len": 4096,
         "spread": 0.95, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64},
        # a full server, short chains
        {"name": "attend_64x5_to_8192", "kind": "attend", "seqs": 64, "rows": 5, "width": 1, "len": 8192, "spread": 0.5,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 128},
        # a large tree behind one very long document
        {"name": "attend_1x63_at_100000", "kind": "attend", "seqs": 1, "rows": 63, "width": 3, "len": 100063,
         "spread": 0.0, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 256},
        # one conversation's chain, and the trees of a batch
        {"name": "softmax_5", "kind": "softmax", "rows": 5, "vocab": 32000, "pad": 0, "kept": 1.0},
        {"name": "softmax_416", "kind": "softmax", "rows": 416, "vocab": 32000, "pad": 64, "kept": 0.01},
        # a full server's chains, drawn from the draft's probabilities
        {"name": "verify_64x5", "kind": "verify", "seqs": 64, "rows": 5, "width": 1, "spread": 0.0, "vocab": 32000,
         "mode": "drawn"},
        # trees whose branches were drawn without repeats
        {"name": "verify_16x26", "kind": "verify", "seqs": 16, "rows": 26, "width": 4, "spread": 0.5, "vocab": 32000,
         "mode": "distinct"},
        # the rows that stand: of one conversation, and of a full server
        {"name": "keep_1x26", "kind": "keep", "seqs": 1, "rows": 26, "kept": 5, "spread": 0.0, "before": 701,
         "layers": 32, "kv_heads": 8, "head_dim": 128, "page": 64},
        {"name": "keep_64x26", "kind": "keep", "seqs": 64, "rows": 26, "kept": 5, "spread": 0.5, "before": 77,
         "layers": 32, "kv_heads": 8, "head_dim": 128, "page": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("turn", "attend", "attend", "attend", "softmax", "verify", "verify", "keep"))
    spread = rng.choice((0.0, rng.uniform(0.1, 0.95)))
    if kind == "softmax":
        vocab = _log(rng, 1, 150000)
        return {"kind": kind, "rows": max(1, min(_log(rng, 1, 3000), 416 * 32000 // vocab)), "vocab": vocab,
                "pad": rng.choice((0, 0, rng.randint(1, 100))), "kept": rng.choice((1.0, rng.uniform(0.001, 0.5)))}
    seqs = _log(rng, 1, 64)
    if kind == "verify":
        mode, rows = rng.choice(_MODES), _log(rng, 1, 64)
        vocab = _log(rng, 100, 150000)
        rows = max(1, min(rows, 416 * 32000 // (seqs * vocab)))
        return {"kind": kind, "seqs": seqs, "rows": rows, "width": rng.choice((1, 1, 2, 3, 4)), "spread": spread,
                "vocab": vocab, "mode": mode}
    hd = rng.choice((32, 64, 64, 96, 128, 128, 128))
    heads = rng.choice((4, 8, 16, 24, 32, 40))
    kv_heads = heads // rng.choice((1, 2, 4))
    page = rng.choice((32, 64, 128, 256))
    if kind == "keep":
        rows = _log(rng, 1, 128)
        layers = max(1, min(_log(rng, 1, 32), 64 * 32 * 8 * 128 * 128 // (seqs * (rows + 128) * kv_heads * hd)))
        return {"kind": kind, "seqs": seqs, "rows": rows, "kept": _log(rng, 1, 12), "spread": spread,
                "before": _log(rng, 1, 128) - 1, "layers": layers, "kv_heads": kv_heads, "head_dim": hd,
                "page": min(page, 64)}
    width = rng.choice((1, 2, 3, 4))
    if kind == "turn":
        rows = _log(rng, 1, 128)
        if rng.random() < 0.4:
            width, rows = 0, _log(rng, 1, 2000)
        rows = max(1, min(rows, 2400 * 32 // (seqs * heads)))
        return {"kind": kind, "seqs": seqs, "rows": rows, "width": width, "spread": spread,
                "before": _log(rng, 1, 120000) - 1, "heads": heads, "kv_heads": kv_heads, "head_dim": hd,
                "dims": rng.choice((hd, hd, hd // 2, hd - 2 * rng.randint(0, hd // 2 - 1))),
                "pairs": rng.choice(("half", "interleaved")), "stretch": rng.choice((1.0, rng.uniform(1.0, 16.0))),
                "keys_out": rng.random() < 0.5, "page": page}
    rows, length = _log(rng, 1, 160), _log(rng, 1, 60000)
    length = max(1, min(length, 64 * 8 * 128 * 6000 // (seqs * kv_heads * hd)))
    rows = max(1, min(rows, length, 63 * 100000 * 32 * 128 // (seqs * length * heads * hd)))
    return {"kind": kind, "seqs": seqs, "rows": rows, "width": width, "len": length, "spread": spread, "heads": heads,
            "kv_heads": kv_heads, "head_dim": hd, "page": page}


# ---- sizes and trees -----------------------------------------------------------------

def _shrunk(longest, spread, n):
    """n whole numbers from `longest` down to (1 - spread) of it."""
    return [max(1, int(longest * (1 - spread * i / max(1, n - 1)))) for i in range(n)]


def _sizes(case):
    """Rows of the call and positions of the cache (these rows among them), by sequence."""
    if case["kind"] == "attend":
        lens = _shrunk(case["len"], case["spread"], case["seqs"])
        return [min(case["rows"], n) for n in lens], lens
    rows = _shrunk(case["rows"], case["spread"], case["seqs"])
    return rows, [case.get("before", 0) + r for r in rows]


def _tree(rows, width, seed):
    """parent of each row: every row has up to `width` behind it, half of the rows follow the one before them."""
    rng, parent, kids = random.Random(seed), [-1], [0]
    for j in range(1, rows):
        p = j - 1
        if rng.random() < 0.5 or kids[p] >= width:
            p = rng.choice([i for i in range(j) if kids[i] < width])
        kids[p] += 1
        parent.append(p)
        kids.append(0)
    return parent


def _depths(parent):
    depth = []
    for p in parent:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _masks(parent, words):
    """By row, its own bit and those of the rows it follows, in 32-bit words."""
    mask = []
    for i, p in enumerate(parent):
        mask.append((mask[p] if p >= 0 else 0) | 1 << i)
    return [[m >> 32 * w & 0xFFFFFFFF for w in range(words)] for m in mask]


def _trees(case, rows):
    return [_tree(r, case["width"], 1000 * i + r) for i, r in enumerate(rows)]


def work(case):
    if case["kind"] == "softmax":
        n = case["rows"] * case["vocab"]
        return {"bytes": 8 * n, "flops": 4 * n}
    rows, lens = _sizes(case)
    if case["kind"] == "verify":
        # the probabilities behind each sequence's last token: the target's, and the draft's where they count
        n = case["seqs"] * case["vocab"] * (1 if case["mode"] == "chosen" else 2)
        return {"bytes": 4 * n + 16 * sum(rows), "flops": 2 * n}
    hd, kv = case["head_dim"], case["kv_heads"]
    row4 = kv * hd * 36 // 32  # a position's keys and values in one layer of the cache
    if case["kind"] == "keep":
        moved = sum(n - 1 if r > n else 0 for r, n in zip(rows, _kept(case, rows)))
        return {"bytes": 2 * moved * case["layers"] * row4 + 4 * (sum(rows) + case["seqs"]), "flops": 0}
    if case["kind"] == "turn":
        b = 8 * case["heads"] * hd + 16 * kv * hd + 2 * row4 + (4 * kv * hd if case["keys_out"] else 0)
        b += 8 + 4 * ((max(rows) + 31) // 32) if case["width"] else 0
        return {"bytes": sum(rows) * b, "flops": sum(rows) * (3 * (case["heads"] + kv) * case["dims"] + 8 * kv * hd)}
    pairs = sum(r * (n - r) + sum(_depths(t)) + r for r, n, t in zip(rows, lens, _trees(case, rows)))
    return {"bytes": sum(lens) * row4 + 8 * sum(rows) * case["heads"] * hd, "flops": 4 * pairs * case["heads"] * hd}


def _kept(case, rows):
    """Rows that stand, by sequence: row 0 and rows behind all places that are written."""
    return [max(1, min(case["kept"], (r + 1) // 2)) for r in rows]


# ---- the 4-bit tiles ------------------------------------------------------------------

def _quantised(x):
    """Codes 0 .. 15 [..., hd] and f16 scales [..., hd / 32] of finite values."""
    b = x.unflatten(-1, (-1, 32))
    low, high = b.amin(-1), b.amax(-1)
    big = torch.maximum(-low, high)
    d = torch.where(-low >= high, 1.0, -1.0) * (big / 8).to(torch.bfloat16).float().clamp(max=2720.0)
    d = d.half()
    # a quotient in 64 bits: in 32 a value next to the middle of two codes could take the wrong one
    c = torch.round(b.double() / d.double().unsqueeze(-1)).clamp(-8, 7)
    c = torch.where(d.unsqueeze(-1) == 0, 0.0, c)
    return (c.flatten(-2) + 8).to(torch.uint8), d


def _values(codes, d):
    return ((codes.unflatten(-1, (-1, 32)).float() - 8) * d.float().unsqueeze(-1)).flatten(-2)


def _words(nibbles):
    """[..., 8] codes into 32-bit words."""
    place = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=nibbles.device)
    return (nibbles.long() << place).sum(-1).to(torch.int32)


def _nibbles(words):
    place = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=words.device, dtype=torch.int32)
    return ((words.unsqueeze(-1) >> place) & 15).to(torch.uint8)


def _k_codes(c):
    """[..., 32, hd] codes as the bytes of K."""
    nb = c.shape[-1] // 32
    c = c.reshape(*c.shape[:-2], 2, 16, 4, nb, 8).movedim(-3, -4)  # half, g, r, j, 8
    return _words(c).contiguous().flatten(-4).view(torch.uint8)


def _v_codes(c):
    """[..., 32, hd] codes as the bytes of V."""
    m = c.shape[-1] // 16
    vw = 4 if m % 4 == 0 else 2
    c = c.reshape(*c.shape[:-2], 2, 4, 4, m // vw, vw, 16)  # half, g, 4, chunk, j, r
    n = c.dim() - 6
    c = c.permute(*range(n), n + 3, n + 1, n + 5, n + 4, n, n + 2).flatten(-2)  # chunk, g, r, j, 8
    return _words(c).contiguous().flatten(-4).view(torch.uint8)


def _packed_tiles(ck, cv, dk, dv):
    """Tiles [..., 36 hd] of bytes from codes [..., 32, hd] and scales [..., 32, nb]."""
    sk = dk.unflatten(-2, (2, 16)).movedim(-1, -3).movedim(-2, -1)  # nb, r, half
    sv = dv.unflatten(-2, (2, 4, 4)).movedim(-1, -4).movedim(-3, -2)  # nb, g, half, 4
    return torch.cat((_k_codes(ck), _v_codes(cv), sk.contiguous().flatten(-3).view(torch.uint8),
                      sv.contiguous().flatten(-4).view(torch.uint8)), -1)


def _unpacked_tiles(t, hd):
    """Codes and scales (as _packed_tiles takes them) of tiles [..., 36 hd] of bytes."""
    nb, lead = hd // 32, t.shape[:-1]
    n = len(lead)
    k, v, sk, sv = (x.contiguous() for x in t.split((16 * hd, 16 * hd, 2 * hd, 2 * hd), -1))
    ck = _nibbles(k.view(torch.int32).reshape(*lead, 2, 4, 16, nb)).movedim(-4, -3).reshape(*lead, 32, hd)
    vw = 4 if nb % 2 == 0 else 2
    cv = _nibbles(v.view(torch.int32).reshape(*lead, 2 * nb // vw, 4, 16, vw)).unflatten(-1, (2, 4))
    cv = cv.permute(*range(n), n + 4, n + 1, n + 5, n, n + 3, n + 2).reshape(*lead, 32, hd)
    dk = sk.view(torch.float16).reshape(*lead, nb, 16, 2).movedim(-1, -3).movedim(-2, -1).reshape(*lead, 32, nb)
    dv = sv.view(torch.float16).reshape(*lead, nb, 4, 2, 4).movedim(-2, -3).movedim(-4, -1).reshape(*lead, 32, nb)
    return ck, cv, dk, dv


# ---- inputs ---------------------------------------------------------------------------

def _pool(s, gen, first_used):
    """Pages in random order behind the sequences' positions from first_used on, of normal keys and values."""
    case, lens = s["case"], s["lens"]
    hd, kv, page = case["head_dim"], case["kv_heads"], case["page"]
    used = [(p // page, -(-n // page)) for p, n in zip(first_used, lens)]
    pages = sum(b - a for a, b in used)
    s["pages"] = pages + 2
    order = torch.randperm(pages + 2, generator=gen, device="cuda").to(torch.int32)
    s["table"] = torch.full((case["seqs"], max(b for _, b in used)), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i, (a, b) in enumerate(used):
        s["table"][i, a:b] = order[at:at + b - a]
        at += b - a
    s["layers"] = case.get("layers", 2 if pages * page < 100000 else 1)
    # keys and values of standard deviation about 1, as a normalised projection gives them
    tiles = []
    for _ in range(s["layers"]):
        shape = (pages + 2, kv, page // 32, 32, hd)
        (ck, dk), (cv, dv) = (_quantised(torch.randn(shape, generator=gen, device="cuda")) for _ in range(2))
        tiles.append(_packed_tiles(ck, cv, dk, dv))
    s["pool"] = torch.stack(tiles, 1)


def _probabilities(s, gen):
    """The target's and the draft's probabilities, and tokens taken from the draft's."""
    case, total, width = s["case"], s["total"], s["case"]["width"]
    z = torch.randn(total, case["vocab"], generator=gen, device="cuda") * 3
    s["target"] = torch.softmax(z, 1)
    z += torch.randn(z.shape, generator=gen, device="cuda")
    s["draft"] = torch.softmax(z, 1)
    del z
    if case["mode"] == "chosen":
        picks = s["draft"].topk(width, 1).indices
    else:
        picks = torch.multinomial(s["draft"], width, case["mode"] == "drawn", generator=gen)
    at, rank, first = [], [], 0
    for t in s["trees"]:
        kids = {}
        for p in t:
            at.append(first + max(p, 0))
            rank.append(kids.get(p, 0) % width)
            kids[p] = kids.get(p, 0) + 1
        first += len(t)
    index = torch.tensor([at, rank], device="cuda")
    s["tokens"] = picks[index[0], index[1]].to(torch.int32)
    s["u"] = torch.rand(total, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    def whole(x):
        return torch.tensor(x, device="cuda", dtype=torch.int64).to(torch.int32)

    s = {"case": case}
    if case["kind"] == "softmax":
        x = normal(case["rows"], case["vocab"] + case["pad"])[:, :case["vocab"]] * 3
        if case["kept"] < 1:  # all but the largest logits taken out
            n = max(1, int(case["kept"] * case["vocab"]))
            x = x.masked_fill(x < x.topk(n, 1).values[:, -1:], -math.inf)
        s["x"] = normal(case["rows"], case["vocab"] + case["pad"])
        s["x"][:, :case["vocab"]] = x
        s["out"], s["scale"] = torch.zeros(case["rows"], case["vocab"], device="cuda"), 1.25
        return s
    rows, lens = _sizes(case)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    s.update(rows=rows, lens=lens, total=cu[-1], cu=whole(cu), words=(max(rows) + 31) // 32)
    if case.get("width"):
        s["trees"] = _trees(case, rows)
        s["parent"] = whole([p for t in s["trees"] for p in t])
    if case["kind"] == "verify":
        _probabilities(s, gen)
        s["path"] = whole([0] * s["total"])
        s["n_path"], s["next"] = whole([0] * case["seqs"]), whole([0] * case["seqs"])
        return s
    hd, kv = case["head_dim"], case["kv_heads"]
    s["len"] = whole(lens)
    if case["kind"] == "keep":
        _pool(s, gen, [0] * case["seqs"])
        s["n_path"], path = whole(_kept(case, rows)), []
        for i, (r, n) in enumerate(zip(rows, _kept(case, rows))):
            behind = random.Random(1000 * seed + i).sample(range(n, r), n - 1) if r > n else list(range(1, n))
            path += [0] + sorted(behind) + [-1] * (r - n)
        s["path"] = whole(path)
        return s
    s["q"] = normal(s["total"], case["heads"] * hd)
    if case["kind"] == "attend":
        _pool(s, gen, [0] * case["seqs"])
        s["mask"] = whole([m for t in s["trees"] for m in _masks(t, s["words"])])
        s["out"] = torch.zeros_like(s["q"])
        return s
    _pool(s, gen, [n - r for r, n in zip(rows, lens)])
    s["k"], s["v"] = normal(s["total"], kv * hd), normal(s["total"], kv * hd)
    s["q_out"], s["k_held"], s["v_held"] = (torch.zeros_like(s[x]) for x in ("q", "k", "v"))
    if case["keys_out"]:
        s["k_out"] = torch.zeros_like(s["k"])
    i = torch.arange(case["dims"] // 2, device="cuda", dtype=torch.float64)
    s["freq"] = 10000.0 ** (-2 * i / case["dims"]) / case["stretch"]
    s["scale"] = 1.0 if case["stretch"] == 1 else float(np.float32(0.1 * math.log(case["stretch"]) + 1))
    if "trees" in s:
        s["depth"] = whole([0] * s["total"])
        s["mask"] = whole([[0] * s["words"]] * s["total"])
    return s


# ---- the framework's calls --------------------------------------------------------------

def _own_state(s):
    """The descriptors that a program fills once: of the cache, the batch and the rotation."""
    holo, case = _holo(), s["case"]
    o = {"holo": holo, "lib": holo.lib()}
    if case["kind"] == "softmax":
        return o
    o["batch"] = holo.Batch(rows=s["total"], n_seqs=case["seqs"], max_rows=max(s["rows"]), max_len=max(s["lens"]),
                            cu_rows=s["cu"].data_ptr())
    if case["kind"] != "verify":
        o["cache"] = holo.KV4(pool=s["pool"].data_ptr(), table=s["table"].data_ptr(), len=s["len"].data_ptr(),
                              n_pages=s["pages"], page_len=case["page"], n_layers=s["layers"],
                              n_kv_heads=case["kv_heads"], head_dim=case["head_dim"], n_seqs=case["seqs"],
                              max_pages=s["table"].shape[1])
    if case["kind"] == "turn":
        o["rope"] = holo.Rope(freq=s["freq"].data_ptr(), dims=case["dims"],
                              interleaved=int(case["pairs"] == "interleaved"), scale=s["scale"])
    return o


def _run_own(s):
    if "own" not in s:
        s["own"] = _own_state(s)
    o, case = s["own"], s["case"]
    lib, kind, ref = o["lib"], case["kind"], ctypes.byref
    if kind == "softmax":
        rc = lib.holo_softmax_rows(s["out"].data_ptr(), s["x"].data_ptr(), case["rows"], case["vocab"],
                                   s["out"].stride(0), s["x"].stride(0), s["scale"])
        out = s["out"]
    elif kind == "verify":
        rc = lib.holo_draft_verify(s["path"].data_ptr(), s["n_path"].data_ptr(), s["next"].data_ptr(),
                                   s["target"].data_ptr(), s["draft"].data_ptr(), s["target"].stride(0),
                                   s["draft"].stride(0), case["vocab"], s["tokens"].data_ptr(), s["parent"].data_ptr(),
                                   s["u"].data_ptr(), _MODES.index(case["mode"]), ref(o["batch"]))
        out = {"path": s["path"], "n_path": s["n_path"], "next": s["next"]}
    elif kind == "keep":
        rc = lib.holo_kv4_keep(ref(o["cache"]), s["path"].data_ptr(), s["n_path"].data_ptr(), ref(o["batch"]))
        out = s["pool"].view(torch.int32)
    elif kind == "attend":
        rc = lib.holo_attention_kv4_draft(ref(o["cache"]), s["layers"] - 1, s["out"].data_ptr(), s["q"].data_ptr(),
                                          s["out"].stride(0), s["q"].stride(0), case["heads"], s["mask"].data_ptr(),
                                          s["words"], ref(o["batch"]))
        out = s["out"]
    else:
        dim, rc, depth = case["kv_heads"] * case["head_dim"], 0, None
        out = {"q": s["q_out"], "k": s["k_held"], "v": s["v_held"]}
        if "trees" in s:
            depth, out["depth"], out["mask"] = s["depth"].data_ptr(), s["depth"], s["mask"]
            rc = lib.holo_draft_plan(s["parent"].data_ptr(), depth, s["mask"].data_ptr(), s["words"], ref(o["batch"]))
        if "k_out" in s:
            out["k_out"] = s["k_out"]
        rc = rc or lib.holo_kv4_append_rope(ref(o["cache"]), s["layers"] - 1, ref(o["rope"]), s["q"].data_ptr(),
                                            s["k"].data_ptr(), s["v"].data_ptr(), s["q"].stride(0), dim, dim,
                                            s["q_out"].data_ptr(), s["k_out"].data_ptr() if "k_out" in s else None,
                                            s["q_out"].stride(0), dim, case["heads"], depth, ref(o["batch"]))
        # the values that the cache holds now
        rc = rc or lib.holo_kv4_read(ref(o["cache"]), s["layers"] - 1, s["k_held"].data_ptr(), s["v_held"].data_ptr(),
                                     dim, dim, ref(o["batch"]))
    if rc:
        o["holo"].check(kind)
    return out


# ---- the plain forms ----------------------------------------------------------------------

def _by_sequence(s):
    """Row numbers [n, longest] (the last row's where a sequence has fewer) and which of them are its own."""
    i = torch.arange(max(s["rows"]), device="cuda")
    at = s["cu"][:-1, None].long() + i
    mine = at < s["cu"][1:, None]
    return at.clamp(max=s["total"] - 1), mine


def _plain_attend(s):
    case, (at, mine) = s["case"], _by_sequence(s)
    hd, kv, heads = case["head_dim"], case["kv_heads"], case["heads"]
    n, rows = at.shape
    g = heads // kv
    tiles = s["pool"][s["table"].long().clamp(min=0), s["layers"] - 1]  # n, pages, kv, tiles, bytes
    ck, cv, dk, dv = _unpacked_tiles(tiles, hd)
    k, v = (_values(c, d).movedim(2, 4).flatten(1, 3) for c, d in ((ck, dk), (cv, dv)))
    del tiles, ck, cv, dk, dv
    # the positions before the entry's rows, and those of the rows that the mask names
    t = torch.arange(k.shape[1], device="cuda")
    j = t - (s["len"].long() - (s["cu"][1:] - s["cu"][:-1]).long())[:, None]  # n, positions
    word = s["mask"][at].gather(2, (j.clamp(0, 32 * s["words"] - 1) // 32)[:, None].expand(-1, rows, -1))
    seen = (word >> (j[:, None] % 32).to(torch.int32) & 1).bool() & (j < 32 * s["words"])[:, None]
    seen = (seen | (j < 0)[:, None]) & (t < s["len"][:, None])[:, None]  # n, rows, positions
    q = s["q"][at].view(n, rows, kv, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, g * rows, hd)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    x = (q @ k).div_(math.sqrt(hd)).view(n, kv, g, rows, -1)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    y = (x.flatten(2, 3) @ v).view(n, kv, g, rows, hd) / x.sum(-1, keepdim=True)
    s["out"][at[mine]] = y.permute(0, 3, 1, 2, 4).reshape(n, rows, -1)[mine]
    return s["out"]


def _turned(s, x, pos):
    """x [total, heads * hd] with its pairs turned to the positions, in 64 bits, rounded to 32."""
    case = s["case"]
    x = x.view(s["total"], -1, case["head_dim"]).clone()
    a = pos.double()[:, None, None] * s["freq"]
    c, d = a.cos() * s["scale"], a.sin() * s["scale"]
    dims, half = case["dims"], case["dims"] // 2
    one, two = ((slice(0, dims, 2), slice(1, dims, 2)) if case["pairs"] == "interleaved"
                else (slice(0, half), slice(half, dims)))
    a, b = x[..., one].double(), x[..., two].double()
    x[..., one], x[..., two] = (a * c - b * d).float(), (a * d + b * c).float()
    return x.flatten(1)


def _store(s, layer, rows, seq, pos, ck, dk, cv, dv):
    """The codes and scales [rows, kv, ..] into the tiles of the positions, which are taken apart and put together
    again; what the tiles then hold of them."""
    case = s["case"]
    page, hd = case["page"], case["head_dim"]
    tile = s["table"][seq, pos // page].long() * (page // 32) + pos % page // 32
    touched, which = tile.unique(return_inverse=True)
    where = (touched // (page // 32), layer, slice(None), touched % (page // 32))
    a, b, da, db = _unpacked_tiles(s["pool"][where], hd)  # touched, kv, 32, ..
    a[which, :, pos % 32], b[which, :, pos % 32] = ck[rows], cv[rows]
    da[which, :, pos % 32], db[which, :, pos % 32] = dk[rows], dv[rows]
    s["pool"][where] = _packed_tiles(a, b, da, db)
    return (_values(a[which, :, pos % 32], da[which, :, pos % 32]).flatten(1),
            _values(b[which, :, pos % 32], db[which, :, pos % 32]).flatten(1))


def _plain_turn(s):
    case, (at, mine) = s["case"], _by_sequence(s)
    first = s["len"][:, None].long() - (s["cu"][1:, None] - s["cu"][:-1, None]).long()
    out = {"q": s["q_out"], "k": s["k_held"], "v": s["v_held"]}
    slot = (first + torch.arange(at.shape[1], device="cuda"))[mine]  # where the cache holds the row, rows in order
    pos = slot
    if "trees" in s:
        # level by level: a row's bits are its own and those of the row it follows
        i = torch.arange(at.shape[1], device="cuda").expand(at.shape)[mine]
        up = s["parent"].long()
        over = (s["cu"][:-1, None].expand(at.shape)[mine].long() + up).clamp(min=0)
        bits = torch.zeros_like(s["mask"])
        bits[torch.arange(s["total"], device="cuda"), i // 32] = (1 << i % 32).to(torch.int32)
        mask, depth = bits, torch.zeros_like(up)
        for _ in range(max(max(_depths(t)) for t in s["trees"])):
            mask = bits | torch.where(up[:, None] >= 0, mask[over], 0)
            depth = torch.where(up >= 0, depth[over] + 1, 0)
        s["mask"][:], s["depth"][:] = mask, depth.to(torch.int32)
        out["depth"], out["mask"] = s["depth"], s["mask"]
        pos = first.expand(at.shape)[mine] + depth
    s["q_out"][:] = _turned(s, s["q"], pos)
    k = _turned(s, s["k"], pos)
    if "k_out" in s:
        s["k_out"][:] = k
        out["k_out"] = s["k_out"]
    (ck, dk), (cv, dv) = (_quantised(x.view(s["total"], case["kv_heads"], case["head_dim"])) for x in (k, s["v"]))
    seq = torch.arange(case["seqs"], device="cuda")[:, None].expand(at.shape)[mine]
    s["k_held"][:], s["v_held"][:] = _store(s, s["layers"] - 1, at[mine], seq, slot, ck, dk, cv, dv)
    return out


def _plain_keep(s):
    case, page = s["case"], s["case"]["page"]
    at, mine = _by_sequence(s)
    i = torch.arange(at.shape[1], device="cuda").expand(at.shape)
    go = mine & (i < s["n_path"][:, None])
    first = s["len"][:, None].long() - (s["cu"][1:, None] - s["cu"][:-1, None]).long()
    to, frm = (first + i)[go], (first + s["path"][at].long())[go]
    seq = torch.arange(case["seqs"], device="cuda")[:, None].expand(at.shape)[go]
    rows = torch.arange(len(seq), device="cuda")
    for layer in range(s["layers"]):
        src = s["table"][seq, frm // page].long(), layer, slice(None), frm % page // 32
        parts = _unpacked_tiles(s["pool"][src], case["head_dim"])  # moved, kv, 32, ..
        ck, cv, dk, dv = (x[rows, :, frm % 32] for x in parts)
        _store(s, layer, rows, seq, to, ck, dk, cv, dv)
    return s["pool"].view(torch.int32)


def _plain_softmax(s):
    x = s["x"][:, :s["case"]["vocab"]]
    x = ((x - x.amax(1, keepdim=True)) * s["scale"]).exp()
    s["out"][:] = x / x.sum(1, keepdim=True)
    return s["out"]


def _plain_verify(s):
    case, (at, mine) = s["case"], _by_sequence(s)
    n, rows = at.shape
    seq = torch.arange(n, device="cuda")
    drawn, distinct = case["mode"] != "chosen", case["mode"] == "distinct"
    node = torch.zeros(n, device="cuda", dtype=torch.int64)
    count = torch.ones_like(node)
    one = torch.ones(n, device="cuda", dtype=torch.float64)
    left, beta, gone = one, one * 0, one * 0
    path = torch.full((n, rows + 1), -1, device="cuda", dtype=torch.int64)
    path[:, 0] = 0
    refused = torch.zeros(n, case["vocab"], device="cuda", dtype=torch.bool)
    u = s["u"].double()
    for j in range(1, rows):
        row = at[:, j]
        judged = mine[:, j] & (s["parent"][row] == node)
        here = at[seq, node]
        x = s["tokens"][row].long()
        p = s["target"][here, x].double()
        if drawn:
            q = s["draft"][here, x].double()
            stands = u[row] * q * left < (p - beta * q).clamp(min=0) * (1 - gone)
        else:
            p = torch.where(refused[seq, x], 0, p)
            stands = u[row] * left < p
        stands = stands & judged
        falls = judged & ~stands
        if drawn:
            beta = torch.where(falls, beta + left / (1 - gone), beta)
            w = s["target"][here].double() - beta[:, None] * s["draft"][here]
            left = torch.where(falls, w.clamp(min=0).sum(1), left)
            if distinct:
                gone = torch.where(falls, gone + q, gone)
        else:
            left = torch.where(falls, left - p, left)
            refused[seq, x] |= falls
        path[seq, torch.where(stands, count, rows)] = j
        count = count + stands
        node = torch.where(stands, j, node)
        left, beta, gone = torch.where(stands, 1, left), torch.where(stands, 0, beta), torch.where(stands, 0, gone)
        refused &= ~stands[:, None]
    here = at[seq, node]
    w = s["target"][here].double()
    w = (w - beta[:, None] * s["draft"][here]).clamp(min=0) if drawn else w.masked_fill(refused, 0)
    total = w.cumsum(1)
    x = (total <= (u[at[:, 0]] * total[:, -1])[:, None]).sum(1)
    last = case["vocab"] - 1 - (w.flip(1) > 0).to(torch.int8).argmax(1)
    s["next"][:] = torch.minimum(x, last).to(torch.int32)
    i = torch.arange(rows, device="cuda").expand(n, -1)
    s["path"][at[mine]] = torch.where(i < count[:, None], path[:, :rows], -1)[mine].to(torch.int32)
    s["n_path"][:] = count.to(torch.int32)
    return {"path": s["path"], "n_path": s["n_path"], "next": s["next"]}


_PLAIN = {"turn": _plain_turn, "attend": _plain_attend, "softmax": _plain_softmax, "verify": _plain_verify,
          "keep": _plain_keep}


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


# ---- the same in 64 bits ------------------------------------------------------------------

def _held64(s, i, head, which):
    """[len, hd] in 64 bits of sequence i's keys (which = 0) or values (1), found byte by byte."""
    case = s["case"]
    hd, page, n = case["head_dim"], case["page"], s["lens"][i]
    nb = hd // 32
    p, d = torch.arange(n, device="cuda")[:, None], torch.arange(hd, device="cuda")[None, :]
    pool = s["pool"].reshape(-1)
    base = ((s["table"][i].long()[p // page] * s["layers"] + s["layers"] - 1) * case["kv_heads"] + head)
    base = (base * (page // 32) + p % page // 32) * (36 * hd)
    p, b = p % 32, d // 32
    if which == 0:
        w, slot = d // 8, d % 8
        word = ((p // 16 * 4 + w // nb) * 16 + p % 16) * nb + w % nb
        scale = 32 * hd + 2 * (b * 32 + p % 16 * 2 + p // 16)
    else:
        vw = 4 if nb % 2 == 0 else 2
        g, slot, m = p % 16 // 4, p // 16 * 4 + p % 4, d // 16
        word = 4 * hd + ((m // vw * 4 + g) * 16 + d % 16) * vw + m % vw
        scale = 34 * hd + 2 * (b * 32 + g * 8 + slot)
    nibble = slot // 2 + 4 * (slot % 2)
    code = (pool[base + 4 * word + nibble // 2].int() >> (4 * (nibble % 2))) & 15
    bits = pool[base + scale].int() | (pool[base + scale + 1].int() << 8)
    return (code.double() - 8) * bits.to(torch.int16).view(torch.float16).double()


def _exact_attend(s):
    case = s["case"]
    hd, kv, at = case["head_dim"], case["kv_heads"], s["cu"].tolist()
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    group = case["heads"] // kv
    for i, tree in enumerate(s["trees"]):
        a, b, n, rows = at[i], at[i + 1], s["lens"][i], len(tree)
        seen = torch.ones(rows, n, dtype=torch.bool)
        seen[:, n - rows:] = False
        for r in range(rows):  # the row, what it follows, and so on
            j = r
            while j >= 0:
                seen[r, n - rows + j] = True
                j = tree[j]
        seen = seen.cuda()
        for j in range(kv):
            k, v = _held64(s, i, j, 0), _held64(s, i, j, 1)
            for h in range(j * group, (j + 1) * group):
                x = s["q"][a:b, h * hd:(h + 1) * hd].double() @ k.t() / math.sqrt(hd)
                out[a:b, h * hd:(h + 1) * hd] = torch.softmax(x.masked_fill_(~seen, -math.inf), 1) @ v
    return out


def _rounded64(x):
    """What the cache holds of x [total, kv * hd]."""
    b = x.double().view(len(x), -1, 32)
    m = b.gather(2, b.abs().argmax(2, keepdim=True))
    m = torch.where((b == -m.abs()).any(2, keepdim=True), -m.abs(), m)
    d = (-m / 8).to(torch.bfloat16).clamp(-2720, 2720).half().double()
    return (torch.round(b / d).clamp(-8, 7) * d).nan_to_num(0.0).view(len(x), -1)


def _exact_turn(s):
    case = s["case"]
    hd, dims = case["head_dim"], case["dims"]
    trees = s["trees"] if "trees" in s else [list(range(-1, r - 1)) for r in s["rows"]]
    depth = [d for t in trees for d in _depths(t)]
    pos = np.repeat(np.array(s["lens"]) - np.array(s["rows"]), s["rows"]) + np.array(depth)
    turn = np.exp(1j * pos[:, None] * s["freq"].cpu().numpy()) * s["scale"]  # pairs as complex numbers

    def turned(x):
        x = x.cpu().numpy().astype(np.float64).reshape(s["total"], -1, hd)
        i = np.arange(dims // 2)
        one, two = (2 * i, 2 * i + 1) if case["pairs"] == "interleaved" else (i, i + dims // 2)
        z = (x[..., one] + 1j * x[..., two]) * turn[:, None]
        x[..., one], x[..., two] = z.real, z.imag
        return torch.from_numpy(x.reshape(s["total"], -1)).cuda()

    k = turned(s["k"])
    out = {"q": turned(s["q"]), "k": _rounded64(k.float()), "v": _rounded64(s["v"])}
    if "trees" in s:
        out["depth"] = torch.tensor(depth)
        out["mask"] = torch.tensor([m for t in trees for m in _masks(t, s["words"])]).to(torch.int32)
    if "k_out" in s:
        out["k_out"] = k
    return out


def _exact_verify(s):
    case, at = s["case"], s["cu"].tolist()
    path, n_path, following = [], [], []
    tokens, u = s["tokens"].tolist(), s["u"].double().tolist()
    for i, tree in enumerate(s["trees"]):
        node, stood, first = 0, [0], at[i]

        def weights():
            p, q = (s[x][first + node].double().cpu().numpy() for x in ("target", "draft"))
            return p, q

        (p, q), left, beta, gone = weights(), 1.0, 0.0, 0.0
        r = p.copy()
        for j in range(1, len(tree)):
            if tree[j] != node:
                continue
            x = tokens[first + j]
            if case["mode"] == "chosen":
                stands = u[first + j] * left < r[x]
            else:
                stands = u[first + j] * q[x] * left < max(p[x] - beta * q[x], 0.0) * (1 - gone)
            if stands:
                node = j
                stood.append(j)
                (p, q), left, beta, gone = weights(), 1.0, 0.0, 0.0
                r = p.copy()
            elif case["mode"] == "chosen":
                left -= r[x]
                r[x] = 0
            else:
                beta += left / (1 - gone)
                r = np.maximum(p - beta * q, 0)
                left = r.sum()
                gone += q[x] if case["mode"] == "distinct" else 0.0
        sums = np.cumsum(r)
        x = int(np.searchsorted(sums, u[first] * sums[-1], side="right"))
        following.append(min(x, int(np.flatnonzero(r)[-1])))
        path += stood + [-1] * (len(tree) - len(stood))
        n_path.append(len(stood))
    return {"path": torch.tensor(path), "n_path": torch.tensor(n_path), "next": torch.tensor(following)}


def exact(case, seed):
    if case["kind"] == "keep":
        return None
    s = prepare(case, seed)
    if case["kind"] == "softmax":
        x = s["x"][:, :case["vocab"]].double()
        return torch.softmax((x - x.amax(1, keepdim=True)) * s["scale"], 1)
    return {"turn": _exact_turn, "attend": _exact_attend, "verify": _exact_verify}[case["kind"]](s)
