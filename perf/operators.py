"""The operators of decoding several sequences at once, as measurable cases.

A program that serves more than one conversation keeps their keys and values in
a cache of fixed-size pages, four bits a value, and runs these calls:

  packed  holo_attention_packed: the prompts of several sequences, their rows
          one behind the other, each attending to its own rows before it
  store   holo_kv4_append and holo_kv4_read: the rows' keys and values into the
          pages of their sequences, and back as the values that the cache holds
  attend  holo_attention_kv4: the last rows of every sequence (one in a decode
          step, a few to many in a chunk of a prompt) over its pages
  copy    holo_kv4_copy_pages: pages copied before a shared one is written to,
          and when the used pages of a cache are moved together

A page holds, for every layer and KV head, tiles of 32 positions of 36 * hd
bytes.  With nb = hd / 32 blocks of 32 dims and lane = 16 g + r, g < 4, r < 16:

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
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _holo():
    path = os.path.join(_ROOT, "google-classic_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import holo_mi355x as holo
    holo.init()
    return holo


def listed():
    return [
        # a decode step of a busy server: one new row of each conversation
        {"name": "store_32x1", "kind": "store", "seqs": 32, "rows": 1, "spread": 0.0, "before": 701, "kv_heads": 8,
         "head_dim": 128, "page": 64},
        # four prompts of a batch, the longest 1000 rows, behind a shared start that ends inside a tile
        {"name": "store_4x1000", "kind": "store", "seqs": 4, "rows": 1000, "spread": 0.8, "before": 77,
         "kv_heads": 8, "head_dim": 128, "page": 128},
        # one short conversation, every query head with keys of its own: where latency counts
        {"name": "attend_1x1_at_512", "kind": "attend", "seqs": 1, "rows": 1, "len": 513, "spread": 0.0, "heads": 32,
         "kv_heads": 32, "head_dim": 128, "page": 64},
        # a decode step over conversations of all lengths, grouped-query heads
        {"name": "attend_16x1_to_4096", "kind": "attend", "seqs": 16, "rows": 1, "len": 4096, "spread": 0.95,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64},
        # one very long document in the cache
        {"name": "attend_1x1_at_100000", "kind": "attend", "seqs": 1, "rows": 1, "len": 100001, "spread": 0.0,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 256},
        # a decode step of a full server
        {"name": "attend_64x1_to_8192", "kind": "attend", "seqs": 64, "rows": 1, "len": 8192, "spread": 0.5,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 128},
        # follow-up messages of four conversations, as chunks over what the cache holds
        {"name": "attend_4x100_at_2000", "kind": "attend", "seqs": 4, "rows": 100, "len": 2100, "spread": 0.5,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64},
        # a handful of short questions in one batch
        {"name": "packed_6x40", "kind": "packed", "seqs": 6, "rows": 40, "spread": 0.9, "heads": 32, "kv_heads": 32,
         "head_dim": 128, "fused": False},
        # prompts of a batch, q, k and v side by side in one buffer
        {"name": "packed_4x1023_fused", "kind": "packed", "seqs": 4, "rows": 1023, "spread": 0.7, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "fused": True},
        # a long document beside nothing else
        {"name": "packed_1x4096", "kind": "packed", "seqs": 1, "rows": 4096, "spread": 0.0, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "fused": False},
        # the last pages of two forked conversations before their next rows
        {"name": "copy_2", "kind": "copy", "pages": 2, "page": 64, "kv_heads": 8, "head_dim": 128, "layers": 8},
        # a cache compacted after many conversations ended
        {"name": "copy_300", "kind": "copy", "pages": 300, "page": 64, "kv_heads": 8, "head_dim": 128, "layers": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("store", "attend", "attend", "attend", "packed", "packed", "copy"))
    hd = rng.choice((32, 64, 64, 96, 128, 128, 128))
    heads = rng.choice((4, 8, 16, 24, 32, 40))
    kv_heads = heads // rng.choice((1, 2, 4))
    page = rng.choice((32, 64, 128, 256))
    spread = rng.choice((0.0, rng.uniform(0.1, 0.95)))
    if kind == "copy":
        layers, pages = _log(rng, 1, 32), _log(rng, 1, 600)
        size = layers * kv_heads * (page // 32) * 36 * hd
        return {"kind": kind, "pages": max(1, min(pages, 300 * 32 * 8 * 2 * 36 * 128 // size)), "page": page,
                "kv_heads": kv_heads, "head_dim": hd, "layers": layers}
    seqs = _log(rng, 1, 64)
    if kind == "store":
        rows = rng.choice((1, _log(rng, 2, 2000)))
        return {"kind": kind, "seqs": seqs, "rows": max(1, min(rows, 8000 // seqs)), "spread": spread,
                "before": _log(rng, 1, 1000) - 1, "kv_heads": kv_heads, "head_dim": hd, "page": page}
    if kind == "attend":
        length = _log(rng, 1, 60000)
        length = max(1, min(length, 64 * 8 * 128 * 6000 // (seqs * kv_heads * hd)))
        rows = rng.choice((1, 1, _log(rng, 2, 300)))
        rows = max(1, min(rows, length, 4096 * 2048 // (seqs * length)))
        return {"kind": kind, "seqs": seqs, "rows": rows, "len": length, "spread": spread, "heads": heads,
                "kv_heads": kv_heads, "head_dim": hd, "page": page}
    rows = _log(rng, 1, 4096)
    most = math.sqrt(4096 * 4096 * 32 * 128 / (seqs * max(heads, 32) * 128))
    return {"kind": kind, "seqs": seqs, "rows": max(1, min(rows, int(most))), "spread": spread, "heads": heads,
            "kv_heads": kv_heads, "head_dim": hd, "fused": rng.random() < 0.5}


# ---- sizes -------------------------------------------------------------------------

def _shrunk(longest, spread, n):
    """n whole numbers from `longest` down to (1 - spread) of it."""
    return [max(1, int(longest * (1 - spread * i / max(1, n - 1)))) for i in range(n)]


def _sizes(case):
    """Rows of the call and positions of the cache (these rows among them), by sequence."""
    rows = _shrunk(case["rows"], case["spread"], case["seqs"])
    if case["kind"] == "store":
        return rows, [case["before"] + r for r in rows]
    if case["kind"] == "packed":
        return rows, rows
    lens = _shrunk(case["len"], case["spread"], case["seqs"])
    return [min(case["rows"], n) for n in lens], lens


def work(case):
    hd, kv = case["head_dim"], case["kv_heads"]
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pages"] * case["layers"] * kv * (case["page"] // 32) * 36 * hd, "flops": 0}
    rows, lens = _sizes(case)
    row4 = kv * hd * 36 // 32  # a position's keys and values in the cache
    if case["kind"] == "store":
        return {"bytes": sum(rows) * (16 * kv * hd + 2 * row4), "flops": sum(rows) * kv * hd * 8}
    pairs = sum(r * (n - r) + r * (r + 1) // 2 for r, n in zip(rows, lens))
    qo = 8 * sum(rows) * case["heads"] * hd
    cache = sum(lens) * row4 if case["kind"] == "attend" else sum(rows) * 8 * kv * hd
    return {"bytes": cache + qo, "flops": 4 * pairs * case["heads"] * hd}


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

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    hd, kv = case["head_dim"], case["kv_heads"]
    s = {"case": case}
    if case["kind"] == "copy":
        size = case["layers"] * kv * (case["page"] // 32) * 36 * hd
        n = case["pages"]
        s["pool"] = torch.randint(-2 ** 31, 2 ** 31, (2 * n + 3, size // 4), generator=gen, device="cuda",
                                  dtype=torch.int64).to(torch.int32)
        order = torch.randperm(2 * n + 3, generator=gen, device="cuda")
        s["src"], s["dst"] = order[:n].tolist(), order[n:2 * n].tolist()
        return s
    rows, lens = _sizes(case)
    n, total = case["seqs"], sum(rows)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    s.update(rows=rows, lens=lens, total=total)
    s["cu"] = torch.tensor(cu, device="cuda", dtype=torch.int32)
    s["len"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
    if case["kind"] != "store":
        q_dim = case["heads"] * hd
        s["out"] = torch.zeros(total, q_dim, device="cuda")
    if case["kind"] == "packed":
        if case["fused"]:
            qkv = normal(total, q_dim + 2 * kv * hd)
            s["q"], s["k"], s["v"] = qkv.split((q_dim, kv * hd, kv * hd), 1)
        else:
            s["q"], s["k"], s["v"] = normal(total, q_dim), normal(total, kv * hd), normal(total, kv * hd)
        return s
    # pages in random order, of a two-layer model where they are few
    page, most = case["page"], -(-max(lens) // case["page"])
    pages = sum(-(-x // page) for x in lens)
    s["layers"], s["pages"] = 2 if pages * page < 100000 else 1, pages + 2
    order = torch.randperm(pages + 2, generator=gen, device="cuda").to(torch.int32)
    s["table"] = torch.full((n, most), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i, x in enumerate(lens):
        k = -(-x // page)
        s["table"][i, :k] = order[at:at + k]
        at += k
    # keys and values of standard deviation about 1, as a normalised projection gives them
    tiles = (pages + 2, s["layers"], kv, page // 32, 32, hd)
    (ck, dk), (cv, dv) = _quantised(normal(*tiles)), _quantised(normal(*tiles))
    s["pool"] = _packed_tiles(ck, cv, dk, dv)
    if case["kind"] == "store":
        s["k"], s["v"] = normal(total, kv * hd), normal(total, kv * hd)
        s["k_held"], s["v_held"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
    else:
        s["q"] = normal(total, case["heads"] * hd)
    return s


# ---- the framework's calls --------------------------------------------------------------

def _own_state(s):
    """The descriptors that a program fills once: of the cache, and of the batch."""
    holo, case = _holo(), s["case"]
    o = {"holo": holo, "lib": holo.lib()}
    if case["kind"] == "copy":
        o["cache"] = holo.KV4(pool=s["pool"].data_ptr(), n_pages=s["pool"].shape[0], page_len=case["page"],
                              n_layers=case["layers"], n_kv_heads=case["kv_heads"], head_dim=case["head_dim"])
        n = case["pages"]
        o["src"], o["dst"] = (ctypes.c_int * n)(*s["src"]), (ctypes.c_int * n)(*s["dst"])
        return o
    o["batch"] = holo.Batch(rows=s["total"], n_seqs=case["seqs"], max_rows=max(s["rows"]), max_len=max(s["lens"]),
                            cu_rows=s["cu"].data_ptr())
    if case["kind"] != "packed":
        o["cache"] = holo.KV4(pool=s["pool"].data_ptr(), table=s["table"].data_ptr(), len=s["len"].data_ptr(),
                              n_pages=s["pages"], page_len=case["page"], n_layers=s["layers"],
                              n_kv_heads=case["kv_heads"], head_dim=case["head_dim"], n_seqs=case["seqs"],
                              max_pages=s["table"].shape[1])
    return o


def _run_own(s):
    if "own" not in s:
        s["own"] = _own_state(s)
    o, case = s["own"], s["case"]
    lib, kind, ref = o["lib"], case["kind"], ctypes.byref
    if kind == "copy":
        rc = lib.holo_kv4_copy_pages(ref(o["cache"]), o["src"], o["dst"], case["pages"])
        out = s["pool"]
    elif kind == "store":
        dim = case["kv_heads"] * case["head_dim"]
        rc = lib.holo_kv4_append(ref(o["cache"]), s["layers"] - 1, s["k"].data_ptr(), s["v"].data_ptr(), dim, dim,
                                 ref(o["batch"]))
        rc = rc or lib.holo_kv4_read(ref(o["cache"]), s["layers"] - 1, s["k_held"].data_ptr(), s["v_held"].data_ptr(),
                                     dim, dim, ref(o["batch"]))
        out = {"k": s["k_held"], "v": s["v_held"]}
    elif kind == "attend":
        rc = lib.holo_attention_kv4(ref(o["cache"]), s["layers"] - 1, s["out"].data_ptr(), s["q"].data_ptr(),
                                    s["out"].stride(0), s["q"].stride(0), case["heads"], ref(o["batch"]))
        out = s["out"]
    else:
        rc = lib.holo_attention_packed(s["out"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                                       s["out"].stride(0), s["q"].stride(0), s["k"].stride(0), s["v"].stride(0),
                                       case["head_dim"], case["heads"], case["kv_heads"], ref(o["batch"]))
        out = s["out"]
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


def _attention(q, k, v, pos, heads, kv_heads):
    """softmax(q k / sqrt(hd)) v of q [n, R, H hd] at positions pos [n, R] over k, v [n, T, KV, hd], t <= pos."""
    n, rows = pos.shape
    hd, g = k.shape[-1], heads // kv_heads
    q = q.view(n, rows, kv_heads, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, g * rows, hd)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    x = (q @ k).div_(math.sqrt(hd)).view(n, kv_heads, g, rows, -1)
    x.masked_fill_(torch.arange(k.shape[-1], device="cuda") > pos[:, None, None, :, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    out = (x.flatten(2, 3) @ v).view(n, kv_heads, g, rows, hd) / total
    return out.permute(0, 3, 1, 2, 4).reshape(n, rows, -1)


def _run_plain(s):
    case = s["case"]
    hd, kv = case["head_dim"], case["kv_heads"]
    if case["kind"] == "copy":
        s["pool"][s["dst"]] = s["pool"][s["src"]]
        return s["pool"]
    at, mine = _by_sequence(s)
    if case["kind"] == "packed":
        k, v = (s[x][at].view(*at.shape, kv, hd) for x in ("k", "v"))
        pos = torch.arange(at.shape[1], device="cuda").expand(at.shape)
        y = _attention(s["q"][at], k, v, pos, case["heads"], kv)
        s["out"][at[mine]] = y[mine]
        return s["out"]
    layer, page = s["layers"] - 1, case["page"]
    first = s["len"][:, None].long() - (s["cu"][1:, None] - s["cu"][:-1, None]).long()
    pos = first + torch.arange(at.shape[1], device="cuda")
    if case["kind"] == "attend":
        tiles = s["pool"][s["table"].long().clamp(min=0), layer]  # n, pages, kv, tiles, bytes
        ck, cv, dk, dv = _unpacked_tiles(tiles, hd)
        k, v = (_values(c, d).movedim(2, 4).flatten(1, 3) for c, d in ((ck, dk), (cv, dv)))
        y = _attention(s["q"][at], k, v, pos, case["heads"], kv)
        s["out"][at[mine]] = y[mine]
        return s["out"]
    # store: the tiles that the rows touch are taken apart, written and put together again
    (ck, dk), (cv, dv) = (_quantised(s[x].view(-1, kv, hd)) for x in ("k", "v"))
    rows = at[mine]
    pos = pos[mine]
    seq = torch.arange(case["seqs"], device="cuda")[:, None].expand(at.shape)[mine]
    tile = s["table"][seq, pos // page].long() * (page // 32) + pos % page // 32
    touched, which = tile.unique(return_inverse=True)
    where = (touched // (page // 32), layer, slice(None), touched % (page // 32))
    a, b, da, db = _unpacked_tiles(s["pool"][where], hd)  # touched, kv, 32, ..
    a[which, :, pos % 32], b[which, :, pos % 32] = ck[rows], cv[rows]
    da[which, :, pos % 32], db[which, :, pos % 32] = dk[rows], dv[rows]
    s["pool"][where] = _packed_tiles(a, b, da, db)
    s["k_held"][rows] = _values(a[which, :, pos % 32], da[which, :, pos % 32]).flatten(1)
    s["v_held"][rows] = _values(b[which, :, pos % 32], db[which, :, pos % 32]).flatten(1)
    return {"k": s["k_held"], "v": s["v_held"]}


def run(s):
    return _run_own(s) if own else _run_plain(s)


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


def _softmax64(q, k, v, first):
    """Rows of q at positions first, first + 1, ... over k and v."""
    x = q @ k.t() / math.sqrt(q.shape[1])
    hidden = torch.arange(k.shape[0], device="cuda") > first + torch.arange(q.shape[0], device="cuda")[:, None]
    return torch.softmax(x.masked_fill_(hidden, -math.inf), 1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        return None
    hd, kv = case["head_dim"], case["kv_heads"]
    if case["kind"] == "store":
        out = {}
        for x in ("k", "v"):
            b = s[x].double().view(s["total"], -1, 32)
            m = b.gather(2, b.abs().argmax(2, keepdim=True))
            m = torch.where((b == -m.abs()).any(2, keepdim=True), -m.abs(), m)
            d = (-m / 8).to(torch.bfloat16).clamp(-2720, 2720).half().double()
            out[x] = (torch.round(b / d).clamp(-8, 7) * d).nan_to_num(0.0).view(s["total"], -1)
        return out
    q, out = s["q"].double(), torch.empty(s["total"], case["heads"] * hd, device="cuda", dtype=torch.float64)
    group, at = case["heads"] // kv, s["cu"].tolist()
    for i in range(case["seqs"]):
        a, b = at[i], at[i + 1]
        for j in range(kv):
            if case["kind"] == "attend":
                k, v = _held64(s, i, j, 0), _held64(s, i, j, 1)
            else:
                k, v = (s[x][a:b, j * hd:(j + 1) * hd].double() for x in ("k", "v"))
            for h in range(j * group, (j + 1) * group):
                out[a:b, h * hd:(h + 1) * hd] = _softmax64(q[a:b, h * hd:(h + 1) * hd], k, v, s["lens"][i] - (b - a))
    return out
