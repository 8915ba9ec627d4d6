"""Attention over the 4-bit cache where its smaller paths are at work: scales
below f16's normal numbers, a chunk among single tokens at far positions, and
partial sums past what the scratch arena holds, eager and captured.

Tolerance 1e-5 normwise, as for the other shapes: a cached value d c is an
exact f16 with a subnormal d too (d has at most 8 significant bits, c three)."""
import numpy as np
import pytest

from kv4_model import Batch, Cache, OnDevice, normwise, quantise, want_attention
from test_gpu_kv4 import TOL, attention, fill, pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("scale", [2e-5, 1e-6, 2e-7])
def test_scales_below_the_normal_numbers(holo, hd, scale):
    """Keys and values so small that their scales are f16 subnormals; q large enough that the
    scores differ, and of ordinary size."""
    print(f"case kv4 subnormal scales hd {hd} {scale}", flush=True)
    rng = np.random.default_rng(hd)
    heads, n_kv, lens, rows = 4, 2, [70, 300], [3, 1]
    d = quantise((scale * rng.standard_normal((50, hd))).astype(np.float32))[1]
    assert (np.abs(d.astype(np.float64)) < 2.0 ** -14).all() and (d != 0).any()
    c = Cache(hd, 32, 1, n_kv, 14, 2, 10)
    pages(c, lens, rng)
    fill(c, rng, lens, 0, scale)
    dev = OnDevice(holo, c)
    for size in (1.0, 1 / scale):
        q = (size * rng.standard_normal((4, heads * hd))).astype(np.float32)
        got = attention(holo, dev, 0, q, rows, heads)
        assert normwise(got, want_attention(c, 0, q, rows, c.len, [0, 1], heads)) <= TOL


def test_a_chunk_among_single_tokens(holo):
    """One entry of many rows beside single tokens of long sequences, in one call and by themselves."""
    print("case kv4 mixed batch", flush=True)
    rng = np.random.default_rng(21)
    hd, heads, n_kv = 64, 8, 2
    lens, rows = [1700, 400, 900, 33], [1, 150, 1, 1]
    c = Cache(hd, 64, 1, n_kv, sum(-(-n // 64) for n in lens), 4, 27)
    pages(c, lens, rng)
    fill(c, rng, lens, 0)
    dev = OnDevice(holo, c)
    q = rng.standard_normal((sum(rows), heads * hd)).astype(np.float32)
    want, at = want_attention(c, 0, q, rows, c.len, [0, 1, 2, 3], heads), 0
    for bound in (1700, 100000):
        got = attention(holo, dev, 0, q, rows, heads, max_len=bound)
        assert normwise(got, want) <= TOL
    for s, n in enumerate(rows):
        assert normwise(got[at:at + n], want[at:at + n]) <= TOL
        alone = attention(holo, dev, 0, q[at:at + n], [n], heads, seqs=[s])
        assert normwise(alone, want[at:at + n]) <= TOL
        at += n


@pytest.mark.parametrize("heads", [2, 4, 16])
def test_partial_sums_past_the_arena(holo, heads):
    """Under a far bound on the lengths two entries have 256 ranges each: 0.5 MiB of partial sums with 2
    heads a KV head of 128, 1.03 with 4, 4.1 with 16.  Eager, and captured on two streams at once, whose
    replays follow the lengths, with eager calls between them."""
    print(f"case kv4 partial sums heads {heads}", flush=True)
    rng = np.random.default_rng(heads)
    lib = holo.lib()
    hd, n_kv, bound = 128, 1, 200000
    assert 2 * heads * 256 * (hd + 4) * 4 > 1 << 19
    sides = []
    before = lib.holo_get_stream()
    streams = [lib.holo_stream_create(), lib.holo_stream_create()]
    try:
        for side in range(2):
            c = Cache(hd, 64, 1, n_kv, 30, 2, 16)
            pages(c, [900, 600], rng)
            fill(c, rng, [900, 600], 0)
            dev = OnDevice(holo, c)
            b = Batch(holo, [1, 1], None, None, bound)
            dq, do = (holo.DeviceBuffer(2 * heads * hd * 4) for _ in range(2))
            lib.holo_set_stream(streams[side])
            assert lib.holo_graph_begin() == 0
            rc = lib.holo_attention_kv4(dev.ref, 0, do.ptr, dq.ptr, heads * hd, heads * hd, heads, b.ref)
            graph = lib.holo_graph_end()
            assert rc == 0 and graph
            holo.check("capture")
            sides.append((c, dev, b, dq, do, graph))
        for lens in ([900, 600], [899, 37], [520, 255], [900, 1]):
            wants = []
            for side, (c, dev, b, dq, do, graph) in enumerate(sides):
                lib.holo_set_stream(streams[side])
                c.len[:] = lens
                dev.refresh()
                q = rng.standard_normal((2, heads * hd)).astype(np.float32)
                dq.upload(q)
                wants.append((q, want_attention(c, 0, q, [1, 1], c.len, [0, 1], heads)))
            lib.cuda_sync()
            for _ in range(2):  # both under way at once, twice
                for side in range(2):
                    lib.holo_set_stream(streams[side])
                    assert lib.holo_graph_launch(sides[side][5]) == 0
            for side in range(2):
                lib.holo_set_stream(streams[side])
                lib.cuda_sync()
            holo.check("replay")
            for side, ((c, dev, b, dq, do, graph), (q, want)) in enumerate(zip(sides, wants)):
                got = do.download(np.float32).reshape(2, -1)
                assert normwise(got, want) <= TOL
                lib.holo_set_stream(streams[side])
                assert np.array_equal(got, attention(holo, dev, 0, q, [1, 1], heads, max_len=bound))
    finally:
        for *_, graph in sides:
            lib.holo_graph_destroy(graph)
        lib.holo_set_stream(before)
        for s in streams:
            lib.holo_stream_destroy(s)
