"""The operators of several sequences together, as a program that serves them
runs them: prompts packed in one call, their keys and values into 4-bit pages,
a conversation forked, decode steps and a chunk over the pages, sequences
ended and the cache compacted.  After every call the outputs are compared with
float64 numpy on the values that a plain model of the cache holds."""
import ctypes as C

import numpy as np
import pytest

from kv4_model import Batch, Cache, OnDevice, attend, normwise, quantise, values

pytestmark = pytest.mark.gpu

TOL = 1e-5  # test_gpu_kv4.py


def ints(x):
    return (C.c_int * max(len(x), 1))(*x)


@pytest.mark.parametrize("hd,heads,n_kv,page_len", [(64, 8, 2, 32), (128, 4, 4, 64)])
def test_serving(holo, hd, heads, n_kv, page_len):
    print(f"case serving hd {hd} heads {heads}/{n_kv} page {page_len}", flush=True)
    rng = np.random.default_rng(hd)
    lib, layers, n_seqs = holo.lib(), 2, 5
    c = Cache(hd, page_len, layers, n_kv, 24, n_seqs, 8)
    dev = OnDevice(holo, c)
    pages = lib.holo_kv4_pages_create(dev.ref)
    assert pages
    q_dim, kv_dim = heads * hd, n_kv * hd
    up = holo.DeviceBuffer.from_array
    # by sequence and layer: the fp32 rows appended so far
    rows_of = {(s, l): [np.zeros((0, kv_dim), np.float32)] * 2 for s in range(n_seqs) for l in range(layers)}

    def held(s, l):
        return [values(*quantise(x)).reshape(-1, n_kv, hd) for x in rows_of[s, l]]

    def heads_of(q, ks, vs, seen):
        return np.concatenate([attend(q[h * hd:(h + 1) * hd], ks[:, h * n_kv // heads], vs[:, h * n_kv // heads], seen)
                               for h in range(heads)])

    def call(seqs, rows, packed=False):
        """One step of the sequences: q, k and v of their new rows, side by side."""
        assert lib.holo_kv4_pages_reserve(pages, ints(seqs), ints(rows), len(seqs)) == 0
        ld = q_dim + 2 * kv_dim
        longest = max(lib.holo_kv4_pages_len(pages, s) for s in seqs)
        b = Batch(holo, rows, seqs, None, longest)
        for layer in range(layers):
            qkv = rng.standard_normal((sum(rows), ld)).astype(np.float32)
            q, k, v = qkv[:, :q_dim], qkv[:, q_dim:q_dim + kv_dim], qkv[:, q_dim + kv_dim:]
            d, out = up(qkv), holo.DeviceBuffer(4 * sum(rows) * q_dim)
            dq, dk, dv = d.ptr, d.ptr + 4 * q_dim, d.ptr + 4 * (q_dim + kv_dim)
            assert lib.holo_kv4_append(dev.ref, layer, dk, dv, ld, ld, b.ref) == 0
            if packed:
                assert lib.holo_attention_packed(out.ptr, dq, dk, dv, q_dim, ld, ld, ld, hd, heads, n_kv, b.ref) == 0
            else:
                assert lib.holo_attention_kv4(dev.ref, layer, out.ptr, dq, q_dim, ld, heads, b.ref) == 0
            lib.cuda_sync()
            holo.check("serving step")
            want, at = np.zeros((sum(rows), q_dim)), 0
            for s, n in zip(seqs, rows):
                new = k[at:at + n], v[at:at + n]
                old = rows_of[s, layer][0].shape[0]
                rows_of[s, layer] = [np.concatenate((a, x)) for a, x in zip(rows_of[s, layer], new)]
                if packed:
                    ks, vs = (x.astype(np.float64).reshape(n, n_kv, hd) for x in new)
                else:
                    ks, vs = held(s, layer)
                for i in range(n):
                    seen = np.arange(len(ks)) <= (i if packed else old + i)
                    want[at + i] = heads_of(q[at + i], ks, vs, seen)
                at += n
            assert normwise(out.download(np.float32).reshape(want.shape), want) <= TOL

    def check_cache():
        """What the pages hold, of every sequence and layer."""
        for s in range(n_seqs):
            n = lib.holo_kv4_pages_len(pages, s)
            assert n == rows_of[s, 0][0].shape[0]
            if not n:
                continue
            b = Batch(holo, [n], [s])
            for layer in range(layers):
                k, v = holo.DeviceBuffer(4 * n * kv_dim), holo.DeviceBuffer(4 * n * kv_dim)
                assert lib.holo_kv4_read(dev.ref, layer, k.ptr, v.ptr, kv_dim, kv_dim, b.ref) == 0
                lib.cuda_sync()
                for got, x in zip((k, v), rows_of[s, layer]):
                    assert np.array_equal(got.download(np.float32).reshape(n, kv_dim), values(*quantise(x)))

    call([0, 3, 1], [45, 1, 70], packed=True)  # the prompts
    check_cache()
    call([0, 1, 3], [1, 1, 1])                 # a decode step
    assert lib.holo_kv4_pages_fork(pages, ints([0, 0]), ints([2, 4]), 2) == 0
    for s in (2, 4):
        for l in range(layers):
            rows_of[s, l] = list(rows_of[0, l])
    check_cache()
    call([4, 0, 2], [1, 1, 1])                 # three ways on from the same rows
    call([2, 1], [37, 5])                      # chunks
    check_cache()
    assert lib.holo_kv4_pages_free(pages, ints([0, 3]), 2) == 0
    for s in (0, 3):
        for l in range(layers):
            rows_of[s, l] = [x[:0] for x in rows_of[s, l]]
    assert lib.holo_kv4_pages_compact(pages) == 0
    used = c.n_pages - lib.holo_kv4_pages_available(pages)
    for s in range(n_seqs):
        got = ints([0] * 8)
        n = lib.holo_kv4_pages_list(pages, s, got, 8)
        assert all(0 <= x < used for x in list(got)[:n])
    check_cache()
    call([1, 4, 3], [1, 1, 20])
    check_cache()
    holo.check("serving")
    # no changes of the tables inside a capture
    before, st = lib.holo_get_stream(), lib.holo_stream_create()
    lib.holo_set_stream(st)
    assert lib.holo_graph_begin() == 0
    assert lib.holo_kv4_pages_reserve(pages, ints([0]), ints([1]), 1) == holo.EINVAL
    assert lib.holo_kv4_pages_compact(pages) == holo.EINVAL and lib.holo_kv4_pages_create(dev.ref) is None
    graph = lib.holo_graph_end()
    lib.holo_graph_destroy(graph)
    lib.holo_set_stream(before)
    lib.holo_stream_destroy(st)
    assert lib.holo_last_error() == holo.EINVAL
    lib.holo_kv4_pages_destroy(pages)
