// kv4.h -- the 4-bit cache's pages as the kernels see them (holo_kv4_t of
// holo_forward.h).
//
// A tile is 32 positions of one layer and KV head, 36 * hd bytes: K codes, V
// codes, K scales, V scales.  Its words lie in the order in which the lanes of
// v_mfma_f32_16x16x32_f16 take them (lane = 16 g + r), so a wave's loads are
// whole lines and nothing crosses lanes:
//   K  [half][lane][NB]: position 16 half + r (the A row r), dims 8 w .. + 7 with
//      w = NB g + j, the slots of lane group g in step j;
//   V  [chunk][lane][VW]: dim 16 m + r (the A row r of V^T), m = VW chunk + j, and
//      the 8 positions 4 g .. + 3, 16 + 4 g .. + 3: those whose scores lane group g
//      holds after the first product, so that the probabilities are the second
//      one's B operand as they stand;
//   scales: K [block][r][half], V [block][g][8], f16.
// Value i of a word is nibble i / 2 + 4 (i % 2): a shift and a mask bring values
// 2 p and 2 p + 1 into the halves of a register.
#pragma once

#include "common.h"

#include "../../include/holo_forward.h"

namespace holo {

struct Kv4View {
    uint8_t *pool;
    const int *table, *len;
    int64_t layer_tiles;  // tiles before this layer in a page
    int64_t page_tiles;   // tiles of a page, every layer
    int n_pages, page_shift, n_kv_heads, n_seqs, max_pages;
};

// The rows of one entry of a batch: first row, how many, how many of them the
// call takes (max_rows), its sequence's positions, its row of the table.
struct Kv4Entry {
    int first, rows, take, len;
    const int *pages;
};

__device__ __forceinline__ Kv4Entry kv4_entry(const Kv4View &c, const holo_batch_t &b, int s)
{
    Kv4Entry e;
    e.first = min(max(b.cu_rows[s], 0), b.rows);
    e.rows = min(max(b.cu_rows[s + 1], e.first), b.rows) - e.first;
    e.take = min(e.rows, b.max_rows);
    const int slot = b.seqs ? b.seqs[s] : s;
    const bool there = slot >= 0 && slot < c.n_seqs;
    e.pages = c.table + (there ? (int64_t)slot * c.max_pages : 0);
    e.len = there ? (int)min((int64_t)max(c.len[slot], 0), (int64_t)c.max_pages << c.page_shift) : 0;
    return e;
}

// Tile t of a sequence and KV head; nullptr where the table has no page.
template <int NB>
__device__ __forceinline__ uint8_t *kv4_tile(const Kv4View &c, const Kv4Entry &e, int kvh, int t)
{
    const int per = c.page_shift - 5;
    const int page = e.pages[t >> per];
    if (page < 0 || page >= c.n_pages) return nullptr;
    const int64_t at = page * c.page_tiles + c.layer_tiles + ((int64_t)kvh << per) + (t & ((1 << per) - 1));
    return c.pool + at * (36 * 32 * NB);
}

// Position of value i of lane group g's V words, and the bit of a word's value i.
__device__ __forceinline__ int v_pos(int g, int i) { return i < 4 ? 4 * g + i : 12 + 4 * g + i; }
__device__ __forceinline__ int word_shift(int i) { return 4 * (i >> 1) + 16 * (i & 1); }

// Host: the layout is in the set; the descriptor, layer and batch may be launched.
bool kv4_layout_ok(const holo_kv4_t *c);
bool kv4_call_ok(const holo_kv4_t *c, int layer, const holo_batch_t *b);
bool batch_ok(const holo_batch_t *b);
bool draft_rows_ok(const holo_batch_t *b, int words);  // an entry's rows have a bit each in so many words
Kv4View kv4_view(const holo_kv4_t *c, int layer);
// run(first, n) for the tiles that `take` rows of an entry can lie in, at most 2^23 a launch: a dimension has
// below 2^32 threads (more are cut off, and no error says so), and take may be a far bound.
template <typename F>
inline void kv4_tile_launches(int take, F run)
{
    constexpr int kAtOnce = 1 << 23;
    const int n = (take + 30) / 32 + 1;
    for (int at = 0; at < n; at += kAtOnce) run(at, n - at < kAtOnce ? n - at : kAtOnce);
}
// Rows at p, ld floats from one to the next, of `dim` floats, in 16-byte pieces.
inline bool rows_ok(const void *p, int ld, int64_t dim) { return p && !((uintptr_t)p & 15) && ld % 4 == 0 && ld >= dim; }

}  // namespace holo
