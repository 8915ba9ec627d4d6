// kv4.hip -- the 4-bit cache (holo_forward.h): rows in and out of its pages,
// page copies, and the host bookkeeping of which page is whose.
#include "kv4_quant.h"

#include <algorithm>
#include <functional>
#include <mutex>
#include <new>
#include <unordered_map>
#include <unordered_set>
#include <vector>

namespace holo {

// Words of V in a tile, and the place of word (m, lane g, r) among them.
template <int NB>
struct VWords {
    static constexpr int W = NB % 2 ? 2 : 4;
    static constexpr int N = 128 * NB;  // 2 NB dims-of-16 times 64 lanes
    // m, g, r of word i
    __device__ static void at(int i, int &m, int &g, int &r)
    {
        const int j = i % W, lane = i / W & 63;
        m = i / (64 * W) * W + j;
        g = lane >> 4;
        r = lane & 15;
    }
};

// ---- append -----------------------------------------------------------------------------
//
// A workgroup takes one tile of one KV head of an entry: groups of eight lanes
// quantise (position, block) pairs, the keys straight into their words (a pair
// of lanes makes one), the values through LDS, because a word of V holds eight
// positions of a dim.  There the codes lie as bytes, the dims r + 16 m of an r side
// by side, so that a thread reads the VW dims of its words for each of the eight
// positions and turns bytes into words by byte permutes.  A word of V with
// positions outside the batch keeps their nibbles; it is loaded with the rows.
// Nothing but the tile is written, so no two workgroups meet.
//
// What bounds it, 8 KV heads of 128: four prompts of up to 1000 rows (2400 in
// all), 20 MB read and 3 written, 9.8-11 us, of which 4.3 at a large copy's rate;
// vector instructions issue in a fifth of the cycles, the waits are for rows that
// come from memory (all of a group's loads at once instead of a block's: no
// faster).  32 single rows 3.6 us: lengths, page, rows one after the other.  (V
// codes as bytes dim by dim and 128 words' nibbles gathered one by one: 16.8 and
// 5.1.)
template <int NB>
__global__ __launch_bounds__(256) void kv4_append_k(Kv4View c, holo_batch_t b, const float *k, const float *v, int ldk,
                                                    int ldv, int first)
{
    constexpr int HD = 32 * NB;
    __shared__ __align__(16) uint8_t lv[32 * HD];
    const Kv4Entry e = kv4_entry(c, b, blockIdx.z);
    const int kvh = blockIdx.y, from = e.len - e.rows;  // position of the entry's first row
    const int nth = first + (int)blockIdx.x;  // of the entry's tiles
    if (nth > (e.take + 30) / 32) return;     // (so that 32 t stays an int)
    const int t = (max(from, 0) >> 5) + nth, p0 = 32 * t;
    // the tile's positions in the batch: lo .. hi - 1
    const int lo = max(from - p0, 0), hi = min(min(from + e.take, e.len) - p0, 32);
    if (lo >= hi) return;
    uint8_t *tile = kv4_tile<NB>(c, e, kvh, t);
    if (!tile) return;
    Kv4VWords<NB> words(tile, lo, hi);
    const int x = threadIdx.x & 7;  // the lane's place in its block
    const int64_t row0 = (int64_t)e.first + p0 - from;
    for (int i = threadIdx.x >> 3; i < (hi - lo) * NB; i += 32) {
        const int p = lo + i / NB, blk = i % NB;
        const float4 kx = *(const float4 *)(k + (row0 + p) * ldk + kvh * HD + 32 * blk + 4 * x);
        const float4 vx = *(const float4 *)(v + (row0 + p) * ldv + kvh * HD + 32 * blk + 4 * x);
        kv4_put<NB>(tile, lv, p, blk, x, kx, vx);
    }
    __syncthreads();
    words.store(lv);
}

// ---- read ---------------------------------------------------------------------------------
//
// Its mirror: V words to bytes in LDS, then groups of eight lanes write (position,
// block) pairs.  2400 rows of 8 heads of 128 take 6.4-7.4 us, 20 MB written (4.3 at a
// large copy's rate), 32 single rows 3.0.

template <int NB>
__global__ __launch_bounds__(256) void kv4_read_k(Kv4View c, holo_batch_t b, float *k, float *v, int ldk, int ldv,
                                                  int first)
{
    constexpr int HD = 32 * NB;
    __shared__ __align__(16) uint8_t lv[32][HD];
    const Kv4Entry e = kv4_entry(c, b, blockIdx.z);
    const int kvh = blockIdx.y, from = e.len - e.rows;
    // rows before position 0 and of a tile without a page are zeros: the tiles are
    // counted from the one of `from`, which may be negative
    const int nth = first + (int)blockIdx.x;
    if (nth > (e.take + 30) / 32) return;
    const int t = (from >> 5) + nth, p0 = 32 * t;
    const int lo = max(from - p0, 0), hi = min(from + e.take - p0, 32);
    if (lo >= hi) return;
    const uint8_t *tile = t < 0 ? nullptr : kv4_tile<NB>(c, e, kvh, t);
    if (tile) {
        const uint32_t *vw = (const uint32_t *)(tile + 16 * HD);
        for (int i = threadIdx.x; i < VWords<NB>::N; i += 256) {
            int m, g, r;
            VWords<NB>::at(i, m, g, r);
            const uint32_t w = vw[i];
#pragma unroll
            for (int j = 0; j < 8; j++) lv[v_pos(g, j)][16 * m + r] = (uint8_t)(w >> word_shift(j) & 15u);
        }
    }
    __syncthreads();
    const int x = threadIdx.x & 7;
    const int64_t row0 = (int64_t)e.first + p0 - from;
    for (int i = threadIdx.x >> 3; i < (hi - lo) * NB; i += 32) {
        const int p = lo + i / NB, blk = i % NB;
        float4 ko = make_float4(0.f, 0.f, 0.f, 0.f), vo = ko;
        if (tile) {
            const uint32_t *kw = (const uint32_t *)tile;
            const _Float16 *ks = (const _Float16 *)(tile + 32 * HD), *vs = (const _Float16 *)(tile + 34 * HD);
            const float kd = (float)ks[32 * blk + 2 * (p & 15) + (p >> 4)];
            const float vd = (float)vs[32 * blk + 8 * ((p & 15) >> 2) + 4 * (p >> 4) + (p & 3)];
            const int word = 4 * blk + (x >> 1), g = word / NB;
            const uint32_t w = kw[(((p >> 4) * 4 + g) * 16 + (p & 15)) * NB + word - g * NB] >> (8 * (x & 1));
            const uint32_t vc = *(const uint32_t *)&lv[p][32 * blk + 4 * x];
            ko = make_float4(kd * (float)((int)(w & 15u) - 8), kd * (float)((int)(w >> 16 & 15u) - 8),
                             kd * (float)((int)(w >> 4 & 15u) - 8), kd * (float)((int)(w >> 20 & 15u) - 8));
            vo = make_float4(vd * (float)((int)(vc & 255u) - 8), vd * (float)((int)(vc >> 8 & 255u) - 8),
                             vd * (float)((int)(vc >> 16 & 255u) - 8), vd * (float)((int)(vc >> 24) - 8));
        }
        *(float4 *)(k + (row0 + p) * ldk + kvh * HD + 32 * blk + 4 * x) = ko;
        *(float4 *)(v + (row0 + p) * ldv + kvh * HD + 32 * blk + 4 * x) = vo;
    }
}

// ---- rows that stand, moved together ----------------------------------------------------------
//
// Row path[i] of an entry becomes its row i, in every layer and KV head: codes and
// scales as they are.  path rises, so a row's source lies at its place or behind it;
// a workgroup takes the tiles that it writes one after the other, reads all that
// goes into one before it writes any of it, and no later source is among what
// earlier tiles wrote.  A thread makes whole words: the keys of a (position, lane
// group), the VW dims of eight positions' values.
//
// What bounds it: one sequence, 32 layers of 8 heads, four rows moved 5.2-5.5 us, a chain of
// lengths, path, pages and words, and code that a CU has not run yet.  64 sequences 24-25 us (20
// in a trace): 16384 workgroups of a wave, two to a place on the chip, each that chain; the
// bytes (28 MB read, 28 written: pieces of 64, where the rows themselves are 9.4 and 9.4)
// would take 11.  With a tile's halves in two waves 28 (27 in a trace; one sequence the same);
// of those, two heads a workgroup 30.5 and 7.5, four 42 and 11.7, loads without branches 31-37.
// Four heads in four waves of a workgroup: 20 in a trace as well, one sequence 6.3 for 5.9.
template <int NB>
__global__ __launch_bounds__(64) void kv4_keep_k(Kv4View c, holo_batch_t b, const int *path, const int *n_path)
{
    constexpr int HD = 32 * NB, VW = VWords<NB>::W, CH = 2 * NB / VW, SC = (NB + 1) / 2;
    __shared__ const uint8_t *src[32];  // the tile that a position's row comes from; nullptr: it stays
    __shared__ int at[32];              // and the place there
    const int s = blockIdx.z, kvh = blockIdx.x;
    c.layer_tiles *= blockIdx.y;
    const Kv4Entry e = kv4_entry(c, b, s);
    const int n = min(n_path[s], e.take), from = e.len - e.rows;
    const int end = min(from + max(n, 0), e.len);  // positions written: up to here
    const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
    for (int t = max(from, 0) >> 5; 32 * (int64_t)t < end; t++) {
        uint8_t *tile = kv4_tile<NB>(c, e, kvh, t);
        const uint8_t *of = nullptr;
        const int i = 32 * t + lane - from;
        if (tile && lane < 32 && i >= 0 && i < n) {
            const int p = path[e.first + i];
            if (p != i && p >= 0 && p < e.rows && from + p >= 0) {
                of = kv4_tile<NB>(c, e, kvh, (from + p) >> 5);
                at[lane] = (from + p) & 31;
            }
        }
        if (!__any(of != nullptr)) continue;
        if (lane < 32) src[lane] = of;
        __syncthreads();
        // keys of position 16 half + r, lane group g
        uint32_t kw[2][NB];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint8_t *f = src[16 * half + r];
            if (!f) continue;
            const int sp = at[16 * half + r];
            const uint32_t *w = (const uint32_t *)f + NB * (64 * (sp >> 4) + 16 * g + (sp & 15));
#pragma unroll
            for (int j = 0; j < NB; j++) kw[half][j] = w[j];
        }
        // values of dims 16 m + r, m = VW chunk .., at eight positions
        uint32_t *vw = (uint32_t *)(tile + 16 * HD);
        uint32_t put[CH][VW] = {}, mask = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint8_t *f = src[v_pos(g, j)];
            if (!f) continue;
            const int sp = at[v_pos(g, j)], slot = 4 * (sp >> 4) + (sp & 3);
            const uint32_t *w = (const uint32_t *)(f + 16 * HD) + VW * (16 * ((sp & 15) >> 2) + r);
            uint32_t x[CH][VW];
#pragma unroll
            for (int ch = 0; ch < CH; ch++)
#pragma unroll
                for (int i = 0; i < VW; i++) x[ch][i] = w[64 * VW * ch + i];
            mask |= 15u << word_shift(j);
#pragma unroll
            for (int ch = 0; ch < CH; ch++)
#pragma unroll
                for (int i = 0; i < VW; i++) put[ch][i] |= (x[ch][i] >> word_shift(slot) & 15u) << word_shift(j);
        }
        if (mask)
#pragma unroll
            for (int ch = 0; ch < CH; ch++)
#pragma unroll
                for (int i = 0; i < VW; i++) put[ch][i] |= vw[VW * (64 * ch + lane) + i] & ~mask;
        // scales of (position, block)
        const int pos = lane & 31;
        const uint8_t *ss = src[pos];
        uint16_t kd[SC], vd[SC];
        if (ss) {
            const int p = at[pos];
#pragma unroll
            for (int k = 0; k < SC; k++) {
                const int blk = min(2 * k + (lane >> 5), NB - 1);
                kd[k] = ((const uint16_t *)(ss + 32 * HD))[32 * blk + 2 * (p & 15) + (p >> 4)];
                vd[k] = ((const uint16_t *)(ss + 34 * HD))[32 * blk + 8 * ((p & 15) >> 2) + 4 * (p >> 4) + (p & 3)];
            }
        }
        __syncthreads();
#pragma unroll
        for (int half = 0; half < 2; half++)
            if (src[16 * half + r])
#pragma unroll
                for (int j = 0; j < NB; j++) ((uint32_t *)tile)[NB * (64 * half + lane) + j] = kw[half][j];
        if (mask)
#pragma unroll
            for (int ch = 0; ch < CH; ch++)
#pragma unroll
                for (int i = 0; i < VW; i++) vw[VW * (64 * ch + lane) + i] = put[ch][i];
        if (ss)
#pragma unroll
            for (int k = 0; k < SC; k++) {
                const int blk = 2 * k + (lane >> 5);
                if (blk >= NB) continue;
                ((uint16_t *)(tile + 32 * HD))[32 * blk + 2 * (pos & 15) + (pos >> 4)] = kd[k];
                ((uint16_t *)(tile + 34 * HD))[32 * blk + 8 * ((pos & 15) >> 2) + 4 * (pos >> 4) + (pos & 3)] = vd[k];
            }
        __syncthreads();
    }
}

// ---- page copies and table updates -----------------------------------------------------------
//
// Pairs travel as kernel arguments: no device memory for them, and no copy that
// the host would have to wait for.  300 pages of 2.36 MB: 261-274 us, 5.2-5.4 TB/s read
// and written, as a large copy; two of 0.6 MB 2.3, a launch.

constexpr int kCopyPairs = 256, kUpdates = 256;
struct CopyPairs {
    int src[kCopyPairs], dst[kCopyPairs];
};

__global__ __launch_bounds__(256) void kv4_copy_k(uint8_t *pool, int64_t page16, CopyPairs pairs)
{
    const uint4 *s = (const uint4 *)pool + pairs.src[blockIdx.y] * page16;
    uint4 *d = (uint4 *)pool + pairs.dst[blockIdx.y] * page16;
    const int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x;
    if (i + 768 < page16) {  // four loads in flight
        const uint4 x0 = s[i], x1 = s[i + 256], x2 = s[i + 512], x3 = s[i + 768];
        d[i] = x0;
        d[i + 256] = x1;
        d[i + 512] = x2;
        d[i + 768] = x3;
    } else {
        for (int64_t j = i; j < page16; j += 256) d[j] = s[j];
    }
}

// Entry at[i] of the table, or of len where it is negative (-1 - sequence), becomes to[i].
struct Updates {
    int64_t at[kUpdates];
    int to[kUpdates];
};

__global__ __launch_bounds__(kUpdates) void kv4_update_k(int *table, int *len, Updates u, int n)
{
    const int i = threadIdx.x;
    if (i >= n) return;
    if (u.at[i] < 0) len[-1 - u.at[i]] = u.to[i];
    else table[u.at[i]] = u.to[i];
}

static void copy_pages(const holo_kv4_t *c, const int *src, const int *dst, int n)
{
    const int64_t page16 = (int64_t)(holo_kv4_page_bytes(c) / 16);
    for (int at = 0; at < n; at += kCopyPairs) {
        const int m = n - at < kCopyPairs ? n - at : kCopyPairs;
        CopyPairs p = {};
        for (int i = 0; i < m; i++) {
            p.src[i] = src[at + i];
            p.dst[i] = dst[at + i];
        }
        hipLaunchKernelGGL(kv4_copy_k, dim3((unsigned)((page16 + 1023) / 1024), m), dim3(256), 0, stream(),
                           (uint8_t *)c->pool, page16, p);
        HOLO_LAUNCH_CHECK();
    }
}

// ---- checks --------------------------------------------------------------------------------

bool kv4_layout_ok(const holo_kv4_t *c)
{
    if (!c || c->n_pages <= 0 || c->n_layers <= 0 || c->n_layers > 65535 || c->n_kv_heads <= 0 || c->n_kv_heads > 65535)
        return false;
    const int p = c->page_len, h = c->head_dim;
    return p >= 32 && p <= 1024 && !(p & (p - 1)) && (h == 32 || h == 64 || h == 96 || h == 128);
}

bool batch_ok(const holo_batch_t *b)
{
    return b && b->rows >= 0 && b->rows <= 0x7FFFF000 && b->n_seqs >= 0 && b->n_seqs <= 65535 &&
           (b->rows == 0 || b->n_seqs == 0 || (b->cu_rows && b->max_rows > 0));
}

bool kv4_call_ok(const holo_kv4_t *c, int layer, const holo_batch_t *b)
{
    return kv4_layout_ok(c) && c->pool && !((uintptr_t)c->pool & 15) && c->table && c->len && c->n_seqs > 0 &&
           c->max_pages > 0 && (int64_t)c->max_pages * c->page_len <= 0x7FFFF000 && layer >= 0 &&
           layer < c->n_layers && batch_ok(b);
}

Kv4View kv4_view(const holo_kv4_t *c, int layer)
{
    int shift = 5;
    while ((1 << shift) < c->page_len) shift++;
    const int64_t layer_tiles = (int64_t)c->n_kv_heads << (shift - 5);
    return Kv4View{(uint8_t *)c->pool, c->table,      c->len,   layer_tiles * layer, layer_tiles * c->n_layers,
                   c->n_pages,         shift,         c->n_kv_heads, c->n_seqs,      c->max_pages};
}

}  // namespace holo

using namespace holo;

// ---- which page is whose ----------------------------------------------------------------------

struct holo_kv4_pages {
    std::mutex mu;
    holo_kv4_t c;
    std::vector<int> table, len, refs;  // [n_seqs][max_pages], [n_seqs], [n_pages]
    std::vector<int> free;              // a heap, the lowest page first
    std::vector<int64_t> at;            // updates of the device's table (see Updates)
    std::vector<int> to, src, dst;      // and page copies before them

    int pages_of(int seq) const { return (len[seq] + c.page_len - 1) / c.page_len; }
    int &entry(int seq, int p) { return table[(size_t)seq * c.max_pages + p]; }
    int take()
    {
        std::pop_heap(free.begin(), free.end(), std::greater<int>());
        const int page = free.back();
        free.pop_back();
        refs[page] = 1;
        return page;
    }
    void drop(int page)
    {
        if (--refs[page]) return;
        free.push_back(page);  // within the capacity that create() reserved
        std::push_heap(free.begin(), free.end(), std::greater<int>());
    }
    void set(int seq, int p, int page)
    {
        entry(seq, p) = page;
        at.push_back((int64_t)seq * c.max_pages + p);
        to.push_back(page);
    }
    void set_len(int seq, int n)
    {
        len[seq] = n;
        at.push_back(-1 - (int64_t)seq);
        to.push_back(n);
    }
    // Room for the changes of a call, before the first of them: past this point
    // nothing allocates.
    void begin(size_t updates, size_t copies)
    {
        at.clear();
        to.clear();
        src.clear();
        dst.clear();
        at.reserve(updates);
        to.reserve(updates);
        src.reserve(copies);
        dst.reserve(copies);
    }
    void end()
    {
        if (!c.pool) return;
        copy_pages(&c, src.data(), dst.data(), (int)src.size());
        for (size_t i = 0; i < at.size(); i += kUpdates) {
            const int m = (int)(at.size() - i < kUpdates ? at.size() - i : kUpdates);
            Updates u = {};
            for (int j = 0; j < m; j++) {
                u.at[j] = at[i + j];
                u.to[j] = to[i + j];
            }
            hipLaunchKernelGGL(kv4_update_k, dim3(1), dim3(kUpdates), 0, stream(), const_cast<int *>(c.table),
                               const_cast<int *>(c.len), u, m);
            HOLO_LAUNCH_CHECK();
        }
    }
    bool seq_ok(int s) const { return s >= 0 && s < c.n_seqs; }
    // Not under capture: a replay would set the tables of then again.
    bool open() const { return !c.pool || !stream_capturing(); }
};

namespace {

int out_of_memory(const char *what)
{
    latch_error((int)hipErrorOutOfMemory, what, __FILE__, __LINE__);
    return (int)hipErrorOutOfMemory;
}

int rejected(const char *what)
{
    HOLO_REJECT(what);
    return HOLO_EINVAL;
}

}  // namespace

extern "C" {

size_t holo_kv4_page_bytes(const holo_kv4_t *c)
{
    if (!kv4_layout_ok(c)) return 0;
    return (size_t)c->n_layers * c->n_kv_heads * (c->page_len / 32) * 36 * c->head_dim;
}

int holo_kv4_append(const holo_kv4_t *c, int layer, const float *k, const float *v, int ldk, int ldv,
                    const holo_batch_t *b)
{
    if (!kv4_call_ok(c, layer, b)) return rejected("holo_kv4_append: cache, layer or batch outside the supported set");
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    const int64_t dim = (int64_t)c->n_kv_heads * c->head_dim;
    if (!rows_ok(k, ldk, dim) || !rows_ok(v, ldv, dim))
        return rejected("holo_kv4_append: null or misaligned rows, or rows that overlap");
    const Kv4View w = kv4_view(c, layer);
    const int take = b->max_rows < b->rows ? b->max_rows : b->rows;
    auto run = [&](auto kern) {
        kv4_tile_launches(take, [&](int first, int n) {
            hipLaunchKernelGGL(kern, dim3(n, c->n_kv_heads, b->n_seqs), dim3(256), 0, stream(), w, *b, k, v, ldk, ldv, first);
        });
    };
    switch (c->head_dim) {
    case 32: run(kv4_append_k<1>); break;
    case 64: run(kv4_append_k<2>); break;
    case 96: run(kv4_append_k<3>); break;
    default: run(kv4_append_k<4>); break;
    }
    HOLO_LAUNCH_CHECK();
    return 0;
}

int holo_kv4_read(const holo_kv4_t *c, int layer, float *k, float *v, int ldk, int ldv, const holo_batch_t *b)
{
    if (!kv4_call_ok(c, layer, b)) return rejected("holo_kv4_read: cache, layer or batch outside the supported set");
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    const int64_t dim = (int64_t)c->n_kv_heads * c->head_dim;
    if (!rows_ok(k, ldk, dim) || !rows_ok(v, ldv, dim))
        return rejected("holo_kv4_read: null or misaligned rows, or rows that overlap");
    const Kv4View w = kv4_view(c, layer);
    const int take = b->max_rows < b->rows ? b->max_rows : b->rows;
    auto run = [&](auto kern) {
        kv4_tile_launches(take, [&](int first, int n) {
            hipLaunchKernelGGL(kern, dim3(n, c->n_kv_heads, b->n_seqs), dim3(256), 0, stream(), w, *b, k, v, ldk, ldv, first);
        });
    };
    switch (c->head_dim) {
    case 32: run(kv4_read_k<1>); break;
    case 64: run(kv4_read_k<2>); break;
    case 96: run(kv4_read_k<3>); break;
    default: run(kv4_read_k<4>); break;
    }
    HOLO_LAUNCH_CHECK();
    return 0;
}

int holo_kv4_keep(const holo_kv4_t *c, const int *path, const int *n_path, const holo_batch_t *b)
{
    if (!kv4_call_ok(c, 0, b)) return rejected("holo_kv4_keep: cache or batch outside the supported set");
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    if (!path || !n_path || ((uintptr_t)path & 3) || ((uintptr_t)n_path & 3))
        return rejected("holo_kv4_keep: a null or misaligned array");
    const Kv4View w = kv4_view(c, 1);  // (the kernel takes layer_tiles times its layer)
    const dim3 grid(c->n_kv_heads, c->n_layers, b->n_seqs);
    switch (c->head_dim) {
    case 32: hipLaunchKernelGGL(kv4_keep_k<1>, grid, dim3(64), 0, stream(), w, *b, path, n_path); break;
    case 64: hipLaunchKernelGGL(kv4_keep_k<2>, grid, dim3(64), 0, stream(), w, *b, path, n_path); break;
    case 96: hipLaunchKernelGGL(kv4_keep_k<3>, grid, dim3(64), 0, stream(), w, *b, path, n_path); break;
    default: hipLaunchKernelGGL(kv4_keep_k<4>, grid, dim3(64), 0, stream(), w, *b, path, n_path); break;
    }
    HOLO_LAUNCH_CHECK();
    return 0;
}

int holo_kv4_copy_pages(const holo_kv4_t *c, const int *src, const int *dst, int n)
{
    if (!kv4_layout_ok(c) || !c->pool || ((uintptr_t)c->pool & 15) || n < 0 || (n > 0 && (!src || !dst)))
        return rejected("holo_kv4_copy_pages: cache outside the supported set, or no pages given");
    try {
        std::unordered_set<int> written;
        for (int i = 0; i < n; i++)
            if (src[i] < 0 || src[i] >= c->n_pages || dst[i] < 0 || dst[i] >= c->n_pages ||
                !written.insert(dst[i]).second)
                return rejected("holo_kv4_copy_pages: a page outside the pool, or written twice");
        for (int i = 0; i < n; i++)
            if (written.count(src[i])) return rejected("holo_kv4_copy_pages: a page that is read and written");
    } catch (const std::bad_alloc &) {
        return out_of_memory("holo_kv4_copy_pages");
    }
    copy_pages(c, src, dst, n);
    return 0;
}

holo_kv4_pages_t *holo_kv4_pages_create(const holo_kv4_t *c)
{
    const bool none = c && !c->pool && !c->table && !c->len;
    if (!kv4_layout_ok(c) || c->n_seqs <= 0 || c->max_pages <= 0 ||
        (int64_t)c->max_pages * c->page_len > 0x7FFFF000 ||
        (!none && (!c->pool || ((uintptr_t)c->pool & 15) || !c->table || !c->len || stream_capturing()))) {
        HOLO_REJECT("holo_kv4_pages_create: cache outside the supported set, or under capture");
        return nullptr;
    }
    holo_kv4_pages *p = nullptr;
    try {
        p = new holo_kv4_pages;
        p->c = *c;
        p->table.assign((size_t)c->n_seqs * c->max_pages, -1);
        p->len.assign(c->n_seqs, 0);
        p->refs.assign(c->n_pages, 0);
        p->free.resize(c->n_pages);
        for (int i = 0; i < c->n_pages; i++) p->free[i] = i;  // ascending: a heap already
    } catch (const std::bad_alloc &) {
        delete p;
        out_of_memory("holo_kv4_pages_create");
        return nullptr;
    }
    if (!none) {
        fill_bytes(const_cast<int *>(c->table), 0xFF, p->table.size() * sizeof(int));
        fill_bytes(const_cast<int *>(c->len), 0, p->len.size() * sizeof(int));
    }
    return p;
}

void holo_kv4_pages_destroy(holo_kv4_pages_t *p) { delete p; }

int holo_kv4_pages_reserve(holo_kv4_pages_t *p, const int *seqs, const int *rows, int n)
{
    if (!p || n < 0 || (n > 0 && (!seqs || !rows))) return rejected("holo_kv4_pages_reserve: null argument");
    std::lock_guard<std::mutex> lk(p->mu);
    try {
        // what the call needs, before anything changes: new pages, and copies of
        // shared last pages (of several sequences that share one, the last keeps it)
        std::unordered_set<int> seen;
        std::unordered_map<int, int> left;  // sequences that keep a shared page
        size_t need = 0, updates = 0, copies = 0;
        for (int i = 0; i < n; i++) {
            const int s = seqs[i];
            if (!p->seq_ok(s) || rows[i] < 0 || !seen.insert(s).second)
                return rejected("holo_kv4_pages_reserve: a sequence outside the cache or given twice, or rows < 0");
            if ((int64_t)p->len[s] + rows[i] > (int64_t)p->c.max_pages * p->c.page_len)
                return rejected("holo_kv4_pages_reserve: a sequence longer than its row of the table");
            if (rows[i] == 0) continue;
            const int had = p->pages_of(s);
            const size_t more = (size_t)((p->len[s] + rows[i] + p->c.page_len - 1) / p->c.page_len - had);
            need += more;
            updates += more + 1;
            if (p->len[s] % p->c.page_len) {
                const int last = p->entry(s, had - 1);
                int &keep = left.emplace(last, p->refs[last]).first->second;
                if (keep > 1) {
                    keep--;
                    need++;
                    copies++;
                    updates++;
                }
            }
        }
        if (!p->open()) return rejected("holo_kv4_pages_reserve: under graph capture");
        if (need > p->free.size()) {
            latch_error(HOLO_ENOPAGES, "holo_kv4_pages_reserve", __FILE__, __LINE__);
            return HOLO_ENOPAGES;
        }
        p->begin(updates, copies);
    } catch (const std::bad_alloc &) {
        return out_of_memory("holo_kv4_pages_reserve");
    }
    for (int i = 0; i < n; i++) {
        const int s = seqs[i];
        if (rows[i] == 0) continue;
        const int had = p->pages_of(s), want = (p->len[s] + rows[i] + p->c.page_len - 1) / p->c.page_len;
        if (p->len[s] % p->c.page_len) {
            const int last = p->entry(s, had - 1);
            if (p->refs[last] > 1) {
                const int page = p->take();
                p->src.push_back(last);
                p->dst.push_back(page);
                p->refs[last]--;
                p->set(s, had - 1, page);
            }
        }
        for (int j = had; j < want; j++) p->set(s, j, p->take());
        p->set_len(s, p->len[s] + rows[i]);
    }
    p->end();
    return 0;
}

int holo_kv4_pages_fork(holo_kv4_pages_t *p, const int *src, const int *dst, int n)
{
    if (!p || n < 0 || (n > 0 && (!src || !dst))) return rejected("holo_kv4_pages_fork: null argument");
    std::lock_guard<std::mutex> lk(p->mu);
    try {
        std::unordered_map<int, int> becomes;  // positions of the sequences forked so far
        size_t updates = 0;
        for (int i = 0; i < n; i++) {
            if (!p->seq_ok(src[i]) || !p->seq_ok(dst[i]) || src[i] == dst[i] || p->len[dst[i]] ||
                becomes.count(dst[i]))
                return rejected("holo_kv4_pages_fork: a sequence outside the cache, or a target that is not empty");
            const auto it = becomes.find(src[i]);
            const int len = it == becomes.end() ? p->len[src[i]] : it->second;
            becomes[dst[i]] = len;
            updates += (size_t)((len + p->c.page_len - 1) / p->c.page_len) + 1;
        }
        if (!p->open()) return rejected("holo_kv4_pages_fork: under graph capture");
        p->begin(updates, 0);
    } catch (const std::bad_alloc &) {
        return out_of_memory("holo_kv4_pages_fork");
    }
    for (int i = 0; i < n; i++) {
        for (int j = 0; j < p->pages_of(src[i]); j++) {
            const int page = p->entry(src[i], j);
            p->refs[page]++;
            p->set(dst[i], j, page);
        }
        p->set_len(dst[i], p->len[src[i]]);
    }
    p->end();
    return 0;
}

int holo_kv4_pages_free(holo_kv4_pages_t *p, const int *seqs, int n)
{
    if (!p || n < 0 || (n > 0 && !seqs)) return rejected("holo_kv4_pages_free: null argument");
    std::lock_guard<std::mutex> lk(p->mu);
    try {
        size_t updates = 0;
        for (int i = 0; i < n; i++) {
            if (!p->seq_ok(seqs[i])) return rejected("holo_kv4_pages_free: a sequence outside the cache");
            updates += (size_t)p->pages_of(seqs[i]) + 1;
        }
        if (!p->open()) return rejected("holo_kv4_pages_free: under graph capture");
        p->begin(updates, 0);
    } catch (const std::bad_alloc &) {
        return out_of_memory("holo_kv4_pages_free");
    }
    for (int i = 0; i < n; i++) {  // one given twice is empty the second time
        for (int j = 0; j < p->pages_of(seqs[i]); j++) {
            p->drop(p->entry(seqs[i], j));
            p->set(seqs[i], j, -1);
        }
        p->set_len(seqs[i], 0);
    }
    p->end();
    return 0;
}

int holo_kv4_pages_trim(holo_kv4_pages_t *p, const int *seqs, const int *rows, int n)
{
    if (!p || n < 0 || (n > 0 && (!seqs || !rows))) return rejected("holo_kv4_pages_trim: null argument");
    std::lock_guard<std::mutex> lk(p->mu);
    try {
        std::unordered_set<int> seen;
        size_t updates = 0;
        for (int i = 0; i < n; i++) {
            const int s = seqs[i];
            if (!p->seq_ok(s) || rows[i] < 0 || !seen.insert(s).second || rows[i] > p->len[s])
                return rejected("holo_kv4_pages_trim: a sequence outside the cache or given twice, or rows that it has not");
            updates += (size_t)p->pages_of(s) + 1;
        }
        if (!p->open()) return rejected("holo_kv4_pages_trim: under graph capture");
        p->begin(updates, 0);
    } catch (const std::bad_alloc &) {
        return out_of_memory("holo_kv4_pages_trim");
    }
    for (int i = 0; i < n; i++) {
        const int s = seqs[i];
        if (rows[i] == 0) continue;
        const int had = p->pages_of(s), keep = (p->len[s] - rows[i] + p->c.page_len - 1) / p->c.page_len;
        for (int j = keep; j < had; j++) {
            p->drop(p->entry(s, j));
            p->set(s, j, -1);
        }
        p->set_len(s, p->len[s] - rows[i]);
    }
    p->end();
    return 0;
}

int holo_kv4_pages_compact(holo_kv4_pages_t *p)
{
    if (!p) return rejected("holo_kv4_pages_compact: null argument");
    std::lock_guard<std::mutex> lk(p->mu);
    const int used = p->c.n_pages - (int)p->free.size();
    std::vector<int> to;  // of each page
    try {
        to.assign(p->c.n_pages, -1);
        size_t updates = 0, copies = 0;
        for (int i = used; i < p->c.n_pages; i++) copies += p->refs[i] > 0;
        for (int s = 0; s < p->c.n_seqs; s++) updates += (size_t)p->pages_of(s);
        if (!p->open()) return rejected("holo_kv4_pages_compact: under graph capture");
        p->begin(updates, copies);
    } catch (const std::bad_alloc &) {
        return out_of_memory("holo_kv4_pages_compact");
    }
    // the used pages past the front, in order, into the free ones of the front, in
    // order: no page is both read and written
    for (int i = used, hole = 0; i < p->c.n_pages; i++) {
        if (!p->refs[i]) continue;
        while (p->refs[hole]) hole++;
        to[i] = hole;
        p->src.push_back(i);
        p->dst.push_back(hole);
        p->refs[hole] = p->refs[i];
        p->refs[i] = 0;
    }
    for (int s = 0; s < p->c.n_seqs; s++)
        for (int j = 0; j < p->pages_of(s); j++) {
            const int page = to[p->entry(s, j)];
            if (page >= 0) p->set(s, j, page);
        }
    for (int i = used; i < p->c.n_pages; i++) p->free[i - used] = i;  // ascending: a heap
    p->end();
    return 0;
}

int holo_kv4_pages_available(holo_kv4_pages_t *p)
{
    if (!p) return 0;
    std::lock_guard<std::mutex> lk(p->mu);
    return (int)p->free.size();
}

int holo_kv4_pages_len(holo_kv4_pages_t *p, int seq)
{
    if (!p) return -1;
    std::lock_guard<std::mutex> lk(p->mu);
    return p->seq_ok(seq) ? p->len[seq] : -1;
}

int holo_kv4_pages_list(holo_kv4_pages_t *p, int seq, int *pages, int n)
{
    if (!p) return -1;
    std::lock_guard<std::mutex> lk(p->mu);
    if (!p->seq_ok(seq)) return -1;
    const int m = p->pages_of(seq);
    for (int j = 0; j < m && j < n && pages; j++) pages[j] = p->entry(seq, j);
    return m;
}

}  // extern "C"
