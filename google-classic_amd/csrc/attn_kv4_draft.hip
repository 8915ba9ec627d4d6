// attn_kv4_draft.hip -- attention of drafted rows over the 4-bit cache
// (holo_attention_kv4_draft).
//
// The mathematics is that of attn_kv4.hip: S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x32_f16, a lane one column (a row and query head) throughout, q and
// the probabilities two f16 halves, one pass with a running maximum that few tiles
// move.  What differs: tiles before the entry's own rows are seen by every column and
// take no mask at all; in the last few a column's 32 bits come out of its row's mask words by
// a shift.  A workgroup has 16 columns or, for much work, 32: a tile is then unpacked once
// for both.  Sequences are cut into ranges of one length (not as many for each), so that a
// batch's long and short ones end together.
//
// What bounds it (32 heads on 8 of 128): 63 rows over 100063 positions take 222-228 us, 465
// TFLOP/s of scores and values, twice that on the matrix cores for the halves: 0.93 of the
// 1.14 PFLOP/s that a large f16 product reaches here.  Matrix and vector instructions of a
// SIMD's two waves hardly overlap: they issue in 40% and 53% of the cycles.  64 x 5 rows of up to
// 8192 140-146 us, 3.2 TB/s, 20 of 32 columns in use, 33% and 44%; 16 x 26 of up to 4096 53-57, the
// longest sequences' workgroups (mean 67 tiles, the longest 128).  Both with the longest entries
// first: workgroups start in the caller's order, and in others it is 149-154 and 63-75.  5 rows of 517 positions 9.0,
// a chain of five tiles of 1.05 each and the launch.
//
// Tried: the tiles unpacked once into LDS for 64 or 128 columns of four waves, a tile
// ahead, with the keys a tile before the values and with matrix and vector instructions
// interleaved by hand: 208 us at 63 rows of 100063 (spills of a few registers among them),
// but 70-90 at 16 x 26 and 230-320 at 64 x 5, where a tile at a time is a chain of 1 us and 2.5.  All
// tiles in equal shares across the sequences' borders: 76 against 57 at 16 x 26, each further entry
// of a share costs its 4 us of first loads.  Pages by scalar loads tile by tile: 250 against 228.
#include "attn_kv4.h"

namespace holo {

struct Draft {
    Kv4Attn a;             // (ctiles: groups of columns of max_rows rows)
    const uint32_t *mask;  // bit j of row i's words: it sees row j of its entry
    int words;
    int cut;               // the workgroups that sequences are cut into ranges for
    int slots;             // ranges of all entries, at most; entries where none is cut
    int2 *ranges;          // of each entry that has rows: its first slot, how many
};

// Which of tile t's positions a drafted row sees, one bit each: those before the
// entry's rows (the first at position `from`), and the rows that its words name.
__device__ __forceinline__ uint32_t draft_sees(const uint32_t *words, int n_words, int t, int from, int len)
{
    const int at = 32 * t - from, left = len - 32 * t;  // the tile's first position among the rows
    uint32_t bits;
    if (at <= -32) bits = 0xFFFFFFFFu;
    else if (at < 0) bits = ((1u << -at) - 1u) | words[0] << -at;
    else {
        const int w = at >> 5, s = at & 31;
        bits = w < n_words ? words[w] >> s : 0u;
        if (s && w + 1 < n_words) bits |= words[w + 1] << (32 - s);
    }
    return left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1u) : 0u;
}

// ---- ranges --------------------------------------------------------------------------------
//
// The tiles of a batch's sequences are cut into ranges of one length, so that long ones
// take as long as short ones: slots count the ranges, entry after entry, and every wave
// finds its own from the lengths.

// Tiles of entry s; -1: it has no rows.  A sequence past max_len has none.
__device__ __forceinline__ int draft_tiles(const Draft &d, int s)
{
    if (s >= d.a.b.n_seqs) return -1;
    const Kv4Entry e = kv4_entry(d.a.c, d.a.b, s);
    return e.take <= 0 ? -1 : e.len > d.a.b.max_len ? 0 : (e.len + 31) >> 5;
}

__device__ __forceinline__ int ranges_of(int tiles, int chunk) { return tiles < 0 ? 0 : tiles == 0 ? 1 : (tiles - 1) / chunk + 1; }

struct Range {
    int entry, at, chunk;  // range `at` of the entry's, each of chunk tiles; entry -1: there is none
};

__device__ __forceinline__ Range draft_range(const Draft &d, int slot, int lane)
{
    const int each = (d.a.b.n_seqs + 63) >> 6;  // entries of a lane
    long long tiles = 0;
    for (int i = 0; i < each; i++) tiles += max(draft_tiles(d, lane * each + i), 0);
    for (int off = 32; off > 0; off >>= 1) tiles += __shfl_xor(tiles, off, 64);
    const long long groups = (long long)d.a.ctiles * d.a.c.n_kv_heads;
    Range r{-1, 0, __builtin_amdgcn_readfirstlane((int)max((tiles * groups + d.cut - 1) / d.cut, (long long)kLeastRange))};
    int n = 0;
    for (int i = 0; i < each; i++) n += ranges_of(draft_tiles(d, lane * each + i), r.chunk);
    int upto = n;
    for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(upto, off, 64);
        if (lane >= off) upto += v;
    }
    const uint64_t past = __ballot(upto > slot);
    if (!past) return r;
    const int l = __ffsll((unsigned long long)past) - 1;
    r.at = slot - __builtin_amdgcn_readlane(upto - n, l);
    r.entry = l * each;
    for (int i = 1; i < each; i++, r.entry++) {  // the lane's entries: their ranges pass r.at
        const int m = ranges_of(draft_tiles(d, r.entry), r.chunk);
        if (r.at < m) break;
        r.at -= m;
    }
    r.at = __builtin_amdgcn_readfirstlane(r.at);  // (scalar registers: the compiler does not see it)
    r.entry = __builtin_amdgcn_readfirstlane(r.entry);
    return r;
}

// The partial sums of a slot's row and head: HD sums, the maximum they are relative to
// and the probabilities' sum.
__device__ __forceinline__ float *draft_partial(const Draft &d, int slot, int row, int h, int hd)
{
    return d.a.part + (((int64_t)slot * d.a.b.max_rows + row) * d.a.n_heads + h) * (hd + 4);
}

// Joins an entry's ranges: one row and head a workgroup.
template <int NB>
__global__ __launch_bounds__(256) void attn_draft_join_k(Draft d)
{
    constexpr int HD = 32 * NB;
    const int row = blockIdx.y, h = blockIdx.x;
    const Kv4Entry e = kv4_entry(d.a.c, d.a.b, blockIdx.z);
    if (row >= e.take) return;
    const int2 r = d.ranges[blockIdx.z];
    if (r.y <= 1) return;
    kv4_join<NB>(draft_partial(d, r.x, row, h, HD), (int64_t)d.a.b.max_rows * d.a.n_heads * (HD + 4), r.y,
                 d.a.out + (int64_t)(e.first + row) * d.a.ldo + (int64_t)h * HD);
}

// The same of many rows, in range order: one row and head a group of HD / 4 lanes.
template <int NB>
__global__ __launch_bounds__(256) void attn_draft_join_rows_k(Draft d)
{
    constexpr int HD = 32 * NB, D = HD / 4, GR = 256 / D, R = 4;
    const int row = blockIdx.y, h = blockIdx.x * GR + (int)threadIdx.x / D, x = 4 * (threadIdx.x % D);
    const Kv4Entry e = kv4_entry(d.a.c, d.a.b, blockIdx.z);
    if (row >= e.take) return;
    const int2 r = d.ranges[blockIdx.z];
    if (r.y <= 1 || h >= d.a.n_heads || (int)threadIdx.x >= GR * D) return;
    const float *pp = draft_partial(d, r.x, row, h, HD);
    const int64_t stride = (int64_t)d.a.b.max_rows * d.a.n_heads * (HD + 4);
    float M = -FLT_MAX, L = 0.f;
    f4 O = f4{};
    for (int s0 = 0; s0 < r.y; s0 += R) {
        f2 ml[R];
        f4 v[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const float *p = pp + min(s0 + i, r.y - 1) * stride;
            ml[i] = *(const f2 *)(p + HD);
            v[i] = *(const f4 *)(p + x);
        }
        float mx = M;
#pragma unroll
        for (int i = 0; i < R; i++) mx = fmaxf(mx, ml[i].x);  // the last range twice does no harm here
        const float was = __builtin_amdgcn_exp2f(M - mx);
        M = mx;
        L *= was;
        O *= was;
#pragma unroll
        for (int i = 0; i < R; i++) {
            if (s0 + i >= r.y) continue;
            const float f = __builtin_amdgcn_exp2f(ml[i].x - M);
            L = fmaf(f, ml[i].y, L);
            O += f * v[i];
        }
    }
    *(f4 *)(d.a.out + (int64_t)(e.first + row) * d.a.ldo + (int64_t)h * HD + x) = O * (L == 0.f ? 0.f : 1.0f / L);
}

// ---- the kernel --------------------------------------------------------------------------------

// A column's q: dims 8 (NB g + j) .. + 7 in step j, scaled to [2^13, 2^14), as two halves;
// the power of two that multiplies its scores.
template <int NB>
__device__ __forceinline__ float load_q(const float *q, h8 (&qh)[NB], h8 (&ql)[NB])
{
    float x[NB][8], big = 0.f;
#pragma unroll
    for (int j = 0; j < NB; j++) {
        const float4 u = *(const float4 *)(q + 8 * j), w = *(const float4 *)(q + 8 * j + 4);
        x[j][0] = u.x, x[j][1] = u.y, x[j][2] = u.z, x[j][3] = u.w;
        x[j][4] = w.x, x[j][5] = w.y, x[j][6] = w.z, x[j][7] = w.w;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[j][i] *= score_scale(32 * NB);
            big = fmaxf(big, fabsf(x[j][i]));
        }
    }
    big = fmaxf(big, __shfl_xor(big, 16, 64));
    big = fmaxf(big, __shfl_xor(big, 32, 64));
    const int ex = scale_exp(big);
#pragma unroll
    for (int j = 0; j < NB; j++) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[j][i] = ldexpf(x[j][i], -ex);
        split8(x[j], qh[j], ql[j]);
    }
    return ldexpf(1.f, ex);
}

// The largest of a lane's scores.
__device__ __forceinline__ float most_of(const f4 (&s)[2])
{
    return fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                 fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
}

// Probabilities of a lane's scores, as two halves; their sum.
__device__ __forceinline__ float probabilities(const f4 (&s)[2], float sc, float m, h8 &ph, h8 &pl)
{
    float p[8], ps[2] = {};
    const float off = kPShift - m;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], sc, off));
        ps[i & 1] += p[i];
    }
    split8(p, ph, pl);
    return ps[0] + ps[1];
}

// NaN scales at positions from `from` on, which not every row sees, become 0; those
// positions, a bit each.
__device__ __forceinline__ uint32_t take_nans(u4 &scales, int g, int from)
{
    h8 d = __builtin_bit_cast(h8, scales);
    uint32_t nan = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int p = v_pos(g, i);
        const bool bad = d[i] != d[i] && p >= from;
        nan |= bad ? 1u << p : 0u;
        d[i] = bad ? (_Float16)0.f : d[i];
    }
    scales = __builtin_bit_cast(u4, d);
    nan |= __shfl_xor(nan, 16, 64);
    return nan | __shfl_xor(nan, 32, 64);
}

// The table's entries of an entry's tiles, 64 pages at a time in the lanes.
struct Pages {
    int first = 0, of = 0;
    __device__ __forceinline__ void load(const Kv4View &c, const Kv4Entry &e, int p, int lane)
    {
        first = p;
        of = e.pages[min(p + lane, c.max_pages - 1)];
        asm volatile("" : "+v"(of));  // waited for here, not wherever it is read
    }
    // Tile t, not below the last one asked for; there: whether it has a page, else the
    // pool's first tile stands for it.
    template <int NB>
    __device__ __forceinline__ const uint8_t *tile(const Kv4View &c, const Kv4Entry &e, int kvh, int t, int lane, bool &there)
    {
        const int per = c.page_shift - 5, p = t >> per;
        if (p >= first + 64) load(c, e, p, lane);
        const int page = __builtin_amdgcn_readlane(of, p - first);
        there = page >= 0 && page < c.n_pages;
        const int64_t i = page * c.page_tiles + c.layer_tiles + ((int64_t)kvh << per) + (t & ((1 << per) - 1));
        return c.pool + (there ? i * (36 * 32 * NB) : 0);
    }
};

// Tiles t0 .. t1 - 1 of an entry, for 16 CT columns of a KV head.  The waves take them in
// turn and meet in LDS.
template <int NB, int CT>
struct DraftLds {
    float o[4][16 * CT][32 * NB + 4], m[4][16 * CT], l[4][16 * CT];
};

template <int NB, int CT>
__device__ __forceinline__ void draft_tiles_of(const Draft &d, const Kv4Entry &e, int kvh, int c0, int t0, int t1, int slot,
                                               DraftLds<NB, CT> &lds)
{
    constexpr int HD = 32 * NB, W = 4, C = 16 * CT;
    auto &lo_ = lds.o;
    auto &lm = lds.m;
    auto &ll = lds.l;
    const Kv4Attn &a = d.a;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int G = a.n_heads / a.c.n_kv_heads, ncols = e.take * G;
    const bool too_long = e.len > a.b.max_len;
    const int from = e.len - e.rows;
    const int ntiles = too_long ? 0 : (e.len + 31) >> 5;
    t1 = min(t1, ntiles);

    h8 qh[CT][NB], ql[CT][NB];
    float sc[CT], m[CT], l[CT];
    int mask_row[CT];
    f4 o[CT][2 * NB], s[CT][2];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const int col = min(c0 + 16 * c + r, ncols - 1);  // past the last: the last again
        mask_row[c] = e.first + col / G;
        sc[c] = load_q<NB>(a.q + (int64_t)mask_row[c] * a.ldq + (int64_t)(kvh * G + col % G) * HD + 8 * NB * g, qh[c], ql[c]);
        m[c] = -FLT_MAX;
        l[c] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) o[c][i] = f4{};
    }
    uint32_t k16;
    asm("v_mov_b32 %0, 0x4C004C00" : "=v"(k16));
    Pages pages;
    auto where = [&](int t, bool &there) { return pages.tile<NB>(a.c, e, kvh, min(t, t1 - 1), lane, there); };
    TileK<NB> xk;
    TileV<NB> xv;
    auto scores = [&]() {
#pragma unroll
        for (int c = 0; c < CT; c++) s[c][0] = s[c][1] = f4{};
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const h2 both = __builtin_bit_cast(h2, xk.s[j]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const h2 dd = {both[h], both[h]}, dm = dd * (_Float16)-24.f;
                const h2 d4[4] = {dd, dd, dd, dd}, m4[4] = {dm, dm, dm, dm};
                const h8 k8 = kv4_unpack(xk.w[h][j], k16, d4, m4);
#pragma unroll
                for (int c = 0; c < CT; c++) {
                    s[c][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[c][j], s[c][h], 0, 0, 0);
                    s[c][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[c][j], s[c][h], 0, 0, 0);
                }
            }
        }
    };
    // Some column may not see the whole tile.
    int poison[CT] = {};  // by block of dims: the column sees a NaN
    auto mask = [&](int t, bool there) {
        uint32_t bits[CT];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            bits[c] = there ? draft_sees(d.mask + (int64_t)mask_row[c] * d.words, d.words, t, from, e.len) : 0u;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (!(bits[c] >> v_pos(g, i) & 1u)) s[c][i >> 2][i & 3] = -INFINITY;
        }
        // scales of values past the sequence's end, and of a tile without a page, become 0
        const int end = there ? e.len - 32 * t : 0;
        uint32_t keep[4];  // of the lane's positions, two a register
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int left = end - v_pos(g, 2 * i);
            keep[i] = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u;
        }
        h2 sum = {};
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                xv.s[b][i] &= keep[i];
                sum += __builtin_bit_cast(h2, (uint32_t)xv.s[b][i]);
            }
        // a NaN's too: the columns that see it take the NaN at the end
        const _Float16 all = sum.x + sum.y;
        if (__builtin_expect(__any(all != all), 0))
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t nan = take_nans(xv.s[b], g, from - 32 * t);
#pragma unroll
                for (int c = 0; c < CT; c++) poison[c] |= (bits[c] & nan) ? 1 << b : 0;
            }
    };
    int t = t0 + wave;
    if (t < t1) {
        // Two tiles under way: keys are loaded a tile ahead of the values, each into
        // the registers that the products have just read.
        bool there, there1;
        pages.load(a.c, e, t >> (a.c.page_shift - 5), lane);
        const uint8_t *at = where(t, there), *at1 = where(t + W, there1);
        load_k<NB>(xk, at, lane);
        load_v<NB>(xv, at, lane);
        scores();
        load_k<NB>(xk, at1, lane);
        // Tiles that leave the maxima alone, in a loop of their own (attn_kv4_k).
        for (;;) {
            for (; t < t1; t += W) {
                if (32 * t + 31 >= from || !there) mask(t, there);
                bool moves = false;
#pragma unroll
                for (int c = 0; c < CT; c++) moves |= sc[c] * most_of(s[c]) > m[c] + kMaxSlack;
                if (__any(moves)) break;
                bool there2;
                const uint8_t *at2 = where(t + 2 * W, there2);
                h8 ph[CT], pl[CT];
#pragma unroll
                for (int c = 0; c < CT; c++) l[c] += probabilities(s[c], sc[c], m[c], ph[c], pl[c]);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    h2 d4[4], m4[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        d4[i] = __builtin_bit_cast(h2, (uint32_t)xv.s[b][i]);
                        m4[i] = d4[i] * (_Float16)-24.f;
                    }
#pragma unroll
                    for (int i = 2 * b; i < 2 * b + 2; i++) {
                        const h8 v8 = kv4_unpack(xv.w[i], k16, d4, m4);
#pragma unroll
                        for (int c = 0; c < CT; c++) {
                            o[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph[c], o[c][i], 0, 0, 0);
                            o[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl[c], o[c][i], 0, 0, 0);
                        }
                    }
                }
                load_v<NB>(xv, at1, lane);
                scores();
                load_k<NB>(xk, at2, lane);
                there = there1, there1 = there2, at1 = at2;
            }
            if (t >= t1) break;
#pragma unroll
            for (int c = 0; c < CT; c++) {
                float mx = sc[c] * most_of(s[c]);
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(m[c], fmaxf(mx, __shfl_xor(mx, 32, 64)));
                const float w = __builtin_amdgcn_exp2f(m[c] - mx);
                m[c] = mx;
                l[c] *= w;
#pragma unroll
                for (int i = 0; i < 2 * NB; i++) o[c][i] *= w;
            }
        }
    }

    // the waves meet: O = sum_w 2^(m_w - M) O_w
#pragma unroll
    for (int c = 0; c < CT; c++) {
        l[c] += __shfl_xor(l[c], 16, 64);
        l[c] += __shfl_xor(l[c], 32, 64);
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            if (poison[c] >> (i >> 1) & 1) o[c][i] = f4{NAN, NAN, NAN, NAN};
            *(f4 *)&lo_[wave][16 * c + r][16 * i + 4 * g] = o[c][i];
        }
        if (g == 0) {
            lm[wave][16 * c + r] = m[c];
            ll[wave][16 * c + r] = l[c];
        }
    }
    __syncthreads();
    const bool whole = t1 - t0 >= ntiles;  // the entry's tiles are all here
    for (int i = threadIdx.x; i < C * (HD / 4); i += 64 * W) {
        const int c = i / (HD / 4), x = 4 * (i % (HD / 4));
        if (c0 + c >= ncols) continue;
        float M = lm[0][c];
#pragma unroll
        for (int w = 1; w < W; w++) M = fmaxf(M, lm[w][c]);
        float L = 0.f;
        f4 O = f4{};
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = __builtin_amdgcn_exp2f(lm[w][c] - M);
            L = fmaf(f, ll[w][c], L);
            O += f * *(const f4 *)&lo_[w][c][x];
        }
        const int row = (c0 + c) / G, h = kvh * G + (c0 + c) % G;
        if (whole) {
            // a row that sees nothing gives zeros (a NaN that it sees is in its sums)
            f4 y = O * (L == 0.f ? 0.f : 1.0f / L);
            if (too_long) y = f4{NAN, NAN, NAN, NAN};
            *(f4 *)(a.out + (int64_t)(e.first + row) * a.ldo + (int64_t)h * HD + x) = y;
        } else {
            float *pp = draft_partial(d, slot, row, h, HD);
            *(f4 *)(pp + x) = O;
            if (x == 0) *(f2 *)(pp + HD) = f2{M, L};
        }
    }
}

// Workgroups go to the 8 XCDs in turn: eight (slot, KV head) pairs side by side, their
// groups of columns behind one another, so that those which read the same tiles share an
// L2.  (CUT: without it the code and registers are smaller, 10.2 -> 9.0 us at 5 rows of
// 517 positions.)
template <int NB, int CT, bool CUT>
__global__ __launch_bounds__(256, CT == 1 && NB < 3 ? 3 : 2) void attn_draft_k(Draft d)
{
    __shared__ __align__(16) DraftLds<NB, CT> lds;
    const Kv4Attn &a = d.a;
    const uint32_t id = blockIdx.x + blockIdx.y * gridDim.x;  // below 2^32 (run_draft)
    const uint32_t in = id % (8u * a.ctiles), pair = id / (8u * a.ctiles) * 8 + (in & 7);
    const int slot = (int)(pair / a.c.n_kv_heads), kvh = (int)(pair % a.c.n_kv_heads), ct = (int)(in >> 3);
    if (slot >= d.slots) return;
    Range r{slot, 0, 0x7FFFFFFF};
    if constexpr (CUT) r = draft_range(d, slot, threadIdx.x & 63);
    if (r.entry < 0) return;
    const Kv4Entry e = kv4_entry(a.c, a.b, r.entry);
    if (CUT && r.at == 0 && kvh == 0 && ct == 0 && threadIdx.x == 0)  // what the join needs to know
        d.ranges[r.entry] = make_int2(slot, ranges_of(draft_tiles(d, r.entry), r.chunk));
    const int t0 = r.at * r.chunk, t1 = r.chunk < 0x7FFFFFFF - t0 ? t0 + r.chunk : 0x7FFFFFFF;
    if (16 * CT * ct < e.take * (a.n_heads / a.c.n_kv_heads)) draft_tiles_of<NB, CT>(d, e, kvh, 16 * CT * ct, t0, t1, slot, lds);
}

// The kernel, and where sequences are cut the join.
template <int NB, int CT>
static int run_draft(Draft d)
{
    const int64_t take = d.a.b.max_rows, cols = take * (d.a.n_heads / d.a.c.n_kv_heads), n = d.a.b.n_seqs;
    const int64_t tiles = (d.a.b.max_len + 31) / 32;
    d.a.ctiles = (int)((cols + 16 * CT - 1) / (16 * CT));
    const int64_t groups = (int64_t)d.a.ctiles * d.a.c.n_kv_heads;
    // For two workgroups a CU, or where the sequences' ends leave more ranges than that, one
    // and a half (16 sequences of 8 rows at up to 4096: 31.1 us, for two 36.6).  Worth
    // the join where a sequence gets some 36 tiles shorter (max_len is all that is known of them): 8 rows
    // at 2000 (45) 19.4 -> 18.9 in eight sequences, 5 rows (21) 20.2 -> 24.6 in sixteen.  Between them,
    // by tiles and us whole and cut: 31 (8 x 8 at 1500) 16.9, 18.7; 32 (4 x 5 at 1200) 14.5, 16.6; 37
    // (1 x 5) 14.4, 13.4; 42 (1 x 26 at 1500) 16.4, 17.1; 43 (16 x 8 at 2048 to 4096, shuffled) 36.8,
    // 38.7; 63 (8 x 8 at 3000) 27.5, 22.7.  A far max_len cuts whatever there is: 5 rows of 517
    // positions 12.3 for 9.5.
    d.cut = n == 1 ? 2 * num_cus() : 3 * num_cus() / 2;
    const bool cuts = n <= 1024 && tiles * (d.cut - n * groups) > (int64_t)36 * d.cut;
    // (ranges: tiles / chunk of them and one more an entry at most)
    d.slots = (int)(cuts ? d.cut / groups + n : n);
    // (65535 entries by 65535 groups at most, rounded up to eight pairs; a row of the grid is whole eights)
    const int64_t blocks = ((int64_t)d.slots * d.a.c.n_kv_heads + 7) / 8 * 8 * d.a.ctiles;
    if (blocks > 0xFFF00000) {
        HOLO_REJECT("holo_attention_kv4_draft: more rows and heads than one launch takes");
        return HOLO_EINVAL;
    }
    const unsigned across = (unsigned)(blocks < 1 << 22 ? blocks : 1 << 22);
    const dim3 grid(across, (unsigned)((blocks + across - 1) / across));
    if (!cuts) {
        hipLaunchKernelGGL((attn_draft_k<NB, CT, false>), grid, dim3(256), 0, stream(), d);
        HOLO_LAUNCH_CHECK();
        return 0;
    }
    const size_t told = ((size_t)n * sizeof(int2) + 15) & ~(size_t)15;
    const StreamScratch scratch(told + (size_t)(d.slots * take * d.a.n_heads * (32 * NB + 4)) * sizeof(float));
    if (!scratch.get()) {
        latch_error((int)hipErrorOutOfMemory, "holo_attention_kv4_draft: partial sums", __FILE__, __LINE__);
        return (int)hipErrorOutOfMemory;
    }
    d.ranges = (int2 *)scratch.get();
    d.a.part = (float *)((uint8_t *)scratch.get() + told);
    hipLaunchKernelGGL((attn_draft_k<NB, CT, true>), grid, dim3(256), 0, stream(), d);
    HOLO_LAUNCH_CHECK();
    // (rows and heads by the workgroup, up to 1024 of them: 4 rows at 100000, 64 ranges, 34.3 us, by groups 43.6; 26 rows of 16 sequences at up
    // to 4096, two to four ranges, 101 us with that join, 86 by groups of lanes)
    constexpr int at_once = 256 / (8 * NB);
    const int heads = d.a.n_heads;
    if (n * take * heads <= 1024)
        hipLaunchKernelGGL(attn_draft_join_k<NB>, dim3(heads, (unsigned)take, (unsigned)n), dim3(256), 0, stream(), d);
    else
        hipLaunchKernelGGL(attn_draft_join_rows_k<NB>, dim3((heads + at_once - 1) / at_once, (unsigned)take, (unsigned)n), dim3(256),
                           0, stream(), d);
    HOLO_LAUNCH_CHECK();
    return 0;
}

template <int NB>
static int run_draft(const Draft &d)
{
    // 16 columns a workgroup; 32, which unpack a tile once for both halves but take twice as long
    // for it, where that makes 256 tiles or more for each of two workgroups a CU (64 x 5 at up to 8192, 512 tiles: 146
    // us, with 16 columns 178; 16 x 26 at up to 4096, 224 tiles: 55.4 and 52.9).  With the entries
    // shuffled, us of 16 and 32 columns: 256 tiles 104 and 84 (64 x 5 at 4096), 276 104 and 91, 329 127
    // and 96; but 32 are ahead below the bound too, 188 83 and 67 (64 x 8 at 3000), 224 77 and 57.
    const int64_t cols = (int64_t)d.a.b.max_rows * (d.a.n_heads / d.a.c.n_kv_heads);
    const int64_t work = (int64_t)d.a.b.n_seqs * d.a.c.n_kv_heads * ((cols + 15) / 16) * ((d.a.b.max_len + 31) / 32);
    return cols > 16 && work >= (int64_t)256 * 2 * num_cus() ? run_draft<NB, 2>(d) : run_draft<NB, 1>(d);
}

}  // namespace holo

using namespace holo;

extern "C" int holo_attention_kv4_draft(const holo_kv4_t *c, int layer, float *out, const float *q, int ldo, int ldq,
                                        int n_heads, const uint32_t *mask, int words, const holo_batch_t *b)
{
    if (!kv4_call_ok(c, layer, b) || n_heads <= 0 || n_heads % c->n_kv_heads != 0) {
        HOLO_REJECT("holo_attention_kv4_draft: cache, layer, heads or batch outside the supported set");
        return HOLO_EINVAL;
    }
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    const int64_t dim = (int64_t)n_heads * c->head_dim;
    Draft d{{kv4_view(c, layer), *b, out, nullptr, q, ldo, ldq, n_heads, 0, 0}, mask, words, 0, 0, nullptr};
    d.a.b.max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    const int64_t cols = (int64_t)d.a.b.max_rows * (n_heads / c->n_kv_heads);
    if (!rows_ok(q, ldq, dim) || !rows_ok(out, ldo, dim) || !draft_rows_ok(&d.a.b, words) || !mask ||
        ((uintptr_t)mask & 3) || b->max_len < 0 || b->max_len > 0x7FFFF000 ||
        (cols + 15) / 16 * c->n_kv_heads > 65535) {
        HOLO_REJECT("holo_attention_kv4_draft: null or misaligned rows or mask, rows that overlap, more rows than a mask or one launch takes");
        return HOLO_EINVAL;
    }
    switch (c->head_dim) {
    case 32: return run_draft<1>(d);
    case 64: return run_draft<2>(d);
    case 96: return run_draft<3>(d);
    default: return run_draft<4>(d);
    }
}
