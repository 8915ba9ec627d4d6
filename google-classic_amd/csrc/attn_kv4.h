// attn_kv4.h -- the attention kernels over the 4-bit cache (attn_kv4.hip: causal
// rows; attn_kv4_draft.hip: rows with masks of their own).
#pragma once

#include "attn_tiles.h"
#include "kv4.h"
#include "stream_scratch.h"

#include <float.h>

namespace holo {

// The 8 values of a word as an MFMA operand; d and d24 = -24 d of the pairs (2 p,
// 2 p + 1).  k16: 0x4C004C00, f16's 16 twice, in a register (v_and_or_b32 takes
// one constant).
__device__ __forceinline__ h8 kv4_unpack(uint32_t w, uint32_t k16, const h2 d[4], const h2 d24[4])
{
    h2 x[4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const uint32_t n = p < 2 ? w << (6 - 4 * p) : w >> (4 * p - 6);
        x[p] = __builtin_elementwise_fma(__builtin_bit_cast(h2, (n & 0x03C003C0u) | k16), d[p], d24[p]);
    }
    return h8{x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
}

// A tile's keys and values in a lane's registers.
template <int NB>
struct TileK {
    uint32_t w[2][NB], s[NB];  // s: the scales of word j of both halves' positions
};
template <int NB>
struct TileV {
    uint32_t w[2 * NB];
    u4 s[NB];
};

template <int NB>
__device__ __forceinline__ void load_k(TileK<NB> &t, const uint8_t *at, uint32_t lane)
{
    const uint32_t r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t *k = (const uint32_t *)(at + 4 * NB * (64 * h + lane));
        if constexpr (NB == 4) *(u4 *)t.w[h] = *(const u4 *)k;
        else if constexpr (NB == 2) *(uint2 *)t.w[h] = *(const uint2 *)k;
        else
#pragma unroll
            for (int j = 0; j < NB; j++) t.w[h][j] = k[j];
    }
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (j > 0 && NB % 4 == 0) t.s[j] = t.s[0];  // one block a lane
        else t.s[j] = *(const uint32_t *)(at + 1024 * NB + 4 * (16 * ((NB * g + j) >> 2) + r));
    }
}

template <int NB>
__device__ __forceinline__ void load_v(TileV<NB> &t, const uint8_t *at, uint32_t lane)
{
    constexpr int W = NB % 2 ? 2 : 4;
#pragma unroll
    for (int c = 0; c < 2 * NB / W; c++) {
        const uint8_t *v = at + 512 * NB + 4 * W * (64 * c + lane);
        if constexpr (W == 4) *(u4 *)(t.w + 4 * c) = *(const u4 *)v;
        else *(uint2 *)(t.w + 2 * c) = *(const uint2 *)v;
    }
#pragma unroll
    for (int b = 0; b < NB; b++) t.s[b] = *(const u4 *)(at + 1088 * NB + 64 * b + 16 * (lane >> 4));
}

constexpr int kLeastRange = 8;  // tiles (of at least 4: 8000 positions of one sequence 12.2 us, of 8 10.1)

struct Kv4Attn {
    Kv4View c;
    holo_batch_t b;
    float *out, *part;
    const float *q;
    int ldo, ldq, n_heads;
    int splits;  // the most ranges that a sequence is cut into
    int ctiles;  // tiles of 16 columns that max_rows rows have
};

// The partial sums of an entry's row and head, range after range: hd sums, the
// maximum they are relative to and the probabilities' sum.
__device__ __forceinline__ float *partial(const Kv4Attn &a, int entry, int row, int h, int hd)
{
    return a.part + ((((int64_t)entry * a.b.max_rows + row) * a.n_heads + h) * a.splits) * (hd + 4);
}

// Tiles of a range of a sequence that has n.
__device__ __forceinline__ int range_of(const Kv4Attn &a, int n)
{
    return a.splits == 1 ? max(n, 1) : max((n + a.splits - 1) / a.splits, kLeastRange);
}

// Column c of an entry and KV head: row c / G, query head kvh * G + c % G.
// Waves: W; the columns of a workgroup: 16.
template <int NB, int W>
__global__ __launch_bounds__(64 * W, NB == 3 ? 2 : 3) void attn_kv4_k(Kv4Attn a)
{
    constexpr int HD = 32 * NB, OS = HD + 4;
    extern __shared__ __align__(16) float kv4_lds[];
    float(*lo_)[16][OS] = (float(*)[16][OS])kv4_lds;
    float(*lm)[16] = (float(*)[16])(kv4_lds + W * 16 * OS), (*ll)[16] = lm + W;
    const int kvh = blockIdx.y / a.ctiles, ct = blockIdx.y % a.ctiles;
    const int G = a.n_heads / a.c.n_kv_heads;
    const Kv4Entry e = kv4_entry(a.c, a.b, blockIdx.z);
    const int ncols = e.take * G, c0 = 16 * ct;
    if (c0 >= ncols) return;
    const bool too_long = e.len > a.b.max_len;
    // the tiles that the tile's last row sees, in ranges
    const int last_row = (min(c0 + 16, ncols) - 1) / G, first_row = c0 / G;
    const int from = e.len - e.rows;
    const int see = max(from + last_row + 1, 0);  // positions the last row sees
    const int ntiles = too_long ? 0 : (see + 31) >> 5;
    const int chunk = range_of(a, ntiles), t0 = blockIdx.x * chunk, t1 = min(t0 + chunk, ntiles);
    if (t0 >= ntiles && blockIdx.x > 0) return;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = min(c0 + r, ncols - 1);  // past the last: the last again
    const int row = col / G, head = kvh * G + col % G;
    const int qpos = from + row;               // the column sees positions 0 .. qpos
    const int all = from + first_row;          // positions 0 .. all are seen by every column

    // q of the column: dims 8 (NB g + j) .. + 7 in step j, scaled to [2^13, 2^14)
    h8 qh[NB], ql[NB];
    float sc;
    {
        float x[NB][8], big = 0.f;
        const float *qp = a.q + (int64_t)(e.first + row) * a.ldq + (int64_t)head * HD + 8 * NB * g;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const float4 u = *(const float4 *)(qp + 8 * j), w = *(const float4 *)(qp + 8 * j + 4);
            x[j][0] = u.x, x[j][1] = u.y, x[j][2] = u.z, x[j][3] = u.w;
            x[j][4] = w.x, x[j][5] = w.y, x[j][6] = w.z, x[j][7] = w.w;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[j][i] *= score_scale(HD);
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
        sc = ldexpf(1.f, ex);
    }

    float m = -FLT_MAX, l = 0.f;  // of log2 units; l: this lane's positions
    f4 o[2 * NB], s[2];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) o[i] = f4{};
    uint32_t k16;
    asm("v_mov_b32 %0, 0x4C004C00" : "=v"(k16));
    // Tile t (past the range: its last); there: whether it has a page, else the
    // pool's first tile stands for it and nobody sees it.
    auto where = [&](int t, bool &there) {
        const uint8_t *at = kv4_tile<NB>(a.c, e, kvh, min(t, t1 - 1));
        there = at != nullptr;
        return there ? at : a.c.pool;
    };
    TileK<NB> xk;
    TileV<NB> xv;
    auto scores = [&]() {
        s[0] = s[1] = f4{};
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const h2 both = __builtin_bit_cast(h2, xk.s[j]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const h2 dd = {both[h], both[h]}, dm = dd * (_Float16)-24.f;
                const h2 d4[4] = {dd, dd, dd, dd}, m4[4] = {dm, dm, dm, dm};
                const h8 k8 = kv4_unpack(xk.w[h][j], k16, d4, m4);
                s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[j], s[h], 0, 0, 0);
                s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[j], s[h], 0, 0, 0);
            }
        }
    };
    // Some column does not see the whole tile.  Its probability is 0 where it does
    // not; the values there must be finite then: scales past the sequence's end (and
    // of a tile without a page) become 0, and a NaN's that some column does not see,
    // the columns that see it taking the NaN at the end.  (Twice changes nothing.)
    int poison = 0;  // by block of dims: this lane's positions have a NaN that the column sees
    auto mask = [&](int t, bool there) {
        const int sees = (there ? qpos : -1) - 32 * t, end = there ? e.len - 32 * t : 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (v_pos(g, i) > sees) s[i >> 2][i & 3] = -INFINITY;
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
        const _Float16 all_of = sum.x + sum.y;
        if (__builtin_expect(__any(all_of != all_of), 0)) {
            const int all_see = all - 32 * t;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                h8 d = __builtin_bit_cast(h8, xv.s[b]);
                int nan = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const bool is = d[i] != d[i];
                    nan |= is && v_pos(g, i) <= sees;
                    if (is && v_pos(g, i) > all_see) d[i] = (_Float16)0.f;
                }
                xv.s[b] = __builtin_bit_cast(u4, d);
                poison |= nan << b;
            }
        }
    };
    auto most = [&]() {
        return sc * fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    };
    int t = t0 + wave;
    if (t < t1) {
        // Two tiles under way: keys are loaded a tile ahead of the values, each into
        // the registers that the products have just read.
        bool there, there1;
        const uint8_t *at = where(t, there), *at1 = where(t + W, there1);
        load_k<NB>(xk, at, lane);
        load_v<NB>(xv, at, lane);
        scores();
        load_k<NB>(xk, at1, lane);
        // Tiles that leave the maximum alone, in a loop of their own: with the scaling
        // of the outputs in it the compiler copied them every tile.
        for (;;) {
            for (; t < t1; t += W) {
                if (32 * t + 31 > all || !there) mask(t, there);
                if (__any(most() > m + kMaxSlack)) break;
                bool there2;
                const uint8_t *at2 = where(t + 2 * W, there2);
                float p[8], ps[2] = {};
                const float off = kPShift - m;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], sc, off));
                    ps[i & 1] += p[i];
                }
                l += ps[0] + ps[1];
                h8 ph, pl;
                split8(p, ph, pl);
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
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph, o[i], 0, 0, 0);
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl, o[i], 0, 0, 0);
                    }
                }
                load_v<NB>(xv, at1, lane);
                scores();
                load_k<NB>(xk, at2, lane);
                there = there1, there1 = there2, at1 = at2;
            }
            if (t >= t1) break;
            float mx = most();
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
            const float w = __builtin_amdgcn_exp2f(m - mx);
            m = mx;
            l *= w;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) o[i] *= w;
        }
    }

    // the waves meet: O = sum_w 2^(m_w - M) O_w
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (__any(poison)) {
        poison |= __shfl_xor(poison, 16, 64);
        poison |= __shfl_xor(poison, 32, 64);
#pragma unroll
        for (int i = 0; i < 2 * NB; i++)
            if (poison >> (i >> 1) & 1) o[i] = f4{NAN, NAN, NAN, NAN};
    }
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) *(f4 *)&lo_[wave][r][16 * i + 4 * g] = o[i];
    if (g == 0) {
        lm[wave][r] = m;
        ll[wave][r] = l;
    }
    __syncthreads();
    // one range: the entry's tiles are all here
    const bool whole = ntiles <= chunk;
    for (int i = threadIdx.x; i < 16 * (HD / 4); i += 64 * W) {
        const int c = i / (HD / 4), d = 4 * (i % (HD / 4));
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
            O += f * *(const f4 *)&lo_[w][c][d];
        }
        const int64_t at = e.first + (c0 + c) / G;
        const int h = kvh * G + (c0 + c) % G;
        if (whole) {
            // a row that sees nothing gives zeros (a NaN that it sees is in its sums)
            const float f = L == 0.f ? 0.f : 1.0f / L;
            f4 y = O * f;
            if (too_long) y = f4{NAN, NAN, NAN, NAN};
            *(f4 *)(a.out + at * a.ldo + (int64_t)h * HD + d) = y;
        } else {
            float *pp = partial(a, blockIdx.z, (c0 + c) / G, h, HD) + (int64_t)blockIdx.x * (HD + 4);
            *(f4 *)(pp + d) = O;
            if (d == 0) *(f2 *)(pp + HD) = f2{M, L};
        }
    }
}

// Joins the n ranges of a row and head, in range order, their partial sums `stride`
// floats apart: groups of HD / 4 lanes take every 256 / (HD / 4)-th range, four dims a
// lane, and meet in LDS in group order.
template <int NB>
__device__ __forceinline__ void kv4_join(const float *pp, int64_t stride, int n, float *out)
{
    constexpr int HD = 32 * NB, D = HD / 4, GR = 256 / D, R = 4;
    __shared__ __align__(16) float lo_[GR][HD];
    __shared__ float lm[GR], ll[GR];
    const int g = threadIdx.x / D, d = 4 * (threadIdx.x % D);
    float M = -FLT_MAX, L = 0.f;
    f4 O = f4{};
    if (g < GR) {
        for (int s0 = g; s0 < n; s0 += R * GR) {
            f2 ml[R];
            f4 x[R];
#pragma unroll
            for (int i = 0; i < R; i++) {
                const float *p = pp + (int64_t)min(s0 + GR * i, n - 1) * stride;
                ml[i] = *(const f2 *)(p + HD);
                x[i] = *(const f4 *)(p + d);
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
                if (s0 + GR * i >= n) continue;
                const float f = __builtin_amdgcn_exp2f(ml[i].x - M);
                L = fmaf(f, ml[i].y, L);
                O += f * x[i];
            }
        }
        *(f4 *)&lo_[g][d] = O;
        if (d == 0) {
            lm[g] = M;
            ll[g] = L;
        }
    }
    __syncthreads();
    if (threadIdx.x >= D) return;
    const int groups = min(n, GR);
    for (int i = 0; i < groups; i++) M = fmaxf(M, lm[i]);
    L = 0.f;
    O = f4{};
    for (int i = 0; i < groups; i++) {
        const float f = __builtin_amdgcn_exp2f(lm[i] - M);
        L = fmaf(f, ll[i], L);
        O += f * *(const f4 *)&lo_[i][d];
    }
    *(f4 *)(out + d) = O * (L == 0.f ? 0.f : 1.0f / L);
}

template <int NB>
__global__ __launch_bounds__(256) void attn_kv4_join_k(Kv4Attn a)
{
    constexpr int HD = 32 * NB;
    const Kv4Entry e = kv4_entry(a.c, a.b, blockIdx.z);
    const int h = blockIdx.x, row = blockIdx.y;
    if (row >= e.take || e.len > a.b.max_len) return;
    const int G = a.n_heads / a.c.n_kv_heads;
    // the ranges of the row's tile of columns, as the workgroups above have it
    const int c0 = (row * G + h % G) & ~15, last_row = (min(c0 + 16, e.take * G) - 1) / G;
    const int ntiles = (max(e.len - e.rows + last_row + 1, 0) + 31) >> 5;
    const int chunk = range_of(a, ntiles), n = (ntiles + chunk - 1) / chunk;
    if (n <= 1) return;
    const int64_t at = e.first + row;
    const float *pp = partial(a, blockIdx.z, row, h, HD);
    kv4_join<NB>(pp, HD + 4, n, a.out + at * a.ldo + (int64_t)h * HD);
}

// Ranges: one where a sequence has few tiles (700 positions of 32 sequences, a
// workgroup a CU: 9.7 us, in two ranges 13.4, the launch that joins them among it;
// 513 of one: 8.5, in three 8.9) or where there are two workgroups a CU without
// ranges (64 sequences of up to 8192: 104, in two 118); else as many as bring it
// there.  max_len only bounds them: each sequence's own tiles are dealt out evenly.
// (Every entry counts with max_rows rows.  Beside a chunk of 512 rows at 2000, 70 us by
// itself, one token at 100000 walks its sequence in one range: 999 us, alone 31; with
// 15 tokens at up to 4096, alone 23.6, the chunk takes 268.)
inline int ranges(int64_t groups, int tiles)
{
    if (tiles <= 24) return 1;
    const int64_t want = (2 * (int64_t)num_cus() + groups - 1) / groups, most = (tiles + kLeastRange - 1) / kLeastRange;
    return (int)(want < most ? want : most);
}

}  // namespace holo
