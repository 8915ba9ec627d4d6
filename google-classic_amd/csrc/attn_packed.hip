// attn_packed.hip -- causal attention over packed sequences (holo_attention_packed).
//
// softmax(q . k_p / sqrt(hd)) . v_p over the rows p of the same sequence up to a
// row's own.  Both products run on v_mfma_f32_32x32x16_f16, transposed (S^T = K
// Q^T, O^T = V^T P^T): lane j + 32 hh holds column j (a row and query head) of its
// wave's 32 throughout, the scores of keys (r % 4) + 8 (r / 4) + 4 hh in
// registers r < 16.  Every operand is two f16 halves, hi hi + hi lo + lo hi in
// fp32 (x - hi - lo within 2^-22 |x|).
//   - A workgroup's four waves take 128 columns (rows times the query heads that
//     share a KV head) and walk the keys together, 32 at a time: a tile is split
//     into halves once, into LDS, and read by all four as the operands they need.
//     Two tiles are in LDS and a third's loads under way.
//   - LDS holds operands in the lanes' order, 16 bytes a lane.  V is turned on the
//     way in: a thread loads four dims of the eight keys that make up a register
//     group of the scores, so that the probabilities are the second product's B
//     operand where they stand.  Pieces are permuted (XOR) so that both the
//     writes and the reads of 16 lanes fall on 64 different banks.
//   - Keys and values are held times 2^8, which suits f16 for rows whose largest
//     value is in [2^-11, 2^8); q rows are scaled to their largest value.  Where
//     the keys that a workgroup walks hold any other row (or an infinity or NaN,
//     which the matrix instructions would hand to the rows that do not see it), it
//     starts over in fp32, value by value: right for anything, and slow.
//   - The softmax is one pass; the running maximum moves only when a score passes
//     it by 2^7 (attn_tiles.h).
// KV heads are the fastest grid index, so that with 8 of them each XCD's L2 holds
// one head's keys and values.
#include "attn_tiles.h"
#include "kv4.h"

namespace holo {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

struct PackedAttn {
    holo_batch_t b;
    float *out;
    const float *q, *k, *v;
    int ldo, ldq, ldk, ldv, n_heads, n_kv_heads;
};

constexpr float kHeld = 256.f;                               // keys and values are held times this
constexpr float kRowLow = 1.f / 2048.f, kRowHigh = 256.f;    // a row's largest value

// The largest magnitude of four values; NaN if one is.
__device__ __forceinline__ float most(const f4 x)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(x.x), fabsf(x.y)),
                                         __builtin_elementwise_maximum(fabsf(x.z), fabsf(x.w)));
}

// Rows lie in LPR lanes.  0 where one of the wave's 64 / LPR rows has no lane with
// its bit in the mask.
template <int LPR>
__device__ __forceinline__ uint32_t every_row(unsigned long long mask)
{
    uint32_t lo = (uint32_t)mask, hi = (uint32_t)(mask >> 32);
    if constexpr (LPR < 32) {
        constexpr uint32_t one = LPR == 16 ? 0xFFFFu : 0xFFu;
        uint32_t all = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < 32; i += LPR) all = min(all, min(lo >> i & one, hi >> i & one));
        return all;
    }
    return min(lo, hi);
}

// Whether a row, in any of the wave's, has a largest value that is not 0 and below kRowLow.
template <int LPR>
__device__ __forceinline__ bool low_row(float m)
{
    const unsigned long long ge = __ballot(m >= kRowLow), pos = __ballot(m > 0.f);
    constexpr unsigned long long one = LPR == 32 ? 0xFFFFFFFFull : LPR == 16 ? 0xFFFFull : 0xFFull;
    bool low = false;
    for (int i = 0; i < 64; i += LPR) low |= (pos >> i & one) != 0 && (ge >> i & one) == 0;
    return low;
}

template <int NB>
struct PackedLds {
    static constexpr int HD = 32 * NB;  // HD / 8 <= 16
    // [hi, lo][dims 8 d8 ..][key ^ (d8 & 15)] and [hi, lo][dims 32 b ..][keys' group][dim]
    h8 k[2][2][HD / 8][32], v[2][2][NB][4][32];
    int odd[2][2][4];  // by half and staging wave: a row that the halves do not suit
};

// One column in fp32 by the two lanes that hold it, half of the dims each.
template <int HD>
__device__ __forceinline__ void packed_fp32(const PackedAttn &a, const float *qp, const float *kb, const float *vb,
                                            int row, int hh, float *out)
{
#pragma clang fp contract(off)  // the largest score less itself has to be 0
    constexpr int H = HD / 2;
    float m = -FLT_MAX, l = 0.f;
    f4 o[H / 4];
#pragma unroll
    for (int i = 0; i < H / 4; i++) o[i] = f4{};
    qp += H * hh, kb += H * hh, vb += H * hh, out += H * hh;
    for (int key = 0; key <= row; key++) {
        const f4 *k = (const f4 *)(kb + (int64_t)key * a.ldk), *v = (const f4 *)(vb + (int64_t)key * a.ldv);
        f4 d4 = f4{};
#pragma unroll 4
        for (int i = 0; i < H / 4; i++) d4 += ((const f4 *)qp)[i] * k[i];
        float s = (d4[0] + d4[1]) + (d4[2] + d4[3]);
        s = (s + __shfl_xor(s, 32, 64)) * score_scale(HD);
        const float mx = fmaxf(m, s), w = __builtin_amdgcn_exp2f(m - mx), p = __builtin_amdgcn_exp2f(s - mx);
        m = mx;
        // the average so far: a sum of values next to the largest float would overflow
        const float was = l * w;
        l = was + p;
        const float keep = was / l, add = p / l;
#pragma unroll
        for (int i = 0; i < H / 4; i++) o[i] = o[i] * keep + add * v[i];
    }
#pragma unroll
    for (int i = 0; i < H / 4; i++) ((f4 *)out)[i] = o[i];
}

template <int NB>
__global__ __launch_bounds__(256, 2) void attn_packed_k(PackedAttn a)
{
    constexpr int HD = 32 * NB, NC = HD / 16, D4 = HD / 4;
    constexpr int LPR = HD == 32 ? 8 : HD == 64 ? 16 : 32;  // lanes of a row (HD 96: the last eight idle)
    constexpr int VW = NB > 2 ? 2 : 1;                       // waves that stage V, the others K
    extern __shared__ __align__(16) uint8_t packed_lds[];
    PackedLds<NB> &S = *(PackedLds<NB> *)packed_lds;
    const int G = a.n_heads / a.n_kv_heads;
    const int kvh = blockIdx.x, ct = gridDim.y - 1 - blockIdx.y;  // the longest first
    const int s0 = min(max(a.b.cu_rows[blockIdx.z], 0), a.b.rows);
    const int n = min(min(max(a.b.cu_rows[blockIdx.z + 1], s0), a.b.rows) - s0, a.b.max_rows);
    const int ncols = n * G, c0 = 128 * ct;
    if (c0 >= ncols) return;
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ntiles = ((min(c0 + 128, ncols) - 1) / G + 32) >> 5;
    // the wave's columns, from row w_first on
    const int w0 = c0 + 32 * wave;
    const int w_first = w0 / G;
    const int col = min(w0 + j, ncols - 1);
    const int row = col / G, head = kvh * G + col % G;
    const float *qp = a.q + (int64_t)(s0 + row) * a.ldq + (int64_t)head * HD;
    const float *kb = a.k + (int64_t)s0 * a.ldk + (int64_t)kvh * HD;
    const float *vb = a.v + (int64_t)s0 * a.ldv + (int64_t)kvh * HD;

    // ---- staging: a tile's pieces from memory to registers, and into LDS.  Buffer
    // loads from the tile's first row: rows past the sequence, and the idle lanes
    // of HD 96, read zeros.
    f4 ld[4];
    const bool stages_v = wave < VW;
    const int x4 = lane % LPR;  // the thread's four dims
    const bool on = HD != 96 || x4 < D4;
    // V: group vg of eight keys (register group vg / 2, half vg % 2): 4 (vg & 1) + 16 (vg >> 1) + 0..3 and + 8..11;
    // K: row kr and every KS-th, KH of them a half
    constexpr int KS = 64 * (4 - VW) / LPR, KH = (32 + 2 * KS - 1) / (2 * KS);
    const int vg = tid / LPR, kr = (tid - 64 * VW) / LPR;
    const float *xb = stages_v ? vb : kb;
    const uint32_t rowb = 4u * (uint32_t)(stages_v ? a.ldv : a.ldk);
    const bool mine = on && (!stages_v || vg < 4);
    const uint32_t vo = mine ? (uint32_t)(stages_v ? 16 * (vg >> 1) + 4 * (vg & 1) : kr) * rowb + 16u * x4 : 0x80000000u;
    // Half f of a tile: a thread's first or last four keys of V, or its first or
    // last pieces of K (a whole tile in registers spilled, HD 128).
    auto load = [&](int t, int f) {
        const int rows = min(n - 32 * t, 32);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(xb + (int64_t)32 * t * (rowb >> 2)), (short)0, (int)((uint32_t)(rows - 1) * rowb + 4u * HD),
            kRawBufWord3);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (!stages_v && i >= KH) continue;
            const uint32_t r = stages_v ? i + 8 * f : KS * (KH * f + i);
            ld[i] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)vo, (int)(r * rowb), 0));
        }
    };
    auto store = [&](int b, int f) {
        float big = 0.f, m[4];
        uint32_t rows = 0xFFFFFFFFu;
        const int nl = stages_v ? 4 : KH;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i >= nl) continue;
            m[i] = most(ld[i]);
            big = __builtin_elementwise_maximum(big, m[i]);
            rows = min(rows, every_row<LPR>(__ballot(m[i] >= kRowLow)));
        }
        if (stages_v) {
#pragma unroll
            for (int d = 0; d < 4; d++) {
                h2 hi[2], lo[2];
                split2(ld[0][d], ld[1][d], kHeld, hi[0], lo[0]);
                split2(ld[2][d], ld[3][d], kHeld, hi[1], lo[1]);
                if (mine) {
                    const int vb_ = x4 >> 3, at = 4 * (x4 & 7) + (d ^ ((x4 >> 2 & 1) + 2 * (vb_ & 1)));
                    ((h4 *)&S.v[b][0][vb_][vg][at])[f] = h4{hi[0].x, hi[0].y, hi[1].x, hi[1].y};
                    ((h4 *)&S.v[b][1][vb_][vg][at])[f] = h4{lo[0].x, lo[0].y, lo[1].x, lo[1].y};
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < KH; i++) {
                const int r = kr + KS * (KH * f + i), d8 = x4 >> 1;
                h2 hi[2], lo[2];
                split2(ld[i][0], ld[i][1], kHeld, hi[0], lo[0]);
                split2(ld[i][2], ld[i][3], kHeld, hi[1], lo[1]);
                if (mine && (2 * KH * KS == 32 || r < 32)) {
                    ((h4 *)&S.k[b][0][d8][r ^ (d8 & 15)])[x4 & 1] = h4{hi[0].x, hi[0].y, hi[1].x, hi[1].y};
                    ((h4 *)&S.k[b][1][d8][r ^ (d8 & 15)])[x4 & 1] = h4{lo[0].x, lo[0].y, lo[1].x, lo[1].y};
                }
            }
        }
        bool odd = __any(!(big < kRowHigh));
        if (rows == 0)  // a row of small values, or of zeros
            for (int i = 0; i < nl; i++) odd |= low_row<LPR>(i == 0 ? m[0] : i == 1 ? m[1] : i == 2 ? m[2] : m[3]);
        if (lane == 0) S.odd[b][f][wave] = odd;
    };
    load(0, 0);

    h8 qh[NC], ql[NC];
    float sc;
    {
        float x[NC][8], big = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const float4 u = *(const float4 *)(qp + 16 * c + 8 * hh), w = *(const float4 *)(qp + 16 * c + 8 * hh + 4);
            x[c][0] = u.x, x[c][1] = u.y, x[c][2] = u.z, x[c][3] = u.w;
            x[c][4] = w.x, x[c][5] = w.y, x[c][6] = w.z, x[c][7] = w.w;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c][i] *= score_scale(HD);
                big = fmaxf(big, fabsf(x[c][i]));
            }
        }
        big = fmaxf(big, __shfl_xor(big, 32, 64));
        // to [2^13, 2^14); rows of zeros, and rows with an infinity (whose halves make NaN of it), as they are
        const int ex = big > 0.f && big <= FLT_MAX ? ilogbf(big) - 13 : 0;
#pragma unroll
        for (int c = 0; c < NC; c++) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[c][i] = ldexpf(x[c][i], -ex);
            split8(x[c], qh[c], ql[c]);
        }
        sc = ldexpf(1.f / kHeld, ex);
    }
    store(0, 0);
    load(0, 1);
    store(0, 1);
    __syncthreads();

    float m = -FLT_MAX, l = 0.f;
    f16v o[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) o[i] = f16v{};

    // operand x of a tile's values: dims 32 (x % NB) .., keys 16 (x / NB) ..
    h8 vh, vl;
    auto read_v = [&](int b, int x) {
        const int i = x % NB, at = j ^ ((j >> 4 & 1) + 2 * (i & 1)), g = 2 * (x / NB) + hh;
        vh = S.v[b][0][i][g][at];
        vl = S.v[b][1][i][g][at];
    };
    // the probabilities of a tile's scores, and their values
    auto values = [&](int b, f16v s) {
        read_v(b, 0);
        float ps[4] = {};
        const float off = kPShift - m;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, off));
            ps[r & 3] += s[r];
        }
        l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        h8 ph[2], pl[2];
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const float p8[8] = {s[8 * ks],     s[8 * ks + 1], s[8 * ks + 2], s[8 * ks + 3],
                                 s[8 * ks + 4], s[8 * ks + 5], s[8 * ks + 6], s[8 * ks + 7]};
            split8(p8, ph[ks], pl[ks]);
        }
#pragma unroll
        for (int x = 0; x < 2 * NB; x++) {
            const int i = x % NB, ks = x / NB;
            const h8 h = vh, l = vl;
            if (x + 1 < 2 * NB) read_v(b, x + 1);
            __builtin_amdgcn_sched_barrier(0);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, ph[ks], o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, pl[ks], o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l, ph[ks], o[i], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto rest = [&](int t) {  // of a tile: the second half of the next one into LDS
        if (t + 1 < ntiles) store((t + 1) & 1, 1);
        __syncthreads();
    };
    bool over = false;  // a tile that the halves do not suit
    int t = 0;
    for (;;) {
        f16v s;
        bool moves = false;  // the running maximum, at tile t
        // Tiles that leave the maximum alone, in a loop of their own: with the
        // scaling of the outputs in it the compiler copied them every tile.
        for (; t < ntiles; t++) {
            const int b = t & 1, key0 = 32 * t;
            const int4 odd0 = *(const int4 *)S.odd[b][0], odd1 = *(const int4 *)S.odd[b][1];
            over = __builtin_amdgcn_readfirstlane(odd0.x | odd0.y | odd0.z | odd0.w | odd1.x | odd1.y | odd1.z | odd1.w);
            if (over) break;
            const bool more = t + 1 < ntiles;
            if (more) load(t + 1, 0);
            s = f16v{};
            // (opaque: a step's address is one XOR, not a register kept for it)
            int jh = j ^ hh;
            asm volatile("" : "+v"(jh));
            // a step's operands are read under the step before
            h8 kh = S.k[b][0][hh][jh], kl = S.k[b][1][hh][jh];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const h8 h = kh, l = kl;
                if (c + 1 < NC) {
                    const int d8 = 2 * (c + 1);
                    kh = S.k[b][0][d8 + hh][jh ^ d8];
                    kl = S.k[b][1][d8 + hh][jh ^ d8];
                }
                __builtin_amdgcn_sched_barrier(0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, qh[c], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, ql[c], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(l, qh[c], s, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (key0 + 31 > w_first) {
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (key0 + (r & 3) + 8 * (r >> 2) + 4 * hh > row) s[r] = -INFINITY;
            }
            if (more) {
                store(b ^ 1, 0);  // last read a tile ago, before the barrier
                load(t + 1, 1);
            }
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
            moves = __any(mx * sc > m + kMaxSlack);
            if (moves) break;
            values(b, s);
            rest(t);
        }
        if (!moves || over) break;
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
        mx = fmaxf(m, sc * fmaxf(mx, __shfl_xor(mx, 32, 64)));
        const float w = __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l *= w;
#pragma unroll
        for (int i = 0; i < NB; i++) o[i] *= w;
        values(t & 1, s);
        rest(t++);
    }
    if (over) {
        if (w0 + j < ncols) packed_fp32<HD>(a, qp, kb, vb, row, hh, a.out + (int64_t)(s0 + row) * a.ldo + (int64_t)head * HD);
        return;
    }
    l += __shfl_xor(l, 32, 64);
    if (w0 + j >= ncols) return;
    const float f = 1.0f / (kHeld * l);  // a row sees itself
    float *op = a.out + (int64_t)(s0 + row) * a.ldo + (int64_t)head * HD + 4 * hh;
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *(f4 *)(op + 32 * i + 2 * r) = f4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]} * f;
}

template <int NB>
static void run_packed(const PackedAttn &a, int ctiles)
{
    constexpr size_t lds = sizeof(PackedLds<NB>);
    static bool attr = false;
    if (!attr) {
        HOLO_CHECK(hipFuncSetAttribute((const void *)attn_packed_k<NB>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)lds));
        attr = true;
    }
    hipLaunchKernelGGL(attn_packed_k<NB>, dim3(a.n_kv_heads, ctiles, a.b.n_seqs), dim3(256), lds, stream(), a);
    HOLO_LAUNCH_CHECK();
}

}  // namespace holo

using namespace holo;

extern "C" int holo_attention_packed(float *out, const float *q, const float *k, const float *v, int ldo, int ldq,
                                     int ldk, int ldv, int head_dim, int n_heads, int n_kv_heads,
                                     const holo_batch_t *b)
{
    if (!batch_ok(b) || n_kv_heads <= 0 || n_kv_heads > 65535 || n_heads <= 0 || n_heads % n_kv_heads != 0 ||
        !(head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128)) {
        HOLO_REJECT("holo_attention_packed: heads, head_dim or batch outside the supported set");
        return HOLO_EINVAL;
    }
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    const int64_t q_dim = (int64_t)n_heads * head_dim, kv_dim = (int64_t)n_kv_heads * head_dim;
    PackedAttn a{*b, out, q, k, v, ldo, ldq, ldk, ldv, n_heads, n_kv_heads};
    a.b.max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    const int64_t ctiles = ((int64_t)a.b.max_rows * (n_heads / n_kv_heads) + 127) / 128;
    const int most_ld = 1 << 24;  // 32 rows' bytes in 31 bits
    if (!rows_ok(out, ldo, q_dim) || !rows_ok(q, ldq, q_dim) || !rows_ok(k, ldk, kv_dim) || !rows_ok(v, ldv, kv_dim) ||
        ctiles > 65535 || ldk >= most_ld || ldv >= most_ld) {
        HOLO_REJECT("holo_attention_packed: null or misaligned rows, rows that overlap, or more than one launch takes");
        return HOLO_EINVAL;
    }
    switch (head_dim) {
    case 32: run_packed<1>(a, (int)ctiles); break;
    case 64: run_packed<2>(a, (int)ctiles); break;
    case 96: run_packed<3>(a, (int)ctiles); break;
    default: run_packed<4>(a, (int)ctiles); break;
    }
    return 0;
}
