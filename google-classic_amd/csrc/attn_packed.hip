// attn_packed.hip -- causal attention over packed sequences (holo_attention_packed).
//
// softmax(q . k_p / sqrt(hd)) . v_p over the rows p of the same sequence up to a
// row's own.  Both products run on v_mfma_f32_32x32x16_f16, transposed (S^T = K
// Q^T, O^T = V^T P^T): lane j + 32 hh holds column j (a row and query head) of its
// wave's 32 throughout, the scores of keys (r % 4) + 8 (r / 4) + 4 hh in
// registers r < 16.  Every operand is two f16 halves, hi hi + hi lo + lo hi in
// fp32 (x - hi - lo within 2^-22 |x|).
//   - A workgroup's waves take 128 or 256 columns (rows times the query heads that
//     share a KV head) and walk the keys together, 32 at a time: a tile is split
//     into halves once, into LDS, and read by all of them as the operands they need.
//     Two tiles are in LDS and a third's loads under way.
//   - LDS holds operands in the lanes' order, 16 bytes a lane.  V is turned on the
//     way in: a thread loads four dims of keys that make up a register group of the
//     scores, so that the probabilities are the second product's B operand where
//     they stand.  Pieces are permuted (XOR) so that the writes and the reads of 16
//     lanes fall on 64 different banks.
//   - Keys and values are held times 2^8, which suits f16 for rows whose largest
//     value is in [2^-11, 255.9375); q rows are scaled to their largest value.  Smaller
//     rows are held within 2^-33, which does no harm to scores of ordinary q rows, nor
//     to outputs that other rows have a part in.  The columns that it harms, and
//     every column of a workgroup that walks a row of larger values (or of infinities
//     or NaN, which the matrix instructions would hand to the rows that do not see
//     it), start over in fp32, value by value: right for anything, and slow (1024
//     rows with two small ones 68 us, as without them; 4096 with one of 300: 11.7 ms).
//   - The softmax is one pass; the running maximum moves only when a score passes
//     it by 2^7 (attn_tiles.h).
// KV heads are the fastest grid index, so that with 8 of them each XCD's L2 holds
// one head's keys and values.
//
// What bounds it: 4096 rows, 32 heads on 8 of 128, take 357 us (355-425 on several
// cards), three products of 137 GFLOP each at 1.15 PFLOP/s; a large f16 product of the
// library runs at 1.22 on such values, the chip's power setting both (the matrix cores
// are busy 64% of the cycles, at 1.7 GHz).  Below that, the steps that led here: 16 columns a workgroup
// and every tile split by each 2703 us, 128 columns 622, nothing spilled 463,
// cheaper halves and checks 437.  Short prompts: one chain of loads, scores,
// exponentials and products a tile, 7.4 us with one tile.
#include "attn_tiles.h"
#include "block_reduce.h"
#include "kv4.h"

namespace holo {

struct PackedAttn {
    holo_batch_t b;
    float *out;
    const float *q, *k, *v;
    int ldo, ldq, ldk, ldv, n_heads, n_kv_heads;
};

constexpr float kHeld = 256.f;  // keys and values are held times this
// A row's largest value; from kRowHigh up, times kHeld it is 65520 and more, which f16 rounds to infinity.
constexpr float kRowLow = 1.f / 2048.f, kRowHigh = 255.9375f;
// What a workgroup's staged rows hold that the halves do not suit.  Low rows are
// held within 2^-33: no harm to a column whose scores that moves by 2^-22 at most (hd
// values of q below 16 in log2 units, sc below kLowSc), or whose output's
// largest value is not low itself.
enum { kHighRow = 1, kLowKey = 2, kLowValue = 4 };
constexpr float kLowSc = 0x1p-17f;

// The largest magnitude of four values; NaN if one is.
__device__ __forceinline__ float most(const f4 x)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(x.x), fabsf(x.y)),
                                         __builtin_elementwise_maximum(fabsf(x.z), fabsf(x.w)));
}

// Whether some row has no value from kRowLow up.  Rows lie in LPR lanes each, m[i]
// the lane's largest of the i-th: a bit for each, joined across the row's lanes.
template <int LPR, int N>
__device__ __forceinline__ bool some_low(const float (&m)[N])
{
    int bits = 0;
#pragma unroll
    for (int i = 0; i < N; i++) bits |= m[i] >= kRowLow ? 1 << i : 0;
    bits |= __builtin_amdgcn_update_dpp(0, bits, 0xB1, 0xF, 0xF, false);   // quad [1,0,3,2]
    bits |= __builtin_amdgcn_update_dpp(0, bits, 0x4E, 0xF, 0xF, false);   // quad [2,3,0,1]
    bits |= __builtin_amdgcn_update_dpp(0, bits, 0x141, 0xF, 0xF, false);  // half mirror
    if constexpr (LPR >= 16) bits |= __builtin_amdgcn_update_dpp(0, bits, 0x140, 0xF, 0xF, false);  // mirror
    if constexpr (LPR == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
        bits = r[0] | r[1];
    }
    return __any(bits != (1 << N) - 1);
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
    int odd[8];  // by wave: of the rows that it staged
};

// One column in fp32 by the two lanes that hold it, half of the dims each, four
// keys at a time.
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
    auto keys = [&]<int N>(int key) {
        f4 d[N];
        float s[N], mx = m;
#pragma unroll
        for (int n = 0; n < N; n++) d[n] = f4{};
        const float *k = kb + (int64_t)key * a.ldk, *v = vb + (int64_t)key * a.ldv;
#pragma unroll 4
        for (int i = 0; i < H / 4; i++) {
            const f4 x = ((const f4 *)qp)[i];
#pragma unroll
            for (int n = 0; n < N; n++)
                d[n] = __builtin_elementwise_fma(x, ((const f4 *)(k + (int64_t)n * a.ldk))[i], d[n]);
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            s[n] = (d[n][0] + d[n][1]) + (d[n][2] + d[n][3]);
            s[n] = (s[n] + __shfl_xor(s[n], 32, 64)) * score_scale(HD);
            mx = fmaxf(mx, s[n]);
        }
        // the average so far: a sum of values next to the largest float would overflow
        const float was = l * __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l = was;
#pragma unroll
        for (int n = 0; n < N; n++) l += s[n] = __builtin_amdgcn_exp2f(s[n] - mx);
        // (while every score is -infinity no key has weight, and the average stays 0)
        const float sum = l == 0.f ? 1.f : l, keep = was / sum;
#pragma unroll
        for (int n = 0; n < N; n++) s[n] /= sum;
#pragma unroll
        for (int i = 0; i < H / 4; i++) {
            f4 y = o[i] * keep;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const f4 x = ((const f4 *)(v + (int64_t)n * a.ldv))[i];
                y = __builtin_elementwise_fma(f4{s[n], s[n], s[n], s[n]}, x, y);
            }
            o[i] = y;
        }
    };
    int key = 0;
    for (; key + 3 <= row; key += 4) keys.template operator()<4>(key);
    for (; key <= row; key++) keys.template operator()<1>(key);
#pragma unroll
    for (int i = 0; i < H / 4; i++) ((f4 *)out)[i] = l == 0.f ? f4{NAN, NAN, NAN, NAN} : o[i];
}

// W = 4: 128 columns a workgroup, each wave doing all of a tile's work, the next
// tile's staging between the matrix instructions; two workgroups a CU.
// W = 8: 256 columns, two groups of four waves, one of each on a SIMD, half a
// tile apart: while the waves of one multiply (the values of tile t, the keys of
// t + 1), those of the other do what is not multiplication (probabilities, and
// staging, the first group the keys and the second the values), and a barrier
// lets them change places.
template <int NB, int W>
__global__ __launch_bounds__(64 * W, 2) void attn_packed_k(PackedAttn a)
{
    constexpr int HD = 32 * NB, NC = HD / 16, D4 = HD / 4;
    constexpr int LPR = HD == 32 ? 8 : HD == 64 ? 16 : 32;  // lanes of a row (HD 96: the last eight idle)
    extern __shared__ __align__(16) uint8_t packed_lds[];
    PackedLds<NB> &S = *(PackedLds<NB> *)packed_lds;
    const int G = a.n_heads / a.n_kv_heads;
    const int kvh = blockIdx.x, ct = gridDim.y - 1 - blockIdx.y;  // the longest first
    const int s0 = min(max(a.b.cu_rows[blockIdx.z], 0), a.b.rows);
    const int n = min(min(max(a.b.cu_rows[blockIdx.z + 1], s0), a.b.rows) - s0, a.b.max_rows);
    const int ncols = n * G, c0 = 32 * W * ct;
    if (c0 >= ncols) return;
    const int tid = threadIdx.x & 255, lane = tid & 63, j = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int ntiles = ((min(c0 + 32 * W, ncols) - 1) / G + 32) >> 5;
    // the wave's columns, from row w_first on
    const int w0 = c0 + 32 * wave;
    const int w_first = w0 / G;
    const int col = min(w0 + j, ncols - 1);
    const int row = col / G, head = kvh * G + col % G;
    const float *qp = a.q + (int64_t)(s0 + row) * a.ldq + (int64_t)head * HD;
    const float *kb = a.k + (int64_t)s0 * a.ldk + (int64_t)kvh * HD;
    const float *vb = a.v + (int64_t)s0 * a.ldv + (int64_t)kvh * HD;

    // ---- staging: a tile's pieces from memory to registers, and into LDS: the keys
    // in one half of a tile's work, the values in the other.  Buffer loads from the
    // tile's first row: rows past the sequence, and the idle lanes of HD 96, read
    // zeros.  The thread's four dims: 4 x4 ..; its keys: row kr and every KS-th; its
    // values: VK keys from 32 / GS * .. (GS groups of lanes), which are half or less
    // of a register group of the scores, 16 (vg / 2) + 4 (vg % 2) + 0..3 and + 8..11.
    constexpr int KS = 256 / LPR, KP = 32 / KS, VK = KP;  // rows a pass, pieces a thread
    const int x4 = lane % LPR, kr = tid / LPR;
    const bool mine = HD != 96 || x4 < D4;
    // of the thread's VK values: their group, first place in it, and first key
    const int vg = kr * VK / 8, vi = kr * VK % 8, v_key = 16 * (vg >> 1) + 4 * (vg & 1) + (vi & 3) + 8 * (vi >> 2);
    const uint32_t kvo = mine ? kr * 4u * (uint32_t)a.ldk + 16u * x4 : 0x80000000u;
    const uint32_t vvo = mine ? v_key * 4u * (uint32_t)a.ldv + 16u * x4 : 0x80000000u;
    f4 ld[KP];
    auto load = [&](const float *base, int ldx, uint32_t vo, int step, int t) {
        const uint32_t rowb = 4u * (uint32_t)ldx;
        const int rows = min(n - 32 * t, 32);  // none past the sequence
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(base + (int64_t)32 * t * ldx), (short)0, rows > 0 ? (int)((uint32_t)(rows - 1) * rowb + 4u * HD) : 0,
            kRawBufWord3);
#pragma unroll
        for (int i = 0; i < KP; i++)
            ld[i] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)vo, (int)(step * i * rowb), 0));
    };
    auto load_k = [&](int t) { load(kb, a.ldk, kvo, KS, t); };
    auto load_v = [&](int t) { load(vb, a.ldv, vvo, 1, t); };
    // piece i of the keys, dim i of the values
    auto store_k = [&](int b, int i) {
        const int r = kr + KS * i, d8 = x4 >> 1;
        h2 hi[2], lo[2];
        split2(ld[i][0], ld[i][1], kHeld, hi[0], lo[0]);
        split2(ld[i][2], ld[i][3], kHeld, hi[1], lo[1]);
        if (mine) {
            ((h4 *)&S.k[b][0][d8][r ^ (d8 & 15)])[x4 & 1] = h4{hi[0].x, hi[0].y, hi[1].x, hi[1].y};
            ((h4 *)&S.k[b][1][d8][r ^ (d8 & 15)])[x4 & 1] = h4{lo[0].x, lo[0].y, lo[1].x, lo[1].y};
        }
    };
    auto store_v = [&](int b, int d) {
        const int vb_ = x4 >> 3, at = 4 * (x4 & 7) + (d ^ ((x4 >> 2 & 1) + 2 * (vb_ & 1)));
        _Float16 *ph = (_Float16 *)&S.v[b][0][vb_][vg][at] + vi, *pl = (_Float16 *)&S.v[b][1][vb_][vg][at] + vi;
        h2 hi, lo, hi2, lo2;
        split2(ld[0][d], ld[VK > 1 ? 1 : 0][d], kHeld, hi, lo);
        if constexpr (VK == 4) split2(ld[2][d], ld[3][d], kHeld, hi2, lo2);
        if (mine) {
            if constexpr (VK == 4) {
                *(h4 *)ph = h4{hi.x, hi.y, hi2.x, hi2.y};
                *(h4 *)pl = h4{lo.x, lo.y, lo2.x, lo2.y};
            } else if constexpr (VK == 2) {
                *(h2 *)ph = hi;
                *(h2 *)pl = lo;
            } else {
                *ph = hi.x;
                *pl = lo.x;
            }
        }
    };
    // whether the loaded rows suit the halves; low: of the keys', or of the values
    bool high = false, low_k = false, low_v = false;
    auto check = [&](bool &low) {
        float big = 0.f, m[KP];
#pragma unroll
        for (int i = 0; i < KP; i++) {
            m[i] = most(ld[i]);
            big = __builtin_elementwise_maximum(big, m[i]);
        }
        high |= __any(!(big < kRowHigh));
        if (some_low<LPR>(m)) {  // a row of small values, or of zeros
#pragma unroll
            for (int i = 0; i < KP; i++) low |= low_row<LPR>(m[i]);
        }
    };
    const bool second = W == 8 && wave >= 4;
    if (second) load_v(0);
    else load_k(0);

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
        const int ex = scale_exp(max_halves(big));
#pragma unroll
        for (int c = 0; c < NC; c++) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[c][i] = ldexpf(x[c][i], -ex);
            split8(x[c], qh[c], ql[c]);
        }
        sc = ldexpf(1.f / kHeld, ex);
    }
    check(low_k);
    if (second) {
#pragma unroll
        for (int i = 0; i < 4; i++) store_v(0, i);
        load_v(1);  // (past the sequence: zeros)
    } else {
#pragma unroll
        for (int i = 0; i < KP; i++) store_k(0, i);
        if constexpr (W == 4) {
            load_v(0);
            check(low_v);
#pragma unroll
            for (int i = 0; i < 4; i++) store_v(0, i);
        }
        load_k(1);
    }
    __syncthreads();

    float m = -FLT_MAX, l = 0.f;
    f16v o[NB], s;
#pragma unroll
    for (int i = 0; i < NB; i++) o[i] = f16v{};

    // s = the scores of the tile in buffer b; between(c) goes between step c's instructions
    auto scores = [&](int b, auto between) {
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
            between(c);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(l, qh[c], s, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Whether tile t's scores move the running maximum; they are masked here.
    auto moves = [&](int t) {
        const int key0 = 32 * t;
        if (key0 + 31 > w_first) {
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (key0 + (r & 3) + 8 * (r >> 2) + 4 * hh > row) s[r] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
        return (bool)__any(mx * sc > m + kMaxSlack);
    };
    auto move = [&]() {
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
        mx = fmaxf(m, sc * max_halves(mx));
        const float w = __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l *= w;
#pragma unroll
        for (int i = 0; i < NB; i++) o[i] *= w;
    };
    // the probabilities of the scores, as operands
    h8 ph[2], pl[2];
    auto probabilities = [&]() {
        float ps[4] = {};
        const float off = kPShift - m;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, off));
            ps[r & 3] += s[r];
        }
        l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const float p8[8] = {s[8 * ks],     s[8 * ks + 1], s[8 * ks + 2], s[8 * ks + 3],
                                 s[8 * ks + 4], s[8 * ks + 5], s[8 * ks + 6], s[8 * ks + 7]};
            split8(p8, ph[ks], pl[ks]);
        }
    };
    // o += the values of the tile in buffer b, in steps x: dims 32 (x % NB) .., keys 16 (x / NB) ..
    h8 vh, vl;
    auto read_v = [&](int b, int x) {
        const int i = x % NB, at = j ^ ((j >> 4 & 1) + 2 * (i & 1)), g = 2 * (x / NB) + hh;
        vh = S.v[b][0][i][g][at];
        vl = S.v[b][1][i][g][at];
    };
    auto values = [&](int b, auto between) {
#pragma unroll
        for (int x = 0; x < 2 * NB; x++) {
            const int i = x % NB, ks = x / NB;
            const h8 h = vh, l = vl;
            if (x + 1 < 2 * NB) read_v(b, x + 1);
            __builtin_amdgcn_sched_barrier(0);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, ph[ks], o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, pl[ks], o[i], 0, 0, 0);
            between(x);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l, ph[ks], o[i], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto nothing = [](int) {};
    // Tiles that leave the maximum alone, in a loop of their own: with the scaling
    // of the outputs in it the compiler copied them every tile.
    int t = 0;
    if constexpr (W == 4) {
        auto front = [&](int t) {
            const int b = t & 1;
            scores(b, [&](int c) {
                // the next tile's keys into LDS, once their loads are there
                constexpr int H = NC / 2;
                if (c == H) check(low_k);
#pragma unroll
                for (int i = KP * (c - H) / H; c >= H && i < KP * (c - H + 1) / H; i++) store_k(b ^ 1, i);
            });
            load_v(t + 1);
        };
        front(0);
        for (;;) {
            for (; t < ntiles && !moves(t);) {
                const int b = t & 1;
                read_v(b, 0);
                probabilities();
                values(b, [&](int x) {
                    if (x == NB) check(low_v);
#pragma unroll
                    for (int d = 4 * (x - NB) / NB; x >= NB && d < 4 * (x - NB + 1) / NB; d++) store_v(b ^ 1, d);
                });
                load_k(t + 2);
                __syncthreads();
                if (++t < ntiles) front(t);
            }
            if (t == ntiles) break;
            move();
        }
    } else {
        if (second) __syncthreads();
        scores(0, nothing);
        __syncthreads();
        for (;;) {
            for (; t < ntiles && !moves(t); t++) {
                const int b = t & 1;
                probabilities();
                check(low_k);  // (of the values, in the second group)
                if (second) {
#pragma unroll
                    for (int i = 0; i < 4; i++) store_v(b ^ 1, i);
                    load_v(t + 2);
                } else {
#pragma unroll
                    for (int i = 0; i < KP; i++) store_k(b ^ 1, i);
                    load_k(t + 2);
                }
                __syncthreads();
                __builtin_amdgcn_s_setprio(1);
                read_v(b, 0);
                values(b, nothing);
                scores(b ^ 1, nothing);
                __builtin_amdgcn_s_setprio(0);
                __syncthreads();
            }
            if (t == ntiles) break;
            move();
        }
        if (!second) __syncthreads();
    }
    // columns that the halves do not suit: over again
    if (second) low_v = low_k, low_k = false;
    if (lane == 0) S.odd[wave] = (high ? kHighRow : 0) | (low_k ? kLowKey : 0) | (low_v ? kLowValue : 0);
    __syncthreads();
    int odd = 0;
#pragma unroll
    for (int w = 0; w < W; w++) odd |= S.odd[w];
    l += __shfl_xor(l, 32, 64);
    const float f = 1.0f / (kHeld * l);  // a row sees itself
    bool over = odd & kHighRow || (odd & kLowKey && sc >= kLowSc);
    if (odd & kLowValue) {
        float big = 0.f;
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) big = fmaxf(big, fabsf(o[i][r]));
        over |= max_halves(big) * f < kRowLow;
    }
    if (w0 + j >= ncols) return;
    float *op = a.out + (int64_t)(s0 + row) * a.ldo + (int64_t)head * HD;
    if (over) {
        packed_fp32<HD>(a, qp, kb, vb, row, hh, op);
        return;
    }
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *(f4 *)(op + 4 * hh + 32 * i + 2 * r) = f4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]} * f;
}

// ---- few columns: the keys shared by the waves ----------------------------------------
//
// 32 columns a workgroup; its W waves take the 32-key tiles in turn and meet in
// LDS at the end.  Every wave loads and splits its own tiles: more work a tile,
// but a short prompt has as many waves at work as it has tiles.  Keys come in
// whole rows and reach their lanes through a stage of the wave's; a lane's values
// are dims NB * i .. of its 16 keys, the operand rows of NB blocks i of 32 dims.
template <int NB, int W>
struct SplitLds {
    static constexpr int HD = 32 * NB, DH = HD == 96 ? 32 : HD < 64 ? HD : 64;  // dims in a stage
    static constexpr int QS = HD + 8, KS = DH + 4, OS = HD + 1;                  // strides: distinct banks
    union {
        struct {
            _Float16 q[2][32][QS];
            float k[W][32][KS];
        };
        float o[W][32][OS];
    };
    float m[W][32], l[W][32], w[W][32];
    int odd[W];
};

template <int NB, int W>
__global__ __launch_bounds__(64 * W, 8 / W) void attn_packed_split_k(PackedAttn a)
{
    using Lds = SplitLds<NB, W>;
    constexpr int HD = 32 * NB, NC = HD / 16, DH = Lds::DH, LR = DH / 4, RPI = 64 / LR, NI = 32 / RPI;
    extern __shared__ __align__(16) uint8_t packed_lds[];
    Lds &S = *(Lds *)packed_lds;
    const int G = a.n_heads / a.n_kv_heads;
    const int kvh = blockIdx.x, ct = gridDim.y - 1 - blockIdx.y;
    const int s0 = min(max(a.b.cu_rows[blockIdx.z], 0), a.b.rows);
    const int n = min(min(max(a.b.cu_rows[blockIdx.z + 1], s0), a.b.rows) - s0, a.b.max_rows);
    const int ncols = n * G, c0 = 32 * ct;
    if (c0 >= ncols) return;
    const int lane = threadIdx.x & 63, j = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int first = c0 / G, last = (min(c0 + 32, ncols) - 1) / G, ntiles = (last + 32) >> 5;
    const int col = min(c0 + j, ncols - 1);
    const int row = col / G, head = kvh * G + col % G;
    const float *kb = a.k + (int64_t)s0 * a.ldk + (int64_t)kvh * HD;
    const float *vb = a.v + (int64_t)s0 * a.ldv + (int64_t)kvh * HD;
    const float *qp = a.q + (int64_t)(s0 + row) * a.ldq + (int64_t)head * HD;

    // a tile's loads: rows past the sequence read zeros
    f4 kr[HD / DH][NI];
    float vr[16][NB];
    const uint32_t krowb = 4u * (uint32_t)a.ldk, vrowb = 4u * (uint32_t)a.ldv;
    const uint32_t ko = (uint32_t)(lane / LR) * krowb + 16u * (uint32_t)(lane % LR);
    const uint32_t vo = 4u * (uint32_t)hh * vrowb + 4u * NB * (uint32_t)j;
    auto load = [&](int t) {
        const int rows = min(n - 32 * t, 32);
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(kb + (int64_t)32 * t * a.ldk), (short)0, rows > 0 ? (int)((uint32_t)(rows - 1) * krowb + 4u * HD) : 0,
            kRawBufWord3);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(vb + (int64_t)32 * t * a.ldv), (short)0, rows > 0 ? (int)((uint32_t)(rows - 1) * vrowb + 4u * HD) : 0,
            kRawBufWord3);
#pragma unroll
        for (int f = 0; f < HD / DH; f++)
#pragma unroll
            for (int i = 0; i < NI; i++)
                kr[f][i] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(
                                                      rk, (int)(ko + 4 * DH * f), (int)((uint32_t)(RPI * i) * krowb), 0));
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int so = (int)((uint32_t)((r & 3) + 8 * (r >> 2)) * vrowb);
            if constexpr (NB == 4) {
                const f4 x = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rv, (int)vo, so, 0));
#pragma unroll
                for (int i = 0; i < 4; i++) vr[r][i] = x[i];
            } else if constexpr (NB == 3) {
                const auto x = __builtin_amdgcn_raw_buffer_load_b96(rv, (int)vo, so, 0);
#pragma unroll
                for (int i = 0; i < 3; i++) vr[r][i] = __uint_as_float(x[i]);
            } else if constexpr (NB == 2) {
                const f2 x = __builtin_bit_cast(f2, __builtin_amdgcn_raw_buffer_load_b64(rv, (int)vo, so, 0));
                vr[r][0] = x.x;
                vr[r][1] = x.y;
            } else {
                vr[r][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rv, (int)vo, so, 0));
            }
        }
    };
    if (wave < ntiles) load(wave);

    // q: the halves into LDS, a column in QL lanes (HD 96: the last eight idle)
    constexpr int QL = HD == 96 ? 32 : HD / 4, QC = 64 * W / QL, QP = 32 / QC > 0 ? 32 / QC : 1;
    {
        const int x4 = lane % QL;
        f4 x[QP];
#pragma unroll
        for (int i = 0; i < QP; i++) {
            const int c = min(c0 + (int)threadIdx.x / QL + QC * i, ncols - 1), h = kvh * G + c % G;
            x[i] = f4{};
            if (4 * x4 < HD) x[i] = *(const f4 *)(a.q + (int64_t)(s0 + c / G) * a.ldq + (int64_t)h * HD + 4 * x4);
        }
#pragma unroll
        for (int i = 0; i < QP; i++) {
            const int c = (int)threadIdx.x / QL + QC * i;
            x[i] *= score_scale(HD);
            float big = fmaxf(fmaxf(fabsf(x[i][0]), fabsf(x[i][1])), fmaxf(fabsf(x[i][2]), fabsf(x[i][3])));
#pragma unroll
            for (int y = 1; y < QL; y <<= 1) big = fmaxf(big, __shfl_xor(big, y, 64));
            const int ex = scale_exp(big);
#pragma unroll
            for (int y = 0; y < 4; y++) x[i][y] = ldexpf(x[i][y], -ex);
            h2 hi[2], lo[2];
            split2(x[i][0], x[i][1], hi[0], lo[0]);
            split2(x[i][2], x[i][3], hi[1], lo[1]);
            if (c < 32 && 4 * x4 < HD) {
                *(h4 *)&S.q[0][c][4 * x4] = h4{hi[0].x, hi[0].y, hi[1].x, hi[1].y};
                *(h4 *)&S.q[1][c][4 * x4] = h4{lo[0].x, lo[0].y, lo[1].x, lo[1].y};
                if (x4 == 0) S.w[0][c] = ldexpf(1.f / kHeld, ex);
            }
        }
    }
    __syncthreads();
    const float sc = S.w[0][j];
    float *const kput = &S.k[wave][lane / LR][4 * (lane % LR)];
    const float *const kget = &S.k[wave][j][8 * hh];

    float m = -FLT_MAX, l = 0.f;
    int odd = 0;
    f16v o[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) o[i] = f16v{};
    for (int t = wave; t < ntiles; t += W) {
        const int key0 = 32 * t;
        {  // whether the rows suit the halves
            float big = 0.f;
            float mk[NI], mv[16];
#pragma unroll
            for (int i = 0; i < NI; i++) {
                mk[i] = most(kr[0][i]);
#pragma unroll
                for (int f = 1; f < HD / DH; f++) mk[i] = __builtin_elementwise_maximum(mk[i], most(kr[f][i]));
                big = __builtin_elementwise_maximum(big, mk[i]);
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                mv[r] = fabsf(vr[r][0]);
#pragma unroll
                for (int i = 1; i < NB; i++) mv[r] = __builtin_elementwise_maximum(mv[r], fabsf(vr[r][i]));
                big = __builtin_elementwise_maximum(big, mv[r]);
            }
            odd |= __any(!(big < kRowHigh)) ? kHighRow : 0;
            if (some_low<LR>(mk) || some_low<32>(mv)) {
#pragma unroll
                for (int i = 0; i < NI; i++) odd |= low_row<LR>(mk[i]) ? kLowKey : 0;
#pragma unroll
                for (int r = 0; r < 16; r++) odd |= low_row<32>(mv[r]) ? kLowValue : 0;
            }
        }
        f16v s = f16v{};
#pragma unroll
        for (int c = 0; c < NC; c++) {
            if (c % (DH / 16) == 0) {
                // the wave's own stage: no barrier
                wave_lds_fence();
#pragma unroll
                for (int i = 0; i < NI; i++) *(f4 *)(kput + RPI * i * Lds::KS) = kr[c / (DH / 16)][i];
                wave_lds_fence();
            }
            const f4 x = *(const f4 *)(kget + 16 * (c % (DH / 16))), y = *(const f4 *)(kget + 16 * (c % (DH / 16)) + 4);
            h2 h[4], w[4];
            split2(x[0], x[1], kHeld, h[0], w[0]);
            split2(x[2], x[3], kHeld, h[1], w[1]);
            split2(y[0], y[1], kHeld, h[2], w[2]);
            split2(y[2], y[3], kHeld, h[3], w[3]);
            const h8 kh = {h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
            const h8 kl = {w[0].x, w[0].y, w[1].x, w[1].y, w[2].x, w[2].y, w[3].x, w[3].y};
            const h8 qh = *(const h8 *)&S.q[0][j][16 * c + 8 * hh], ql = *(const h8 *)&S.q[1][j][16 * c + 8 * hh];
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh, s, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (key0 + 31 > first) {
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (key0 + (r & 3) + 8 * (r >> 2) + 4 * hh > row) s[r] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
        mx = fmaxf(m, sc * max_halves(mx));
        const float corr = __builtin_amdgcn_exp2f(m - mx), off = kPShift - mx;
        m = mx;
        float ps[4] = {};
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, off));
            ps[r & 3] += s[r];
        }
        l = fmaf(l, corr, (ps[0] + ps[1]) + (ps[2] + ps[3]));
#pragma unroll
        for (int i = 0; i < NB; i++) o[i] *= corr;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const float p8[8] = {s[8 * ks],     s[8 * ks + 1], s[8 * ks + 2], s[8 * ks + 3],
                                 s[8 * ks + 4], s[8 * ks + 5], s[8 * ks + 6], s[8 * ks + 7]};
            h8 ph, pl;
            split8(p8, ph, pl);
#pragma unroll
            for (int i = 0; i < NB; i++) {
                h2 h[4], w[4];
#pragma unroll
                for (int x = 0; x < 4; x++)
                    split2(vr[8 * ks + 2 * x][i], vr[8 * ks + 2 * x + 1][i], kHeld, h[x], w[x]);
                const h8 vh = {h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
                const h8 vl = {w[0].x, w[0].y, w[1].x, w[1].y, w[2].x, w[2].y, w[3].x, w[3].y};
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph, o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl, o[i], 0, 0, 0);
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph, o[i], 0, 0, 0);
            }
        }
        if (t + W < ntiles) load(t + W);
    }
    // the waves meet: O = sum_w 2^(m_w - M) O_w / (kHeld L)
    l += __shfl_xor(l, 32, 64);
    __syncthreads();  // every wave is done with the queries and its stage
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) S.o[wave][j][NB * ((r & 3) + 8 * (r >> 2) + 4 * hh) + i] = o[i][r];
    if (hh == 0) {
        S.m[wave][j] = m;
        S.l[wave][j] = l;
    }
    if (lane == 0) S.odd[wave] = odd;
    __syncthreads();
    if (threadIdx.x < 32) {
        float M = S.m[0][j], L = 0.f;
#pragma unroll
        for (int w = 1; w < W; w++) M = fmaxf(M, S.m[w][j]);
        float f[W];
#pragma unroll
        for (int w = 0; w < W; w++) {
            f[w] = __builtin_amdgcn_exp2f(S.m[w][j] - M);
            L = fmaf(f[w], S.l[w][j], L);
        }
#pragma unroll
        for (int w = 0; w < W; w++) S.w[w][j] = f[w] / (kHeld * L);
    }
    odd = 0;
#pragma unroll
    for (int w = 0; w < W; w++) odd |= S.odd[w];
    __syncthreads();
    auto at = [&](int c, int d) {
        float O = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) O = fmaf(S.w[w][c], S.o[w][c][d], O);
        return O;
    };
    if (odd) {  // columns that the halves do not suit: over again
        if (wave == 0) {
            bool over = odd & kHighRow || (odd & kLowKey && sc >= kLowSc);
            if (odd & kLowValue) {
                float big = 0.f;
                for (int d = 0; d < HD / 2; d++) big = fmaxf(big, fabsf(at(j, HD / 2 * hh + d)));
                over |= max_halves(big) < kRowLow;
            }
            if (hh == 0) S.m[0][j] = over ? 1.f : 0.f;
            if (over && c0 + j < ncols)
                packed_fp32<HD>(a, qp, kb, vb, row, hh, a.out + (int64_t)(s0 + row) * a.ldo + (int64_t)head * HD);
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < 32 * HD; e += 64 * W) {
        const int c = e / HD, d = e % HD;
        if (c0 + c >= ncols || (odd && S.m[0][c] != 0.f)) continue;
        a.out[(int64_t)(s0 + (c0 + c) / G) * a.ldo + (int64_t)(kvh * G + (c0 + c) % G) * HD + d] = at(c, d);
    }
}

template <int NB, int W>
static void launch_split(const PackedAttn &a, int64_t cols)
{
    constexpr size_t lds = sizeof(SplitLds<NB, W>);
    static bool attr = false;
    if (!attr) {
        HOLO_CHECK(hipFuncSetAttribute((const void *)attn_packed_split_k<NB, W>,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        attr = true;
    }
    const dim3 grid(a.n_kv_heads, (unsigned)((cols + 31) / 32), a.b.n_seqs);
    hipLaunchKernelGGL((attn_packed_split_k<NB, W>), grid, dim3(64 * W), lds, stream(), a);
    HOLO_LAUNCH_CHECK();
}

template <int NB, int W>
static void launch_packed(const PackedAttn &a, int64_t cols)
{
    constexpr size_t lds = sizeof(PackedLds<NB>);
    static bool attr = false;
    if (!attr) {
        HOLO_CHECK(hipFuncSetAttribute((const void *)attn_packed_k<NB, W>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)lds));
        attr = true;
    }
    const dim3 grid(a.n_kv_heads, (unsigned)((cols + 32 * W - 1) / (32 * W)), a.b.n_seqs);
    hipLaunchKernelGGL((attn_packed_k<NB, W>), grid, dim3(64 * W), lds, stream(), a);
    HOLO_LAUNCH_CHECK();
}

// Which form (us; head_dim 128, 32 heads on 8 unless said):
//   keys shared by eight waves, up to a workgroup a CU: one prompt of 256 rows 13.3,
//   the forms below 15.1 21.2 26.6;
//   by four, up to three: one of 384 rows 18.4 (21.6 27.7 33.6), of 768 41.8 (46.5
//   47.0 53.8), two of 512 43.7 (51.0 36.4 41.8); not for up to two tiles of keys (16
//   of 64 rows 26.0, 35.1 14.3 19.2), where there is nothing to share;
//   128 columns, with 32 keys at most (one row 7.4; 8.9 8.5 9.2) and from there on;
//   256 in two groups where they fill the chip with long prompts: 4096 rows 365-391
//   (436-464 with 128), two of 1000 72.7 (90.4), four 128.5 (129.9), 16 of 999 475
//   (496); 16 of 256 rows 61.9 (59.9), eight of 384 63.2 (59.6), and with head_dim 64,
//   where more waves of 128 fit a SIMD, four of 1024 92.6 (81.1).  Between 500 and
//   1000 rows, which take 128 columns, the two are level (four of 640 65.7, 64.4;
//   head_dim 96, eight of 768 134.8, 132.3) or 256 are faster (four of 512 46.5,
//   54.0; four of 768 86.3, 95.2; two of 999 73.0, 90.7).
template <int NB>
static void run_packed(const PackedAttn &a, int64_t cols)
{
    const int64_t heads = (int64_t)a.n_kv_heads * a.b.n_seqs, cus = num_cus(), groups = (cols + 31) / 32 * heads;
    if (a.b.max_rows > 32 && groups <= cus) launch_split<NB, 8>(a, cols);
    else if (a.b.max_rows > 64 && groups <= 3 * cus) launch_split<NB, 4>(a, cols);
    else if (NB >= 3 && a.b.max_rows >= 1000 && (cols + 255) / 256 * heads >= cus) launch_packed<NB, 8>(a, cols);
    else launch_packed<NB, 4>(a, cols);
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
    const int64_t cols = (int64_t)a.b.max_rows * (n_heads / n_kv_heads);
    const int most_ld = 1 << 24;  // 32 rows' bytes in 31 bits
    if (!rows_ok(out, ldo, q_dim) || !rows_ok(q, ldq, q_dim) || !rows_ok(k, ldk, kv_dim) || !rows_ok(v, ldv, kv_dim) ||
        cols > 65535 * 32 || ldk >= most_ld || ldv >= most_ld) {
        HOLO_REJECT("holo_attention_packed: null or misaligned rows, rows that overlap, or more than one launch takes");
        return HOLO_EINVAL;
    }
    switch (head_dim) {
    case 32: run_packed<1>(a, cols); break;
    case 64: run_packed<2>(a, cols); break;
    case 96: run_packed<3>(a, cols); break;
    default: run_packed<4>(a, cols); break;
    }
    return 0;
}
