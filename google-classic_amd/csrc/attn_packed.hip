// attn_packed.hip -- causal attention over packed sequences (holo_attention_packed).
//
// softmax(q . k_p / sqrt(hd)) . v_p over the rows p of the same sequence up to a
// row's own.  Both products run on v_mfma_f32_16x16x32_f16, transposed (S^T = K
// Q^T, O^T = V^T P^T), a lane holding one column (a row and query head); every
// operand is two f16 halves, hi hi + hi lo + lo hi in fp32: x - hi - lo within
// 2^-22 |x|.  q rows, and tiles of 32 keys and values, are scaled by a power of
// two to their largest value first, so that no value is too large or small for
// f16.
//
// A tile that holds an infinity or NaN is multiplied in fp32, value by value:
// the matrix instructions would hand it to the rows that do not see it.
#include "attn_tiles.h"
#include "kv4.h"

namespace holo {

struct PackedAttn {
    holo_batch_t b;
    float *out;
    const float *q, *k, *v;
    int ldo, ldq, ldk, ldv, n_heads, n_kv_heads;
    int ctiles;  // tiles of 16 columns that max_rows rows have
};

// The exponent that brings a largest value to [2^13, 2^14).
__device__ __forceinline__ int scale_exp(float big) { return big > 0.f ? ilogbf(big) - 13 : -4000; }

template <int NB, int W>
__global__ __launch_bounds__(64 * W) void attn_packed_k(PackedAttn a)
{
    constexpr int HD = 32 * NB, OS = HD + 4;
    __shared__ __align__(16) float lo_[W][16][OS];
    __shared__ float lm[W][16], ll[W][16];
    __shared__ int le[W];
    const int G = a.n_heads / a.n_kv_heads;
    const int kvh = blockIdx.y, ct = gridDim.x - 1 - blockIdx.x;  // the longest first
    const int s0 = min(max(a.b.cu_rows[blockIdx.z], 0), a.b.rows);
    const int n = min(min(max(a.b.cu_rows[blockIdx.z + 1], s0), a.b.rows) - s0, a.b.max_rows);
    const int ncols = n * G, c0 = 16 * ct;
    if (c0 >= ncols) return;
    const int last_row = (min(c0 + 16, ncols) - 1) / G, first_row = c0 / G;
    const int ntiles = (last_row + 32) >> 5;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int col = c0 + r;
    const bool valid = col < ncols;
    const int row = valid ? col / G : first_row, head = kvh * G + (valid ? col % G : 0);
    const float *qp = a.q + (int64_t)(s0 + row) * a.ldq + (int64_t)head * HD;
    const float *kb = a.k + (int64_t)s0 * a.ldk + (int64_t)kvh * HD;
    const float *vb = a.v + (int64_t)s0 * a.ldv + (int64_t)kvh * HD;

    h8 qh[NB], ql[NB];
    float sc;
    {
        float x[NB][8], big = 0.f;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const float4 u = *(const float4 *)(qp + 8 * (NB * g + j)), w = *(const float4 *)(qp + 8 * (NB * g + j) + 4);
            x[j][0] = u.x, x[j][1] = u.y, x[j][2] = u.z, x[j][3] = u.w;
            x[j][4] = w.x, x[j][5] = w.y, x[j][6] = w.z, x[j][7] = w.w;
#pragma unroll
            for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[j][i]));
        }
        big = fmaxf(big, __shfl_xor(big, 16, 64));
        big = fmaxf(big, __shfl_xor(big, 32, 64));
        const int ex = big > 0.f && big <= FLT_MAX ? scale_exp(big) : 0;
#pragma unroll
        for (int j = 0; j < NB; j++) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[j][i] = ldexpf(x[j][i], -ex);
            split8(x[j], qh[j], ql[j]);
        }
        sc = ldexpf(1.4426950408889634f / sqrtf((float)HD), ex);
    }

    float m = -FLT_MAX, l = 0.f;
    int E = -4000;  // the outputs are held times 2^-E
    f4 o[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) o[i] = f4{};

    for (int t = wave; t < ntiles; t += W) {
        const int p0 = 32 * t;
        // keys: rows p0 + 16 h + r (past the sequence: its last row, not seen)
        float kx[2][NB][8], big = 0.f;
        bool bad = false;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int pos = min(p0 + 16 * h + r, n - 1);
            const float *kp = kb + (int64_t)pos * a.ldk + 8 * NB * g;
#pragma unroll
            for (int j = 0; j < NB; j++) {
                const float4 u = *(const float4 *)(kp + 8 * j), w = *(const float4 *)(kp + 8 * j + 4);
                float *x = kx[h][j];
                x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    bad |= !(fabsf(x[i]) <= FLT_MAX);
                    big = fmaxf(big, fabsf(x[i]));
                }
            }
        }
        float p[8];
        if (__any(bad)) {
            for (int i = 0; i < 8; i++) {
                const int pos = p0 + v_pos(g, i);
                float d = 0.f;
                if (pos <= row)
                    for (int j = 0; j < HD; j++) d = fmaf(qp[j], kb[(int64_t)pos * a.ldk + j], d);
                p[i] = d * (1.4426950408889634f / sqrtf((float)HD));
            }
        } else {
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) big = fmaxf(big, __shfl_xor(big, x, 64));
            const int ek = big > 0.f ? scale_exp(big) : 0;
            f4 s[2] = {f4{}, f4{}};
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < NB; j++) {
                    h8 kh, kl;
#pragma unroll
                    for (int i = 0; i < 8; i++) kx[h][j][i] = ldexpf(kx[h][j][i], -ek);
                    split8(kx[h][j], kh, kl);
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[j], s[h], 0, 0, 0);
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[j], s[h], 0, 0, 0);
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[j], s[h], 0, 0, 0);
                }
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = ldexpf(s[i >> 2][i & 3] * sc, ek);
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (p0 + v_pos(g, i) > row) p[i] = -INFINITY;
        float mx = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
        if (__any(mx > m + kMaxSlack)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
            const float w = __builtin_amdgcn_exp2f(m - mx);
            m = mx;
            l *= w;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) o[i] *= w;
        }
        float ps = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[i] = __builtin_amdgcn_exp2f(p[i] - m + kPShift);
            ps += p[i];
        }
        l += ps;
        // values: dim 16 i + r of the lane's eight positions
        float vx[2 * NB][8];
        big = 0.f;
        bad = false;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int pos = p0 + v_pos(g, j);
            const bool in = pos <= last_row;
            const float *vp = vb + (int64_t)min(pos, last_row) * a.ldv + r;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) {
                const float y = in ? vp[16 * i] : 0.f;
                vx[i][j] = y;
                bad |= !(fabsf(y) <= FLT_MAX);
                big = fmaxf(big, fabsf(y));
            }
        }
        if (__any(bad)) {
            if (E < -2000) E = 0;
            for (int x = 0; x <= last_row - p0 && x < 32; x++) {
                // x's probability: value 4 (x / 16) + x % 4 of lane group (x / 4) % 4
                float w = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i == 4 * (x >> 4) + (x & 3)) w = p[i];
                w = __shfl(w, ((x >> 2) & 3) * 16 + r, 64);
                if (p0 + x > row) continue;
                const float *vp = vb + (int64_t)(p0 + x) * a.ldv + 4 * g;
#pragma unroll
                for (int i = 0; i < 2 * NB; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[i][j] = fmaf(w, ldexpf(vp[16 * i + j], -E), o[i][j]);
            }
            continue;
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) big = fmaxf(big, __shfl_xor(big, x, 64));
        const int ev = scale_exp(big);
        if (ev <= -4000) continue;  // values of zero
        if (ev > E) {
#pragma unroll
            for (int i = 0; i < 2 * NB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[i][j] = ldexpf(o[i][j], E - ev);
            E = ev;
        }
        h8 ph, pl;
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = ldexpf(p[i], ev - E);
        split8(p, ph, pl);
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            h8 vh, vl;
#pragma unroll
            for (int j = 0; j < 8; j++) vx[i][j] = ldexpf(vx[i][j], -ev);
            split8(vx[i], vh, vl);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph, o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl, o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph, o[i], 0, 0, 0);
        }
    }

    // the waves meet: O = sum_w 2^(m_w - M + E_w) O_w
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) *(f4 *)&lo_[wave][r][16 * i + 4 * g] = o[i];
    if (g == 0) {
        lm[wave][r] = m;
        ll[wave][r] = l;
    }
    if (lane == 0) le[wave] = E;
    __syncthreads();
    int top = le[0];
#pragma unroll
    for (int w = 1; w < W; w++) top = max(top, le[w]);
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
            O += ldexpf(f, le[w] - top) * *(const f4 *)&lo_[w][c][d];
        }
        const float f = 1.0f / L;  // a row sees itself
        f4 y = O * f;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = ldexpf(y[j], top);
        const int h = kvh * G + (c0 + c) % G;
        *(f4 *)(a.out + (int64_t)(s0 + (c0 + c) / G) * a.ldo + (int64_t)h * HD + d) = y;
    }
}

template <int NB>
static void run_packed(const PackedAttn &a)
{
    constexpr int W = 4;
    hipLaunchKernelGGL((attn_packed_k<NB, W>), dim3(a.ctiles, a.n_kv_heads, a.b.n_seqs), dim3(64 * W), 0, stream(), a);
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
    PackedAttn a{*b, out, q, k, v, ldo, ldq, ldk, ldv, n_heads, n_kv_heads, 0};
    a.b.max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    const int64_t cols = (int64_t)a.b.max_rows * (n_heads / n_kv_heads);
    if (!rows_ok(out, ldo, q_dim) || !rows_ok(q, ldq, q_dim) || !rows_ok(k, ldk, kv_dim) || !rows_ok(v, ldv, kv_dim) ||
        cols > 0x7FFFFF00) {
        HOLO_REJECT("holo_attention_packed: null or misaligned rows, or rows that overlap");
        return HOLO_EINVAL;
    }
    a.ctiles = (int)((cols + 15) / 16);
    switch (head_dim) {
    case 32: run_packed<1>(a); break;
    case 64: run_packed<2>(a); break;
    case 96: run_packed<3>(a); break;
    default: run_packed<4>(a); break;
    }
    return 0;
}
