// kv4_rope.hip -- rows rotated to their positions on the way into the 4-bit cache
// (holo_kv4_append_rope), and the pairs' frequencies (holo_rope_freqs).
#include "kv4_quant.h"

#include <cmath>

namespace holo {

struct RopeRows {
    holo_rope_t r;
    const float *q, *k, *v;
    float *q_out, *k_out;
    int ldq, ldk, ldv, ldqo, ldko, n_heads;
    const int *depth;
};

// Query heads of a workgroup.
constexpr int kRopeHeads = 4;

// A workgroup takes the rows of one tile of positions, one KV head and up to four of
// the query heads that share it (its first workgroup of them the keys and values
// too).  The angle of a (position, pair) is computed once for all of these, in 64
// bits: position * freq reaches 10^5 and more, and a key next to the border of two
// codes must fall to the same side at every caller.  A thread has both values of its
// pairs, so rows may be rotated in place; the keys go to the quantisation, which
// takes whole blocks of 32, through LDS.
template <int NB>
__global__ __launch_bounds__(256) void kv4_append_rope_k(Kv4View c, holo_batch_t b, RopeRows a)
{
    constexpr int HD = 32 * NB, P = HD / 2, GROUPS = 256 / P, KS = HD + 4;
    __shared__ __align__(16) float lk[32 * KS];
    __shared__ __align__(16) uint8_t lv[32 * HD];
    const Kv4Entry e = kv4_entry(c, b, blockIdx.z);
    const int kvh = blockIdx.y % c.n_kv_heads, part = blockIdx.y / c.n_kv_heads;
    const int G = a.n_heads / c.n_kv_heads, h0 = part * kRopeHeads, heads = min(G - h0, kRopeHeads);
    const int from = e.len - e.rows;  // position of the entry's first row, which may be negative
    if ((int)blockIdx.x > (e.take + 30) / 32) return;
    const int t = (from >> 5) + (int)blockIdx.x, p0 = 32 * t;
    const int lo = max(from - p0, 0), hi = min(from + e.take - p0, 32);
    if (lo >= hi) return;
    const int64_t row0 = (int64_t)e.first + p0 - from;
    const bool keys = part == 0;
    uint8_t *tile = keys && t >= 0 ? kv4_tile<NB>(c, e, kvh, t) : nullptr;

    const int i = threadIdx.x % P, g = threadIdx.x / P;
    const bool turns = 2 * i < a.r.dims;
    // the pair's values: dims d0 and d1 of a head
    const int d0 = turns && !a.r.interleaved ? i : 2 * i, d1 = turns && !a.r.interleaved ? i + a.r.dims / 2 : 2 * i + 1;
    const double freq = turns ? a.r.freq[i] * M_1_PI : 0.0;
    // groups of P threads take rows, and where there are few rows each some of the heads
    const int n = hi - lo, slots = min(max(GROUPS / n, 1), max(heads + keys, 1)), rows = GROUPS / slots;
    if (g < rows * slots)
        for (int p = lo + g / slots; p < hi; p += rows) {
            const int64_t row = row0 + p;
            const float *qp = a.q + row * a.ldq + (int64_t)(kvh * G + h0) * HD;
            float *qo = a.q_out + row * a.ldqo + (int64_t)(kvh * G + h0) * HD;
            const float *kp = a.k + row * a.ldk + kvh * HD;
            float x[kRopeHeads + 1], y[kRopeHeads + 1];
#pragma unroll
            for (int j = 0; j <= kRopeHeads; j++) {  // head h0 + s; behind the last, the key
                const int s = g % slots + j * slots;
                if (s > heads || (s == heads && !keys)) break;
                const float *at = s < heads ? qp + s * HD : kp;
                x[j] = at[d0];
                y[j] = at[d1];
            }
            double cs = 1.0, sn = 0.0;
            if (turns) {
                double turn = ((double)from + (double)(a.depth ? a.depth[row] : p + p0 - from)) * freq;  // half turns
                turn -= 2.0 * rint(0.5 * turn);
                sincospi(turn, &sn, &cs);
                cs *= a.r.scale;
                sn *= a.r.scale;
            }
#pragma unroll
            for (int j = 0; j <= kRopeHeads; j++) {
                const int s = g % slots + j * slots;
                if (s > heads || (s == heads && !keys)) break;
                float u = x[j], w = y[j];
                if (turns) {
                    u = (float)(x[j] * cs - y[j] * sn);
                    w = (float)(x[j] * sn + y[j] * cs);
                }
                if (s < heads) {
                    qo[s * HD + d0] = u;
                    qo[s * HD + d1] = w;
                } else {
                    lk[p * KS + d0] = u;
                    lk[p * KS + d1] = w;
                    if (a.k_out) {
                        a.k_out[row * a.ldko + kvh * HD + d0] = u;
                        a.k_out[row * a.ldko + kvh * HD + d1] = w;
                    }
                }
            }
        }
    if (!tile) return;
    Kv4VWords<NB> words(tile, lo, hi);
    __syncthreads();
    const int lane = threadIdx.x & 7;
    for (int j = threadIdx.x >> 3; j < n * NB; j += 32) {
        const int p = lo + j / NB, blk = j % NB;
        const float4 kx = *(const float4 *)&lk[p * KS + 32 * blk + 4 * lane];
        const float4 vx = *(const float4 *)(a.v + (row0 + p) * a.ldv + kvh * HD + 32 * blk + 4 * lane);
        kv4_put<NB>(tile, lv, p, blk, lane, kx, vx);
    }
    __syncthreads();
    words.store(lv);
}

}  // namespace holo

using namespace holo;

extern "C" {

int holo_kv4_append_rope(const holo_kv4_t *c, int layer, const holo_rope_t *r, const float *q, const float *k,
                         const float *v, int ldq, int ldk, int ldv, float *q_out, float *k_out, int ldqo, int ldko,
                         int n_heads, const int *depth, const holo_batch_t *b)
{
    if (!kv4_call_ok(c, layer, b)) {
        HOLO_REJECT("holo_kv4_append_rope: cache, layer or batch outside the supported set");
        return HOLO_EINVAL;
    }
    if (!r || !r->freq || ((uintptr_t)r->freq & 7) || r->dims < 2 || r->dims % 2 || r->dims > c->head_dim ||
        !std::isfinite(r->scale)) {
        HOLO_REJECT("holo_kv4_append_rope: rotation outside the supported set");
        return HOLO_EINVAL;
    }
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    const int64_t dim = (int64_t)c->n_kv_heads * c->head_dim, qdim = (int64_t)n_heads * c->head_dim;
    if (!rows_ok(k, ldk, dim) || !rows_ok(v, ldv, dim) || (k_out && !rows_ok(k_out, ldko, dim)) ||
        ((uintptr_t)depth & 3)) {
        HOLO_REJECT("holo_kv4_append_rope: null or misaligned keys or values, or rows that overlap");
        return HOLO_EINVAL;
    }
    const int G = n_heads < 0 || n_heads % c->n_kv_heads ? -1 : n_heads / c->n_kv_heads;
    const int64_t parts = G > kRopeHeads ? (G + kRopeHeads - 1) / kRopeHeads : 1;
    if (G < 0 || (G > 0 && (!rows_ok(q, ldq, qdim) || !rows_ok(q_out, ldqo, qdim))) || parts * c->n_kv_heads > 65535) {
        HOLO_REJECT("holo_kv4_append_rope: query heads, or their rows, outside the supported set");
        return HOLO_EINVAL;
    }
    const Kv4View w = kv4_view(c, layer);
    const int take = b->max_rows < b->rows ? b->max_rows : b->rows;
    const dim3 grid((unsigned)(take + 30) / 32 + 1, (unsigned)(parts * c->n_kv_heads), b->n_seqs);
    const RopeRows a{*r, q, k, v, q_out, k_out, ldq, ldk, ldv, ldqo, ldko, n_heads, depth};
    auto run = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream(), w, *b, a); };
    switch (c->head_dim) {
    case 32: run(kv4_append_rope_k<1>); break;
    case 64: run(kv4_append_rope_k<2>); break;
    case 96: run(kv4_append_rope_k<3>); break;
    default: run(kv4_append_rope_k<4>); break;
    }
    HOLO_LAUNCH_CHECK();
    return 0;
}

int holo_rope_freqs(double *freq, float *scale, const holo_rope_scaling_t *s)
{
    const bool known = s && s->kind >= HOLO_ROPE_PLAIN && s->kind <= HOLO_ROPE_RAMP;
    if (!freq || !known || s->dims < 2 || s->dims % 2 || s->dims > 128 || !(s->base > 1.0) || !std::isfinite(s->base) ||
        (s->kind != HOLO_ROPE_PLAIN && (!(s->factor >= 1.0) || !std::isfinite(s->factor))) ||
        (s->kind == HOLO_ROPE_BASE && s->dims == 2) ||
        (s->kind >= HOLO_ROPE_BANDS && (s->trained <= 0 || !(s->low > 0.0) || !(s->high > s->low) || !std::isfinite(s->high)))) {
        HOLO_REJECT("holo_rope_freqs: a null pointer, or parameters outside the supported set");
        return HOLO_EINVAL;
    }
    const int n = s->dims / 2;
    for (int i = 0; s->divisors && i < n; i++)
        if (!(s->divisors[i] > 0.f) || !std::isfinite(s->divisors[i])) {
            HOLO_REJECT("holo_rope_freqs: a divisor that is not positive and finite");
            return HOLO_EINVAL;
        }
    const double two_pi = 2.0 * M_PI, f = s->factor;
    const double base = s->kind == HOLO_ROPE_BASE ? s->base * pow(f, s->dims / (s->dims - 2.0)) : s->base;
    // RAMP: the pair that turns `turns` times over the trained positions
    auto pair_of = [&](double turns) { return s->dims * log(s->trained / (turns * two_pi)) / (2.0 * log(s->base)); };
    for (int i = 0; i < n; i++) {
        double w = pow(base, -2.0 * i / s->dims);
        if (s->divisors) w /= s->divisors[i];
        if (s->kind == HOLO_ROPE_LINEAR) w /= f;
        double keep = 1.0;  // the share of w left as it is
        if (s->kind == HOLO_ROPE_BANDS) {
            keep = (s->trained * w / two_pi - s->low) / (s->high - s->low);
        } else if (s->kind == HOLO_ROPE_RAMP) {
            const double first = fmax(floor(pair_of(s->high)), 0.0);
            const double last = fmin(ceil(pair_of(s->low)), s->dims - 1.0);
            keep = 1.0 - (i - first) / fmax(last - first, 0.001);
        }
        keep = fmin(fmax(keep, 0.0), 1.0);
        if (s->kind >= HOLO_ROPE_BANDS) w = keep * w + (1.0 - keep) * (w / f);
        freq[i] = w;
    }
    if (scale) *scale = s->kind == HOLO_ROPE_RAMP ? (float)(0.1 * log(f) + 1.0) : 1.f;
    return 0;
}

}  // extern "C"
