// kv4_rope.hip -- rows rotated to their positions on the way into the 4-bit cache
// (holo_kv4_append_rope), and the pairs' frequencies (holo_rope_freqs).
#include "kv4_quant.h"

#include <cmath>
#include <type_traits>

namespace holo {

struct RopeRows {
    holo_rope_t r;
    const float *q, *k, *v;
    float *q_out, *k_out;
    int ldq, ldk, ldv, ldqo, ldko, n_heads;
    const int *depth;
};

// Query heads of a workgroup (one: 43.1 us for the prompts below with the read back; two
// 39.7, four 46.2).
constexpr int kRopeHeads = 2;

// The sine and cosine of position * freq, times the scale.  half_turns: of the freq.
__device__ __forceinline__ void turn_by(double position, double half_turns, float scale, double &cs, double &sn)
{
    double t = position * half_turns;
    t -= 2.0 * rint(0.5 * t);
    sincospi(t, &sn, &cs);
    cs *= scale;
    sn *= scale;
}

__device__ __forceinline__ void turn_pair(float &x, float &y, double cs, double sn)
{
    const float u = (float)(x * cs - y * sn);
    y = (float)(x * sn + y * cs);
    x = u;
}

// A workgroup takes the rows of one tile of positions, one KV head and up to two of
// the query heads that share it (its first workgroup of them the keys and values
// too).  The angle of a (position, pair) is computed once for all of these, in 64
// bits: position * freq reaches 10^5 and more, and a key next to the border of two
// codes must fall to the same side at every caller.  A thread has both values of its
// pairs, so rows may be rotated in place; the keys go to the quantisation, which
// takes whole blocks of 32, through LDS.  WIDE: four pairs a thread, in 16-byte pieces
// (dims a multiple of 8); else one.
//
// What bounds it: prompts of up to 1000 rows (2400 in all), 32 heads on 8 of 128, 96 dims
// turning, rotated keys out as well: 109 MB, 21-23 us at a large copy's rate, take 26-28 in a kernel
// trace; vector instructions (a third in 64 bits) issue in about a third of the cycles, the rest is
// memory, the rows written among it at the launch's end (past the caches they take 37.4 us with
// the read back, through them 39.7).  Four sequences of 8 rows 6.6: lengths, page, rows, angles one
// after the other.  (Of other
// dims, one pair a thread: from call to call 98 dims take 25.7 us in halves and 32.0 interleaved,
// 96 dims 25.0 and 28.2.  The pairs' layout not a template, 55 with the read back.)
template <int NB, bool WIDE, bool INTERLEAVED>
__global__ __launch_bounds__(256) void kv4_append_rope_k(Kv4View c, holo_batch_t b, RopeRows a, int first)
{
    constexpr int HD = 32 * NB, N = WIDE ? 4 : 1, P = HD / (2 * N), GROUPS = 256 / P, KS = HD + 4;
    typedef float vec __attribute__((ext_vector_type(N)));
    __shared__ __align__(16) float lk[32 * KS];
    __shared__ __align__(16) uint8_t lv[32 * HD];
    const Kv4Entry e = kv4_entry(c, b, blockIdx.z);
    const int kvh = blockIdx.y % c.n_kv_heads, part = blockIdx.y / c.n_kv_heads;
    const int G = a.n_heads / c.n_kv_heads, h0 = part * kRopeHeads, heads = min(G - h0, kRopeHeads);
    const int from = e.len - e.rows;  // position of the entry's first row, which may be negative
    const int nth = first + (int)blockIdx.x;  // of the entry's tiles
    if (nth > (e.take + 30) / 32) return;
    const int t = (from >> 5) + nth, p0 = 32 * t;
    const int lo = max(from - p0, 0), hi = min(from + e.take - p0, 32), n = hi - lo;
    if (n <= 0) return;
    const int64_t row0 = (int64_t)e.first + p0 - from;
    const bool keys = part == 0;
    uint8_t *tile = keys && t >= 0 ? kv4_tile<NB>(c, e, kvh, t) : nullptr;

    const int i = threadIdx.x % P, g = threadIdx.x / P;
    const bool turns = 2 * N * i < a.r.dims;
    // the pairs' values: N of a head from d0 on, and N from d1 on
    const int d0 = turns && !INTERLEAVED ? N * i : 2 * N * i, d1 = turns && !INTERLEAVED ? N * i + a.r.dims / 2 : 2 * N * i + N;
    double freq[N], cs[N], sn[N];
#pragma unroll
    for (int k = 0; k < N; k++) freq[k] = turns ? a.r.freq[N * i + k] * M_1_PI : 0.0;
    auto angles = [&](int p) {
        if (!turns) return;
        const double position = (double)from + (double)(a.depth ? a.depth[row0 + p] : p + p0 - from);
#pragma unroll
        for (int k = 0; k < N; k++) turn_by(position, freq[k], a.r.scale, cs[k], sn[k]);
    };
    auto turn = [&](vec &x, vec &y) {
        if (!turns) return;
        float v[2 * N];
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = x[k], v[N + k] = y[k];
#pragma unroll
        for (int k = 0; k < N; k++)
            if (INTERLEAVED && N > 1) turn_pair(v[2 * k], v[2 * k + 1], cs[k], sn[k]);
            else turn_pair(v[k], v[N + k], cs[k], sn[k]);
#pragma unroll
        for (int k = 0; k < N; k++) x[k] = v[k], y[k] = v[N + k];
    };
    auto put_key = [&](int p, const vec &x, const vec &y) {
        *(vec *)(lk + p * KS + d0) = x;
        *(vec *)(lk + p * KS + d1) = y;
        if (a.k_out) {
            *(vec *)(a.k_out + (row0 + p) * a.ldko + kvh * HD + d0) = x;
            *(vec *)(a.k_out + (row0 + p) * a.ldko + kvh * HD + d1) = y;
        }
    };
    const float *q = a.q + (int64_t)(kvh * G + h0) * HD, *key = a.k + kvh * HD;
    float *q_out = a.q_out + (int64_t)(kvh * G + h0) * HD;
    if (g >= GROUPS) {
    } else if (n >= GROUPS) {  // many rows: a group takes whole rows
        for (int p = lo + g; p < hi; p += GROUPS) {
            const float *in = q + (row0 + p) * a.ldq, *kin = key + (row0 + p) * a.ldk;
            float *out = q_out + (row0 + p) * a.ldqo;
            vec x[kRopeHeads], y[kRopeHeads], kx, ky;
#pragma unroll
            for (int j = 0; j < kRopeHeads; j++)
                if (j < heads) {
                    x[j] = *(const vec *)(in + j * HD + d0);
                    y[j] = *(const vec *)(in + j * HD + d1);
                }
            if (keys) {
                kx = *(const vec *)(kin + d0);
                ky = *(const vec *)(kin + d1);
            }
            angles(p);
#pragma unroll
            for (int j = 0; j < kRopeHeads; j++)
                if (j < heads) {
                    turn(x[j], y[j]);
                    __builtin_nontemporal_store(x[j], (vec *)(out + j * HD + d0));
                    __builtin_nontemporal_store(y[j], (vec *)(out + j * HD + d1));
                }
            if (keys) {
                turn(kx, ky);
                put_key(p, kx, ky);
            }
        }
    } else {  // few: a head of a row
        const int units = max(heads, 0) + keys;
        for (int u = g; u < n * units; u += GROUPS) {
            const int p = lo + u / units, s = u % units;
            const float *in = s < heads ? q + (row0 + p) * a.ldq + s * HD : key + (row0 + p) * a.ldk;
            vec x = *(const vec *)(in + d0), y = *(const vec *)(in + d1);
            angles(p);
            turn(x, y);
            if (s < heads) {
                float *out = q_out + (row0 + p) * a.ldqo + s * HD;
                *(vec *)(out + d0) = x;
                *(vec *)(out + d1) = y;
            } else {
                put_key(p, x, y);
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
    const RopeRows a{*r, q, k, v, q_out, k_out, ldq, ldk, ldv, ldqo, ldko, n_heads, depth};
    const bool wide = r->dims % 8 == 0;
    auto run = [&](auto kern) {
        kv4_tile_launches(take, [&](int first, int n) {
            hipLaunchKernelGGL(kern, dim3(n, (unsigned)(parts * c->n_kv_heads), b->n_seqs), dim3(256), 0, stream(), w, *b, a, first);
        });
    };
    auto pick = [&](auto nb) {
        if (r->interleaved) wide ? run(kv4_append_rope_k<nb, true, true>) : run(kv4_append_rope_k<nb, false, true>);
        else wide ? run(kv4_append_rope_k<nb, true, false>) : run(kv4_append_rope_k<nb, false, false>);
    };
    switch (c->head_dim) {
    case 32: pick(std::integral_constant<int, 1>()); break;
    case 64: pick(std::integral_constant<int, 2>()); break;
    case 96: pick(std::integral_constant<int, 3>()); break;
    default: pick(std::integral_constant<int, 4>()); break;
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
