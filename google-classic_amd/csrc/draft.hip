// draft.hip -- drafted tokens (holo_forward.h): what the rows of a tree follow, and
// which of them stand against the target's probabilities.
#include "block_reduce.h"
#include "kv4.h"

#include <float.h>

namespace holo {

bool draft_rows_ok(const holo_batch_t *b, int words)
{
    return words > 0 && words <= 32 && b->max_rows <= 32 * words;
}

// The rows of an entry, without a cache.
__device__ __forceinline__ void batch_rows(const holo_batch_t &b, int s, int &first, int &take)
{
    first = min(max(b.cu_rows[s], 0), b.rows);
    take = min(min(max(b.cu_rows[s + 1], first), b.rows) - first, b.max_rows);
}

// ---- depth and mask of a tree's rows -------------------------------------------------------
//
// A thread climbs from its row; the rows that it meets come in falling order, so
// each word of the mask is whole when the next one begins.
__global__ __launch_bounds__(1024) void draft_plan_k(const int *parent, int *depth, uint32_t *mask, int words,
                                                     holo_batch_t b)
{
    __shared__ int up[1024];
    int first, take;
    batch_rows(b, blockIdx.x, first, take);
    const int i = threadIdx.x;
    if (i < take) {
        const int p = parent[first + i];
        up[i] = p >= 0 && p < i ? p : -1;
    }
    __syncthreads();
    if (i >= take) return;
    uint32_t *out = mask + (int64_t)(first + i) * words, bits = 0;
    int w = words - 1, n = -1;
    for (int j = i; j >= 0; j = up[j], n++) {
        for (; w > j >> 5; w--) {
            out[w] = bits;
            bits = 0;
        }
        bits |= 1u << (j & 31);
    }
    for (; w >= 0; w--) {
        out[w] = bits;
        bits = 0;
    }
    depth[first + i] = n;
}

// ---- verification ----------------------------------------------------------------------------

struct Verify {
    int *path, *n_path, *next;
    const float *target, *draft;
    int ldt, ldd, vocab, mode;
    const int *tokens, *parent;
    const float *u;
    int block;  // tokens of a partial sum, a multiple of 256
};

constexpr int kVerifyThreads = 1024, kVerifyWaves = kVerifyThreads / 64, kVerifySums = 2048;

__device__ __forceinline__ double wave_sum(double v)
{
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// The sum of the lanes up to this one.
__device__ __forceinline__ double wave_scan(double v, int lane)
{
    for (int off = 1; off < 64; off <<= 1) {
        const double w = __shfl_up(v, off, 64);
        if (lane >= off) v += w;
    }
    return v;
}

// A probability; 0 for what is negative or no finite number (only +denormal and
// +normal values pass).
__device__ __forceinline__ float probability(float p) { return __builtin_amdgcn_classf(p, 0x180) ? p : 0.f; }

// max(p - beta q, 0)
__device__ __forceinline__ double weight(float p, float q, double beta)
{
    const double w = (double)probability(p) - beta * (double)probability(q);
    return w > 0.0 ? w : 0.0;
}

// What the walk has reached, and the weights that it wants the sums of.
struct VerifyStep {
    double beta;
    int node, refused;  // refused: tokens, of a chosen draft
    bool sum, end;
};

// An entry's walk (the formulas: holo_forward.h) by one workgroup.  The first wave
// judges, 64 rows in its lanes: what a row needs of the two distributions depends on
// its parent alone and is loaded ahead.  Where the sum of a whole row of weights is
// needed, all waves sum blocks of tokens, in 64 bits; the same sums then lead to the
// next token's block.  Every sum has one order.
__global__ __launch_bounds__(kVerifyThreads) void draft_verify_k(Verify a, holo_batch_t b)
{
    __shared__ double sums[kVerifySums];
    __shared__ int refused_tok[1024];
    __shared__ VerifyStep step;
    int first, take;
    batch_rows(b, blockIdx.x, first, take);
    if (take <= 0) {
        if (threadIdx.x == 0) {
            a.n_path[blockIdx.x] = 0;
            a.next[blockIdx.x] = -1;
        }
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool drawn = a.mode != HOLO_DRAFT_CHOSEN;
    const int nsums = (a.vocab + a.block - 1) / a.block, per = (nsums + 63) / 64;

    // the first wave's: row judged last, rows that stand, N, beta, Q
    int node = 0, last = 0, count = 1, refused = 0;
    double left = 1.0, beta = 0.0, gone = 0.0;
    bool summed = false;  // sums are of this node and beta
    // its lanes' rows: base + lane
    int base = -1, r_up = -1, r_tok = -1;
    float r_p = 0.f, r_q = 0.f, r_u = 0.f;
    auto load_rows = [&](int at) {
        base = at;
        const int i = at + lane;
        r_up = i > 0 && i < take ? a.parent[first + i] : -1;
        if (r_up >= i) r_up = -1;
        r_tok = -1;
        r_p = r_q = 0.f;
        if (r_up < 0) return;
        r_tok = a.tokens[first + i];
        r_u = a.u[first + i];
        if (r_tok < 0 || r_tok >= a.vocab) {
            r_tok = -1;
            return;
        }
        r_p = a.target[(int64_t)(first + r_up) * a.ldt + r_tok];
        if (drawn) r_q = a.draft[(int64_t)(first + r_up) * a.ldd + r_tok];
    };
    // The next row behind `last` whose parent is the node; -1: none.
    auto next_row = [&]() {
        for (int at = (last + 1) & ~63; at < take; at += 64) {
            if (at != base) load_rows(at);
            const uint64_t hit = __ballot(r_up == node && at + lane > last);
            if (hit) return at + __ffsll((unsigned long long)hit) - 1;
        }
        return -1;
    };
    // Sum of all blocks; upto: of those up to the end of this lane's.
    auto total = [&](double &upto) {
        double s = 0.0;
        for (int i = lane * per; i < min((lane + 1) * per, nsums); i++) s += sums[i];
        upto = wave_scan(s, lane);
        return __shfl(upto, 63, 64);
    };
    // Judges rows until a sum is needed (true) or none is left.
    auto walk = [&]() {
        for (int j; (j = next_row()) >= 0;) {
            last = j;
            const int tok = __shfl(r_tok, j & 63, 64);
            const float p = __shfl(r_p, j & 63, 64), q = __shfl(r_q, j & 63, 64), u = __shfl(r_u, j & 63, 64);
            const double qx = probability(q);
            double px = weight(p, drawn ? q : 0.f, beta);
            bool stands;
            if (drawn) {
                stands = (double)u * qx * left < px * (1.0 - gone);
            } else {
                bool again = false;  // a token refused at this node before: nothing is left of it
                for (int i = lane; i < refused; i += 64) again |= refused_tok[i] == tok;
                if (__any(again)) px = 0.0;
                stands = (double)u * left < px;
            }
            if (stands) {
                if (lane == 0) a.path[first + count] = j;
                count++;
                node = j;
                left = 1.0;
                beta = gone = 0.0;
                refused = 0;
                summed = false;
            } else if (!drawn) {
                if (lane == 0) refused_tok[refused] = tok;
                wave_lds_fence();
                refused++;
                left -= px;
            } else if (tok >= 0 && gone < 1.0) {
                beta += left / (1.0 - gone);
                if (a.mode == HOLO_DRAFT_DISTINCT) gone += qx;
                return true;
            }
        }
        return false;
    };

    if (threadIdx.x == 0) a.path[first] = 0;
    for (;;) {
        if (wave == 0) {
            const bool more = walk();
            if (lane == 0) step = VerifyStep{beta, node, refused, more || !summed, !more};
        }
        __syncthreads();
        const VerifyStep s = step;
        const float *p = a.target + (int64_t)(first + s.node) * a.ldt;
        const float *q = drawn ? a.draft + (int64_t)(first + s.node) * a.ldd : p;
        const double w = drawn ? s.beta : 0.0;
        if (s.sum) {
            constexpr int U = 4;
            for (int e = wave; e < nsums; e += U * kVerifyWaves) {
                double sum[U] = {};
                for (int o = lane; o < a.block; o += 256) {
                    float x[U][4], y[U][4];
#pragma unroll
                    for (int i = 0; i < U; i++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int64_t at = (int64_t)(e + i * kVerifyWaves) * a.block + o + 64 * k;
                            x[i][k] = at < a.vocab ? p[at] : 0.f;
                            y[i][k] = at < a.vocab && w != 0.0 ? q[at] : 0.f;
                        }
#pragma unroll
                    for (int i = 0; i < U; i++)
#pragma unroll
                        for (int k = 0; k < 4; k++) sum[i] += weight(x[i][k], y[i][k], w);
                }
#pragma unroll
                for (int i = 0; i < U; i++) {
                    sum[i] = wave_sum(sum[i]);
                    if (lane == 0 && e + i * kVerifyWaves < nsums) sums[e + i * kVerifyWaves] = sum[i];
                }
            }
        }
        __syncthreads();
        if (s.end) break;
        if (wave == 0) {
            double upto;
            left = total(upto);
            summed = true;
        }
    }

    // Chosen: blocks with refused tokens once more, without them.
    const VerifyStep s = step;
    const float *p = a.target + (int64_t)(first + s.node) * a.ldt;
    const float *q = drawn ? a.draft + (int64_t)(first + s.node) * a.ldd : p;
    auto weight_at = [&](int64_t x) {
        if (x >= a.vocab) return 0.0;
        for (int i = 0; i < s.refused; i++)
            if (refused_tok[i] == x) return 0.0;
        return weight(p[x], s.beta != 0.0 ? q[x] : 0.f, s.beta);
    };
    for (int r = wave; r < s.refused; r += kVerifyWaves) {
        const int e = refused_tok[r] / a.block;
        if (refused_tok[r] < 0) continue;
        double sum = 0.0;
        for (int o = lane; o < a.block; o += 64) sum += weight_at((int64_t)e * a.block + o);
        sum = wave_sum(sum);
        if (lane == 0) sums[e] = sum;  // (a block of several: the same sum each time)
    }
    __syncthreads();
    if (wave != 0) return;
    for (int i = count + lane; i < take; i += 64) a.path[first + i] = -1;
    double upto;
    const double all = total(upto), at = (double)a.u[first] * all;
    int token = -1;
    if (all > 0.0) {
        // the first lane, block and token whose sum passes; past them by rounding: the last with a weight
        const double mine = upto - __shfl_up(upto, 1, 64);
        const uint64_t some = __ballot(lane == 0 ? upto > 0.0 : mine > 0.0), pass = __ballot(upto > at) & some;
        const int l = pass ? __ffsll((unsigned long long)pass) - 1 : 63 - __clzll((long long)some);
        double run = __shfl(upto, max(l - 1, 0), 64);
        if (l == 0) run = 0.0;
        int e = -1;
        for (int i = l * per; i < min((l + 1) * per, nsums); i++) {
            if (sums[i] == 0.0) continue;
            if (e >= 0) run += sums[e];
            e = i;
            if (run + sums[i] > at) break;
        }
        for (int o = 0; o < a.block; o += 64) {
            const int64_t x = (int64_t)e * a.block + o + lane;
            const double v = weight_at(x), to = run + wave_scan(v, lane);
            const uint64_t pos = __ballot(v > 0.0), in = __ballot(to > at) & pos;
            if (pos) token = e * a.block + o + (in ? __ffsll((unsigned long long)in) - 1 : 63 - __clzll((long long)pos));
            if (in) break;
            run = __shfl(to, 63, 64);
        }
    } else {
        // nothing weighs: the target's most probable token, the lowest of equals
        float best = -FLT_MAX;
        for (int x = lane; x < a.vocab; x += 64)
            if (p[x] > best || (token < 0 && p[x] == p[x])) {
                best = p[x];
                token = x;
            }
        for (int off = 32; off > 0; off >>= 1) {
            const float v = __shfl_xor(best, off, 64);
            const int x = __shfl_xor(token, off, 64);
            if (x >= 0 && (token < 0 || v > best || (v == best && x < token))) {
                best = v;
                token = x;
            }
        }
        token = max(token, 0);
    }
    if (lane == 0) {
        a.n_path[blockIdx.x] = count;
        a.next[blockIdx.x] = token;
    }
}

}  // namespace holo

using namespace holo;

extern "C" {

int holo_draft_plan(const int *parent, int *depth, uint32_t *mask, int words, const holo_batch_t *b)
{
    if (!batch_ok(b)) {
        HOLO_REJECT("holo_draft_plan: batch outside the supported set");
        return HOLO_EINVAL;
    }
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    holo_batch_t v = *b;
    v.max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    if (!parent || !depth || !mask || ((uintptr_t)parent & 3) || ((uintptr_t)depth & 3) || ((uintptr_t)mask & 3) ||
        !draft_rows_ok(&v, words)) {
        HOLO_REJECT("holo_draft_plan: a null or misaligned array, or more rows than the masks hold");
        return HOLO_EINVAL;
    }
    const int threads = (v.max_rows + 63) / 64 * 64;
    hipLaunchKernelGGL(draft_plan_k, dim3(b->n_seqs), dim3(threads), 0, stream(), parent, depth, mask, words, v);
    HOLO_LAUNCH_CHECK();
    return 0;
}

int holo_draft_verify(int *path, int *n_path, int *next, const float *target, const float *draft, int ldt, int ldd,
                      int vocab, const int *tokens, const int *parent, const float *u, int mode, const holo_batch_t *b)
{
    if (!batch_ok(b) || mode < HOLO_DRAFT_CHOSEN || mode > HOLO_DRAFT_DISTINCT) {
        HOLO_REJECT("holo_draft_verify: batch or mode outside the supported set");
        return HOLO_EINVAL;
    }
    if (b->n_seqs == 0 || b->rows == 0) return 0;
    holo_batch_t v = *b;
    v.max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    const void *all[] = {path, n_path, next, target, tokens, parent, u};
    bool ok = vocab > 0 && vocab <= 1 << 24 && ldt >= vocab && v.max_rows <= 1024;
    for (const void *p : all) ok = ok && p && !((uintptr_t)p & 3);
    if (mode != HOLO_DRAFT_CHOSEN) ok = ok && draft && !((uintptr_t)draft & 3) && ldd >= vocab;
    if (!ok) {
        HOLO_REJECT("holo_draft_verify: a null or misaligned array, rows that overlap, more than 1024 rows an entry or 2^24 tokens");
        return HOLO_EINVAL;
    }
    const int block = (int)(((int64_t)vocab + 256 * kVerifySums - 1) / (256 * kVerifySums)) * 256;
    const Verify a{path, n_path, next, target, draft, ldt, ldd, vocab, mode, tokens, parent, u, block};
    hipLaunchKernelGGL(draft_verify_k, dim3(b->n_seqs), dim3(kVerifyThreads), 0, stream(), a, v);
    HOLO_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
