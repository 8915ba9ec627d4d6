// draft.hip -- drafted tokens (holo_forward.h): what the rows of a tree follow, and
// which of them stand against the target's probabilities.
#include "kv4.h"
#include "stream_scratch.h"

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
//
// Probabilities are given, so that what stands and the next token do not depend on how a
// kernel rounds an exponential: products and sums of them are in 64 bits, where two orders
// of a sum differ by 10^-16 and a token's border is hit once in 10^11 calls.  After
// refusals the weights left are max(p - beta q, 0) in closed form, so that a sum N over the row is
// all that a refusal costs.
//
// What bounds it: latency.  64 chains of 5 rows, 32000 tokens, 16.4 MB of the rows that the
// walks end at (3.4 us at a large copy's rate): 12.7-13.1 us (chosen 13.6; 128256 tokens 20.7), two launches of 5 and 4.4 with loads
// that depend on each other (rows, tokens, probabilities; then the row); with one workgroup an entry for
// all of it 42.  16 trees of up to 26 rows 26-32 (78; chosen, where a refusal costs no sum, 13.8;
// of 128256 tokens 83-97): the second launch goes from refusal to refusal, some 4 us each, half of it 64-bit arithmetic; with the row's probabilities kept in registers
// the compiler spills them (50-57).

struct Verify {
    int *path, *n_path, *next;
    const float *target, *draft;
    int ldt, ldd, vocab, mode;
    const int *tokens, *parent;
    const float *u;
    int block;  // tokens of a partial sum, a multiple of 256
    struct WalkState *states;  // of each entry: where its walk stands, and the sums of the weights there
    double *sums;
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

// max(p - beta q, 0), of one rounding: every place that asks for a token's weight gets the same.
__device__ __forceinline__ double weight(float p, float q, double beta)
{
    const double w = fma(-beta, (double)probability(q), (double)probability(p));
    return w > 0.0 ? w : 0.0;
}

// A random number: what lies outside [0, 1) is the nearest number inside, NaN is 0.
__device__ __forceinline__ float unit(float u) { return fminf(fmaxf(u, 0.f), 0x1.fffffep-1f); }

// Where a walk stands (the formulas: holo_forward.h).
struct WalkState {
    double left, beta, gone;  // N, beta, Q
    int node, last, count;    // the row that it is at, the row judged last, rows that stand
    int asks;                 // the row judged last is refused, another follows, and N is wanted for it
};

// A walk over an entry's rows by one wave, 64 rows in its lanes: what a row needs of
// the two distributions depends on its parent alone and is loaded ahead.
struct Walk {
    const Verify &a;
    int first, take, lane;
    WalkState s;
    int base = -1, up = -1, tok = -1;  // the lanes' rows: base + lane
    float p = 0.f, q = 0.f, u = 0.f;

    __device__ __forceinline__ Walk(const Verify &a, int first, int take, int lane) : a(a), first(first), take(take), lane(lane)
    {
        s = WalkState{1.0, 0.0, 0.0, 0, 0, 1, 0};
    }
    __device__ __forceinline__ bool drawn() const { return a.mode != HOLO_DRAFT_CHOSEN; }
    __device__ __forceinline__ void load_rows(int at)
    {
        base = at;
        const int i = at + lane;
        up = i > 0 && i < take ? a.parent[first + i] : -1;
        if (up >= i) up = -1;
        tok = -1;
        p = q = 0.f;
        if (up < 0) return;
        tok = a.tokens[first + i];
        u = unit(a.u[first + i]);
        if (tok < 0 || tok >= a.vocab) {
            tok = -1;
            return;
        }
        p = a.target[(int64_t)(first + up) * a.ldt + tok];
        if (drawn()) q = a.draft[(int64_t)(first + up) * a.ldd + tok];
    }
    // The next row behind the last one whose parent is the node; -1: none.
    __device__ __forceinline__ int next_row()
    {
        for (int at = (s.last + 1) & ~63; at < take; at += 64) {
            if (at != base) load_rows(at);
            const uint64_t hit = __ballot(up == s.node && at + lane > s.last);
            if (hit) return at + __ffsll((unsigned long long)hit) - 1;
        }
        return -1;
    }
    // Chosen: whether row j's token is that of an earlier row behind the node, which was refused.
    __device__ __forceinline__ bool again(int j, int t)
    {
        bool same = __any(up == s.node && base + lane < j && tok == t);
        for (int at = 0; at < base && !same; at += 64)
            same = __any(a.parent[first + at + lane] == s.node && at + lane > s.node && a.tokens[first + at + lane] == t);
        return same;
    }
    // Judges rows until N is wanted (asks) or none is left; stood(i, row): row i of the path.
    template <typename F>
    __device__ __forceinline__ void go(F stood)
    {
        s.asks = 0;
        for (int j; (j = next_row()) >= 0;) {
            s.last = j;
            const int t = __shfl(tok, j & 63, 64);
            const float pj = __shfl(p, j & 63, 64), qj = __shfl(q, j & 63, 64), uj = __shfl(u, j & 63, 64);
            const double qx = probability(qj);
            double px = weight(pj, qj, s.beta);
            bool stands;
            if (drawn()) {
                stands = (double)uj * qx * s.left < px * (1.0 - s.gone);
            } else {
                if (t >= 0 && again(j, t)) px = 0.0;
                stands = (double)uj * s.left < px;
            }
            if (stands) {
                stood(s.count, j);
                s = WalkState{1.0, 0.0, 0.0, j, j, s.count + 1, 0};
            } else if (!drawn()) {
                s.left -= px;
            } else if (t >= 0 && s.gone < 1.0) {
                s.beta += s.left / (1.0 - s.gone);
                if (a.mode == HOLO_DRAFT_DISTINCT) s.gone += qx;
                s.asks = next_row() >= 0;  // (behind the last one the sum is part of finding the next token)
                return;
            }
        }
    }
};

// The sums of the weights of blocks e, e + stride, .. (U of them), by a wave: the loads
// of all of them under way at once.
template <int U>
__device__ __forceinline__ void block_sums(const Verify &a, const float *p, const float *q, double beta, int e, int stride, int lane,
                                           double *to, int nsums)
{
    double sum[U] = {};
    for (int o = lane; o < a.block; o += 256) {
        float x[U][4], y[U][4];
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t at = (uint32_t)((e + i * stride) * a.block + o + 64 * k);  // (vocab up to 2^24)
                x[i][k] = at < (uint32_t)a.vocab ? p[at] : 0.f;
                y[i][k] = at < (uint32_t)a.vocab && beta != 0.0 ? q[at] : 0.f;
            }
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) sum[i] += weight(x[i][k], y[i][k], beta);
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
        const double s = wave_sum(sum[i]);
        if (lane == 0 && e + i * stride < nsums) to[e + i * stride] = s;
    }
}

// The start of every entry's walk, up to where a sum over a row is wanted, which for a
// chain is where it ends: each of an entry's workgroups walks by itself and sums some of
// the row's blocks, the first one writes down where the walk stands.
__global__ __launch_bounds__(256) void draft_verify_start_k(Verify a, holo_batch_t b)
{
    __shared__ WalkState state;
    const int e = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int first, take;
    batch_rows(b, e, first, take);
    if (take <= 0) return;
    if (wave == 0) {
        Walk w(a, first, take, lane);
        const bool writes = blockIdx.x == 0 && lane == 0;
        if (writes) a.path[first] = 0;
        w.go([&](int i, int row) {
            if (writes) a.path[first + i] = row;
        });
        if (writes) a.states[e] = w.s;
        if (lane == 0) state = w.s;
    }
    __syncthreads();
    const WalkState s = state;
    const float *p = a.target + (int64_t)(first + s.node) * a.ldt;
    const float *q = a.mode != HOLO_DRAFT_CHOSEN ? a.draft + (int64_t)(first + s.node) * a.ldd : p;
    const int nsums = (a.vocab + a.block - 1) / a.block;
    double *sums = a.sums + (int64_t)e * nsums;
    for (int i = 4 * blockIdx.x + wave; i < nsums; i += 4 * gridDim.x) block_sums<1>(a, p, q, s.beta, i, 1, lane, sums, nsums);
}

// The rest, a workgroup an entry: more rows behind a refused one (the branches of a
// tree), and the next token.  Sums are in 64 bits, each in one order.
__global__ __launch_bounds__(kVerifyThreads) void draft_verify_k(Verify a, holo_batch_t b)
{
    __shared__ double sums[kVerifySums];
    __shared__ int refused_tok[1024];
    __shared__ WalkState state;
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
    for (int i = threadIdx.x; i < nsums; i += kVerifyThreads) sums[i] = a.sums[(int64_t)blockIdx.x * nsums + i];
    // Sum of all blocks; own: of this lane's, upto: of those up to the end of this lane's.
    auto total = [&](double &own, double &upto) {
        own = 0.0;
        for (int i = lane * per; i < min((lane + 1) * per, nsums); i++) own += sums[i];
        upto = wave_scan(own, lane);
        return __shfl(upto, 63, 64);
    };

    Walk w(a, first, take, lane);
    w.s = a.states[blockIdx.x];
    __syncthreads();
    const float *p, *q;
    auto rows = [&]() {
        p = a.target + (int64_t)(first + w.s.node) * a.ldt;
        q = drawn ? a.draft + (int64_t)(first + w.s.node) * a.ldd : p;
    };
    while (w.s.asks) {  // (the same for every wave)
        const int node = w.s.node;
        const double beta = w.s.beta;
        if (wave == 0) {
            double own, upto;
            w.s.left = total(own, upto);
            w.go([&](int i, int row) {
                if (lane == 0) a.path[first + i] = row;
            });
            if (lane == 0) state = w.s;
        }
        __syncthreads();
        if (wave != 0) w.s = state;
        if (w.s.node == node && w.s.beta == beta) break;  // sums are of these
        rows();
        constexpr int U = 2;
        for (int e = wave; e < nsums; e += U * kVerifyWaves)
            block_sums<U>(a, p, q, w.s.beta, e, kVerifyWaves, lane, sums, nsums);
        __syncthreads();
    }
    rows();
    // Chosen: every row behind the node was refused; blocks with such tokens once more, without them.
    int refused = 0;
    if (!drawn) {
        if (wave == 0) {
            for (int at = 0; at < take; at += 64) {
                const int i = at + lane;
                const bool is = i > w.s.node && i < take && a.parent[first + i] == w.s.node;
                const uint64_t hits = __ballot(is);
                if (is) refused_tok[refused + __popcll(hits & ((1ull << lane) - 1))] = a.tokens[first + i];
                refused += __popcll(hits);
            }
            if (lane == 0) state.count = refused;
        }
        __syncthreads();
        refused = state.count;
    }
    auto weight_at = [&](int64_t t) {
        if (t >= a.vocab) return 0.0;
        for (int i = 0; i < refused; i++)
            if (refused_tok[i] == t) return 0.0;
        return weight(p[t], w.s.beta != 0.0 ? q[t] : 0.f, w.s.beta);
    };
    for (int r = wave; r < refused; r += kVerifyWaves) {
        const int t = refused_tok[r], e = t / a.block;
        if (t < 0 || t >= a.vocab) continue;
        double sum = 0.0;
        for (int o = lane; o < a.block; o += 64) sum += weight_at((int64_t)e * a.block + o);
        sum = wave_sum(sum);
        if (lane == 0) sums[e] = sum;  // (a block of several: the same sum each time)
    }
    __syncthreads();
    if (wave != 0) return;
    for (int i = w.s.count + lane; i < take; i += 64) a.path[first + i] = -1;
    double own, upto;
    const double all = total(own, upto), at = (double)unit(a.u[first]) * all;
    int token = -1;
    if (all > 0.0) {
        // The first lane, block and token whose sum passes; past them by rounding: the last with
        // a weight.  Only lanes whose own blocks weigh count: the scan adds in another order in
        // every lane, and one without any weight can have a sum a rounding above its neighbour's.
        const uint64_t some = __ballot(own > 0.0), pass = __ballot(upto > at) & some;
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
            const int64_t t = (int64_t)e * a.block + o + lane;
            const double v = weight_at(t), to = run + wave_scan(v, lane);
            const uint64_t pos = __ballot(v > 0.0), in = __ballot(to > at) & pos;
            if (pos) token = e * a.block + o + (in ? __ffsll((unsigned long long)in) - 1 : 63 - __clzll((long long)pos));
            if (in) break;
            run = __shfl(to, 63, 64);
        }
    } else {
        // nothing weighs: the target's most probable token, the lowest of equals
        float best = -1.f;
        for (int t = lane; t < a.vocab; t += 64) {
            const float v = probability(p[t]);
            if (v > best) {
                best = v;
                token = t;
            }
        }
        for (int off = 32; off > 0; off >>= 1) {
            const float v = __shfl_xor(best, off, 64);
            const int t = __shfl_xor(token, off, 64);
            if (v > best || (v == best && t < token)) {
                best = v;
                token = t;
            }
        }
    }
    if (lane == 0) {
        a.n_path[blockIdx.x] = w.s.count;
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
    const int nsums = (vocab + block - 1) / block;
    const size_t told = (size_t)b->n_seqs * sizeof(WalkState);
    const StreamScratch scratch(told + (size_t)b->n_seqs * nsums * sizeof(double));
    if (!scratch.get()) {
        latch_error((int)hipErrorOutOfMemory, "holo_draft_verify: sums", __FILE__, __LINE__);
        return (int)hipErrorOutOfMemory;
    }
    const Verify a{path,   n_path, next,  target, draft, ldt,  ldd, vocab, mode,
                   tokens, parent, u,     block,  (WalkState *)scratch.get(), (double *)((uint8_t *)scratch.get() + told)};
    const int want = 2048 / b->n_seqs, most = (nsums + 3) / 4, parts = want < 1 ? 1 : want < most ? want : most;
    hipLaunchKernelGGL(draft_verify_start_k, dim3(parts, b->n_seqs), dim3(256), 0, stream(), a, v);
    HOLO_LAUNCH_CHECK();
    hipLaunchKernelGGL(draft_verify_k, dim3(b->n_seqs), dim3(kVerifyThreads), 0, stream(), a, v);
    HOLO_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
