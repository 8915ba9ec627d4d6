// attn_kv4.hip -- attention over the 4-bit cache (holo_attention_kv4).
//
// softmax(q . k_p / sqrt(hd)) . v_p over the positions p a row sees, for the last
// rows of several sequences.  Both products run on v_mfma_f32_16x16x32_f16,
// transposed: S^T = K Q^T and O^T = V^T P^T, so that a lane holds one column (a
// query row and head) throughout.
//   - The columns of a KV head are its entry's rows times the query heads that
//     share it, 16 of them a tile: all the heads of a grouped-query decode step
//     at once.
//   - A cached value d * c is an exact f16 (kv4.h, holo_forward.h): a code's
//     four bits shifted into an f16's mantissa under the exponent of 16 are 16 +
//     c + 8, and one packed fma with d and -24 d makes d * c of it.
//   - q (scaled by a power of two to its row's largest value) and the
//     probabilities are two f16 halves, x - hi - lo within 2^-22 |x|: fp32's
//     class with two matrix instructions.  Probabilities are held times 2^7.5, so
//     that a small one's lo stays above f16's smallest step.
//   - The softmax is one pass: the running maximum of a column moves only when a
//     score passes it by 2^7 (p then stays below 2^15), which few tiles do.
//   - A lane's scores are those of the eight positions that its V words hold:
//     P is the second product's operand without crossing lanes.
// A workgroup's waves take the tiles of a range in turn and meet in LDS; ranges
// of a long sequence are workgroups of their own, whose partial sums a second
// launch joins in range order.
//
// What bounds it (32 heads on 8 of 128): 64 sequences of up to 8192 positions, 455
// MB, take 100-116 us, 3.9-4.6 TB/s; vector instructions (300 a tile, 192 of
// them unpacking) issue in 56% of the cycles, 72% of those in which a CU has work,
// the rest is the lengths' imbalance.  One wave's tile is a chain of 1.2 us: 513
// positions of one sequence (four tiles a wave) 8.5 us.  16 sequences of up to 4096
// (up to eight) 17.8: 15.3 and 4.8 for the ranges' join in a kernel trace, whose
// times hold each launch's start and end.  100000 positions of one sequence 32-34,
// the join 5.1 of them.  Chunks: 16 columns unpack every tile again, four
// sequences of 100 rows at 2000 take 37-40 us at 260 TFLOP/s.  With the tiles in LDS
// for 128 columns that was 62, with 32 columns a wave as fast or slower (the second
// operand's registers), with q in LDS or eight waves 5-15% slower.
#include "attn_kv4.h"

namespace holo {

template <int NB>
static int run_attn(Kv4Attn a)
{
    constexpr int W = 4;  // (eight: 64 sequences 119 us, 513 positions of one 9.2)
    const int G = a.n_heads / a.c.n_kv_heads, take = a.b.max_rows;
    a.ctiles = (int)(((int64_t)take * G + 15) / 16);
    const int tiles = (a.b.max_len + 31) / 32;
    const int64_t groups = (int64_t)a.ctiles * a.c.n_kv_heads * a.b.n_seqs;
    a.splits = ranges(groups, tiles);
    const dim3 grid(a.splits, a.ctiles * a.c.n_kv_heads, a.b.n_seqs);
    constexpr size_t lds = (size_t)W * 16 * (32 * NB + 4 + 2) * sizeof(float);
    if (a.splits == 1) {
        hipLaunchKernelGGL((attn_kv4_k<NB, W>), grid, dim3(64 * W), lds, stream(), a);
        HOLO_LAUNCH_CHECK();
        return 0;
    }
    // (a small buffer: ranges are for fewer than two workgroups a CU, and make fewer than
    // four.  At two, with 4 heads a KV head of 128 dims, it is 1.03 MiB, which a captured call
    // allocates by nodes of its graph: 16 sequences of up to 4096 20.1 us eager, 29-31 replayed.)
    const StreamScratch scratch((size_t)a.b.n_seqs * take * a.n_heads * a.splits * (32 * NB + 4) * sizeof(float));
    a.part = (float *)scratch.get();
    if (!a.part) {
        latch_error((int)hipErrorOutOfMemory, "holo_attention_kv4: partial sums", __FILE__, __LINE__);
        return (int)hipErrorOutOfMemory;
    }
    hipLaunchKernelGGL((attn_kv4_k<NB, W>), grid, dim3(64 * W), lds, stream(), a);
    HOLO_LAUNCH_CHECK();
    hipLaunchKernelGGL(attn_kv4_join_k<NB>, dim3(a.n_heads, take, a.b.n_seqs), dim3(256), 0, stream(), a);
    HOLO_LAUNCH_CHECK();
    return 0;
}

}  // namespace holo

using namespace holo;

extern "C" int holo_attention_kv4(const holo_kv4_t *c, int layer, float *out, const float *q, int ldo, int ldq,
                                  int n_heads, const holo_batch_t *b)
{
    if (!kv4_call_ok(c, layer, b) || n_heads <= 0 || n_heads % c->n_kv_heads != 0) {
        HOLO_REJECT("holo_attention_kv4: cache, layer, heads or batch outside the supported set");
        return HOLO_EINVAL;
    }
    if (b->rows == 0 || b->n_seqs == 0) return 0;
    const int64_t dim = (int64_t)n_heads * c->head_dim;
    Kv4Attn a{kv4_view(c, layer), *b, out, nullptr, q, ldo, ldq, n_heads, 0, 0};
    a.b.max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    const int64_t cols = (int64_t)a.b.max_rows * (n_heads / c->n_kv_heads);
    if (!rows_ok(q, ldq, dim) || !rows_ok(out, ldo, dim) || b->max_len < 0 || b->max_len > 0x7FFFF000 ||
        (cols + 15) / 16 * c->n_kv_heads > 65535 || a.b.max_rows > 65535) {
        HOLO_REJECT("holo_attention_kv4: null or misaligned rows, rows that overlap, or more rows than one launch takes");
        return HOLO_EINVAL;
    }
    switch (c->head_dim) {
    case 32: return run_attn<1>(a);
    case 64: return run_attn<2>(a);
    case 96: return run_attn<3>(a);
    default: return run_attn<4>(a);
    }
}
