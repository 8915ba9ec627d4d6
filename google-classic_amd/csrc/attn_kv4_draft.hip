// attn_kv4_draft.hip -- attention of drafted rows over the 4-bit cache
// (holo_attention_kv4_draft).
#include "attn_kv4.h"

namespace holo {

template <int NB>
static int run_draft(Kv4Attn a)
{
    constexpr int W = 4;
    const int G = a.n_heads / a.c.n_kv_heads, take = a.b.max_rows;
    a.ctiles = (int)(((int64_t)take * G + 15) / 16);
    const int tiles = (a.b.max_len + 31) / 32;
    const int64_t groups = (int64_t)a.ctiles * a.c.n_kv_heads * a.b.n_seqs;
    a.splits = ranges(groups, tiles);
    const dim3 grid(a.splits, a.ctiles * a.c.n_kv_heads, a.b.n_seqs);
    constexpr size_t lds = (size_t)W * 16 * (32 * NB + 4 + 2) * sizeof(float);
    if (a.splits == 1) {
        hipLaunchKernelGGL((attn_kv4_k<NB, W, true>), grid, dim3(64 * W), lds, stream(), a);
        HOLO_LAUNCH_CHECK();
        return 0;
    }
    const StreamScratch scratch((size_t)a.b.n_seqs * take * a.n_heads * a.splits * (32 * NB + 4) * sizeof(float));
    a.part = (float *)scratch.get();
    if (!a.part) {
        latch_error((int)hipErrorOutOfMemory, "holo_attention_kv4_draft: partial sums", __FILE__, __LINE__);
        return (int)hipErrorOutOfMemory;
    }
    hipLaunchKernelGGL((attn_kv4_k<NB, W, true>), grid, dim3(64 * W), lds, stream(), a);
    HOLO_LAUNCH_CHECK();
    hipLaunchKernelGGL((attn_kv4_join_k<NB, true>), dim3(a.n_heads, take, a.b.n_seqs), dim3(256), 0, stream(), a);
    HOLO_LAUNCH_CHECK();
    return 0;
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
    Kv4Attn a{kv4_view(c, layer), *b, out, nullptr, q, ldo, ldq, n_heads, 0, 0, mask, words};
    a.b.max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    const int64_t cols = (int64_t)a.b.max_rows * (n_heads / c->n_kv_heads);
    if (!rows_ok(q, ldq, dim) || !rows_ok(out, ldo, dim) || !draft_rows_ok(&a.b, words) || !mask ||
        ((uintptr_t)mask & 3) || b->max_len < 0 || b->max_len > 0x7FFFF000 ||
        (cols + 15) / 16 * c->n_kv_heads > 65535) {
        HOLO_REJECT("holo_attention_kv4_draft: null or misaligned rows or mask, rows that overlap, more rows than a mask or one launch takes");
        return HOLO_EINVAL;
    }
    switch (c->head_dim) {
    case 32: return run_draft<1>(a);
    case 64: return run_draft<2>(a);
    case 96: return run_draft<3>(a);
    default: return run_draft<4>(a);
    }
}
