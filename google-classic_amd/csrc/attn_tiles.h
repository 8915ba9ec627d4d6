// attn_tiles.h -- what the attention kernels on 16-column tiles share: operand
// types of v_mfma_f32_16x16x32_f16, the split of fp32 values into two f16 halves,
// and the softmax's scale.
#pragma once

#include <hip/hip_runtime.h>

#include <float.h>

namespace holo {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Scores are in log2 units.  q is multiplied by this before it is split: what is
// left to multiply a score by is a power of two, so that the largest one less
// itself is 0 at any magnitude.
constexpr float score_scale(int hd)
{
    return hd == 32 ? 0.25503486f : hd == 64 ? 0.18033688f : hd == 96 ? 0.14724444f : 0.12751743f;  // log2(e) / sqrt(hd)
}

// Probabilities are held times 2^kPShift; a running maximum moves when a score
// passes it by kMaxSlack: they stay below 2^15.  (7.5: where 8 is half of the
// maximum's last place, the sum of the two could round to 16.)
constexpr float kPShift = 7.5f, kMaxSlack = 7.f;

// x = hi + lo, two values at a time (x - hi is exact in fp32).
__device__ __forceinline__ void split8(const float x[8], h8 &hi, h8 &lo)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const h2 h = __builtin_convertvector((f2){x[2 * i], x[2 * i + 1]}, h2);
        const h2 l = __builtin_convertvector((f2){x[2 * i] - (float)h.x, x[2 * i + 1] - (float)h.y}, h2);
        hi[2 * i] = h.x;
        hi[2 * i + 1] = h.y;
        lo[2 * i] = l.x;
        lo[2 * i + 1] = l.y;
    }
}

}  // namespace holo
