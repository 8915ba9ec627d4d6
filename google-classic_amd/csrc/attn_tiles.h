// attn_tiles.h -- what the attention kernels on the matrix cores share: operand
// types of v_mfma_f32_16x16x32_f16 and v_mfma_f32_32x32x16_f16, the split of fp32 values into two f16 halves,
// and the softmax's scale.
#pragma once

#include <hip/hip_runtime.h>

#include <float.h>

namespace holo {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Scores are in log2 units.  q is multiplied by this before it is split: what is
// left to multiply a score by is a power of two, so that the largest one less
// itself is 0 at any magnitude.
constexpr float score_scale(int hd)
{
    return hd == 32 ? 0.25503486f : hd == 64 ? 0.18033688f : hd == 96 ? 0.14724444f : 0.12751743f;  // log2(e) / sqrt(hd)
}

// The exponent by which a row of q is scaled down, its largest value to [2^13,
// 2^14); rows of zeros, and rows with an infinity (whose halves make NaN of it), as
// they are.  (-100: a power of two that multiplies scores is not 0.)
__device__ __forceinline__ int scale_exp(float big)
{
    return big > 0.f && big <= FLT_MAX ? max(ilogbf(big) - 13, -100) : 0;
}

// Probabilities are held times 2^kPShift; a running maximum moves when a score
// passes it by kMaxSlack: they stay below 2^15.  (7.5: where 8 is half of the
// maximum's last place, the sum of the two could round to 16.)
constexpr float kPShift = 7.5f, kMaxSlack = 7.f;

// The f16 halves of two values, x = hi + lo within 2^-22 |x|: a packed conversion
// and two mixed fused multiply-adds (x - hi is exact in fp32), which the compiler
// otherwise takes apart into conversions and subtractions.
__device__ __forceinline__ void split2(float x, float y, h2 &hi, h2 &lo)
{
    hi = __builtin_convertvector((f2){x, y}, h2);
    uint32_t l;
    asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x), "v"(hi));
    asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(y), "v"(hi));
    lo = __builtin_bit_cast(h2, l);
}

// The same of x times s (a power of two).
__device__ __forceinline__ void split2(float x, float y, float s, h2 &hi, h2 &lo)
{
    uint32_t h, l;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(x), "s"(s));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(y), "s"(s));
    asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x), "s"(s), "v"(h));
    asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(y), "s"(s), "v"(h));
    hi = __builtin_bit_cast(h2, h);
    lo = __builtin_bit_cast(h2, l);
}

__device__ __forceinline__ void split8(const float x[8], h8 &hi, h8 &lo)
{
    h2 h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) split2(x[2 * i], x[2 * i + 1], h[i], l[i]);
    hi = h8{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
    lo = h8{l[0].x, l[0].y, l[1].x, l[1].y, l[2].x, l[2].y, l[3].x, l[3].y};
}

// The larger of the two lanes j and j + 32.
__device__ __forceinline__ float max_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

}  // namespace holo
