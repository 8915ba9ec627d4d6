// kv4_quant.h -- fp32 values to the 4-bit cache's codes and scales.
#pragma once

#include "kv4.h"

#include <float.h>

namespace holo {

// ---- quantisation of a block of 32 ----------------------------------------------------
//
// Eight lanes hold a block, four values each.  The code is the nearest integer
// to x / d.  x * (1 / d) is within 2^-20 of it, so its nearest integer is the code
// unless it lies that near to the middle of two; there the remainder x - c d
// decides (exact: c d has 12 bits and x lies within a factor of c d).

// The larger (or smaller) of the eight lanes' values; NaN if one is.
template <bool MAX>
__device__ __forceinline__ float of_eight(float v)
{
    auto pick = [](float a, float b) { return MAX ? __builtin_elementwise_maximum(a, b) : __builtin_elementwise_minimum(a, b); };
    v = pick(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));   // quad [1,0,3,2]
    v = pick(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));   // quad [2,3,0,1]
    return pick(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false)));  // half mirror
}

// f16 bits of the block's scale: bfloat16(|m| / 8), at most 2720, and m's sign
// reversed; NaN where a value is not finite.
__device__ __forceinline__ uint16_t kv4_scale(const float4 x)
{
    auto least = [](float a, float b) { return __builtin_elementwise_minimum(a, b); };
    auto most = [](float a, float b) { return __builtin_elementwise_maximum(a, b); };
    const float lo = of_eight<false>(least(least(x.x, x.y), least(x.z, x.w)));
    const float hi = of_eight<true>(most(most(x.x, x.y), most(x.z, x.w)));
    const float big = most(-lo, hi);
    const uint32_t u = __float_as_uint(big * 0.125f);
    const float b = __uint_as_float((u + 0x7FFFu + ((u >> 16) & 1u)) & 0xFFFF0000u);  // bfloat16, ties to even
    const float d = fminf(b, 2720.f);
    const uint16_t h = __builtin_bit_cast(uint16_t, (_Float16)(-lo >= hi ? d : -d));
    return big <= FLT_MAX ? h : (uint16_t)0x7E00;
}

// The lane's four codes, one a byte.
__device__ __forceinline__ uint32_t kv4_codes(const float4 x4, uint16_t scale)
{
    const float d = (float)__builtin_bit_cast(_Float16, scale);
    if (!(fabsf(d) > 0.f)) return 0x08080808u;  // zeros, and blocks of NaN
    const float inv = 1.0f / d, x[4] = {x4.x, x4.y, x4.z, x4.w};
    float c[4];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float q = fminf(fmaxf(x[i] * inv, -9.f), 9.f);
        c[i] = rintf(q);
        near |= fabsf(q - c[i]) > 0.5f - 0x1p-16f;
    }
    if (near) {
        const float h = 0.5f * fabsf(d);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float r = fmaf(-c[i], d, x[i]);
            r = d < 0.f ? -r : r;
            const bool odd = (int)c[i] & 1;
            if (r > h || (r == h && odd)) c[i] += 1.f;
            else if (r < -h || (r == -h && odd)) c[i] -= 1.f;
        }
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) w |= (uint32_t)((int)fminf(fmaxf(c[i], -8.f), 7.f) + 8) << (8 * i);
    return w;
}

// ---- a tile's positions lo .. hi - 1, by 256 threads ------------------------------------

// Position p's block blk of a tile: lane x of eight has four values of the key and
// of the value.  The key's codes go into their words (a pair of lanes makes one), the
// value's as bytes into lv, [position][16 r's][2 NB dims r + 16 m], and both scales.
template <int NB>
__device__ __forceinline__ void kv4_put(uint8_t *tile, uint8_t *lv, int p, int blk, int x, float4 kx, float4 vx)
{
    constexpr int HD = 32 * NB, M = 2 * NB;
    uint32_t *kw = (uint32_t *)tile;
    uint16_t *ks = (uint16_t *)(tile + 32 * HD), *vs = (uint16_t *)(tile + 34 * HD);
    const uint16_t kd = kv4_scale(kx), vd = kv4_scale(vx);
    const uint32_t kc = kv4_codes(kx, kd), vcodes = kv4_codes(vx, vd);
    // codes of values 0..3 (even lane) or 4..7 (odd): nibbles 0, 4, 1, 5 or 2, 6, 3, 7
    uint32_t w = (kc & 15u) | (kc >> 8 & 15u) << 16 | (kc >> 16 & 15u) << 4 | (kc >> 24) << 20;
    w <<= 8 * (x & 1);
    w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xF, 0xF, false);
    const int word = 4 * blk + (x >> 1), g = word / NB;
    if (!(x & 1)) kw[(((p >> 4) * 4 + g) * 16 + (p & 15)) * NB + word - g * NB] = w;
    uint8_t *to = lv + p * HD + 4 * (x & 3) * M + 2 * blk + (x >> 2);
#pragma unroll
    for (int y = 0; y < 4; y++) to[y * M] = (uint8_t)(vcodes >> (8 * y));
    if (x == 0) {
        ks[32 * blk + 2 * (p & 15) + (p >> 4)] = kd;
        vs[32 * blk + 8 * ((p & 15) >> 2) + 4 * (p >> 4) + (p & 3)] = vd;
    }
}

// A thread's words of V, VW of lane group vg, and which of their nibbles are new:
// loaded before the tile's blocks are put, stored behind a barrier after them.
template <int NB>
struct Kv4VWords {
    static constexpr int VW = NB % 2 ? 2 : 4, M = 2 * NB;
    uint32_t *vw;
    int vg, vr, vc;
    uint32_t mask = 0, old[VW] = {};
    __device__ __forceinline__ Kv4VWords(uint8_t *tile, int lo, int hi)
        : vw((uint32_t *)(tile + 16 * 32 * NB)), vg(threadIdx.x >> 4 & 3), vr(threadIdx.x & 15), vc(threadIdx.x >> 6)
    {
        if (VW * vc >= M) return;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (v_pos(vg, j) >= lo && v_pos(vg, j) < hi) mask |= 15u << word_shift(j);
        if (mask != 0 && mask != 0xFFFFFFFFu)
#pragma unroll
            for (int i = 0; i < VW; i++) old[i] = vw[VW * threadIdx.x + i];
    }
    __device__ __forceinline__ void store(const uint8_t *lv)
    {
        if (mask == 0) return;
        uint32_t q[8];  // the codes of position j, dim i in byte i (of positions outside the batch: any four bits)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint8_t *at = lv + v_pos(vg, j) * (32 * NB) + vr * M + VW * vc;
            q[j] = (VW == 4 ? *(const uint32_t *)at : *(const uint16_t *)at) & 0x0F0F0F0Fu;
        }
        // nibbles 0 and 1, 2 and 3, 4 and 5, 6 and 7 of the words: positions 0 2, 4 6, 1 3, 5 7
        const uint32_t n0 = q[0] | q[2] << 4, n1 = q[4] | q[6] << 4, n2 = q[1] | q[3] << 4, n3 = q[5] | q[7] << 4;
#pragma unroll
        for (int i = 0; i < VW; i++) {
            const uint32_t w = (n0 >> (8 * i) & 255u) | (n1 >> (8 * i) & 255u) << 8 | (n2 >> (8 * i) & 255u) << 16 |
                               (n3 >> (8 * i) & 255u) << 24;
            old[i] = (old[i] & ~mask) | (w & mask);
        }
        if constexpr (VW == 4) *(uint4 *)(vw + 4 * threadIdx.x) = make_uint4(old[0], old[1], old[2], old[3]);
        else *(uint2 *)(vw + 2 * threadIdx.x) = make_uint2(old[0], old[1]);
    }
};

}  // namespace holo
