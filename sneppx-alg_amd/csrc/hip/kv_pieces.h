// kv_pieces.h - what the attention kernels' matrix products are fed with: int8 rows as bf16,
// weights as bf16 pieces, and lanes that have parts of one query.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "codec.h"

namespace snx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// x of this lane and of the one 32 lanes away
__device__ __forceinline__ float swap32(float x, float& y) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
    y = u2f(r[1]);
    return u2f(r[0]);
}

// and of the one 16 lanes away
__device__ __forceinline__ float swap16(float x, float& y) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
    y = u2f(r[1]);
    return u2f(r[0]);
}

// eight int8 as bf16 (exact)
__device__ __forceinline__ u32x4 bytes_to_bf16(uint32_t a, uint32_t b) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t w = i ? b : a;
        const float f0 = (float)(int8_t)w, f1 = (float)(int8_t)(w >> 8);
        const float f2 = (float)(int8_t)(w >> 16), f3 = (float)(int8_t)(w >> 24);
        o[2 * i] = __builtin_amdgcn_perm(f2u(f1), f2u(f0), 0x07060302u);
        o[2 * i + 1] = __builtin_amdgcn_perm(f2u(f3), f2u(f2), 0x07060302u);
    }
    return o;
}

// Eight weights as three bf16 pieces each, exactly (24 significant bits cut into 8 + 8 + 8):
// the products with bf16 values then sum as fp32 ones would, whatever the results' type.
// Of a bf16 cache weights are not negative and values may be infinite, and a zero second or
// third piece would make NaN of that: they are 2^-40 of the first at least (and normal),
// which no sum shows, but zero where the weight is zero, so that a token of no weight adds
// nothing to any value.  Of int8 weights have the sign of their token's scale, and the codes
// are finite; where the weight is not (an infinite scale) it is all in the first piece.
template <bool I8>
__device__ __forceinline__ void split3(const float* x, bf16x8 (&piece)[3]) {
    u32x4 o[3];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float a[2] = {x[e], x[e + 1]}, least[2];
#pragma unroll
        for (int i = 0; i < 3; i++) {
            o[i][e >> 1] = __builtin_amdgcn_perm(f2u(a[1]), f2u(a[0]), 0x07060302u);
            if (i == 2) break;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float high = u2f(f2u(a[j]) & 0xFFFF0000u), low = a[j] - high;
                if (!I8 && i == 0) least[j] = __builtin_amdgcn_fmed3f(high, high * 0x1p-40f, 0x1p-126f);
                a[j] = I8 ? (low == low ? low : 0.0f) : fmaxf(low, least[j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 3; i++) piece[i] = __builtin_bit_cast(bf16x8, o[i]);
}

}  // namespace snx
