// kv_rows.h - rows of a head (keys, values, queries) held by 8, 16 or 32 lanes,
// eight elements each: reductions over them, and the int8 rule of the cache.
#pragma once

#include <hip/hip_runtime.h>

#include <cfloat>
#include <cstdint>

#include "codec.h"
#include "kv_pool.h"

namespace snx {

// max over non-NaN values, as the reference's `if (a > m) m = a`
__device__ __forceinline__ float nanless_max(float a, float b) { return b > a ? b : a; }

// An operation that does not mind the order of two operands over LR lanes, to all of
// them: exchanges of neighbours, pairs, halves of 8, of 16 and of 32 lanes.  Every
// lane gets the same bits.
template <int LR, typename F>
__device__ __forceinline__ float row_all(float m, F op) {
    m = op(m, lane_step<0xB1, 0xf>(m, m));
    m = op(m, lane_step<0x4E, 0xf>(m, m));
    m = op(m, lane_step<0x141, 0xf>(m, m));
    if (LR >= 16) m = op(m, lane_step<0x140, 0xf>(m, m));
    if (LR >= 32) m = op(m, __shfl_xor(m, 16));
    return m;
}
template <int LR>
__device__ __forceinline__ float row_max(float m) {
    return row_all<LR>(m, nanless_max);
}
template <int LR>
__device__ __forceinline__ float row_sum(float m) {
    return row_all<LR>(m, [](float a, float b) { return a + b; });
}

// The rule of SNEPPX_quantize_int8_channel (quantize_int8.c:157-177) for a row: its
// scale, the lane's codes (eight bytes in the order of f), and f as the cache gives
// it back.  Needs IEEE divisions and no contraction.
template <int LR>
__device__ __forceinline__ float quantize_row(float (&f)[8], uint32_t (&q)[2]) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) m = nanless_max(m, fabsf(f[e]));
    m = row_max<LR>(m);
    const float s = m < FLT_MIN ? 1.0f : m / 127.0f, inv = 1.0f / s;
    // Numbers below 128 round half away by adding the number below 1/2 and
    // cutting; what the rule gives for others (an infinity or NaN in the row, a
    // scale whose reciprocal is infinite) takes the long way.
    float all = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) all += fabsf(f[e]);
    const bool plain = all < INFINITY && m < INFINITY && inv < INFINITY;
    q[0] = q[1] = 0u;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float v = f[e] * inv;
        const int c = plain ? (int)(v + copysignf(0.49999997f, v)) : clampi(round_i32(v), -128, 127);
        q[e >> 2] |= (uint32_t)(c & 0xFF) << (8 * (e & 3));
        f[e] = (float)c * s;
    }
    return s;
}

}  // namespace snx
