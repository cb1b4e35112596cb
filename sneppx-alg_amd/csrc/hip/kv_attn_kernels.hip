// kv_attn_kernels.hip - attention of one new token per row over the paged
// key-value cache (include/sneppx_kv.h).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "codec.h"
#include "kv_pool.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

struct Attn {
    const uint16_t* q;
    size_t q_stride, out_stride;
    void* out;
    const int32_t* lengths;
    float* ws;
    uint32_t rows, q_heads, max_length;
    float scale;
    int out_f32, accumulate;
};

template <bool I8>
__device__ __forceinline__ float element(const uint8_t* pool, size_t at) {
    if (I8) return (float)reinterpret_cast<const int8_t*>(pool)[at];
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(pool)[at]);
}

// One workgroup per (row, key-value head): for each of its query heads the
// logits into scratch, their maximum and sum, then the weighted values.
template <bool I8>
__global__ void __launch_bounds__(256) k_kv_attention(const KVPool p, const Attn a) {
    __shared__ float sh[4];
    const uint32_t b = blockIdx.x / p.heads, h = blockIdx.x - b * p.heads, group = a.q_heads / p.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t L = kv_length(a.lengths, b, a.max_length), D = p.dim;
    for (uint32_t g = 0; g < group; g++) {
        const uint32_t hq = h * group + g;
        const uint16_t* q = a.q + b * a.q_stride + (size_t)hq * D;
        float* s = a.ws + ((size_t)b * a.q_heads + hq) * a.max_length;
        float top = -INFINITY;
        bool any = false;
        for (uint32_t t = wave; t < L; t += 4) {
            uint32_t r;
            float x = -INFINITY;
            if (p.row(b, h, t, r)) {
                x = 0.0f;
                for (uint32_t d = lane; d < D; d += 64) x += bf16_to_f32(q[d]) * element<I8>(p.k, (size_t)r * D + d);
                for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
                if (I8) x *= p.ks[r];
                x *= a.scale;
                any = true;
            }
            if (lane == 0) s[t] = x;
            top = fmaxf(top, x);
        }
        any = __syncthreads_or(any);
        if (lane == 0) sh[wave] = top;
        __syncthreads();
        top = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
        __syncthreads();
        float sum = 0.0f;
        for (uint32_t t = tid; t < L; t += 256) {
            uint32_t r;
            const float e = p.row(b, h, t, r) ? expf(s[t] - top) : 0.0f;
            s[t] = e;
            sum += e;
        }
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) sh[wave] = sum;
        __syncthreads();
        sum = sh[0] + sh[1] + sh[2] + sh[3];
        const float inv = any ? 1.0f / sum : 0.0f;
        float o = 0.0f;
        if (tid < D)
            for (uint32_t t = 0; t < L; t++) {
                uint32_t r;
                if (p.row(b, h, t, r)) o += s[t] * (I8 ? p.vs[r] : 1.0f) * element<I8>(p.v, (size_t)r * D + tid);
            }
        if (tid < D) {
            const size_t at = b * a.out_stride + (size_t)hq * D + tid;
            o = any ? o * inv : 0.0f;
            if (a.out_f32) static_cast<float*>(a.out)[at] = o;
            else static_cast<uint16_t*>(a.out)[at] = bf16_out(o);
        }
        __syncthreads();
        if (a.accumulate)
            for (uint32_t t = tid; t < L; t += 256) s[t] *= inv;
        __syncthreads();
    }
    // the heads' sum first, then one addition to what the cache has
    if (a.accumulate)
        for (uint32_t t = tid; t < L; t += 256) {
            uint32_t r;
            if (!p.row(b, h, t, r)) continue;
            float w = 0.0f;
            for (uint32_t g = 0; g < group; g++) w += a.ws[((size_t)b * a.q_heads + h * group + g) * a.max_length + t];
            p.weights[r] += w;
        }
}

}  // namespace

extern "C" {

size_t snx_kv_attention_ws(const SNEPPXKVCache* c, size_t rows, size_t q_heads, size_t max_length, int accumulate) {
    (void)c;
    (void)accumulate;
    return rows * q_heads * max_length * sizeof(float);
}

int snx_k_kv_attention(const SNEPPXKVCache* c, const uint16_t* q, size_t q_stride, void* out, size_t out_stride,
                       int out_f32, const int32_t* tables, size_t width, const int32_t* lengths, size_t rows,
                       size_t q_heads, size_t max_length, float scale, int accumulate, void* ws, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    const Attn a{q, q_stride, out_stride, out, lengths, static_cast<float*>(ws), (uint32_t)rows, (uint32_t)q_heads,
                 (uint32_t)max_length, scale, out_f32, accumulate};
    const unsigned grid = (unsigned)(rows * c->kv_heads);
    if (c->dtype == SNEPPX_INT8)
        k_kv_attention<true><<<grid, 256, 0, S(st)>>>(p, a);
    else
        k_kv_attention<false><<<grid, 256, 0, S(st)>>>(p, a);
    return snx_launch_check("k_kv_attention");
}

}  // extern "C"
