/*
 * rotary.c - entry points of include/sneppx_rotary.h: argument checks, and the
 * frequencies of the scalings, computed on the host.
 */
#include <math.h>
#include <stdint.h>

#include "sneppx_rotary.h"
#include "../snx_internal.h"

#define REQUIRE(cond, ...)               \
    do {                                 \
        if (!(cond)) {                   \
            snx_set_error(__VA_ARGS__);  \
            return -1;                   \
        }                                \
    } while (0)

#define PI 3.14159265358979323846

int snx_rotary_check(const char* who, const SNEPPXRotary* r, size_t head_dim) {
    REQUIRE(r, "%s: NULL rotary", who);
    REQUIRE(r->dims % 8 == 0 && r->dims <= head_dim, "%s: %zu rotated elements are not a multiple of 8 up to head_dim %zu",
            who, r->dims, head_dim);
    REQUIRE(!r->dims || r->freqs, "%s: NULL freqs", who);
    REQUIRE((((uintptr_t)r->freqs | (uintptr_t)r->q_norm | (uintptr_t)r->k_norm) & 15u) == 0,
            "%s: freqs, q_norm and k_norm must be 16-byte aligned", who);
    return 0;
}

int SNEPPX_rotary_frequencies(double* freqs, float* magnitude, size_t dims, double base, SNEPPXRotaryScaling kind,
                              double factor, double original, double low, double high) {
    static const char who[] = "rotary_frequencies";
    REQUIRE(freqs || !dims, "%s: NULL freqs", who);
    REQUIRE(dims % 2 == 0, "%s: %zu elements do not pair", who, dims);
    REQUIRE(base > 1.0 && isfinite(base), "%s: base %g must be above 1", who, base);
    REQUIRE(kind >= SNEPPX_ROTARY_PLAIN && kind <= SNEPPX_ROTARY_RAMP, "%s: unknown scaling %d", who, (int)kind);
    REQUIRE(kind == SNEPPX_ROTARY_PLAIN || (factor >= 1.0 && isfinite(factor)), "%s: factor %g must be 1 or more", who,
            factor);
    REQUIRE(kind != SNEPPX_ROTARY_BASE || dims != 2, "%s: the base of a single pair cannot be scaled", who);
    const int bands = kind == SNEPPX_ROTARY_BANDS || kind == SNEPPX_ROTARY_RAMP;
    REQUIRE(!bands || (original > 0.0 && isfinite(original)), "%s: original %g must be above 0", who, original);
    REQUIRE(!bands || (low > 0.0 && low < high && isfinite(high)), "%s: low %g must be between 0 and high %g", who, low,
            high);
    if (kind == SNEPPX_ROTARY_BASE) base *= pow(factor, (double)dims / ((double)dims - 2.0));
    /* RAMP: the (fractional) pairs that make `high` and `low` turns over `original` positions, whole pairs outwards */
    double first = 0.0, last = 0.0;
    if (kind == SNEPPX_ROTARY_RAMP && dims) {
        const double most = (double)dims - 1.0;
        first = floor((double)dims * log(original / (2.0 * PI * high)) / (2.0 * log(base)));
        last = ceil((double)dims * log(original / (2.0 * PI * low)) / (2.0 * log(base)));
        first = first < 0.0 ? 0.0 : first;
        last = last > most ? most : last;
        if (last <= first) last = first + 0.001;
    }
    for (size_t i = 0; i < dims / 2; i++) {
        double f = pow(base, -2.0 * (double)i / (double)dims);
        double keep = 1.0;
        if (kind == SNEPPX_ROTARY_LINEAR) keep = 0.0;
        if (kind == SNEPPX_ROTARY_BANDS) keep = (original * f / (2.0 * PI) - low) / (high - low);
        if (kind == SNEPPX_ROTARY_RAMP) keep = 1.0 - ((double)i - first) / (last - first);
        keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        freqs[i] = keep == 1.0 ? f : f * (keep + (1.0 - keep) / factor);
    }
    if (magnitude) *magnitude = kind == SNEPPX_ROTARY_RAMP ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    snx_clear_error();
    return 0;
}

int SNEPPX_rotary_apply(const SNEPPXRotary* rotary, const uint16_t* q, size_t q_stride, uint16_t* q_out,
                        size_t q_out_stride, size_t q_heads, const uint16_t* k, size_t k_stride, uint16_t* k_out,
                        size_t k_out_stride, size_t kv_heads, size_t head_dim, const int32_t* positions,
                        size_t tokens, SNEPPXStream stream) {
    static const char who[] = "rotary_apply";
    REQUIRE(head_dim && head_dim <= 256 && head_dim % 8 == 0, "%s: head_dim %zu is not a multiple of 8 up to 256", who,
            head_dim);
    if (snx_rotary_check(who, rotary, head_dim)) return -1;
    REQUIRE(q_heads <= 65535 && kv_heads <= 65535, "%s: %zu and %zu heads are too many", who, q_heads, kv_heads);
    REQUIRE(tokens <= (size_t)1 << 30, "%s: %zu tokens are too many", who, tokens);
    const int none = !tokens || !(q_heads + kv_heads);
    REQUIRE(none || positions, "%s: NULL positions", who);
    REQUIRE(none || !q_heads || (q && q_out), "%s: NULL q or q_out", who);
    REQUIRE(none || !kv_heads || (k && k_out), "%s: NULL k or k_out", who);
    const size_t nq = q_heads * head_dim, nk = kv_heads * head_dim;
    REQUIRE(tokens < 2 || (q_stride >= nq && q_out_stride >= nq && k_stride >= nk && k_out_stride >= nk),
            "%s: a stride (%zu, %zu, %zu, %zu) is below its row of %zu or %zu", who, q_stride, q_out_stride, k_stride,
            k_out_stride, nq, nk);
    REQUIRE(!nq || tokens < 2 || q != q_out || q_stride == q_out_stride, "%s: q in place with another stride", who);
    REQUIRE(!nk || tokens < 2 || k != k_out || k_stride == k_out_stride, "%s: k in place with another stride", who);
    snx_clear_error();
    if (none) return 0;
    return snx_k_rotary(rotary, q, q_stride, q_out, q_out_stride, q_heads, k, k_stride, k_out, k_out_stride, kv_heads,
                        head_dim, positions, tokens, stream);
}
