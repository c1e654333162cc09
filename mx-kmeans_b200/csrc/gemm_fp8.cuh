// Shared pieces of the E4M3 product with a float32 scale per block of 128.
#pragma once

#include "cache_rows.cuh"

namespace mxk {

struct QuantizeFp8 {
    int dtype, block_rows;
    int64_t rows, k;
    const void* x;
    int64_t stride;  // elements
    uint8_t* values;
    float* scales;
};
int launch_quantize_fp8(const QuantizeFp8& q, cudaStream_t stream);

struct GemmFp8 {
    int dtype;  // of out
    int64_t m, n, k;
    const uint8_t* a;
    const float* a_scales;
    const uint8_t* b;
    const float* b_scales;
    void* out;
    int64_t out_stride;  // elements
};

namespace dev {

// x / s, given t = x * (1 / s), which is within four units of the last place of it, or a value
// that rounds to the same code as the exact quotient.  Where a middle between two codes is as near
// as that, the sign of x - middle * s, which fma gives exactly, says on which side of it the
// quotient lies; subnormal codes have other middles, and there the quotient is divided out and
// rounded to odd.
__device__ __forceinline__ bool fp8_in_doubt(float t) {
    return ((__float_as_uint(t) - 0x7fffcu) & 0xfffffu) <= 8u;
}
__device__ __forceinline__ bool fp8_subnormal(float t) {  // from 2^-11 to 2^-6
    return (__float_as_uint(t) & 0x7fffffffu) - 0x3a000000u < 0x02800000u;
}
static __device__ __noinline__ float fp8_quotient(float x, float s, float t) {
    if (fp8_subnormal(t)) {
        t = __fdiv_rn(x, s);
        const float rest = __fmaf_rn(-t, s, x);
        uint32_t bits = __float_as_uint(t);
        if (rest != 0.0f && !(bits & 1u)) bits += (rest > 0.0f) == (t > 0.0f) ? 1u : ~0u;
        return __uint_as_float(bits);
    }
    const uint32_t middle = ((__float_as_uint(t) - 0x7fffcu) & ~0xfffffu) + 0x80000u;
    const float rest = __fmaf_rn(-__uint_as_float(middle), s, x);
    return __uint_as_float(middle + (rest == 0.0f ? 0u : ((rest > 0.0f) == (t > 0.0f) ? 1u : ~0u)));
}

__device__ __forceinline__ uint4 fp8_pack16(const float (&t)[16]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = e4m3x2_encode(t[4 * i], t[4 * i + 1]) | (e4m3x2_encode(t[4 * i + 2], t[4 * i + 3]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Codes of the exact quotients x / s, s the scale of a block with the largest magnitude amax.
__device__ __forceinline__ uint4 fp8_codes16(float (&x)[16], float s, float) {
    if (s < 9.1e-13f) {  // 2^-40: times 2^80, so that remainders stay representable
        s *= 1.2089258e24f;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= 1.2089258e24f;
    }
    const float inv = __frcp_rn(s);
    float t[16];
    bool any = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = x[i] * inv, any |= fp8_in_doubt(t[i]) || fp8_subnormal(t[i]);
    if (any) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (fp8_in_doubt(t[i]) || fp8_subnormal(t[i])) t[i] = fp8_quotient(x[i], s, t[i]);
    }
    return fp8_pack16(t);
}

// The same of 16-bit elements.  x / (amax / 448) then is a middle between two codes exactly, or off
// it by 2^-16 at least: x * 448 and middle * amax are products of 3 and 11 and of 5 and 11 bits.  In
// the middle, x / s lies above if s was rounded down and below if up, for the whole block: so the
// reciprocal is shifted by 2^-21 that way.  Where s is exact (amax has a factor 7) such quotients are
// divided out.
__device__ __forceinline__ uint4 fp8_codes16_narrow(const float (&x)[16], float s, float amax) {
    const float rest = __fmaf_rn(s, 448.0f, -amax), inv = __frcp_rn(s);
    // (the smallest scale is a power of two, and quotients by it are exact)
    const bool exact = rest == 0.0f && s > 1.17549435e-38f;
    const float shifted = s > 1.17549435e-38f && rest != 0.0f ? fmaf(inv, rest > 0.0f ? -4.76837158e-7f : 4.76837158e-7f, inv) : inv;
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = x[i] * shifted;
    if (exact) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (fp8_in_doubt(t[i]) || fp8_subnormal(t[i])) t[i] = __fdiv_rn(x[i], s);
    }
    return fp8_pack16(t);
}
template <class T>
__device__ __forceinline__ uint4 fp8_codes16(float (&x)[16], float s, float amax) {
    if constexpr (sizeof(T) == 2)
        return fp8_codes16_narrow(x, s, amax);
    else
        return fp8_codes16(x, s, amax);
}

__device__ __forceinline__ float fp8_scale(float amax) { return fmaxf(__fdiv_rn(amax, 448.0f), 1.17549435e-38f); }

__device__ __forceinline__ float largest16(const float (&x)[16]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(x[i]));  // a NaN sets no scale
    return m;
}

}  // namespace dev
}  // namespace mxk
