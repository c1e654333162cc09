// Rows of the paged MX cache on their way in and out: accesses of 16 elements, block scales,
// packing of codes.
#pragma once

#include <string.h>

#include "cache.cuh"
#include "mx_codec.cuh"

namespace mxk::dev {

// 32 bytes in one access (sm_100): a thread's 16 two-byte elements then are whole
// sectors.  As two 16-byte accesses every sector is moved in two halves (65,536 tokens
// read back: 8 bits to float32 156 us instead of 117).
__device__ __forceinline__ void load32(const void* p, uint4& a, uint4& b) {
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(p));
}
__device__ __forceinline__ void store32(void* p, uint4 a, uint4 b) {
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
                 "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w), "l"(p)
                 : "memory");
}

// 16 elements as they lie in memory.  VEC: bytes of one access, 0: one element.
template <class T, int VEC>
struct Raw16 {
    uint4 w[sizeof(T)];  // 16 * sizeof(T) bytes
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC == 32) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); i += 2) load32(reinterpret_cast<const uint4*>(p) + i, w[i], w[i + 1]);
        } else if constexpr (VEC == 16) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        } else {
            T e[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) e[i] = p[i];
            memcpy(w, e, sizeof(w));
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (VEC == 32) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); i += 2) store32(reinterpret_cast<uint4*>(p) + i, w[i], w[i + 1]);
        } else if constexpr (VEC == 16) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
        } else {
            T e[16];
            memcpy(e, w, sizeof(w));
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = e[i];
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void to_float(float (&x)[16]) const {
        T e[16];
        memcpy(e, w, sizeof(w));
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = dev::to_float(e[i]);
    }
    __device__ __forceinline__ void from_float(const float (&x)[16]) {
        T e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = dev::from_float<T>(x[i]);
        memcpy(w, e, sizeof(w));
    }
};

// The largest of three, NaN if one is NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The hardware conversions round to nearest even and saturate as quantize_rows
// does.  Below 8 bits a NaN becomes the largest magnitude with the NaN's sign
// there, which the conversions do not promise, so the caller replaces NaNs first.

// Two E2M3 codes, one byte each, `lo` in the low byte.
__device__ __forceinline__ uint32_t e2m3x2_pack(float lo, float hi) {
    uint16_t out;
    asm("cvt.rn.satfinite.e2m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(hi), "f"(lo));
    return out;
}

// Eight E2M1 codes, x[0] in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8_pack(const float* x) {
    uint32_t out;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(out)
        : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return out;
}

// Scale byte of a block with the largest magnitude amax.
template <int BITS>
__device__ __forceinline__ uint32_t block_scale(float amax) {
    if constexpr (BITS == 8)
        return ue8m0_mxfp8_scale(amax);
    else
        return ue8m0_encode(amax > 0.0f ? amax / (BITS == 6 ? 7.5f : 6.0f) : 1.0f);
}

// Packs 16 elements x / 2^(e - 127) as piece `at` (of 16) of rows of elements.  nans: there
// may be NaNs among them.
template <int BITS>
__device__ __forceinline__ void pack16(float (&x)[16], uint32_t e, bool nans, uint8_t* values, int64_t at) {
    const float rcp = ue8m0_reciprocal(e);
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] *= rcp;  // the exact quotient by a power of two
    if (BITS < 8 && nans) {
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = x[k] == x[k] ? x[k] : copysignf(BITS == 6 ? 7.5f : 6.0f, x[k]);
    }
    if constexpr (BITS == 8) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = e4m3x2_encode(x[4 * k], x[4 * k + 1]) | (e4m3x2_encode(x[4 * k + 2], x[4 * k + 3]) << 16);
        reinterpret_cast<uint4*>(values)[at] = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (BITS == 6) {
        // four 6-bit codes in three bytes, lowest first
        uint32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t a = e2m3x2_pack(x[4 * k], x[4 * k + 1]), b = e2m3x2_pack(x[4 * k + 2], x[4 * k + 3]);
            v[k] = (a & 0x3fu) | ((a >> 2) & 0xfc0u) | ((b & 0x3fu) << 12) | ((b & 0x3f00u) << 10);
        }
        uint32_t* out = reinterpret_cast<uint32_t*>(values) + at * 3;
        out[0] = v[0] | (v[1] << 24);
        out[1] = (v[1] >> 8) | (v[2] << 16);
        out[2] = (v[2] >> 16) | (v[3] << 8);
    } else {
        // low nibble = even feature
        reinterpret_cast<uint2*>(values)[at] = make_uint2(e2m1x8_pack(x), e2m1x8_pack(x + 8));
    }
}

}  // namespace mxk::dev
