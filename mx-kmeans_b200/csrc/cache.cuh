// Shared pieces of the paged MX cache: argument checks and the device-side view.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mxk {

// Checks the cache's fields (mxk.h).
int check_cache(const mxk_cache* c, const char* who);

inline int64_t cache_slots(const mxk_cache& c) { return c.pages * c.page_size; }

// Bytes of one row of elements of one head and token.
__host__ __device__ constexpr int cache_row_bytes(int head_dim, int bits) { return head_dim * bits / 8; }

// Whether rows of 2- or 4-byte elements can be moved `bytes` at a time.
inline bool rows_aligned(const mxk_rows& r, int elem_size, int bytes) {
    return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && (r.token_stride * elem_size) % bytes == 0 &&
           (r.head_stride * elem_size) % bytes == 0;
}

namespace dev {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four 6-bit codes packed in 24 bits, lowest first, spread to one byte each.
__device__ __forceinline__ uint32_t spread6(uint32_t v) {
    return (v & 0x3fu) | ((v << 2) & 0x3f00u) | ((v << 4) & 0x3f0000u) | ((v << 6) & 0x3f000000u);
}

// f16 pair (low half from the low byte) of two one-byte element codes; exact.
template <int BITS>
__device__ __forceinline__ uint32_t codes_to_f16x2(uint32_t two) {
    static_assert(BITS == 8 || BITS == 6, "4-bit codes are converted eight at a time");
    uint32_t h2;
    const uint16_t c = (uint16_t)two;
    if constexpr (BITS == 8)
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(c));
    else
        asm("cvt.rn.f16x2.e2m3x2 %0, %1;" : "=r"(h2) : "h"(c));
    return h2;
}

// f16 pairs of the eight E2M1 codes of w, one pair per byte, low nibble first; exact.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h2)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h2[0]), "=r"(h2[1]), "=r"(h2[2]), "=r"(h2[3])
        : "r"(w));
}

}  // namespace dev
}  // namespace mxk
