// Shared pieces of the E4M3 product with a float32 scale per block of 128.
#pragma once

#include "common.cuh"

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

}  // namespace mxk
