// Rows as E4M3 elements with a float32 scale per block of 128 features (no counterpart in
// the reference, whose blocks have 32 features and power-of-two scales).
//
//     s = max(fl(max |x| / 448), 2^-126),   code = RNE_E4M3(x / s)
//
// over 1 row (activations) or 128 rows (weights) by 128 features.  The codes are those of
// the exact quotients (gemm_fp8.cuh): with 16-bit elements quotients in the middle between two
// codes are common, and s is rounded, so one that lies a hair beside the middle must not be
// rounded onto it first.
//
// A thread converts 16 features; 2 or 4 bytes are read and one is written per element, so
// HBM bounds both kernels.  Measured, 16,384 x 8192, by row and in blocks of 128 rows: bfloat16 98 and 87 us (4.1
// and 4.7 TB/s), f16 93 and 83, float32 116 and 118 (5.8).  With 16-bit elements a thread by row asks
// for 32 bytes and then waits for them, half of what it has under way in float32; in blocks of 128 rows for
// 128.
#include <algorithm>
#include <limits>

#include "gemm_fp8.cuh"

namespace mxk {
namespace {

using dev::Raw16;

// Eight threads to a block of 128 features of a row.
template <class T, int VEC>
__global__ void __launch_bounds__(256) quantize_fp8_rows_kernel(const T* x, int64_t stride, int64_t rows, int k,
                                                                int blocks, uint8_t* values, float* scales) {
    dev::let_next_start();  // (linear_fp8's product)
    const int64_t at = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    const int sub = threadIdx.x & 7;
    const int64_t row = at / blocks;
    const int b = (int)(at - row * blocks), f = b * 128 + sub * 16;
    const bool real = row < rows && f < k;
    Raw16<T, VEC> raw;
    if (real)
        raw.load(x + row * stride + f);
    else
        raw.zero();
    float v[16];
    raw.to_float(v);
    float amax = dev::largest16(v);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float s = dev::fp8_scale(amax);
    if (!real) return;
    *reinterpret_cast<uint4*>(values + row * k + f) = dev::fp8_codes16<T>(v, s, amax);
    if (sub == 0) scales[row * blocks + b] = s;
}

// A thread block to 128 rows by 128 features; a thread has features 16 (tid % 8) of rows
// tid / 8 + 32 i.
template <class T, int VEC>
__global__ void __launch_bounds__(256) quantize_fp8_tiles_kernel(const T* x, int64_t stride, int64_t rows, int k,
                                                                 uint8_t* values, float* scales) {
    __shared__ float tops[8];
    const int tid = threadIdx.x, f = (int)blockIdx.x * 128 + (tid & 7) * 16;
    const int64_t row0 = (int64_t)blockIdx.y * 128 + (tid >> 3);
    Raw16<T, VEC> raw[4];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (row0 + 32 * i < rows && f < k)
            raw[i].load(x + (row0 + 32 * i) * stride + f);
        else
            raw[i].zero();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[16];
        raw[i].to_float(v);
        amax = fmaxf(amax, dev::largest16(v));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((tid & 31) == 0) tops[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, tops[i]);
    const float s = dev::fp8_scale(amax);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[16];
        raw[i].to_float(v);
        if (row0 + 32 * i < rows && f < k) *reinterpret_cast<uint4*>(values + (row0 + 32 * i) * k + f) = dev::fp8_codes16<T>(v, s, amax);
    }
    if (tid == 0) scales[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

template <class T, int VEC>
int launch(const QuantizeFp8& q, cudaStream_t stream) {
    const T* x = static_cast<const T*>(q.x);
    const int blocks = (int)((q.k + 127) / 128);
    LaunchScope scope("quantize_fp8", stream);
    if (q.block_rows == 1) {
        const int64_t grid = (q.rows * blocks + 31) / 32;
        MXK_REQUIRE(grid <= std::numeric_limits<int>::max(), "quantize_fp8: too many rows for one call");
        quantize_fp8_rows_kernel<T, VEC><<<(unsigned)grid, 256, 0, stream>>>(x, q.stride, q.rows, (int)q.k, blocks, q.values, q.scales);
    } else {
        const int64_t tiles = (q.rows + 127) / 128;
        MXK_REQUIRE(tiles <= 65535, "quantize_fp8: too many rows for one call");
        quantize_fp8_tiles_kernel<T, VEC><<<dim3((unsigned)blocks, (unsigned)tiles), 256, 0, stream>>>(x, q.stride, q.rows, (int)q.k, q.values, q.scales);
    }
    MXK_CUDA(cudaGetLastError());
    return MXK_OK;
}

template <class T>
int launch_typed(const QuantizeFp8& q, cudaStream_t stream) {
    const uint64_t at = reinterpret_cast<uintptr_t>(q.x) | (uint64_t)(q.stride * (int64_t)sizeof(T));
    if (at % 32 == 0) return launch<T, 32>(q, stream);
    if (at % 16 == 0) return launch<T, 16>(q, stream);
    return launch<T, 0>(q, stream);
}

}  // namespace

int launch_quantize_fp8(const QuantizeFp8& q, cudaStream_t stream) {
    if (q.dtype == MXK_F32) return launch_typed<float>(q, stream);
    if (q.dtype == MXK_F16) return launch_typed<__half>(q, stream);
    return launch_typed<__nv_bfloat16>(q, stream);
}

}  // namespace mxk

extern "C" int mxk_quantize_fp8(int dtype, int64_t rows, int64_t k, const void* x, int64_t row_stride, int block_rows,
                                uint8_t* values, float* scales, void* stream) {
    using namespace mxk;
    MXK_REQUIRE(dtype == MXK_F32 || dtype == MXK_F16 || dtype == MXK_BF16, "quantize_fp8: unknown dtype");
    MXK_REQUIRE(block_rows == 1 || block_rows == 128, "quantize_fp8: block_rows must be 1 or 128");
    MXK_REQUIRE(rows >= 0 && k >= 0 && k % 16 == 0 && k < (1ll << 30),
                "quantize_fp8: k must be a multiple of 16 below 2^30, rows not negative");
    if (rows == 0 || k == 0) return MXK_OK;
    MXK_REQUIRE(x && values && scales, "quantize_fp8: x, values and scales must be non-null");
    const int size = dtype == MXK_F32 ? 4 : 2;
    MXK_REQUIRE(reinterpret_cast<uintptr_t>(x) % size == 0 && reinterpret_cast<uintptr_t>(values) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                "quantize_fp8: x must be aligned to its elements, values to 16 bytes, scales to 4");
    return launch_quantize_fp8({dtype, block_rows, rows, k, x, row_stride, values, scales}, as_stream(stream));
}
