// Paged MX cache: quantising keys and values as they are written, and reading
// them back (no counterpart in the reference; the rows are those of
// quantize_rows, src/kernels/quantize.cu:13-72).
//
// Both kernels stream: a thread moves 16 features of one row, two of them own a
// 32-feature block and join their maxima with one shuffle.  Per row of D
// features the write reads D elements and stores D * bits / 8 + D / 32 bytes,
// the read the reverse, and neither does more than a few operations per element,
// so HBM bounds both.
//
// Measured: 16,384 tokens of 8 heads of 128 in bf16 written as 8 bits and read back (203 MB)
// in 39 us, 5.2 TB/s; 65,536 tokens read back from 4 bits (340 MB) in 62 us, 5.5 TB/s.  One by
// one with a cold L2, 65,536 tokens: 4 bits from bf16 written 74 us (4.6 TB/s) and read 66,
// 6 bits from float32 111 both ways (5.8 TB/s), where a copy of the rows runs at 5.5 to 6.1.  A
// token or a few take a launch's time, 3 us on the device.
#include <limits>

#include "cache_rows.cuh"

namespace mxk {

using dev::max3_nan;
using dev::Raw16;

int check_cache(const mxk_cache* c, const char* who) {
    const std::string w(who);
    MXK_REQUIRE(c, w + ": cache is null");
    MXK_REQUIRE(c->bits == 4 || c->bits == 6 || c->bits == 8, w + ": bits must be 4, 6 or 8");
    MXK_REQUIRE(c->head_dim >= 32 && c->head_dim % 32 == 0 && c->head_dim <= 512,
                w + ": head_dim must be a multiple of 32, at most 512");
    MXK_REQUIRE(c->page_size >= 16 && c->page_size % 16 == 0, w + ": page_size must be a multiple of 16");
    MXK_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 65535, w + ": kv_heads must be in [1, 65535]");
    MXK_REQUIRE(c->pages >= 1 && c->pages <= std::numeric_limits<int>::max(), w + ": pages must be in [1, 2^31)");
    MXK_REQUIRE(c->k_values && c->v_values && c->k_scales && c->v_scales, w + ": a cache buffer is null");
    MXK_REQUIRE((reinterpret_cast<uintptr_t>(c->k_values) | reinterpret_cast<uintptr_t>(c->v_values) |
                 reinterpret_cast<uintptr_t>(c->k_scales) | reinterpret_cast<uintptr_t>(c->v_scales)) % 16 == 0,
                w + ": cache buffers must be 16-byte aligned");
    return MXK_OK;
}

namespace {

// Tokens that a thread handles at once.  65,536 tokens of 8 heads of 128, in us: written as
// 8 bits from bf16 and read back 144 with 1 and 2, 159 with 2 and 3, 161 with 2 and 4 (a
// second row's registers cost the write the occupancy that hides its loads); read back
// from 4 bits 70, 63.5 and 65.5 with 1, 2 and 4.
constexpr int kWritePasses = 1, kReadPasses = 2;

struct Side {
    uint8_t* values;
    uint8_t* scales;
    char* data;  // rows of the caller
    int64_t token_stride, head_stride;
};

struct CacheMove {
    Side side[2];  // keys, values
    const int64_t* slots;
    int64_t tokens, n_slots;
    int chunks;      // 16-feature pieces of a row
    int block_rows;  // tokens of one pass of a block
    int kv_heads, page_size;
    int64_t page_pieces;  // pieces of a page, all heads
    // Divisions without a divide (each took 20 of the 300 instructions of a thread): thread
    // numbers by `chunks` as a product and a shift by 16, exact below 256; numbers below 2^31
    // by page_size with the rounded-up reciprocal 2^(31 + l) / page_size, 2^l >= page_size,
    // whose error times 2^31 stays below one part of the quotient.
    unsigned chunk_factor, page_factor;
    int page_shift;
};

// A block moves `passes` times block_rows tokens of head blockIdx.y, keys (blockIdx.z = 0)
// or values; a thread the same 16-feature piece of as many rows, all requested before the
// first is converted.
struct Mover {
    Side side;
    int head, row, chunk;
    bool active;
    __device__ __forceinline__ explicit Mover(const CacheMove& m) {
        side = blockIdx.z ? m.side[1] : m.side[0];
        head = blockIdx.y;
        row = (int)(threadIdx.x * m.chunk_factor >> 16);
        chunk = (int)threadIdx.x - row * m.chunks;
        active = row < m.block_rows;
    }
    __device__ __forceinline__ int64_t token(const CacheMove& m, int pass, int passes) const {
        return ((int64_t)blockIdx.x * passes + pass) * m.block_rows + row;
    }
    // Piece number of a slot's row in the cache, -1 if the slot lies outside.
    __device__ __forceinline__ int64_t piece(const CacheMove& m, int64_t slot) const {
        if (slot < 0 || slot >= m.n_slots) return -1;
        int64_t page;
        int place;
        if ((slot >> 31) == 0) {
            const unsigned p = __umulhi((unsigned)slot, m.page_factor) >> m.page_shift;
            page = p;
            place = (int)((unsigned)slot - p * (unsigned)m.page_size);
        } else {
            page = slot / m.page_size;
            place = (int)(slot - page * m.page_size);
        }
        return page * m.page_pieces + (int64_t)head * m.page_size * m.chunks + ((int64_t)place * m.chunks + chunk);
    }
    template <class T>
    __device__ __forceinline__ T* rows(int64_t token) const {
        return reinterpret_cast<T*>(side.data) + token * side.token_stride + (int64_t)head * side.head_stride +
               chunk * 16;
    }
};

template <int BITS, class T, int VEC>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheMove m) {
    constexpr int kPasses = kWritePasses;
    const Mover mv(m);
    int64_t at[kPasses];
    Raw16<T, VEC> raw[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int64_t token = mv.token(m, i, kPasses);
        at[i] = mv.active && token < m.tokens ? mv.piece(m, __ldg(m.slots + token)) : -1;
        if (at[i] >= 0)
            raw[i].load(mv.template rows<const T>(token));
        else
            raw[i].zero();
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        float x[16];
        raw[i].to_float(x);
        // The block's largest magnitude, NaN if it holds one: then once more without it.
        // (The two pieces of a block share the token, so both are kept or neither.)
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k += 2) amax = max3_nan(amax, fabsf(x[k]), fabsf(x[k + 1]));
        amax = max3_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1), 0.0f);
        const bool nans = amax != amax;
        if (nans) {
            amax = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; ++k) amax = fmaxf(amax, fabsf(x[k]));
            amax = fmaxf(amax, __shfl_xor_sync(3u << (threadIdx.x & 30u), amax, 1));
        }
        if (at[i] < 0) continue;
        const uint32_t e = dev::block_scale<BITS>(amax);
        dev::pack16<BITS>(x, e, nans, mv.side.values, at[i]);
        if ((mv.chunk & 1) == 0) mv.side.scales[at[i] >> 1] = (uint8_t)e;
    }
}

template <int BITS, class T, int VEC>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheMove m) {
    constexpr int kPasses = kReadPasses;
    const Mover mv(m);
    if (!mv.active) return;
    int64_t at[kPasses];
    uint32_t codes[kPasses][BITS / 2];
    uint32_t scales[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int64_t token = mv.token(m, i, kPasses);
        at[i] = token < m.tokens ? mv.piece(m, __ldg(m.slots + token)) : -1;
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
#pragma unroll
        for (int k = 0; k < BITS / 2; ++k) codes[i][k] = 0;
        scales[i] = 127;
        if (at[i] < 0) continue;
        if constexpr (BITS == 8) {
            const uint4 w = reinterpret_cast<const uint4*>(mv.side.values)[at[i]];
            codes[i][0] = w.x, codes[i][1] = w.y, codes[i][2] = w.z, codes[i][3] = w.w;
        } else if constexpr (BITS == 6) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(mv.side.values) + at[i] * 3;
#pragma unroll
            for (int k = 0; k < 3; ++k) codes[i][k] = p[k];
        } else {
            const uint2 w = reinterpret_cast<const uint2*>(mv.side.values)[at[i]];
            codes[i][0] = w.x, codes[i][1] = w.y;
        }
        scales[i] = mv.side.scales[at[i] >> 1];
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int64_t token = mv.token(m, i, kPasses);
        if (token >= m.tokens) break;
        uint32_t h2[8];  // the 16 elements
        if constexpr (BITS == 4) {
            uint32_t lo[4], hi[4];
            dev::e2m1x8_to_f16(codes[i][0], lo);
            dev::e2m1x8_to_f16(codes[i][1], hi);
#pragma unroll
            for (int k = 0; k < 4; ++k) h2[k] = lo[k], h2[4 + k] = hi[k];
        } else {
            constexpr int kCode = BITS == 4 ? 8 : BITS;
            uint32_t v[4];
            if constexpr (BITS == 8) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = codes[i][k];
            } else {
                const uint32_t a = codes[i][0], b = codes[i][1], c = codes[i][2];
                v[0] = dev::spread6(a), v[1] = dev::spread6((a >> 24) | (b << 8));
                v[2] = dev::spread6((b >> 16) | (c << 16)), v[3] = dev::spread6(c >> 8);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h2[2 * k] = dev::codes_to_f16x2<kCode>(v[k]);
                h2[2 * k + 1] = dev::codes_to_f16x2<kCode>(v[k] >> 16);
            }
        }
        const float scale = dev::ue8m0_value(scales[i]);
        float x[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2[k]));
            x[2 * k] = f.x * scale, x[2 * k + 1] = f.y * scale;
        }
        Raw16<T, VEC> out;
        out.from_float(x);
        out.store(mv.template rows<T>(token));
    }
}

template <bool WRITE, int BITS, class T, int VEC>
int launch_vec(const CacheMove& m, cudaStream_t stream) {
    const int64_t block_tokens = (int64_t)m.block_rows * (WRITE ? kWritePasses : kReadPasses);
    const int64_t blocks = (m.tokens + block_tokens - 1) / block_tokens;
    MXK_REQUIRE(blocks <= std::numeric_limits<int>::max(), "cache: too many tokens for one call");
    const dim3 grid((unsigned)blocks, (unsigned)m.kv_heads, 2);
    if constexpr (WRITE)
        cache_write_kernel<BITS, T, VEC><<<grid, 256, 0, stream>>>(m);
    else
        cache_read_kernel<BITS, T, VEC><<<grid, 256, 0, stream>>>(m);
    MXK_CUDA(cudaGetLastError());
    return MXK_OK;
}

template <bool WRITE, int BITS, class T>
int launch_typed(const CacheMove& m, int vec, cudaStream_t stream) {
    if (vec == 32) return launch_vec<WRITE, BITS, T, 32>(m, stream);
    if (vec == 16) return launch_vec<WRITE, BITS, T, 16>(m, stream);
    return launch_vec<WRITE, BITS, T, 0>(m, stream);
}

template <bool WRITE, int BITS>
int launch_bits(const CacheMove& m, int dtype, int vec, cudaStream_t stream) {
    if (dtype == MXK_F32) return launch_typed<WRITE, BITS, float>(m, vec, stream);
    if (dtype == MXK_F16) return launch_typed<WRITE, BITS, __half>(m, vec, stream);
    return launch_typed<WRITE, BITS, __nv_bfloat16>(m, vec, stream);
}

template <bool WRITE>
int cache_move(const char* who, const mxk_cache* c, int dtype, int64_t tokens, const mxk_rows* k, const mxk_rows* v,
               const int64_t* slots, cudaStream_t stream) {
    const std::string w(who);
    MXK_CHECK(check_cache(c, who));
    MXK_REQUIRE(dtype == MXK_F32 || dtype == MXK_F16 || dtype == MXK_BF16, w + ": unknown dtype");
    MXK_REQUIRE(tokens >= 0, w + ": tokens must not be negative");
    if (tokens == 0) return MXK_OK;
    MXK_REQUIRE(k && v && k->data && v->data && slots, w + ": k, v and slots must be non-null");
    const int size = dtype == MXK_F32 ? 4 : 2;
    MXK_REQUIRE(reinterpret_cast<uintptr_t>(k->data) % size == 0 && reinterpret_cast<uintptr_t>(v->data) % size == 0 &&
                    reinterpret_cast<uintptr_t>(slots) % 8 == 0,
                w + ": k, v and slots must be aligned to their elements");
    CacheMove m{};
    const mxk_rows* rows[2] = {k, v};
    for (int i = 0; i < 2; ++i)
        m.side[i] = {static_cast<uint8_t*>(i ? c->v_values : c->k_values), i ? c->v_scales : c->k_scales,
                     static_cast<char*>(rows[i]->data), rows[i]->token_stride, rows[i]->head_stride};
    m.slots = slots;
    m.tokens = tokens;
    m.n_slots = cache_slots(*c);
    m.chunks = c->head_dim / 16;
    m.block_rows = 256 / m.chunks;
    m.kv_heads = c->kv_heads;
    m.page_size = c->page_size;
    m.page_pieces = (int64_t)m.kv_heads * m.page_size * m.chunks;
    m.chunk_factor = (65536 + m.chunks - 1) / m.chunks;
    int bits = 0;  // 2^bits >= page_size
    while ((1ll << bits) < m.page_size) ++bits;
    m.page_shift = bits - 1;
    m.page_factor = (unsigned)(((1ull << (31 + bits)) + m.page_size - 1) / m.page_size);
    const int vec = rows_aligned(*k, size, 32) && rows_aligned(*v, size, 32)   ? 32
                    : rows_aligned(*k, size, 16) && rows_aligned(*v, size, 16) ? 16
                                                                               : 0;
    LaunchScope scope(WRITE ? "cache_write" : "cache_read", stream);
    if (c->bits == 8) return launch_bits<WRITE, 8>(m, dtype, vec, stream);
    if (c->bits == 6) return launch_bits<WRITE, 6>(m, dtype, vec, stream);
    return launch_bits<WRITE, 4>(m, dtype, vec, stream);
}

}  // namespace
}  // namespace mxk

extern "C" {

int mxk_cache_write(const mxk_cache* cache, int dtype, int64_t tokens, const mxk_rows* k, const mxk_rows* v,
                    const int64_t* slots, void* stream) {
    return mxk::cache_move<true>("cache_write", cache, dtype, tokens, k, v, slots, mxk::as_stream(stream));
}

int mxk_cache_read(const mxk_cache* cache, int dtype, int64_t tokens, const int64_t* slots, const mxk_rows* k,
                   const mxk_rows* v, void* stream) {
    return mxk::cache_move<false>("cache_read", cache, dtype, tokens, k, v, slots, mxk::as_stream(stream));
}

}  // extern "C"
