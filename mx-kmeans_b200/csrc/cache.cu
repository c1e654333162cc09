// Paged MX cache: quantising keys and values as they are written, and reading
// them back (no counterpart in the reference; the rows are those of
// quantize_rows, src/kernels/quantize.cu:13-72).
//
// Both kernels stream: a thread moves 16 features of one row, two of them own a
// 32-feature block and join their maxima with one shuffle.  Per row of D
// features the write reads D elements and stores D * bits / 8 + D / 32 bytes,
// the read the reverse, and neither does more than a few operations per element,
// so HBM bounds both.
#include <limits>

#include "cache.cuh"
#include "mx_codec.cuh"

namespace mxk {

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

struct Side {
    uint8_t* values;
    uint8_t* scales;
    char* data;  // rows of the caller
    int64_t token_stride, head_stride;
};

struct CacheMove {
    Side side[2];  // keys, values
    const int64_t* slots;
    int64_t n_slots;
    unsigned items;      // (token, side, head, chunk) of this launch
    unsigned per_token;  // 2 * kv_heads * chunks
    unsigned chunks;     // head_dim / 16
    int kv_heads, page_size;
};

// Where an item's 16 features lie: `data` in the caller's rows (in elements),
// `row` the cached row's index ((page * kv_heads + head) * page_size + place).
struct Item {
    int side, chunk;
    int64_t data, row, slot;
};

__device__ __forceinline__ Item locate(const CacheMove& m, unsigned g) {
    Item it;
    const unsigned token = g / m.per_token;
    const unsigned in = g - token * m.per_token;
    const unsigned row = in / m.chunks;
    it.chunk = (int)(in - row * m.chunks);
    it.side = row >= (unsigned)m.kv_heads;
    const int head = (int)row - (it.side ? m.kv_heads : 0);
    it.slot = __ldg(m.slots + token);
    const Side s = it.side ? m.side[1] : m.side[0];
    it.data = (int64_t)token * s.token_stride + (int64_t)head * s.head_stride + it.chunk * 16;
    int64_t page;
    int place;
    if ((it.slot >> 31) == 0) {
        const unsigned p = (unsigned)it.slot / (unsigned)m.page_size;
        page = p;
        place = (int)((unsigned)it.slot - p * (unsigned)m.page_size);
    } else {
        page = it.slot / m.page_size;
        place = (int)(it.slot - page * m.page_size);
    }
    it.row = (page * m.kv_heads + head) * m.page_size + place;
    return it;
}

template <class T, bool VEC>
__device__ __forceinline__ void load16(const T* p, float (&x)[16]) {
    if constexpr (VEC) {
        constexpr int n = 16 / sizeof(T);  // elements of one 16-byte load
#pragma unroll
        for (int i = 0; i < 16 / n; ++i) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(p) + i);
            T e[n];
            memcpy(e, &w, 16);
#pragma unroll
            for (int j = 0; j < n; ++j) x[i * n + j] = dev::to_float(e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = dev::to_float(p[i]);
    }
}

template <class T, bool VEC>
__device__ __forceinline__ void store16(T* p, const float (&x)[16]) {
    if constexpr (VEC) {
        constexpr int n = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16 / n; ++i) {
            T e[n];
#pragma unroll
            for (int j = 0; j < n; ++j) e[j] = dev::from_float<T>(x[i * n + j]);
            uint4 w;
            memcpy(&w, e, 16);
            reinterpret_cast<uint4*>(p)[i] = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = dev::from_float<T>(x[i]);
    }
}

// The hardware conversions round to nearest even and saturate as quantize_rows
// does.  Below 8 bits a NaN becomes the largest magnitude with the NaN's sign
// there, which the conversions do not promise, so it is replaced first.
__device__ __forceinline__ float nan_to_most(float x, float most) { return x == x ? x : copysignf(most, x); }

// Two E2M3 codes, one byte each, `lo` in the low byte.
__device__ __forceinline__ uint32_t e2m3x2_pack(float lo, float hi) {
    uint16_t out;
    asm("cvt.rn.satfinite.e2m3x2.f32 %0, %1, %2;"
        : "=h"(out)
        : "f"(nan_to_most(hi, 7.5f)), "f"(nan_to_most(lo, 7.5f)));
    return out;
}

// Eight E2M1 codes, x[0] in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8_pack(const float* x) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = nan_to_most(x[i], 6.0f);
    uint32_t out;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(out)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return out;
}

template <int BITS, class T, bool VEC>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheMove m) {
    const unsigned g = blockIdx.x * 256u + threadIdx.x;
    const bool in_range = g < m.items;
    const Item it = locate(m, in_range ? g : 0u);
    // A pair of threads shares a token, so both leave the block's maximum alike.
    const bool valid = in_range && it.slot >= 0 && it.slot < m.n_slots;
    const Side s = it.side ? m.side[1] : m.side[0];
    float x[16];
    if (valid) {
        load16<T, VEC>(reinterpret_cast<const T*>(s.data) + it.data, x);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    if (!valid) return;
    uint32_t e;
    if constexpr (BITS == 8)
        e = dev::ue8m0_mxfp8_scale(amax);
    else
        e = dev::ue8m0_encode(amax > 0.0f ? amax / (BITS == 6 ? 7.5f : 6.0f) : 1.0f);
    const float rcp = dev::ue8m0_reciprocal(e);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= rcp;  // the exact quotient by a power of two
    const int64_t at = it.row * m.chunks + it.chunk;  // in units of 16 features
    if constexpr (BITS == 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = dev::e4m3x2_encode(x[4 * i], x[4 * i + 1]) | (dev::e4m3x2_encode(x[4 * i + 2], x[4 * i + 3]) << 16);
        reinterpret_cast<uint4*>(s.values)[at] = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (BITS == 6) {
        // four 6-bit codes in three bytes, lowest first
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = e2m3x2_pack(x[4 * i], x[4 * i + 1]), b = e2m3x2_pack(x[4 * i + 2], x[4 * i + 3]);
            v[i] = (a & 0x3fu) | ((a >> 2) & 0xfc0u) | ((b & 0x3fu) << 12) | ((b & 0x3f00u) << 10);
        }
        uint32_t* out = reinterpret_cast<uint32_t*>(s.values) + at * 3;
        out[0] = v[0] | (v[1] << 24);
        out[1] = (v[1] >> 8) | (v[2] << 16);
        out[2] = (v[2] >> 16) | (v[3] << 8);
    } else {
        // low nibble = even feature
        reinterpret_cast<uint2*>(s.values)[at] = make_uint2(e2m1x8_pack(x), e2m1x8_pack(x + 8));
    }
    if ((it.chunk & 1) == 0) s.scales[at >> 1] = (uint8_t)e;
}

template <int BITS, class T, bool VEC>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheMove m) {
    const unsigned g = blockIdx.x * 256u + threadIdx.x;
    if (g >= m.items) return;
    const Item it = locate(m, g);
    const Side s = it.side ? m.side[1] : m.side[0];
    float x[16];
    if (it.slot >= 0 && it.slot < m.n_slots) {
        const int64_t at = it.row * m.chunks + it.chunk;
        uint32_t h2[8];  // the 16 elements
        if constexpr (BITS == 8) {
            const uint4 w = reinterpret_cast<const uint4*>(s.values)[at];
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h2[2 * i] = dev::codes_to_f16x2<8>(v[i]);
                h2[2 * i + 1] = dev::codes_to_f16x2<8>(v[i] >> 16);
            }
        } else if constexpr (BITS == 6) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(s.values) + at * 3;
            const uint32_t a = p[0], b = p[1], c = p[2];
            const uint32_t v[4] = {a, (a >> 24) | (b << 8), (b >> 16) | (c << 16), c >> 8};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = dev::spread6(v[i]);
                h2[2 * i] = dev::codes_to_f16x2<6>(w);
                h2[2 * i + 1] = dev::codes_to_f16x2<6>(w >> 16);
            }
        } else {
            const uint2 w = reinterpret_cast<const uint2*>(s.values)[at];
            uint32_t lo[4], hi[4];
            dev::e2m1x8_to_f16(w.x, lo);
            dev::e2m1x8_to_f16(w.y, hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) h2[i] = lo[i], h2[4 + i] = hi[i];
        }
        const float scale = dev::ue8m0_value(s.scales[at >> 1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2[i]));
            x[2 * i] = f.x * scale, x[2 * i + 1] = f.y * scale;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    }
    store16<T, VEC>(reinterpret_cast<T*>(s.data) + it.data, x);
}

template <bool WRITE, int BITS, class T>
void launch_typed(const CacheMove& m, bool vec, cudaStream_t stream) {
    const unsigned blocks = (m.items + 255u) / 256u;
    if constexpr (WRITE) {
        if (vec)
            cache_write_kernel<BITS, T, true><<<blocks, 256, 0, stream>>>(m);
        else
            cache_write_kernel<BITS, T, false><<<blocks, 256, 0, stream>>>(m);
    } else {
        if (vec)
            cache_read_kernel<BITS, T, true><<<blocks, 256, 0, stream>>>(m);
        else
            cache_read_kernel<BITS, T, false><<<blocks, 256, 0, stream>>>(m);
    }
}

template <bool WRITE, int BITS>
void launch_bits(const CacheMove& m, int dtype, bool vec, cudaStream_t stream) {
    if (dtype == MXK_F32)
        launch_typed<WRITE, BITS, float>(m, vec, stream);
    else if (dtype == MXK_F16)
        launch_typed<WRITE, BITS, __half>(m, vec, stream);
    else
        launch_typed<WRITE, BITS, __nv_bfloat16>(m, vec, stream);
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
    m.chunks = (unsigned)c->head_dim / 16u;
    m.per_token = 2u * (unsigned)c->kv_heads * m.chunks;
    m.kv_heads = c->kv_heads;
    m.page_size = c->page_size;
    m.n_slots = cache_slots(*c);
    const bool vec = rows_aligned(*k, size, 16) && rows_aligned(*v, size, 16);
    // item numbers are 32 bits: more tokens go in several launches
    const int64_t most = (int64_t)(0x7fffff00u / m.per_token);
    for (int64_t first = 0; first < tokens; first += most) {
        const int64_t n = tokens - first < most ? tokens - first : most;
        const mxk_rows* rows[2] = {k, v};
        for (int i = 0; i < 2; ++i) {
            m.side[i].values = static_cast<uint8_t*>(i ? c->v_values : c->k_values);
            m.side[i].scales = i ? c->v_scales : c->k_scales;
            m.side[i].data = static_cast<char*>(rows[i]->data) + first * rows[i]->token_stride * size;
            m.side[i].token_stride = rows[i]->token_stride;
            m.side[i].head_stride = rows[i]->head_stride;
        }
        m.slots = slots + first;
        m.items = (unsigned)n * m.per_token;
        LaunchScope scope(WRITE ? "cache_write" : "cache_read", stream);
        if (c->bits == 8)
            launch_bits<WRITE, 8>(m, dtype, vec, stream);
        else if (c->bits == 6)
            launch_bits<WRITE, 6>(m, dtype, vec, stream);
        else
            launch_bits<WRITE, 4>(m, dtype, vec, stream);
        MXK_CUDA(cudaGetLastError());
    }
    return MXK_OK;
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
