// Appending to the paged MX cache with the rotation by position on the way (no
// counterpart in the reference; the kept rows are those of quantize_rows,
// src/kernels/quantize.cu:13-72, of the rotated keys).
//
//     y_i = x_i cos_i - x_j sin_i,   y_j = x_j cos_i + x_i sin_i,   i < r / 2,
//
// with (i, j) = (i, i + r / 2) or, interleaved, (2 i, 2 i + 1), the cosines and sines from
// the row of the token's position in the caller's table; features from r on stay.
//
// One launch takes queries (rotated, rounded once, written back), keys (rotated and
// quantised) and values (quantised).  Per token it reads (Hq + 2 Hk) D elements, writes
// Hq D elements and 2 Hk rows of D * bits / 8 + D / 32 bytes, and does a few operations per
// element of q and some 25 per element of k, so HBM bounds it.  A thread owns 16 features of a
// row and goes through several heads of its token, with the table's row in registers.  Queries
// may be rotated in place, so a thread owns both ends of its pairs there: features 8 c .. and
// r / 2 + 8 c ...  Keys are cut as cache_write cuts them, so that a block's 32 features lie in two
// neighbouring threads, and the other ends of the pairs are loaded beside them (from L1: they
// are another thread's own).
//
// A key's codes are those of the exact rotation of its features: keys next to a border
// between two codes, or a block's largest next to a border between two scales, would
// otherwise go by the rounding of the float32 sum.  The sum is taken with its rounding
// errors (products split by fma, sums by two-sum), and rounded to odd: a value with 24 bits
// of which the last says "not exactly", which compares with every border, all of which have
// fewer bits, as the exact one does.
//
// Measured: 16,384 tokens of 32 + 8 + 8 heads of 128 in bf16, 8 bits (370 MB) in 88 us, 4.2
// TB/s, interleaved 82, in float32 (706 MB) 120, 5.9 TB/s; 6 bits 89, 83 and 120, 4 bits 87, 80 and 118; 8 tokens
// 3.3.  Threads wait for three loads one after the other (position, table, rows), so occupancy counts: with
// 2, 3 and 4 blocks an SM 123, 98 and 88 us.  At four a thread has 64 registers, of which 24 bytes spill in
// this case (up to 108 where float32 rows are not aligned).  Testing by an interval whether a code is in doubt before taking the
// sum exactly cost the registers of a block and gave nothing (90 us).
#include <algorithm>
#include <cstdlib>
#include <limits>

#include "cache_rows.cuh"

namespace mxk {
namespace {

using dev::Raw16;

struct AppendRows {
    char* data;
    int64_t token_stride, head_stride;
};

struct AppendParams {
    AppendRows q, q_out, k, v;
    uint8_t *k_values, *k_scales, *v_values, *v_scales;
    const int64_t* slots;
    const int64_t* positions;
    const float* cos_sin;  // [table_rows][rot]: cosines, then sines
    int64_t table_rows, tokens, n_slots;
    int rot, heads, kv_heads, page_size;
    int chunks, block_rows;  // 16-feature pieces of a row, tokens of a block
    int span;                // heads that a thread goes through
    int q_blocks, kv_blocks; // blocks of the same tokens that take queries; keys; values
    unsigned chunk_factor;   // thread number / chunks as a product and a shift by 16, exact below 256
};

// x c + p s rounded to odd (above); infinite or no number where the plain sum is.
__device__ __forceinline__ float turn_to_odd(float x, float c, float p, float s) {
    const float a = x * c, b = p * s;
    const float ea = __fmaf_rn(x, c, -a), eb = __fmaf_rn(p, s, -b);
    const float d = __fadd_rn(a, b), bb = __fsub_rn(d, a);
    const float tail = __fadd_rn(__fadd_rn(__fsub_rn(a, __fsub_rn(d, bb)), __fsub_rn(b, bb)), __fadd_rn(ea, eb));
    const float t = __fadd_rn(d, tail);
    if (!(fabsf(t) <= 3.402823466e38f)) return d;
    const float rest = __fadd_rn(__fsub_rn(d, t), tail);
    uint32_t bits = __float_as_uint(t);
    if (rest != 0.0f && !(bits & 1u)) bits += (rest > 0.0f) == (t > 0.0f) ? 1u : ~0u;
    return __uint_as_float(bits);
}

// N elements (8 or 16) as they lie in memory, in accesses of VEC bytes (0: one element) or as
// many as they have.  Plain loads: the rows may be those that the kernel writes.
template <class T, int N, int VEC>
struct Piece {
    uint4 w[N * sizeof(T) / 16];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC >= 16) {
#pragma unroll
            for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
            T e[N];
#pragma unroll
            for (int i = 0; i < N; ++i) e[i] = p[i];
            memcpy(w, e, sizeof(w));
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void to_float(float (&x)[N]) const {
        T e[N];
        memcpy(e, w, sizeof(w));
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = dev::to_float(e[i]);
    }
};

template <class T, int N, int VEC>
__device__ __forceinline__ void store_piece(T* p, const float (&x)[N]) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = dev::from_float<T>(x[i]);
    constexpr int kBytes = N * sizeof(T);
    if constexpr (VEC >= 16) {
        uint4 w[kBytes / 16];
        memcpy(w, e, sizeof(e));
        if constexpr (VEC == 32 && kBytes % 32 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; i += 2) dev::store32(reinterpret_cast<uint4*>(p) + i, w[i], w[i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = e[i];
    }
}

// Eight floats of the table.
__device__ __forceinline__ void load_angles(const float* p, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// Quantises a thread's 16 features, half of a block whose other half the neighbour has, and
// stores them as piece `at` of a side.  The two agree on `kept`.
template <int BITS>
__device__ __forceinline__ void keep16(float (&x)[16], uint8_t* values, uint8_t* scales, int64_t at, bool first,
                                       bool kept) {
    float amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; k += 2) amax = dev::max3_nan(amax, fabsf(x[k]), fabsf(x[k + 1]));
    amax = dev::max3_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1), 0.0f);
    const bool nans = amax != amax;
    if (nans) {
        amax = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) amax = fmaxf(amax, fabsf(x[k]));
        amax = fmaxf(amax, __shfl_xor_sync(3u << (threadIdx.x & 30u), amax, 1));
    }
    if (!kept) return;
    const uint32_t e = dev::block_scale<BITS>(amax);
    dev::pack16<BITS>(x, e, nans, values, at);
    if (first) scales[at >> 1] = (uint8_t)e;
}

template <int BITS, class T, int VEC, bool PAIRS>
__global__ void __launch_bounds__(256, 4) cache_append_kernel(const AppendParams m) {
    const int row = (int)(threadIdx.x * m.chunk_factor >> 16);
    const int c = (int)threadIdx.x - row * m.chunks;
    // (The blocks of some tokens run at about the same time: a fused projection's rows are read
    // together, and the keys' arithmetic goes on beside the queries' streaming.)
    const unsigned parts = m.q_blocks + 2 * m.kv_blocks, at_block = blockIdx.x / parts;
    const int64_t token = (int64_t)at_block * m.block_rows + row;
    const bool active = row < m.block_rows && token < m.tokens;
    const int64_t position = active ? __ldg(m.positions + token) : -1;
    const bool known = position >= 0 && position < m.table_rows;
    const float* table = m.cos_sin + (known ? position : 0) * m.rot;
    const int half = m.rot >> 1, y = (int)(blockIdx.x - at_block * parts);

    if (y < m.q_blocks) {
        if (!active) return;
        // Features a .. a + 7 and b .. b + 7: with PAIRS 16 in a row, else the two ends of 8 pairs.
        const bool turned = 16 * c < m.rot;
        const int a = PAIRS || !turned ? 16 * c : 8 * c, b = PAIRS || !turned ? a + 8 : half + 8 * c;
        const int last = min((y + 1) * m.span, m.heads);
        const T* in = reinterpret_cast<const T*>(m.q.data) + token * m.q.token_stride + (int64_t)y * m.span * m.q.head_stride;
        T* out = reinterpret_cast<T*>(m.q_out.data) + token * m.q_out.token_stride + (int64_t)y * m.span * m.q_out.head_stride;
        Piece<T, PAIRS ? 16 : 8, VEC> next[PAIRS ? 1 : 2];  // (under way while the table's row is, or a head's sums)
        auto ask = [&]() {
            next[0].load(in + a);
            if constexpr (!PAIRS) next[1].load(in + b);
        };
        ask();
        float cosine[8], sine[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cosine[i] = 1.0f, sine[i] = 0.0f;
        if (turned && known) load_angles(table + 8 * c, cosine), load_angles(table + half + 8 * c, sine);
        for (int h = y * m.span; h < last; ++h) {
            if constexpr (PAIRS) {
                float x[16];
                next[0].to_float(x);
                in += m.q.head_stride;
                if (h + 1 < last) ask();
                if (turned) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float u = x[2 * i], v = x[2 * i + 1];
                        x[2 * i] = u * cosine[i] - v * sine[i], x[2 * i + 1] = v * cosine[i] + u * sine[i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = known ? x[i] : 0.0f;
                store_piece<T, 16, VEC>(out + a, x);
            } else {
                float u[8], v[8];
                next[0].to_float(u), next[1].to_float(v);
                in += m.q.head_stride;
                if (h + 1 < last) ask();
                if (turned) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x = u[i];
                        u[i] = x * cosine[i] - v[i] * sine[i], v[i] = v[i] * cosine[i] + x * sine[i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = known ? u[i] : 0.0f, v[i] = known ? v[i] : 0.0f;
                store_piece<T, 8, VEC>(out + a, u);
                store_piece<T, 8, VEC>(out + b, v);
            }
            out += m.q_out.head_stride;
        }
        return;
    }

    const bool values = y >= m.q_blocks + m.kv_blocks;
    const int64_t slot = active ? __ldg(m.slots + token) : -1;
    const bool kept = known && slot >= 0 && slot < m.n_slots;
    const int64_t page = kept ? slot / m.page_size : 0, place = kept ? slot - page * m.page_size : 0;
    const int first = (y - m.q_blocks - (values ? m.kv_blocks : 0)) * m.span, last = min(first + m.span, m.kv_heads);
    const AppendRows& rows = values ? m.v : m.k;
    uint8_t* to_values = values ? m.v_values : m.k_values;
    uint8_t* to_scales = values ? m.v_scales : m.k_scales;
    const int f = 16 * c;
    const bool turned = !values && f < m.rot;
    // The table's numbers for this thread's features: of its 8 pairs (PAIRS), or of its two
    // halves of 8 features, each of which lies at one end of its pairs or stays.
    float cosine[PAIRS ? 8 : 16], sine[PAIRS ? 8 : 16];
    int other[2] = {0, 0};  // the halves' distance to the other ends of their pairs
    if constexpr (PAIRS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) cosine[i] = 1.0f, sine[i] = 0.0f;
        if (turned && kept) load_angles(table + 8 * c, cosine), load_angles(table + half + 8 * c, sine);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = f + 8 * i;
            float cs[8], sn[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) cs[k] = 1.0f, sn[k] = 0.0f;
            if (!values && at < m.rot) {
                const bool upper = at >= half;
                other[i] = upper ? -half : half;
                if (kept) {
                    load_angles(table + at - (upper ? half : 0), cs);
                    load_angles(table + at + (upper ? 0 : half), sn);
                }
                if (!upper) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) sn[k] = -sn[k];
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) cosine[8 * i + k] = cs[k], sine[8 * i + k] = sn[k];
        }
    }
    const int64_t piece0 = (page * m.kv_heads * m.page_size + place) * m.chunks + c;
    for (int h = first; h < last; ++h) {
        const T* in = reinterpret_cast<const T*>(rows.data) + token * rows.token_stride + (int64_t)h * rows.head_stride + f;
        float x[16];
        Raw16<T, VEC> raw;
        if (kept)
            raw.load(in);
        else
            raw.zero();
        raw.to_float(x);
        if (turned) {
            if constexpr (PAIRS) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = x[2 * i], v = x[2 * i + 1];
                    x[2 * i] = turn_to_odd(u, cosine[i], v, -sine[i]);
                    x[2 * i + 1] = turn_to_odd(v, cosine[i], u, sine[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (other[i] == 0) continue;
                    float p[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) p[k] = 0.0f;
                    if (kept) {
                        Piece<T, 8, VEC> piece;
                        piece.load(in + 8 * i + other[i]);
                        piece.to_float(p);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        x[8 * i + k] = turn_to_odd(x[8 * i + k], cosine[8 * i + k], p[k], sine[8 * i + k]);
                }
            }
        }
        keep16<BITS>(x, to_values, to_scales, piece0 + (int64_t)h * m.page_size * m.chunks, (c & 1) == 0, kept);
    }
}

// Heads that a thread goes through, which load the table's row once, by how often the blocks for one
// head each would fill the SMs.  In us for 1, 2, 3, 4 and 5, 32 + 8 + 8 heads of 128 in bf16: 8 tokens 3.8, 5.6,
// 7.2, 9.0, 10.8; 1500 (fill 3.8) 12.4, 12.6, 13.9, 13.6, 16.2; 2048 (5.2) 15.6, 14.6, 15.9, 18.0, 18.9; 4096 (10.4)
// 30.1, 26.3, 26.7, 27.2, 28.8; 8192 (20.8) 60.4, 50.4, 48.9, 48.9, 50.3; 16,384 116, 94, 89, 87, 88.
int heads_of_thread(int64_t blocks) {
    const int64_t fill = blocks / (4 * sm_count());
    return fill >= 16 ? 4 : (fill >= 4 ? 2 : 1);
}

template <int BITS, class T, int VEC, bool PAIRS>
int launch(AppendParams& m, cudaStream_t stream) {
    const int64_t blocks = (m.tokens + m.block_rows - 1) / m.block_rows;
    MXK_REQUIRE(blocks <= std::numeric_limits<int>::max(), "cache_append: too many tokens for one call");
    m.span = heads_of_thread(blocks * (m.heads + 2 * m.kv_heads));
    m.q_blocks = (m.heads + m.span - 1) / m.span, m.kv_blocks = (m.kv_heads + m.span - 1) / m.span;
    const int64_t grid = blocks * (m.q_blocks + 2 * m.kv_blocks);
    MXK_REQUIRE(grid <= std::numeric_limits<int>::max(), "cache_append: too many tokens for one call");
    LaunchScope scope("cache_append", stream);
    cache_append_kernel<BITS, T, VEC, PAIRS><<<(unsigned)grid, 256, 0, stream>>>(m);
    MXK_CUDA(cudaGetLastError());
    return MXK_OK;
}

template <int BITS, class T, int VEC>
int launch_style(AppendParams& m, bool pairs, cudaStream_t stream) {
    return pairs ? launch<BITS, T, VEC, true>(m, stream) : launch<BITS, T, VEC, false>(m, stream);
}

template <int BITS, class T>
int launch_typed(AppendParams& m, bool pairs, int vec, cudaStream_t stream) {
    if (vec == 32) return launch_style<BITS, T, 32>(m, pairs, stream);
    if (vec == 16) return launch_style<BITS, T, 16>(m, pairs, stream);
    return launch_style<BITS, T, 0>(m, pairs, stream);
}

template <int BITS>
int launch_bits(AppendParams& m, int dtype, bool pairs, int vec, cudaStream_t stream) {
    if (dtype == MXK_F32) return launch_typed<BITS, float>(m, pairs, vec, stream);
    if (dtype == MXK_F16) return launch_typed<BITS, __half>(m, pairs, vec, stream);
    return launch_typed<BITS, __nv_bfloat16>(m, pairs, vec, stream);
}

AppendRows rows_of(const mxk_rows& r) { return {static_cast<char*>(r.data), r.token_stride, r.head_stride}; }

}  // namespace
}  // namespace mxk

extern "C" int mxk_cache_append(const mxk_cache* cache, const mxk_append* a, void* stream) {
    using namespace mxk;
    MXK_CHECK(check_cache(cache, "cache_append"));
    MXK_REQUIRE(a, "cache_append: args is null");
    MXK_REQUIRE(a->dtype == MXK_F32 || a->dtype == MXK_F16 || a->dtype == MXK_BF16, "cache_append: unknown dtype");
    MXK_REQUIRE(a->tokens >= 0, "cache_append: tokens must not be negative");
    MXK_REQUIRE(a->heads >= 0 && a->heads <= 65535, "cache_append: heads must be in [0, 65535]");
    MXK_REQUIRE(a->rot_dim >= 16 && a->rot_dim % 16 == 0 && a->rot_dim <= cache->head_dim,
                "cache_append: rot_dim must be a multiple of 16 in [16, head_dim]");
    MXK_REQUIRE(a->table_rows >= 0, "cache_append: table_rows must not be negative");
    if (a->tokens == 0) return MXK_OK;
    MXK_REQUIRE(a->k.data && a->v.data && a->slots && a->positions && (a->cos_sin || a->table_rows == 0),
                "cache_append: k, v, slots, positions and cos_sin must be non-null");
    MXK_REQUIRE(a->heads == 0 || (a->q.data && a->q_out.data), "cache_append: q and q_out must be non-null");
    const int size = a->dtype == MXK_F32 ? 4 : 2;
    const mxk_rows none{};
    const mxk_rows& q = a->heads ? a->q : none;
    const mxk_rows& q_out = a->heads ? a->q_out : none;
    MXK_REQUIRE((reinterpret_cast<uintptr_t>(q.data) | reinterpret_cast<uintptr_t>(q_out.data) |
                 reinterpret_cast<uintptr_t>(a->k.data) | reinterpret_cast<uintptr_t>(a->v.data)) % size == 0 &&
                    (reinterpret_cast<uintptr_t>(a->slots) | reinterpret_cast<uintptr_t>(a->positions)) % 8 == 0,
                "cache_append: q, q_out, k, v, slots and positions must be aligned to their elements");
    MXK_REQUIRE(reinterpret_cast<uintptr_t>(a->cos_sin) % 16 == 0, "cache_append: cos_sin must be 16-byte aligned");
    // (Broadcast queries can be read but not written.)
    MXK_REQUIRE((a->heads <= 1 || std::abs(q_out.head_stride) >= cache->head_dim) &&
                    (a->heads == 0 || a->tokens == 1 || std::abs(q_out.token_stride) >= cache->head_dim),
                "cache_append: rows of q_out must not overlap");
    AppendParams m{};
    m.q = rows_of(q), m.q_out = rows_of(q_out), m.k = rows_of(a->k), m.v = rows_of(a->v);
    m.k_values = static_cast<uint8_t*>(cache->k_values), m.k_scales = cache->k_scales;
    m.v_values = static_cast<uint8_t*>(cache->v_values), m.v_scales = cache->v_scales;
    m.slots = a->slots;
    m.positions = a->positions;
    m.cos_sin = a->cos_sin;
    m.table_rows = a->table_rows;
    m.tokens = a->tokens;
    m.n_slots = cache_slots(*cache);
    m.rot = a->rot_dim;
    m.heads = a->heads, m.kv_heads = cache->kv_heads;
    m.page_size = cache->page_size;
    m.chunks = cache->head_dim / 16;
    m.block_rows = 256 / m.chunks;
    m.chunk_factor = (65536 + m.chunks - 1) / m.chunks;
    int vec = 32;
    for (const mxk_rows* r : {&q, &q_out, &a->k, &a->v}) {
        if (!rows_aligned(*r, size, 32)) vec = std::min(vec, 16);
        if (!rows_aligned(*r, size, 16)) vec = 0;
    }
    const bool pairs = a->interleaved != 0;
    const cudaStream_t st = as_stream(stream);
    if (cache->bits == 8) return launch_bits<8>(m, a->dtype, pairs, vec, st);
    if (cache->bits == 6) return launch_bits<6>(m, a->dtype, pairs, vec, st);
    return launch_bits<4>(m, a->dtype, pairs, vec, st);
}
