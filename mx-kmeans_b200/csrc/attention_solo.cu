// Attention of single query tokens over their sequences' own tokens, behind shared prefixes (no
// counterpart in the reference).
//
// Such parts are many and short: 64 to 256 sequences of some hundred tokens times the key heads.  In
// attention_rows_kernel, which shares a part's tokens among four warps and keeps 16 query rows, a part
// of one token takes a CTA as long as one of 128 (7 us): what there is to start and to end.  Here a
// warp takes a part alone, waits for no other, and its products have
// the tokens as M and up to eight query rows as N, so that no half of them is empty:
//
//   S^T (16 tokens x 8 rows) += K (16 x 16) Q^T (16 x 8), by blocks of 32 features, whose scales go onto
//       the finished sums, in float32: relative to the token's largest, then that with the row's factor
//   P^T, from S^T as it lies in the registers, transposed within the warp (movmatrix), is the right operand
//   O^T (D x 8 rows) += V^T (16 features x 16 tokens) P^T, a lane holding 16 (D = 64: 8) neighbouring features
//
// The weights are rounded to f16 for the product with the values, by at most 2^-11 of each (the instruction
// takes 16-bit operands at this rate, and of those f16 the most exact, as weights are held between 2^15 and
// what no longer counts); the sums that they are divided by take them in float32.  As in the other
// kernels of a call, so that a row does not depend on which of them it meets.
//
// All rows see the same tokens, so scales and NaNs need none of the rows kernel's care about what some
// rows do not see.  Value scales become f16 factors relative to a reference of the lane's block, which
// goes up with the largest; blocks of zeros count for none where that would cost the others bits.
//
// A warp has a ring of four granules of 16 tokens in shared memory, three of them on their way
// (asynchronous copies of 16 bytes); 12 warps an SM.  Long parts are cut into chunks
// (attention_parts_kernel), which the merge joins like any others; warps take them from a counter, as
// some start late (where the kernel before ends late) and chunks differ.
#include <limits>

#include "attention.cuh"
#include "mx_codec.cuh"

namespace mxk {
namespace {

using dev::ex2;
using dev::hmul2;
using dev::kExactDown;
using dev::kExpShift;
using dev::kMaxSlack;
using dev::kQueryExp;
using dev::kScaleOfZeros;
using dev::kValueLift;
using dev::kValueMax;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kGranule = 16;
constexpr int kThreads = 128;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The transpose of an 8 x 8 matrix of 16-bit elements, two of a row a lane.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint32_t f16x2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// N words of shared memory in one access.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t at, uint32_t (&w)[N]) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at));
}
__device__ __forceinline__ int lds_u8(uint32_t at) {
    int v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    return v;
}

// A granule in shared memory: keys, values, scales of the keys, of the values.
template <int D, int BITS>
struct Ring {
    static constexpr int row = D * BITS / 8;        // bytes of a cached row
    static constexpr int blocks = D / 32;           // scales of a row
    static constexpr int k_words = BITS / 4;        // of a lane's 8 features of a block
    static constexpr int v_words = D * BITS / 256;  // of its D / 8 features
    static constexpr int v_at = kGranule * row, ks_at = 2 * v_at, vs_at = ks_at + kGranule * blocks;
    static constexpr int stage = vs_at + kGranule * blocks, stages = 4;
    static constexpr int smem = kThreads / 32 * stages * stage;
    // Byte `at` of row r: 16-byte pieces are permuted, so that the lanes of a load (keys: rows 0 .. 3
    // or 4 .. 7, two pieces; values: every other row, two pieces) meet different banks.
    static __device__ __forceinline__ int place(int r, int at) {
        const int turn = row == 128 ? ((r + ((r >> 2) & 1)) & 3) << 1 : (row == 64 ? r & 2 : 0);
        return r * row + (at ^ (turn << 4));
    }
};

template <int D, int BITS>
__global__ void __launch_bounds__(kThreads, 3) attention_solo_kernel(const SharedParams p) {
    using L = Ring<D, BITS>;
    constexpr int kSteps = D / 16, kTiles = D / 16;  // products of S^T and of O^T
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int warps = gridDim.x * (kThreads / 32), warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const uint32_t ring = dev::smem_addr(smem) + (threadIdx.x >> 5) * (L::stages * L::stage);
    const float neg_inf = __int_as_float(0xff800000);
    dev::let_next_start();
    const int items = __ldg(p.solo_count) * p.kv_heads;
    auto chunk_of = [&](int item, int4& chunk, int4& rest) {
        if (item >= items) return;
        chunk = __ldg(p.solo + 2 * (item / p.kv_heads)), rest = __ldg(p.solo + 2 * (item / p.kv_heads) + 1);
    };
    // A warp's first item goes by its number, the others are taken from a counter, one ahead.
    int4 chunk = make_int4(0, 0, 0, 0), rest = chunk, next_chunk = chunk, next_rest = chunk;
    int next_item = 0;
    chunk_of(warp, chunk, rest);
    for (int item = warp; item < items; item = next_item, chunk = next_chunk, rest = next_rest) {
        if (lane == 0) next_item = warps + atomicAdd(p.solo_count + 1, 1);
        const int head = item % p.kv_heads;
        const int seq = chunk.x, query = chunk.y, begin = chunk.z, end = chunk.w;  // tokens [begin, end)
        const int number = rest.x, chunks = rest.y;                                // of the part
        const int granules = (end - begin + kGranule - 1) / kGranule;
        const int* table = p.page_table + (int64_t)seq * p.table_stride;
        const int per_page = p.page_size / kGranule;
        int at = begin / kGranule / per_page, in = begin / kGranule - at * per_page, issued = 0, to = 0;
        int page = granules > 0 ? __ldg(table + at) : 0;
        auto issue = [&]() {  // the next granule; and the number of the page after it
            if (issued < granules) {
                const uint32_t first = ((uint32_t)min(max(page, 0), p.pages - 1) * p.kv_heads + head) * p.page_size + in * kGranule;
                const int valid = end - begin - issued * kGranule;
                const uint8_t* k = p.k_values + (uint64_t)first * L::row;
                const uint8_t* v = p.v_values + (uint64_t)first * L::row;
#pragma unroll
                for (int i = 0; i < L::row / 32; ++i) {
                    const int piece = lane + 32 * i, r = piece / (L::row / 16), byte = piece % (L::row / 16) * 16;
                    const uint32_t dst = ring + to + L::place(r, byte);
                    copy16(dst, k + piece * 16, r < valid);
                    copy16(dst + L::v_at, v + piece * 16, r < valid);
                }
                constexpr int sc = L::blocks;  // 16-byte pieces of a side's scales
                if (lane < 2 * sc)
                    copy16(ring + to + L::ks_at + lane * 16,
                           (lane < sc ? p.k_scales : p.v_scales - sc * 16) + (uint64_t)first * L::blocks + lane * 16, true);
                ++issued;
                to = to == (L::stages - 1) * L::stage ? 0 : to + L::stage;
                if (++in == per_page) {
                    in = 0, ++at;
                    if (issued < granules) page = __ldg(table + at);
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < L::stages - 1; ++i) issue();
        next_item = __shfl_sync(kFull, next_item, 0);
        chunk_of(next_item, next_chunk, next_rest);

        // Q^T as the right operand: features 8 c + 4 s + (0, 1 | 2, 3) of block b at step 2 b + s.
        uint32_t q[kSteps][2];
        float factor[2];  // of rows 2 c and 2 c + 1
        {
            float x[kSteps][4];
            const uint16_t* from = static_cast<const uint16_t*>(p.q) + (int64_t)query * p.q_token +
                                   (int64_t)(head * p.group + g) * p.q_head + 8 * c;
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t a = 0, b = 0;
                if (g < p.group) {
                    const uint16_t* f = from + (k >> 1) * 32 + (k & 1) * 4;
                    if (p.q_vec) {
                        const uint2 v = __ldg(reinterpret_cast<const uint2*>(f));
                        a = v.x, b = v.y;
                    } else {
                        a = f[0] | ((uint32_t)f[1] << 16), b = f[2] | ((uint32_t)f[3] << 16);
                    }
                }
                if (p.dtype == MXK_F16) {
                    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&a));
                    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&b));
                    x[k][0] = u.x, x[k][1] = u.y, x[k][2] = v.x, x[k][3] = v.y;
                } else {
                    x[k][0] = __uint_as_float(a << 16), x[k][1] = __uint_as_float(a & 0xffff0000u);
                    x[k][2] = __uint_as_float(b << 16), x[k][3] = __uint_as_float(b & 0xffff0000u);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[k][i]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
            // 2^(12 - exponent) in two factors, each a normal float
            int e = amax > 0.0f ? (int)(__float_as_uint(amax) >> 23) - 127 : 0;
            e = max(e, -126);
            const int down = (kQueryExp - e) / 2, up = kQueryExp - e - down;
            const float f0 = __uint_as_float((uint32_t)(down + 127) << 23), f1 = __uint_as_float((uint32_t)(up + 127) << 23);
            const float mine = p.scale_log2 * __uint_as_float((uint32_t)(127 - down) << 23) * __uint_as_float((uint32_t)(127 - up) << 23);
            factor[0] = __shfl_sync(kFull, mine, 8 * c), factor[1] = __shfl_sync(kFull, mine, 8 * c + 4);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                q[k][0] = f16x2(x[k][0] * f0 * f1, x[k][1] * f0 * f1);
                q[k][1] = f16x2(x[k][2] * f0 * f1, x[k][3] * f0 * f1);
            }
        }

        float o[kTiles][4];  // features 2 t and 2 t + 1 of the lane's, rows 2 c and 2 c + 1
#pragma unroll
        for (int t = 0; t < kTiles; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
        float run_max[2] = {neg_inf, neg_inf}, base[2] = {-kExpShift, -kExpShift}, sum[2] = {0.0f, 0.0f};
        int vref = 0;  // the lane's values are relative to 2^(vref - 127), at first to the least scale there is

        auto step = [&](uint32_t here, int t0) {
            // keys of tokens g and g + 8: scales, a byte a block; values of tokens 2 c, 2 c + 1, 2 c + 8 and
            // 2 c + 9: the scales of the lane's block (0: no such token)
            uint32_t ks[2];
            int vs[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (L::blocks == 4) {
                    uint32_t w[1];
                    lds_words<1>(here + L::ks_at + (g + 8 * i) * 4, w);
                    ks[i] = w[0];
                } else {
                    ks[i] = lds_u16(here + L::ks_at + (g + 8 * i) * 2);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 2 * c + (i & 1) + 8 * (i >> 1);
                vs[i] = lds_u8(here + L::vs_at + t * L::blocks + g * L::blocks / 8);
                if (t0 + t >= end) vs[i] = 0;
            }
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            float largest[2];
            uint32_t below[2];  // octaves of the blocks' scales below the token's largest, a byte each
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t m = ks[i];
                if (L::blocks == 4) m = __vmaxu4(m, m >> 16);
                m = max(m & 255u, (m >> 8) & 255u);
                below[i] = m * (L::blocks == 4 ? 0x01010101u : 0x0101u) - ks[i];
                largest[i] = dev::ue8m0_value(m);
            }
#pragma unroll
            for (int b = 0; b < L::blocks; ++b) {
                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t h[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t k[L::k_words];
                    lds_words<L::k_words>(here + L::place(g + 8 * i, (4 * b + c) * BITS), k);
                    if constexpr (BITS == 4) {
                        dev::e2m1x8_to_f16(k[0], h[i]);
                    } else {
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            h[i][2 * w] = dev::codes_to_f16x2<8>(k[w]);
                            h[i][2 * w + 1] = dev::codes_to_f16x2<8>(k[w] >> 16);
                        }
                    }
                }
                mma16816(part, h[0][0], h[1][0], h[0][1], h[1][1], q[2 * b][0], q[2 * b][1]);
                mma16816(part, h[0][2], h[1][2], h[0][3], h[1][3], q[2 * b + 1][0], q[2 * b + 1][1]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f = __uint_as_float((uint32_t)max(127 - (int)((below[i] >> (8 * b)) & 255u), 0) << 23);
                    s[2 * i] = fmaf(part[2 * i], f, s[2 * i]), s[2 * i + 1] = fmaf(part[2 * i + 1], f, s[2 * i + 1]);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool there = t0 + g + 8 * i < end;
                s[2 * i] = there ? s[2 * i] * (factor[0] * largest[i]) : neg_inf;
                s[2 * i + 1] = there ? s[2 * i + 1] * (factor[1] * largest[i]) : neg_inf;
            }

            // A row's maximum is raised when a score exceeds it by more than the slack.
            float m[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
            if (__any_sync(kFull, m[0] > run_max[0] + kMaxSlack || m[1] > run_max[1] + kMaxSlack)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) m[i] = fmaxf(m[i], __shfl_xor_sync(kFull, m[i], d));
                    if (!(m[i] > run_max[i] + kMaxSlack)) m[i] = run_max[i];
                    const float f = m[i] == run_max[i] ? 1.0f : ex2(run_max[i] - m[i]);
                    run_max[i] = m[i];
                    base[i] = (m[i] == neg_inf ? 0.0f : m[i]) - kExpShift;
                    sum[i] *= f;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) o[t][i] *= f, o[t][2 + i] *= f;
                }
            }
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = ex2(s[i] - base[i & 1]);
            sum[0] += w[0] + w[2], sum[1] += w[1] + w[3];
            const uint32_t p0 = transposed(f16x2(w[0], w[1])), p1 = transposed(f16x2(w[2], w[3]));

            uint32_t v[4][L::v_words];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                lds_words<L::v_words>(here + L::v_at + L::place(2 * c + (i & 1) + 8 * (i >> 1), g * (L::row / 8)), v[i]);

            // The values' reference: at or above the largest scale less kValueMax.
            auto over_tokens = [&](int v) {
                v = max(v, __shfl_xor_sync(kFull, v, 1));
                return max(v, __shfl_xor_sync(kFull, v, 2));
            };
            int top = over_tokens(max(max(vs[0], vs[1]), max(vs[2], vs[3])));
            const int some = min(min(vs[0] ? vs[0] : 255, vs[1] ? vs[1] : 255), min(vs[2] ? vs[2] : 255, vs[3] ? vs[3] : 255));
            if (__any_sync(kFull, top > vref + kValueMax || some < vref - kExactDown<BITS>)) {
                // Blocks of zeros have no magnitude: scales without them, where they matter.
                if (__any_sync(kFull, top == kScaleOfZeros || vref - kExactDown<BITS> > some)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t any = 0;
#pragma unroll
                        for (int k = 0; k < L::v_words; ++k) any |= v[i][k] & dev::magnitude_bits<BITS>(k);
                        any |= __shfl_xor_sync(kFull, any, 4);  // half a block a lane, or a quarter
                        if (D == 64) any |= __shfl_xor_sync(kFull, any, 8);
                        if (!any) vs[i] = 0;
                    }
                    top = over_tokens(max(max(vs[0], vs[1]), max(vs[2], vs[3])));
                }
                if (top > vref + kValueMax) {
                    const int ref = top - kValueLift;
                    const float f = __uint_as_float((uint32_t)max(vref - ref + 127, 0) << 23);
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[t][i] *= f;
                    vref = ref;
                }
            }
            const uint32_t f0 = dev::pow2_f16x2(vs[0] - vref, vs[1] - vref), f1 = dev::pow2_f16x2(vs[2] - vref, vs[3] - vref);
            if constexpr (BITS == 4) {
#pragma unroll
                for (int j = 0; j < L::v_words; ++j) {
                    uint32_t lo[2][4], hi[2][4];  // [pair of tokens]: even features, odd ones
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t a = v[2 * i][j], b = v[2 * i + 1][j];
                        dev::e2m1x8_to_f16((a & 0x0f0f0f0fu) | ((b << 4) & 0xf0f0f0f0u), lo[i]);
                        dev::e2m1x8_to_f16(((a >> 4) & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u), hi[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma16816(o[4 * j + i], hmul2(lo[0][i], f0), hmul2(hi[0][i], f0), hmul2(lo[1][i], f1), hmul2(hi[1][i], f1), p0, p1);
                }
            } else {
#pragma unroll
                for (int j = 0; j < L::v_words; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // features 4 j + 2 i and the next
                        const uint32_t a = __byte_perm(v[0][j], v[1][j], i ? 0x7362 : 0x5140);
                        const uint32_t b = __byte_perm(v[2][j], v[3][j], i ? 0x7362 : 0x5140);
                        mma16816(o[2 * j + i], hmul2(dev::codes_to_f16x2<8>(a), f0), hmul2(dev::codes_to_f16x2<8>(a >> 16), f0),
                                 hmul2(dev::codes_to_f16x2<8>(b), f1), hmul2(dev::codes_to_f16x2<8>(b >> 16), f1), p0, p1);
                    }
            }
        };
        int from = 0;
        for (int i = 0; i < granules; ++i) {
            copy_wait<L::stages - 2>();
            __syncwarp();  // the copies of all lanes; and the stage before is done with
            issue();
            step(ring + from, begin + i * kGranule);
            from = from == (L::stages - 1) * L::stage ? 0 : from + L::stage;
        }
        copy_wait<0>();
        __syncwarp();

        // The rows: means, maxima and sums.
        const float vfactor = dev::ue8m0_value(vref);
        const int64_t out_row = p.tokens + query;  // (the sequences' side)
        const int64_t slot = (int64_t)rest.w * p.kv_heads + (int64_t)head * chunks;  // of the part's first chunk
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum[i] += __shfl_xor_sync(kFull, sum[i], d);
            const int r = 2 * c + i;
            if (r >= p.group) continue;
            const float inv = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
            const int h = head * p.group + r;
            float* to = chunks == 1 ? static_cast<float*>(p.out) + out_row * p.out_token + (int64_t)h * p.out_head
                                    : p.part + ((slot + number) * kSoloRows + r) * D;
            to += g * (D / 8);
#pragma unroll
            for (int t = 0; t < kTiles; t += 2) {
                float4 v = make_float4(o[t][i] * inv * vfactor, o[t][2 + i] * inv * vfactor, o[t + 1][i] * inv * vfactor,
                                       o[t + 1][2 + i] * inv * vfactor);
                if (sum[i] == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                *reinterpret_cast<float4*>(to + 2 * t) = v;
            }
            if (g == 0) {
                const dev::PartView view{0, 1, 0, 0, rest.z};
                if (chunks == 1) {
                    dev::store_stat(p, view, out_row, h, run_max[i], sum[i]);
                } else {
                    p.part_stat[(slot + number) * kSoloRows + r] = make_float2(run_max[i], sum[i]);
                    if (number == 0)
                        p.where[out_row * p.heads + h] = make_int4(p.kernel, (int)slot, chunks - 1, r | (rest.z > 0 ? kHasPrefix : 0));
                }
            }
        }
    }
    dev::wait_for_previous();
}

template <int D, int BITS>
int launch(const SharedParams& p, AttentionCall<SharedParams>& call) {
    constexpr int smem = Ring<D, BITS>::smem;
    static thread_local int ready_device = -1;
    int dev = 0;
    MXK_CUDA(cudaGetDevice(&dev));
    if (ready_device != dev) {
        MXK_CUDA(cudaFuncSetAttribute(attention_solo_kernel<D, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ready_device = dev;
    }
    static const int sms = sm_count();
    return call.launch("attention_solo", attention_solo_kernel<D, BITS>, (unsigned)(3 * sms), kThreads, smem, p);
}

}  // namespace

int launch_attention_solo(int bits, int head_dim, SharedParams p, int64_t slots, AttentionCall<SharedParams>& call) {
    MXK_CHECK(call.take_slots(p, slots, kSoloRows, head_dim));
    MXK_CHECK(head_dim == 128 ? (bits == 8 ? launch<128, 8>(p, call) : launch<128, 4>(p, call))
                              : (bits == 8 ? launch<64, 8>(p, call) : launch<64, 4>(p, call)));
    call.slots_later(p, slots, kSoloRows);
    return MXK_OK;
}

}  // namespace mxk
