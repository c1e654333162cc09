// Attention of new tokens over the paged MX cache: the kernel for few query rows
// and the entry point (no counterpart in the reference).
//
//     out_r = sum_t exp(s_rt) v_t / sum_t exp(s_rt),   s_rt = scale * q_r . k_t
//
// With few rows per key head (decoding: one token times the heads of a group) the
// cached rows are read once and used for a handful of products each, so their
// bytes over HBM bandwidth bound it: 2 * (D * bits / 8 + D / 32) per token and key
// head.  attention_rows_kernel keeps that stream busy:
//
//  * A CTA of four warps; every warp streams its own pairs of 16-token granules through
//    its own ring of shared-memory stages (16-byte asynchronous copies, no barrier
//    between warps) and keeps its own running maximum, sum and output rows in
//    registers.  The warps join once per unit.
//  * Products are m16n8k16 f16 with the 16 query rows as M.  Tensor throughput is
//    no concern here (tcgen05 needs 64 or more rows to pay), fragments straight
//    from the raw bytes are: the order of features inside a product is free as
//    long as q and k agree, so a lane reads a contiguous quarter of a key row, and
//    a contiguous eighth of four value rows, and converts in registers.  The row
//    pitches in shared memory keep those reads free of bank conflicts.
//  * The MX scale of a key block becomes an f16 factor relative to the step's
//    largest scale, which goes onto the finished scores.  Where that would not be
//    exact (blocks that differ by more than 2^21 with 8 bits), each token's scores
//    are relative to that token's largest scale instead, so one token's magnitude
//    does not touch another's score.  Value blocks are scaled relative to a power of
//    two that follows the largest scale of the steps; an output row is kept relative to
//    the largest such power that the row itself met, and its weights are lowered by the
//    difference.  Steps of which the rows see different tokens, with scales too far
//    apart, are multiplied in bands of 8 octaves, each for the rows that see one of its
//    tokens.
//
// Measured: 64 sequences of 1 to 8192 tokens (32 heads of 128 on 8, 8 bits, 555 MB) in
// 138 to 147 us, 3.8 to 4.0 TB/s; two of 131,072 (4 bits, 285 MB) in 101 to 102, 2.8 TB/s.
// Counters of the two: DRAM 50 and 35 % of its peak, instructions issued in 50 and 56 % of the
// cycles, ALU pipe 39 and 44 %, tensor pipe 25 and 34 %, so no unit is the bound: three
// warps a scheduler wait for their own chains (scales, conversion to f16, products,
// maximum, weights).  4 bits hold twice the elements a byte, and the instructions go by
// elements.  Finer shares did not help, neither a grid of twice as many CTAs nor short
// shares taken by CTAs as they got done: every start costs more than it evens out.  Looking
// for scales that are too far apart costs 4 to 5 % (133 and 97 us on the card with 138 and
// 101); the times beside the choices below are from before it.
#include <algorithm>
#include <limits>
#include <type_traits>

#include "attention.cuh"

namespace mxk {
namespace {

using dev::ex2;
using dev::four6;
using dev::hmul2;
using dev::kExactDown;
using dev::kKeyLift;
using dev::kQueryExp;
using dev::kScaleOfZeros;
using dev::kValueLift;
using dev::kValueMax;
using dev::pow2_f16x2;
using dev::kExpShift;
using dev::kMaxSlack;
using dev::kMostLift;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kRows = 16;     // query rows of a unit
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kGranule = 16;     // tokens of one product, contiguous in their page
constexpr int kGranules = 2;     // of one step of a warp
constexpr int kPair = kGranule * kGranules;
constexpr int kKeys = kPair * kWarps;
// Key tiles that starting and ending a unit is taken to be worth.  In us for 0, 1, 2, 4 and
// 6: 64 sequences of 1 to 8192 tokens 150, 142, 140, 144, 146; 24 sequences with 2 to 5
// query tokens and windows 35, 29, 27, 29, 29.
constexpr int kUnitCost = 2;
// CTAs that an SM holds (168 registers a thread, 75 KB of rings).  With two: 64 sequences of
// 1 to 8192 tokens 146 us instead of 142.
constexpr int kCtasPerSm = 3;
// Rows per key head up to which this kernel is taken, one pass over the keys for every 16
// of them.  In us, this and the tiles kernel, over 16,384 tokens (32 heads of 128 on 8): 32
// rows 39, 45; 48 rows 47, 47; 64 rows 56, 47; 24 sequences with 2 to 5 query tokens of 8
// heads a key head and windows 27, 54.
constexpr int kMostFewRows = 32;

// Shared-memory row pitches (bytes) of the key and value granules.  Keys are read row by
// row, a quarter per lane; values four rows per lane, an eighth each.  The pitches make the
// lanes of one load touch all banks once; 128-byte rows, for which a gap would cost the
// third CTA of an SM, have their 16-byte chunks permuted by row instead.
template <int D, int BITS>
struct Pitch;
template <> struct Pitch<128, 8> { static constexpr int k = 128, v = 128; static constexpr bool swizzled = true; };
template <> struct Pitch<128, 6> { static constexpr int k = 96, v = 112; static constexpr bool swizzled = false; };
template <> struct Pitch<128, 4> { static constexpr int k = 64, v = 80; static constexpr bool swizzled = false; };
template <> struct Pitch<64, 8> { static constexpr int k = 64, v = 80; static constexpr bool swizzled = false; };
template <> struct Pitch<64, 6> { static constexpr int k = 48, v = 48; static constexpr bool swizzled = false; };
template <> struct Pitch<64, 4> { static constexpr int k = 32, v = 48; static constexpr bool swizzled = false; };

template <int D, int BITS>
struct Stage {
    static constexpr int row = D * BITS / 8;
    static constexpr int chunks = row / 16;       // 16-byte copies of a row
    static constexpr int scale_bytes = D / 32;    // of a row
    static constexpr int v_at = kGranule * Pitch<D, BITS>::k;
    static constexpr int ks_at = v_at + kGranule * Pitch<D, BITS>::v;
    static constexpr int vs_at = ks_at + kGranule * scale_bytes;
    static constexpr int granule = vs_at + kGranule * scale_bytes;
    static constexpr int bytes = kGranules * granule;
    static constexpr int stages = 2;
    static constexpr int ring = kWarps * stages * bytes;
    static constexpr int join = kWarps * kRows * D * 4;  // the warps' outputs, after the ring is done
    static constexpr int smem = ring > join ? ring : join;
    static_assert(granule % 16 == 0, "granules start on 16-byte boundaries");
};

// 16 bytes to shared memory, the first `bytes` of them from src, the rest zero.  The
// offsets are immediates of the instruction.
template <int TO, int FROM>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(TO),
                 "n"(FROM)
                 : "memory");
}
template <int TO, int FROM>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(TO), "n"(FROM)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// N bytes of shared memory at `at` + OFF into words (the last one zero-extended), in
// accesses of W bytes, the widest that divides N and so the alignment of `at` + OFF.
constexpr int widest(int n) { return n % 16 == 0 ? 16 : (n % 8 == 0 ? 8 : (n % 4 == 0 ? 4 : 2)); }
template <int N, int OFF, int W = widest(N)>
__device__ __forceinline__ void lds_bytes(uint32_t at, uint32_t* w) {
    static_assert(N % W == 0 && OFF % W == 0, "aligned accesses");
    if constexpr (W == 16) {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(at), "n"(OFF));
    } else if constexpr (W == 8) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(w[0]), "=r"(w[1]) : "r"(at), "n"(OFF));
    } else if constexpr (W == 4) {
        asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(w[0]) : "r"(at), "n"(OFF));
    } else {
        static_assert(N == 6, "rows end on even bytes");
        uint16_t a, b, c;
        asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(a) : "r"(at), "n"(OFF));
        asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(b) : "r"(at), "n"(OFF + 2));
        asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(c) : "r"(at), "n"(OFF + 4));
        w[0] = a | ((uint32_t)b << 16);
        w[1] = c;
    }
    if constexpr (W >= 4 && N > W) lds_bytes<N - W, OFF + W, W>(at, w + W / 4);
}

__device__ __forceinline__ void lds_at(uint32_t at, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
}

template <int OFF>
__device__ __forceinline__ int lds_u8(uint32_t at) {
    int v;
    asm volatile("ld.shared.u8 %0, [%1 + %2];" : "=r"(v) : "r"(at), "n"(OFF));
    return v;
}

// c += a (16 x 16, row) * b (16 x 8, column), f16 operands, f32 sums.
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The magnitude bits of word k of a lane's N bytes of a packed row.
template <int BITS, int N>
__device__ __forceinline__ uint32_t share_bits(int k) {
    if constexpr (BITS != 6) {
        return dev::magnitude_bits<BITS>(k);
    } else if constexpr (N % 12 == 0) {
        return dev::magnitude_bits<6>(k);
    } else {  // six bytes, from the first code of a group of four
        static_assert(N == 6, "");
        return k == 0 ? 0xdf7df7dfu : 0x7df7u;
    }
}

template <int D, int BITS>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_rows_kernel(const AttentionParams p) {
    using S = Stage<D, BITS>;
    using P = Pitch<D, BITS>;
    constexpr int kSteps = D / 16;       // k-steps of q . k
    constexpr int kTiles = D / 8;        // 8-feature tiles of the output
    constexpr int kShare = S::row / 4;   // bytes of a key row a lane reads
    constexpr int vShare = S::row / 8;   // bytes of a value row a lane reads
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int scratch[2 * kWarps + 2];
    __shared__ float stat_max[kWarps][kRows], stat_sum[kWarps][kRows];
    __shared__ __align__(16) uint4 query[kSteps][32];  // the A operand of every k-step, lane by lane
    __shared__ int2 row_range[kRows];                  // tokens [x, y) take part in the row

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, c = lane & 3;
    const uint32_t ring = dev::smem_addr(smem) + warp * (S::stages * S::bytes);
    // Where a lane's 16 bytes of a granule go: the i-th of them lie 512 bytes further in the
    // cache, and a constant further here where rows lie without gaps or 32 pieces fill rows.
    constexpr int kPieces = kGranule * S::chunks;  // of a side
    constexpr int kCopies = (kPieces + 31) / 32;
    constexpr int kStep = P::k == S::row ? 512 : 32 / S::chunks * P::k;
    constexpr int vStep = P::v == S::row ? 512 : 32 / S::chunks * P::v;
    static_assert(P::k == S::row || 32 % S::chunks == 0, "key rows without gaps, or whole rows in a copy");
    constexpr bool vEven = P::v == S::row || 32 % S::chunks == 0;
    constexpr int kPlaces = P::swizzled ? 2 : 1;               // rows of copy i: lane / 8 + 4 i
    constexpr int vPlaces = P::swizzled ? 2 : (vEven ? 1 : kCopies);
    uint32_t k_lane[kPlaces], v_lane[vPlaces];
    if constexpr (P::swizzled) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            k_lane[i] = ring + (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3) + 4 * i)) << 4);
            v_lane[i] = k_lane[i] + S::v_at;
        }
    } else {
        k_lane[0] = ring + (P::k == S::row ? lane * 16 : lane / S::chunks * P::k + lane % S::chunks * 16);
#pragma unroll
        for (int i = 0; i < vPlaces; ++i) {
            const int x = lane + 32 * i;
            v_lane[i] = ring + S::v_at + (P::v == S::row ? lane * 16 : x / S::chunks * P::v + x % S::chunks * 16);
        }
    }
    static_assert(P::k % widest(kShare) == 0 && P::v % widest(vShare) == 0 && S::v_at % 16 == 0 && S::granule % 16 == 0,
                  "reads are aligned to their width");
    // Where this lane reads: 16-byte halves of its key share; its even and odd tokens' values.
    uint32_t k_read[2], v_read[2];
    k_read[0] = ring + g * P::k + (P::swizzled ? (2 * c ^ g) << 4 : c * kShare);
    k_read[1] = ring + g * P::k + ((2 * c + 1) ^ g) * 16;  // swizzled rows only
    v_read[0] = ring + S::v_at + 2 * c * P::v + (P::swizzled ? (g ^ 2 * c) << 4 : g * vShare);
    v_read[1] = ring + S::v_at + (2 * c + 1) * P::v + (P::swizzled ? (g ^ (2 * c + 1)) << 4 : g * vShare);
    const uint32_t ks_read = ring + S::ks_at + g * S::scale_bytes + (D == 128 ? c : c >> 1);
    const uint32_t vs_read = ring + S::vs_at + 2 * c * S::scale_bytes + (D == 128 ? g >> 1 : g >> 2);

    dev::let_next_start();
    const dev::Share share = dev::take_share<kRows, kKeys, kUnitCost, kThreads>(p, scratch);
    if (share.tiles == 0) {
        if (tid == 0) p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0);
        dev::wait_for_previous();
        return;
    }
    dev::Walk w = dev::walk_to<kRows, kKeys>(p, share);
    int left = share.tiles - w.skip;
    bool open = false;

    while (left > 0) {
        const int tile0 = w.tile;
        const int tiles = min(left, w.tiles - tile0);
        const int rows = min(w.view.n * p.group - w.rt * kRows, kRows);
        const int len = w.view.len;

        // This lane's rows are g and g + 8.  Rows past the unit's see everything; they are
        // zero queries and never written.
        int all_lo = 0, all_hi = len, any_lo, any_hi;
        int64_t row_at[2];
        bool real[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = w.rt * kRows + g + 8 * i;
            real[i] = g + 8 * i < rows;
            const int j = r / p.group;
            int lo = 0, hi = len;
            if (real[i]) dev::seen_range(p, w.view, j, j, lo, hi);
            if (warp == 0 && c == 0) row_range[g + 8 * i] = make_int2(lo, hi);
            row_at[i] = (int64_t)(w.view.row0 + j) * p.q_token +
                        (int64_t)(w.head * p.group + (r - j * p.group)) * p.q_head;
        }
        {
            const int r0 = w.rt * kRows, j0 = r0 / p.group, j1 = (r0 + rows - 1) / p.group;
            int x;
            dev::seen_range(p, w.view, j0, j1, any_lo, any_hi);  // seen by some row
            dev::seen_range(p, w.view, j0, j0, x, all_hi);       // the first row ends first,
            dev::seen_range(p, w.view, j1, j1, all_lo, x);       // the last begins last
        }

        // The warp's pairs of granules: numbers pair0, pair0 + 4, ... of the sequence below `end`.
        // A granule is contiguous in its page, so a lane copies 16 bytes every 512.
        const int pair0 = (w.first + tile0) * kWarps + warp;
        const int end = min((w.first + tile0 + tiles) * kWarps, any_hi <= any_lo ? 0 : (any_hi + kPair - 1) / kPair);
        const int steps = end > pair0 ? (end - pair0 + kWarps - 1) / kWarps : 0;
        const int* table = p.page_table + (int64_t)w.seq * p.table_stride;
        const int per_page = p.page_size / kGranule;
        // pages and granules from a step's first granule to the next step's
        const int jump = kWarps * kGranules / per_page, rest = kWarps * kGranules - jump * per_page;
        int next_at = pair0 * kGranules / per_page, next_in = pair0 * kGranules - next_at * per_page;
        struct Pages {
            int page[2];
            int in[2];  // the granules' places in them
        };
        auto next_pages = [&](int step) -> Pages {
            Pages n{{0, 0}, {next_in, next_in + 1}};
            if (step < steps) {
                const bool over = n.in[1] == per_page;
                if (over) n.in[1] = 0;
                n.page[0] = n.page[1] = min(max(__ldg(table + next_at), 0), p.pages - 1);
                if (over && (pair0 + step * kWarps) * kPair + kGranule < len)
                    n.page[1] = min(max(__ldg(table + next_at + 1), 0), p.pages - 1);
                next_at += jump, next_in += rest;
                if (next_in >= per_page) next_in -= per_page, ++next_at;
            }
            return n;
        };
        // The lane's first bytes of page 0 of the head, and where the scales go.
        constexpr int sc = kGranule * S::scale_bytes / 16;  // 16-byte pieces of a side's scales
        const int64_t head_row = (int64_t)w.head * p.page_size;
        const uint8_t* k_src = p.k_values + head_row * S::row + lane * 16;
        const uint8_t* v_src = p.v_values + head_row * S::row + lane * 16;
        const uint8_t* s_src = (lane < sc ? p.k_scales : p.v_scales - sc * 16) + head_row * S::scale_bytes + lane * 16;
        const uint32_t page_rows = (uint32_t)p.kv_heads * p.page_size;
        int copy_stage = 0;  // offset of the stage to copy to
        auto copy_piece = [&](auto index, auto granule, const uint8_t* k, const uint8_t* v, int valid) {
            constexpr int i = decltype(index)::value, at = decltype(granule)::value * S::granule;
            if (i < kCopies && (kPieces % 32 == 0 || lane + 32 * i < kPieces)) {
                const uint32_t to_k = k_lane[P::swizzled ? i & 1 : 0] + copy_stage;
                const uint32_t to_v = v_lane[P::swizzled ? i & 1 : (vEven ? 0 : i)] + copy_stage;
                constexpr int v_off = at + (vEven ? i * vStep : 0);
                if (valid >= kGranule) {
                    copy16<at + i * kStep, 512 * i>(to_k, k);
                    copy16<v_off, 512 * i>(to_v, v);
                } else {  // rows past the sequence's end are zeros
                    const int bytes = (lane + 32 * i) / S::chunks < valid ? 16 : 0;
                    copy16<at + i * kStep, 512 * i>(to_k, k, bytes);
                    copy16<v_off, 512 * i>(to_v, v, bytes);
                }
            }
        };
        auto copy_granule = [&](auto granule, int page, int in, int valid) {
            constexpr int gi = decltype(granule)::value;
            const uint32_t row = (uint32_t)page * page_rows + (uint32_t)in * kGranule;
            const uint8_t* k = k_src + (uint64_t)row * S::row;
            const uint8_t* v = v_src + (uint64_t)row * S::row;
            static_assert(kCopies <= 4, "");
            copy_piece(std::integral_constant<int, 0>{}, granule, k, v, valid);
            copy_piece(std::integral_constant<int, 1>{}, granule, k, v, valid);
            copy_piece(std::integral_constant<int, 2>{}, granule, k, v, valid);
            copy_piece(std::integral_constant<int, 3>{}, granule, k, v, valid);
            if (lane < 2 * sc)
                copy16<S::ks_at + gi * S::granule, 0>(ring + copy_stage + lane * 16, s_src + (uint64_t)row * S::scale_bytes);
        };
        auto issue = [&](int step, const Pages& n) {
            if (step < steps) {
                const int valid = len - (pair0 + step * kWarps) * kPair;
                copy_granule(std::integral_constant<int, 0>{}, n.page[0], n.in[0], valid);
                copy_granule(std::integral_constant<int, 1>{}, n.page[1], n.in[1], valid - kGranule);
                copy_stage = copy_stage == (S::stages - 1) * S::bytes ? 0 : copy_stage + S::bytes;
            }
            copy_commit();
        };
#pragma unroll
        for (int s = 0; s < S::stages - 1; ++s) issue(s, next_pages(s));
        Pages pages = next_pages(S::stages - 1);

        // q as the A operand: features c * D/4 + 4 i .. + 3 of rows g, g + 8 at step i.
        uint32_t qa[kSteps / kWarps][4];  // those of this warp's k-steps
        float row_factor[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x[D / 4];
            const uint16_t* q = static_cast<const uint16_t*>(p.q) + (row_at[i] + c * (D / 4));
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t a = 0, b = 0;
                if (real[i]) {
                    if (p.q_vec) {
                        const uint2 v = __ldg(reinterpret_cast<const uint2*>(q) + k);
                        a = v.x, b = v.y;
                    } else {
                        a = q[4 * k] | ((uint32_t)q[4 * k + 1] << 16);
                        b = q[4 * k + 2] | ((uint32_t)q[4 * k + 3] << 16);
                    }
                }
                if (p.dtype == MXK_F16) {
                    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&a));
                    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&b));
                    x[4 * k] = u.x, x[4 * k + 1] = u.y, x[4 * k + 2] = v.x, x[4 * k + 3] = v.y;
                } else {
                    x[4 * k] = __uint_as_float(a << 16), x[4 * k + 1] = __uint_as_float(a & 0xffff0000u);
                    x[4 * k + 2] = __uint_as_float(b << 16), x[4 * k + 3] = __uint_as_float(b & 0xffff0000u);
                }
            }
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 4; ++k) amax = fmaxf(amax, fabsf(x[k]));
            amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
            // 2^(12 - exponent) in two factors, each a normal float
            int e = amax > 0.0f ? (int)(__float_as_uint(amax) >> 23) - 127 : 0;
            e = max(e, -126);
            const int down = (kQueryExp - e) / 2, rest = kQueryExp - e - down;
            const float f0 = __uint_as_float((uint32_t)(down + 127) << 23);
            const float f1 = __uint_as_float((uint32_t)(rest + 127) << 23);
            row_factor[i] = p.scale_log2 * __uint_as_float((uint32_t)(127 - down - kKeyLift / 2) << 23) *
                            __uint_as_float((uint32_t)(127 - rest - kKeyLift / 2) << 23);
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
                if (k / (kSteps / kWarps) == warp) {
                    const __half2 u = __floats2half2_rn(x[4 * k] * f0 * f1, x[4 * k + 1] * f0 * f1);
                    const __half2 v = __floats2half2_rn(x[4 * k + 2] * f0 * f1, x[4 * k + 3] * f0 * f1);
                    qa[k % (kSteps / kWarps)][i] = *reinterpret_cast<const uint32_t*>(&u);
                    qa[k % (kSteps / kWarps)][2 + i] = *reinterpret_cast<const uint32_t*>(&v);
                }
        }
#pragma unroll
        for (int k = 0; k < kSteps / kWarps; ++k)
            query[warp * (kSteps / kWarps) + k][lane] = make_uint4(qa[k][0], qa[k][1], qa[k][2], qa[k][3]);
        __syncthreads();
        const uint32_t q_read = dev::smem_addr(&query[0][lane]);

        float o[kTiles][4];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        const float neg_inf = __int_as_float(0xff800000);
        float run_max[2] = {neg_inf, neg_inf};  // of rows g, g + 8, log2 units
        float base[2] = {-kExpShift, -kExpShift};  // what is subtracted from a score: run_max - kExpShift
        float sum[2] = {0.0f, 0.0f};               // this lane's share of the rows' sums
        int vref = 0;                              // values are held relative to 2^(vref - 127); 0: none yet
        int row_ref[2] = {0, 0};                   // the output rows relative to 2^(row_ref - 127)
        int settled = -1;                          // the vref that all rows have taken note of; -1: not all
        bool lowered = false;                      // some row's reference is above vref

        int stage = 0;  // offset of the stage at hand
        for (int step = 0; step < steps; ++step) {
            copy_wait<S::stages - 2>();
            __syncwarp();
            issue(step + S::stages - 1, pages);
            pages = next_pages(step + S::stages);
            const int now = stage;
            stage = stage == (S::stages - 1) * S::bytes ? 0 : stage + S::bytes;
            const int t0 = (pair0 + step * kWarps) * kPair;
            const bool partly = t0 < all_lo || t0 + kPair > all_hi;  // some row does not see all of it

            // The references of the keys, the step's largest scale, and of the values, which
            // moves with the data.  Tokens that no row sees, before a window or past the end,
            // count for nothing: their pages may have been given away and hold any bytes.
            int ks[4], vs[8];
            ks[0] = lds_u8<0>(ks_read + now), ks[1] = lds_u8<8 * S::scale_bytes>(ks_read + now);
            ks[2] = lds_u8<S::granule>(ks_read + now), ks[3] = lds_u8<S::granule + 8 * S::scale_bytes>(ks_read + now);
            vs[0] = lds_u8<0>(vs_read + now), vs[1] = lds_u8<S::scale_bytes>(vs_read + now);
            vs[2] = lds_u8<8 * S::scale_bytes>(vs_read + now), vs[3] = lds_u8<9 * S::scale_bytes>(vs_read + now);
            vs[4] = lds_u8<S::granule>(vs_read + now), vs[5] = lds_u8<S::granule + S::scale_bytes>(vs_read + now);
            vs[6] = lds_u8<S::granule + 8 * S::scale_bytes>(vs_read + now);
            vs[7] = lds_u8<S::granule + 9 * S::scale_bytes>(vs_read + now);
            int k_least = min(min(ks[0], ks[1]), min(ks[2], ks[3]));
            int v_least = min(min(min(vs[0], vs[1]), min(vs[2], vs[3])), min(min(vs[4], vs[5]), min(vs[6], vs[7])));
            bool leading = false, trailing = false;  // some rows see only its end, or only its beginning
            if (partly) {
                const unsigned seen = (unsigned)(any_hi - any_lo);
                k_least = v_least = 255;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((unsigned)(t0 + g + 8 * i - any_lo) >= seen)
                        ks[i] = 0;
                    else
                        k_least = min(k_least, ks[i]);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if ((unsigned)(t0 + 2 * c + (i & 1) + 8 * (i >> 1) - any_lo) >= seen)
                        vs[i] = 0;
                    else
                        v_least = min(v_least, vs[i]);
                leading = t0 < all_lo && any_lo < all_lo, trailing = t0 + kPair > all_hi && all_hi < any_hi;
            }
            auto largest = [&]() -> int {
                return (int)__reduce_max_sync(kFull, (unsigned)max(max(max(vs[0], vs[1]), max(vs[2], vs[3])),
                                                                   max(max(vs[4], vs[5]), max(vs[6], vs[7]))));
            };
            const int kref = max((int)__reduce_max_sync(kFull, (unsigned)max(max(ks[0], ks[1]), max(ks[2], ks[3]))), 1);
            const int vtop = largest();

            // An output row's reference goes up when the row meets a larger one.
            auto raise_row = [&](int i, int ref) {
                const float f = __uint_as_float((uint32_t)max(row_ref[i] - ref + 127, 0) << 23);
#pragma unroll
                for (int n = 0; n < kTiles; ++n) o[n][2 * i] *= f, o[n][2 * i + 1] *= f;
                row_ref[i] = ref;
            };
            uint32_t key_refs = 0;  // rare: the references of this lane's four tokens, a byte each
            bool bands = false;     // rare: the values are multiplied in bands
            if (__any_sync(kFull, k_least < kref - kKeyLift - kExactDown<BITS> || v_least < vref - kExactDown<BITS>) ||
                (unsigned)(vtop - vref) > (unsigned)kValueMax || vref != settled || leading) {
                // Blocks of zeros have no magnitude: scales without them, where they matter.
                if (__any_sync(kFull, k_least < kref - kKeyLift - kExactDown<BITS>)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t at = now + (i >> 1) * S::granule + (i & 1) * (8 * P::k);
                        uint32_t words[(kShare + 3) / 4], any = 0;
                        if constexpr (P::swizzled)
                            lds_bytes<16, 0>(k_read[0] + at, words), lds_bytes<16, 0>(k_read[1] + at, words + 4);
                        else
                            lds_bytes<kShare, 0>(k_read[0] + at, words);
#pragma unroll
                        for (int k = 0; k < (kShare + 3) / 4; ++k) any |= words[k] & share_bits<BITS, kShare>(k);
                        if (D == 64) any |= __shfl_xor_sync(kFull, any, 1);  // half a block a lane
                        int ref = any ? ks[i] : 0;
                        ks[i] = ref;
                        ref = max(ref, __shfl_xor_sync(kFull, ref, 1));
                        ref = max(max(ref, __shfl_xor_sync(kFull, ref, 2)), 1);
                        key_refs |= (uint32_t)ref << (8 * i);
                        ks[i] += kref - ref;
                    }
                }
                // the smallest but 0; 256 if there is none
                auto lowest = [&]() -> int {
                    unsigned m = 255u;
#pragma unroll
                    for (int i = 0; i < 8; ++i) m = min(m, (unsigned)vs[i] - 1u);
                    return (int)__reduce_min_sync(kFull, m) + 1;
                };
                const int most = leading ? kMostLift : kValueLift + kExactDown<BITS>;
                int top = vtop, low = lowest();
                if (top - low > most || (top == kScaleOfZeros && low == kScaleOfZeros)) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t at = v_read[i & 1] + now + (i >> 2) * S::granule + ((i >> 1) & 1) * (8 * P::v);
                        uint32_t words[(vShare + 3) / 4], any = 0;
                        lds_bytes<vShare, 0>(at, words);
#pragma unroll
                        for (int k = 0; k < (vShare + 3) / 4; ++k) any |= words[k] & share_bits<BITS, vShare>(k);
                        any |= __shfl_xor_sync(kFull, any, 4);  // half a block a lane, or a quarter
                        if (D == 64) any |= __shfl_xor_sync(kFull, any, 8);
                        if (!any) vs[i] = 0;
                    }
                    top = largest(), low = lowest();
                }
                bands = (leading || trailing) && top - low > most;
                // (A reference is at most the step's largest scale, so what earlier steps held,
                // and some rows did not see, does not stay.)
                if (!bands && top > 0 &&
                    (vref == 0 || top > vref + kValueMax || top < vref || low < vref - kExactDown<BITS>))
                    vref = max(top - kValueLift, 1);
                if (bands) {
                    settled = -1;
                } else if (vref > 0 && vref != settled) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        bool sees = true;
                        if (leading || trailing) {
                            const int2 range = row_range[g + 8 * i];
                            sees = range.x < t0 + kPair && range.y > t0;
                        }
                        if (sees && row_ref[i] < vref) raise_row(i, vref);
                    }
                    lowered = __any_sync(kFull, max(row_ref[0], row_ref[1]) > vref);
                    settled = leading || trailing ? -1 : vref;
                }
            }

            // scores: 16 rows x 4 tiles of 8 tokens
            float s[4][4];
            auto multiply_keys = [&]() {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t key_words[2][(kShare + 3) / 4];
                    const uint32_t at = now + h * S::granule;
                    if constexpr (P::swizzled) {
                        lds_bytes<16, 0>(k_read[0] + at, key_words[0]), lds_bytes<16, 0>(k_read[1] + at, key_words[0] + 4);
                        lds_bytes<16, 8 * P::k>(k_read[0] + at, key_words[1]);
                        lds_bytes<16, 8 * P::k>(k_read[1] + at, key_words[1] + 4);
                    } else {
                        lds_bytes<kShare, 0>(k_read[0] + at, key_words[0]);
                        lds_bytes<kShare, 8 * P::k>(k_read[0] + at, key_words[1]);
                    }
                    const int e0 = ks[2 * h] - kref + kKeyLift, e1 = ks[2 * h + 1] - kref + kKeyLift;
                    const uint32_t kf[2] = {pow2_f16x2(e0, e0), pow2_f16x2(e1, e1)};
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
                        s[2 * h + nt][0] = s[2 * h + nt][1] = s[2 * h + nt][2] = s[2 * h + nt][3] = 0.0f;
#pragma unroll
                    for (int k = 0; k < kSteps; k += 2) {
                        uint32_t qa[2][4];
                        lds_at(q_read + 512 * k, qa[0]);
                        lds_at(q_read + 512 * (k + 1), qa[1]);
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            uint32_t x[4];
                            if constexpr (BITS == 4) {
                                dev::e2m1x8_to_f16(key_words[nt][k / 2], x);
                            } else {
                                constexpr int kCode = BITS == 4 ? 8 : BITS;
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const uint32_t four = BITS == 8 ? key_words[nt][k + i] : four6(key_words[nt], k + i);
                                    x[2 * i] = dev::codes_to_f16x2<kCode>(four);
                                    x[2 * i + 1] = dev::codes_to_f16x2<kCode>(four >> 16);
                                }
                            }
                            mma16816(s[2 * h + nt], qa[0], hmul2(x[0], kf[nt]), hmul2(x[1], kf[nt]));
                            mma16816(s[2 * h + nt], qa[1], hmul2(x[2], kf[nt]), hmul2(x[3], kf[nt]));
                        }
                    }
                }
            };
            if (key_refs == 0) {
                multiply_keys();
                const float kfactor = __uint_as_float((uint32_t)kref << 23);
                const float fa = row_factor[0] * kfactor, fb = row_factor[1] * kfactor;
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) s[nt][0] *= fa, s[nt][1] *= fa, s[nt][2] *= fb, s[nt][3] *= fb;
            } else {
                multiply_keys();
                // columns 2c and 2c + 1 of the four tiles: the tokens of lanes 8c and 8c + 4
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t refs = __shfl_sync(kFull, key_refs, 8 * c + 4 * e);
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt) {
                        const float f = __uint_as_float(((refs >> (8 * nt)) & 255u) << 23);
                        s[nt][e] *= row_factor[0] * f, s[nt][2 + e] *= row_factor[1] * f;
                    }
                }
            }
            if (partly) {
                const int2 range[2] = {row_range[g], row_range[g + 8]};
#pragma unroll
                for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = t0 + 8 * nt + 2 * c + (e & 1);
                        if (t < range[e >> 1].x || t >= range[e >> 1].y) s[nt][e] = neg_inf;
                    }
            }

            // Raise the maximum of the rows where some score exceeds it by more than the
            // slack (row by row: a row's result does not depend on its neighbours).
            float m[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                m[i] = fmaxf(fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1])),
                             fmaxf(fmaxf(s[2][2 * i], s[2][2 * i + 1]), fmaxf(s[3][2 * i], s[3][2 * i + 1])));
            if (__any_sync(kFull, m[0] > run_max[0] + kMaxSlack || m[1] > run_max[1] + kMaxSlack)) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    m[i] = fmaxf(m[i], __shfl_xor_sync(kFull, m[i], 1));
                    m[i] = fmaxf(m[i], __shfl_xor_sync(kFull, m[i], 2));
                    if (!(m[i] > run_max[i] + kMaxSlack)) m[i] = run_max[i];
                    const float f = m[i] == run_max[i] ? 1.0f : ex2(run_max[i] - m[i]);
                    run_max[i] = m[i];
                    base[i] = (m[i] == neg_inf ? 0.0f : m[i]) - kExpShift;
                    sum[i] *= f;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) o[n][2 * i] *= f, o[n][2 * i + 1] *= f;
                }
            }
            uint32_t pa[2][4];
            auto make_weights = [&]() {
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) {
                    const float p0 = ex2(s[nt][0] - base[0]), p1 = ex2(s[nt][1] - base[0]);
                    const float p2 = ex2(s[nt][2] - base[1]), p3 = ex2(s[nt][3] - base[1]);
                    sum[0] += p0 + p1, sum[1] += p2 + p3;
                    const __half2 a = __floats2half2_rn(p0, p1), b = __floats2half2_rn(p2, p3);
                    pa[nt >> 1][2 * (nt & 1)] = *reinterpret_cast<const uint32_t*>(&a);
                    pa[nt >> 1][2 * (nt & 1) + 1] = *reinterpret_cast<const uint32_t*>(&b);
                }

            };
            // values: of each granule this lane's tokens 2c, 2c + 1, 2c + 8, 2c + 9, their
            // scales in vs relative to ref
            auto add_values = [&](const int (&vs)[8], int ref) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t at = now + h * S::granule;
                    uint32_t vw[4][(vShare + 3) / 4];
                    lds_bytes<vShare, 0>(v_read[0] + at, vw[0]);
                    lds_bytes<vShare, 0>(v_read[1] + at, vw[1]);
                    lds_bytes<vShare, 8 * P::v>(v_read[0] + at, vw[2]);
                    lds_bytes<vShare, 8 * P::v>(v_read[1] + at, vw[3]);
                    const uint32_t f0 = pow2_f16x2(vs[4 * h] - ref, vs[4 * h + 1] - ref);
                    const uint32_t f1 = pow2_f16x2(vs[4 * h + 2] - ref, vs[4 * h + 3] - ref);
                    bool nans = false;
                    if constexpr (BITS == 8) {
                        // A stored NaN belongs to the rows that see its token: where some row
                        // does not, it is taken out here and put into the others' sums below.
                        if (partly) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int j = 0; j < vShare / 4; ++j) {
                                    const uint32_t bad = __vcmpeq4(vw[i][j] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                                    nans |= bad != 0;
                                    vw[i][j] &= ~bad;
                                }
                            nans = __any_sync(kFull, nans);
                        }
                    }
                    if constexpr (BITS == 4) {
#pragma unroll
                        for (int j = 0; j < vShare / 4; ++j) {
                            // bytes of (token, token + 1) nibbles: even features, then odd ones
                            uint32_t even[2][4], odd[2][4];
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t a = vw[2 * i][j], b = vw[2 * i + 1][j];
                                dev::e2m1x8_to_f16((a & 0x0f0f0f0fu) | ((b << 4) & 0xf0f0f0f0u), even[i]);
                                dev::e2m1x8_to_f16(((a >> 4) & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u), odd[i]);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                mma16816(o[8 * j + 2 * i], pa[h], hmul2(even[0][i], f0), hmul2(even[1][i], f1));
                                mma16816(o[8 * j + 2 * i + 1], pa[h], hmul2(odd[0][i], f0), hmul2(odd[1][i], f1));
                            }
                        }
                    } else {
                        constexpr int kCode = BITS == 4 ? 8 : BITS;
#pragma unroll
                        for (int j = 0; j < D / 32; ++j) {
                            uint32_t four[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) four[i] = BITS == 8 ? vw[i][j] : four6(vw[i], j);
                            // (token, token + 1) bytes of features 0, 1 and of 2, 3
                            const uint32_t a01 = __byte_perm(four[0], four[1], 0x5140);
                            const uint32_t a23 = __byte_perm(four[0], four[1], 0x7362);
                            const uint32_t b01 = __byte_perm(four[2], four[3], 0x5140);
                            const uint32_t b23 = __byte_perm(four[2], four[3], 0x7362);
                            mma16816(o[4 * j], pa[h], hmul2(dev::codes_to_f16x2<kCode>(a01), f0),
                                     hmul2(dev::codes_to_f16x2<kCode>(b01), f1));
                            mma16816(o[4 * j + 1], pa[h], hmul2(dev::codes_to_f16x2<kCode>(a01 >> 16), f0),
                                     hmul2(dev::codes_to_f16x2<kCode>(b01 >> 16), f1));
                            mma16816(o[4 * j + 2], pa[h], hmul2(dev::codes_to_f16x2<kCode>(a23), f0),
                                     hmul2(dev::codes_to_f16x2<kCode>(b23), f1));
                            mma16816(o[4 * j + 3], pa[h], hmul2(dev::codes_to_f16x2<kCode>(a23 >> 16), f0),
                                     hmul2(dev::codes_to_f16x2<kCode>(b23 >> 16), f1));
                        }
                    }
                    if (nans) {
                        for (int t = 0; t < kGranule; ++t)
                            for (int i = 0; i < 2; ++i) {
                                const int2 range = row_range[g + 8 * i];
                                if (t0 + h * kGranule + t < range.x || t0 + h * kGranule + t >= range.y) continue;
#pragma unroll
                                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const int byte = (2 * c + e) * vShare + n;
                                        const int in_row = P::swizzled ? (((byte >> 4) ^ (t & 7)) << 4) + (byte & 15) : byte;
                                        if ((lds_u8<0>(ring + at + S::v_at + t * P::v + in_row) & 0x7f) == 0x7f)
                                            o[n][2 * i + e] = __int_as_float(0x7fc00000);
                                    }
                            }
                    }
                }
            };
            if (!bands && !lowered) {
                make_weights();
                add_values(vs, vref);
            } else {
                make_weights();
                int down[2] = {0, 0};  // octaves that the rows' weights have been lowered by so far
                auto lower_weights = [&](int ref) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int by = max(row_ref[i] - ref, 0) - down[i], part = min(by, 24);
                        down[i] += by;
                        const uint32_t f = pow2_f16x2(-part, -part), rest = pow2_f16x2(part - by, part - by);
#pragma unroll
                        for (int k = 0; k < 4; ++k) pa[k >> 1][2 * (k & 1) + i] = hmul2(hmul2(pa[k >> 1][2 * (k & 1) + i], f), rest);
                    }
                };
                int now_vs[8], ref = vref;
#pragma unroll
                for (int i = 0; i < 8; ++i) now_vs[i] = vs[i];
                while (true) {
                    if (bands) {
                        // The next 8 octaves, from the largest scale left; vs becomes 0 as it is done.
                        const int top = largest();
                        if (top == 0) break;
                        ref = max(top - kValueLift, 1);
                        uint32_t tokens = 0;  // of the step that have a block in the band
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const bool in = vs[i] > max(top - kMostLift, 0);
                            const unsigned lanes = __ballot_sync(kFull, in);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (lanes & (0x11111111u << k)) tokens |= 1u << (2 * k + (i & 1) + 8 * (i >> 1));
                            now_vs[i] = in ? vs[i] : ref - 64;
                            if (in) vs[i] = 0;
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int2 range = row_range[g + 8 * i];
                            const int from = min(max(range.x - t0, 0), kPair), to = min(max(range.y - t0, 0), kPair);
                            const uint32_t seen = to > from ? (0xffffffffu >> (32 - (to - from))) << from : 0u;
                            if ((tokens & seen) && row_ref[i] < ref) raise_row(i, ref);
                        }
                    }
                    lower_weights(ref);
                    add_values(now_vs, ref);
                    if (!bands) break;
                }
            }
        }

        // Join the warps: maxima, sums of weights, and outputs as means in true units.
        copy_wait<0>();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sum[i] += __shfl_xor_sync(kFull, sum[i], 1);
            sum[i] += __shfl_xor_sync(kFull, sum[i], 2);
            if (c == 0) stat_max[warp][g + 8 * i] = run_max[i], stat_sum[warp][g + 8 * i] = sum[i];
        }
        __syncthreads();  // the rings are done with as well
        float* joined = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = g + 8 * i;
            const float vfactor = __uint_as_float((uint32_t)row_ref[i] << 23);
            const float inv = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
            // features (2c + e) * D/8 + n, four at a time; the 16-byte chunks of a row are
            // permuted so that eight lanes write to eight different bank groups
            float4* dst = reinterpret_cast<float4*>(joined + (warp * kRows + r) * D);
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int n = 0; n < kTiles; n += 4) {
                    const int chunk = (2 * c + e) * (D / 32) + n / 4;
                    const float4 v = make_float4(o[n][2 * i + e] * inv * vfactor, o[n + 1][2 * i + e] * inv * vfactor,
                                                 o[n + 2][2 * i + e] * inv * vfactor, o[n + 3][2 * i + e] * inv * vfactor);
                    dst[chunk ^ (c | ((g & 1) << 2))] = v;
                }
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tiles == w.tiles;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (tile0 == 0 ? 1 : 0);
        for (int idx = tid; idx < rows * (D / 4); idx += kThreads) {
            const int r = idx / (D / 4), chunk = idx - r * (D / 4);
            const int at = chunk ^ ((chunk / (D / 16)) | ((r & 1) << 2));
            float top = neg_inf, total = 0.0f, weight[kWarps];
#pragma unroll
            for (int k = 0; k < kWarps; ++k) top = fmaxf(top, stat_max[k][r]);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                weight[k] = stat_sum[k][r] * (stat_max[k][r] == top ? 1.0f : ex2(stat_max[k][r] - top));
                total += weight[k];
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float4 x = reinterpret_cast<const float4*>(joined + (k * kRows + r) * D)[at];
                const float f = weight[k] * inv;
                v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
            }
            if (total == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (whole) {
                const int row = w.rt * kRows + r, j = row / p.group;
                const int head = w.head * p.group + (row - j * p.group);
                dev::store4(p, w.view.row0 + j, head, chunk * 4, v);
                if (p.lse && chunk == 0)
                    p.lse[(int64_t)(w.view.row0 + j) * p.heads + head] = dev::row_lse(top, total);
            } else {
                reinterpret_cast<float4*>(p.part + (slot * kRows + r) * D)[chunk] = v;
                if (chunk == 0) p.part_stat[slot * kRows + r] = make_float2(top, total);
            }
        }
        if (!whole && tile0 == 0) {
            open = true;
            if (tid == 0)
                p.part_open[blockIdx.x] =
                    make_int4(w.seq, w.rt, w.head, share.followers(share.tiles - left, w.tiles));
        }
        __syncthreads();  // before the rings are filled again
        left -= tiles + share.cost;
        if (left > 0) dev::walk_on<kRows, kKeys>(p, w);
    }
    if (tid == 0 && !open) p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0);
    dev::wait_for_previous();
}

template <int D, int BITS>
int launch_rows(AttentionParams p, int64_t most_tiles, int64_t most_rows, AttentionCall& call) {
    using S = Stage<D, BITS>;
    static thread_local int ready_device = -1;
    int dev = 0;
    MXK_CUDA(cudaGetDevice(&dev));
    if (ready_device != dev) {
        MXK_CUDA(cudaFuncSetAttribute(attention_rows_kernel<D, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      S::smem));
        ready_device = dev;
    }
    static const int sms = sm_count();
    const int64_t ctas = std::min<int64_t>(most_tiles, kCtasPerSm * sms);
    MXK_CHECK(call.take(p, ctas, kRows, D));
    MXK_CHECK(call.launch("attention_rows", attention_rows_kernel<D, BITS>, (unsigned)ctas, kThreads, S::smem, p));
    call.join_later(p, ctas, kRows, std::min<int64_t>(most_rows, kRows));
    return MXK_OK;
}

template <int D>
int launch_rows_bits(int bits, const AttentionParams& p, int64_t most_tiles, int64_t most_rows, AttentionCall& call) {
    if (bits == 8) return launch_rows<D, 8>(p, most_tiles, most_rows, call);
    if (bits == 6) return launch_rows<D, 6>(p, most_tiles, most_rows, call);
    return launch_rows<D, 4>(p, most_tiles, most_rows, call);
}

}  // namespace
}  // namespace mxk

extern "C" int mxk_cache_attention(const mxk_cache* cache, const mxk_attention* a, void* stream) {
    using namespace mxk;
    MXK_CHECK(check_cache(cache, "cache_attention"));
    MXK_REQUIRE(a, "cache_attention: args is null");
    MXK_REQUIRE(a->dtype == MXK_F16 || a->dtype == MXK_BF16, "cache_attention: dtype must be MXK_F16 or MXK_BF16");
    MXK_REQUIRE(a->heads >= 1 && a->heads <= 65535 && a->heads % cache->kv_heads == 0,
                "cache_attention: heads must be a positive multiple of the cache's kv_heads");
    MXK_REQUIRE(a->tokens >= 0 && a->tokens <= std::numeric_limits<int>::max() / 2 && a->seqs >= 0,
                "cache_attention: tokens must be in [0, 2^30), seqs in [0, 2^31)");
    MXK_REQUIRE(a->max_q >= 0 && a->max_kv >= 0, "cache_attention: max_q and max_kv must not be negative");
    MXK_REQUIRE((int64_t)a->max_q * a->heads <= std::numeric_limits<int>::max() / 2 &&
                    a->max_kv <= std::numeric_limits<int>::max() / 2,
                "cache_attention: max_q * heads and max_kv must be below 2^30");
    MXK_REQUIRE(a->window >= 0 && (a->window == 0 || a->causal), "cache_attention: a window needs causal");
    MXK_REQUIRE(a->scale == a->scale && a->scale - a->scale == 0.0f, "cache_attention: scale must be finite");
    if (cache->head_dim != 64 && cache->head_dim != 128)
        return fail(MXK_ERR_UNSUPPORTED, "cache_attention: head_dim must be 64 or 128");
    // (The kernels number the cache's rows in 32 bits.)
    if (cache->pages * cache->kv_heads > (1ll << 32) / cache->page_size)
        return fail(MXK_ERR_UNSUPPORTED, "cache_attention: pages * kv_heads * page_size must be at most 2^32");
    if (a->tokens == 0 || a->seqs == 0 || a->max_q == 0) return MXK_OK;
    MXK_REQUIRE(a->q.data && a->out.data && a->cu_q && (a->page_table || a->max_kv == 0) && a->kv_lens,
                "cache_attention: q, out, cu_q, page_table and kv_lens must be non-null");
    MXK_REQUIRE((reinterpret_cast<uintptr_t>(a->q.data) | reinterpret_cast<uintptr_t>(a->out.data)) % 2 == 0 &&
                    (reinterpret_cast<uintptr_t>(a->cu_q) | reinterpret_cast<uintptr_t>(a->page_table) |
                     reinterpret_cast<uintptr_t>(a->kv_lens) | reinterpret_cast<uintptr_t>(a->lse)) % 4 == 0,
                "cache_attention: pointers must be aligned to their elements");
    const int64_t need = (a->max_kv + cache->page_size - 1) / cache->page_size;
    MXK_REQUIRE(a->seqs == 1 || a->page_table_stride >= need,
                "cache_attention: page_table_stride is below the pages of max_kv tokens");

    AttentionParams p{};
    p.k_values = static_cast<const uint8_t*>(cache->k_values);
    p.v_values = static_cast<const uint8_t*>(cache->v_values);
    p.k_scales = cache->k_scales;
    p.v_scales = cache->v_scales;
    p.bits = cache->bits;
    p.kv_heads = cache->kv_heads;
    p.page_size = cache->page_size;
    p.pages = (int)cache->pages;
    p.q = a->q.data;
    p.out = a->out.data;
    p.lse = a->lse;
    p.q_token = a->q.token_stride, p.q_head = a->q.head_stride;
    p.out_token = a->out.token_stride, p.out_head = a->out.head_stride;
    p.tokens = a->tokens;
    p.dtype = a->dtype;
    p.heads = a->heads;
    p.group = a->heads / cache->kv_heads;
    p.seqs = a->seqs;
    p.q_vec = rows_aligned(a->q, 2, 8);
    p.out_vec = rows_aligned(a->out, 2, 8);
    p.cu_q = a->cu_q;
    p.page_table = a->page_table;
    p.table_stride = a->page_table_stride;
    p.max_kv = (int)a->max_kv;
    p.max_q = (int)std::min<int64_t>(a->max_q, a->tokens);
    p.kv_lens = a->kv_lens;
    p.scale_log2 = a->scale * 1.44269504088896f;
    p.causal = a->causal != 0;
    p.window = (int)std::min<int64_t>(a->window, 1 << 30);
    p.min_rows = 1;
    p.max_rows = std::numeric_limits<int>::max();

    // Sequences with few rows per key head go to the rows kernel, the others to the
    // tiles kernel; a single sequence has one kernel chosen by its bound, several are
    // sorted by the kernels themselves.
    AttentionCall call(as_stream(stream));
    const int64_t rows = (int64_t)p.max_q * p.group;
    const bool many = rows > kMostFewRows;
    if (many) {
        AttentionParams q = p;
        if (a->seqs > 1) q.min_rows = kMostFewRows + 1;
        MXK_CHECK(launch_attention_tiles(cache->bits, cache->head_dim, q, p.max_q, call));
        p.max_rows = kMostFewRows;
    }
    if (!many || a->seqs > 1) {
        const int64_t few = std::min<int64_t>(rows, kMostFewRows);
        const int64_t most = attention_tile_bound(p, (int)((few + p.group - 1) / p.group), kRows, kKeys);
        MXK_REQUIRE(most <= std::numeric_limits<int>::max() / (1 + kUnitCost), "cache_attention: too much work for one call");
        MXK_CHECK(cache->head_dim == 128 ? launch_rows_bits<128>(cache->bits, p, most, few, call)
                                         : launch_rows_bits<64>(cache->bits, p, most, few, call));
    }
    return call.join_all(cache->head_dim);
}
