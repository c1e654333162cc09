// Attention of new tokens over the paged MX cache: the kernels for many query rows
// per key head (no counterpart in the reference).
//
// With many rows the two products bound it (4 * rows * keys * D operations), with
// the exponentials close behind: one per row and key, 16 a cycle and SM, against
// 4 * D / 8192 cycles of tensor time.  A row tile is 128 rows, with its scores and its
// output in TMEM; a key tile goes through in two halves of 64 tokens, so the tensor
// core multiplies for one while the other is in the softmax.
//
//   softmax     a warpgroup per row tile; a thread owns one row: its running maximum
//               and sum, its weights and its output row
//   products    one warp, whose elected lane issues S = Q K^T from shared memory and
//               O += P V with P from TMEM
//   keys and    two stages each of f16 tiles in shared memory (SWIZZLE_128B), filled
//   values      by eight converter warps from the packed pages (attention_tiles_kernel,
//               one row tile), or, when a key head has more rows than two row tiles, by
//               bulk copies of tiles that attention_unpack_kernel has converted once for
//               all of them (attention_ready_kernel, two row tiles)
//
// Measured at 32 heads of 128 on 8 key heads, 8 bits, 16,384 tokens cached:
//   4096 query tokens   975 to 996 us one after the other, 966 to 986 Tflop/s, 59 % of a
//                       library product's rate; 912 us on an idle card (the power cap).
//                       The ready kernel takes 2.2 to 2.4 us for 256 rows x 128 keys where
//                       the products need 0.57 x 2 and the exponentials 1.0 (1800 MHz, one
//                       pair in eight on the FMA pipe): two softmax warps a scheduler leave
//                       the waits between the steps of a row (scores, maximum, weights,
//                       store) half uncovered.  Tensor pipe 52 % of the cycles, MUFU 46 %.
//   512 query tokens    176 to 187 us; one by one 21 converting, 156 multiplying, 15 joining
//   16 query tokens     58 us with a cold L2 (42 and the join): the packed kernel converts a
//                       key tile for one row tile in the time that tile's softmax takes
// More query rows per thread, or two row tiles beside converters, ran out of registers; as
// it is, the softmax spills some 280 (ready) and 380 (packed) bytes a thread.  The times beside
// the choices below are from when they were made.
//
// P (f16) overwrites the S it came from, so TMEM holds S0 S1 O0 O1, 512 columns at
// D = 128.  Values are the right operand as they lie in the cache (one row per
// token), read by the tensor core as an N-major operand, so nothing is transposed.
//
// Scales: the keys of a 128-token tile are held relative to the tile's largest
// scale, which goes into the factor of the scores (per tile and row).  Where that would
// not be exact (scales that differ by more than 2^21 with 8 bits) the tile is "wide":
// each of its tokens has its own reference, and the softmax takes a slower path, so one
// token's magnitude does not touch another's score.  Values are
// held relative to a reference of their tile, a multiple of kRefStep octaves at or
// above its largest scale; an output row is kept relative to the largest reference of the
// tiles that the row saw something of, and a tile with a smaller one has its weights
// scaled down by the difference, so a row is rescaled only when the reference goes up or
// its maximum does.  A tile of which the rows see different tokens and whose value scales
// are too far apart for one reference is multiplied by hand (exact_values), in float32,
// relative to what each row sees.  Blocks of zeros, whose scale byte stands for 1, are
// left out where they would set a reference.
#include <limits>
#include <type_traits>

#include "attention.cuh"

namespace mxk {
namespace {

using dev::ex2;
using dev::kExactDown;
using dev::kExpShift;
using dev::kKeyLift;
using dev::kMaxSlack;
using dev::kMostLift;
using dev::kQueryExp;
using dev::kScaleOfZeros;
using dev::kValueLift;
using dev::kValueMax;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kTileRows = 128;           // M of one product
constexpr int kKeys = 128;               // tokens of a key tile
constexpr int kHalf = kKeys / 2;         // tokens of one step of the softmax
constexpr int kStages = 2;               // of keys and of values
constexpr int kMeta = 4;                 // key tiles whose references are kept (converter warps)
constexpr int kWide = 1 << 17;           // in place of a tile's key reference: every token has its own;
                                         // beside its value reference: rows that see part of it work by hand
constexpr int kWideRef = 200;            // what scales relative to a token's own reference are added to
constexpr int kRefStep = 4;              // value references are multiples of this many octaves
constexpr int kMostDown = 64;            // octaves that a float32 weight may be scaled down by
// The most memory that converting may take: above it the packed kernel goes over the keys
// once for every 128 rows.
constexpr int64_t kReadyBytes = 4ll << 30;

// The two kernels' row tiles, warps and registers.  Warpgroups give up or take registers
// of those the block was launched with.  Next to converter warps there are registers for
// one row tile only (two, at 96 registers a thread, spilled: the kernel took 55 us instead
// of 46 for 16 query tokens over 16,384, 32 heads of 128 on 8 key heads).
// unit_cost: key tiles that starting and ending a unit is taken to be worth (queries in,
// output out, and the pipeline between: 10 us against 1 to 2 a tile).  In us for 0, 3, 10
// and 15 in Packed and 0, 3, 8 and 12 in Ready, over the same 16,384 tokens: 16 query
// tokens 62, 54, 47, 47; 64: 86, 78, 70, 72; 512: 185, 181, 176, 178; nine sequences of 1
// to 701 query tokens and 333 to 5003 cached ones 182, 153, 141, 143.
// join_split: blocks that join a unit.  In us for 8, 16, 32 and 64: 64 query tokens (units
// in 18 parts) 89, 74, 68, 70; 512 (2 to 3 parts) 183, 179, 181, 181; the nine sequences
// 128, 128, 132, 137.
struct Packed {
    static constexpr int row_tiles = 1, rows = row_tiles * kTileRows;
    static constexpr int softmax_warps = 4 * row_tiles;
    static constexpr int convert_warps = 8;
    static constexpr int product_warp = softmax_warps + convert_warps;
    static constexpr int unit_cost = 10, join_split = 32;
    static constexpr int threads = 512;
    static constexpr int launch_regs = 128, softmax_regs = 168, convert_regs = 128, product_regs = 88;
    static_assert(128 * softmax_regs + 256 * convert_regs + 128 * product_regs <= threads * launch_regs, "");
};
struct Ready {
    static constexpr int row_tiles = 2, rows = row_tiles * kTileRows;
    static constexpr int softmax_warps = 4 * row_tiles;
    static constexpr int product_warp = softmax_warps, load_warp = softmax_warps + 1;
    static constexpr int unit_cost = 8, join_split = 16;
    static constexpr int threads = 384;
    static constexpr int launch_regs = 168, softmax_regs = 200, product_regs = 104;
    static_assert(256 * softmax_regs + 128 * product_regs <= threads * launch_regs, "");
};

template <int D, int TILES = 2>
struct Smem {
    static constexpr int half = kKeys * 128;        // 128 rows x 64 features
    static constexpr int tile = (D / 64) * half;    // 128 rows x D features
    static constexpr int q = 0;                     // the row tiles' queries
    static constexpr int k = TILES * tile;
    static constexpr int v = k + kStages * tile;
    static constexpr int total = v + kStages * tile + 1024;  // 1024: alignment
};

struct Shared {
    uint64_t q_ready[2];       // the tile's queries are in shared memory
    uint64_t k_full[kStages], v_full[kStages], k_empty[kStages], v_empty[kStages];
    uint64_t s_full[2][2];     // [row tile][half of the key tile] scores are in TMEM
    uint64_t p_ready[2][2];    // the half's weights are in TMEM, the output may be added to
    uint64_t o_done[2][2];     // the half's product with the values has finished
    uint64_t rows_out[2];      // the tile's output rows have left the queries' shared memory
    uint64_t drain;
    int2 meta[kMeta];          // converter warps: the key tile's references
    uint8_t key_refs[kMeta][kKeys];  // those of its tokens, in wide tiles
    float row_factor[2][kTileRows];
    int kept[2];               // the output row tile holds values by hand before the unit's first product
    int nan_unit[4];           // converter warps: unit in which a NaN was taken out of a partly seen tile
    int abort_word;
    uint32_t tmem;
};

// What the roles of a CTA share.
struct Block {
    uint8_t* smem;
    Shared* sh;
    uint32_t tmem;
    unsigned* err;
    dev::Share share;
    __device__ __forceinline__ volatile int* abort_flag() const { return &sh->abort_word; }
    // Bounded wait of a whole warp; false: it gave up, leave for the end of the kernel.
    __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) const {
        return __all_sync(kFull, dev::mbar_wait(bar, parity, abort_flag(), err));
    }
    // One arrival for the whole warp, after all its lanes' writes.
    __device__ __forceinline__ void arrive(uint64_t* bar) const {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) dev::mbar_arrive(bar);
    }
    __device__ __forceinline__ bool wait_lean(uint64_t* bar, uint32_t parity) const {
        return __all_sync(kFull, dev::mbar_wait_lean(bar, parity, abort_flag(), err));
    }
};

// A pass over the CTA's share: every role makes the same one.
template <class Cfg, class P>
struct Cursor {
    dev::Walk<P> w;
    int left;          // tiles of the share from the current unit's on
    int tile0, tiles;  // key tiles of the current unit that are this CTA's
    int unit;          // units begun so far
    int cost;          // tiles that the next unit counts as before its own

    __device__ __forceinline__ void take() {
        tile0 = w.tile;
        tiles = min(left, w.tiles - tile0);
    }
    __device__ __forceinline__ bool next(const P& p) {
        left -= tiles + cost;
        if (left <= 0) return false;
        dev::walk_on<Cfg::rows, kKeys>(p, w);
        ++unit;
        take();
        return true;
    }
    __device__ __forceinline__ int rows(const P& p) const {
        return min(w.view.n * p.group - w.rt * Cfg::rows, Cfg::rows);
    }
    __device__ __forceinline__ bool whole() const { return tile0 == 0 && tiles == w.tiles; }
};

// Key tiles [from, to) of the cursor's share of its unit are seen whole by all its rows.
struct Whole {
    int from, to;
};
template <class Cfg, class P>
__device__ __forceinline__ Whole whole_tiles(const P& p, const Cursor<Cfg, P>& c) {
    const int r0 = c.w.rt * Cfg::rows, j0 = r0 / p.group, j1 = (r0 + c.rows(p) - 1) / p.group;
    int lo, hi, x;
    dev::seen_range(p, c.w.view, j0, j0, x, hi);   // the first row ends first,
    dev::seen_range(p, c.w.view, j1, j1, lo, x);   // the last begins last
    const int first = c.w.first + c.tile0;
    Whole wt;
    wt.from = min(max((lo + kKeys - 1) / kKeys - first, 0), c.tiles);
    wt.to = min(max(max(hi, 0) / kKeys - first, 0), c.tiles);
    return wt;
}

// ---------------------------------------------------------------- key and value tiles

template <int N>
__device__ __forceinline__ void ldg_bytes(const uint8_t* src, uint32_t* w) {
    if constexpr (N == 16) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 8) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
        w[0] = v.x, w[1] = v.y;
    } else {
        static_assert(N == 12, "16 elements of 4, 6 or 8 bits");
#pragma unroll
        for (int i = 0; i < 3; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(src) + i);
    }
}

// 16 packed elements to f16 pairs times f.
template <int BITS>
__device__ __forceinline__ void convert16(const uint32_t* w, uint32_t f, uint32_t (&h)[8]) {
    if constexpr (BITS == 4) {
        uint32_t a[4], b[4];
        dev::e2m1x8_to_f16(w[0], a);
        dev::e2m1x8_to_f16(w[1], b);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = dev::hmul2(a[i], f), h[4 + i] = dev::hmul2(b[i], f);
    } else {
        constexpr int kCode = BITS == 4 ? 8 : BITS;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t four = BITS == 8 ? w[i] : dev::four6(w, i);
            h[2 * i] = dev::hmul2(dev::codes_to_f16x2<kCode>(four), f);
            h[2 * i + 1] = dev::hmul2(dev::codes_to_f16x2<kCode>(four >> 16), f);
        }
    }
}

// The scales s of a tile's rows lane + 32 i (place, [from, to): as in Converter), without
// those of blocks whose elements are all zero: they have no magnitude.
template <int D, int BITS>
__device__ __noinline__ uint4 magnitude_scales(const uint8_t* values, uint32_t place, int from, int to, uint4 s) {
    constexpr int kBlock = BITS;  // words of 32 elements
    uint32_t out[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (threadIdx.x & 31) + 32 * i;
        const uint32_t row = __shfl_sync(kFull, place, r >> 4) + (r & 15);
        if (r < from || r >= to) continue;
        const uint8_t* at = values + (uint64_t)row * (D * BITS / 8);
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            uint32_t w[kBlock], any = 0;
#pragma unroll
            for (int k = 0; k < kBlock; k += kBlock % 4 ? 2 : 4) ldg_bytes<kBlock % 4 ? 8 : 16>(at + 4 * (b * kBlock + k), w + k);
#pragma unroll
            for (int k = 0; k < kBlock; ++k) any |= w[k] & dev::magnitude_bits<BITS>(k);
            if (!any) out[i] &= ~(255u << (8 * b));
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// Eight warps turning a tile of 128 packed rows into f16: a thread converts 16-element
// piece `u` of every kStep-th row.  Eight neighbouring lanes cover the 16-byte chunks of
// two rows, so the swizzled stores meet no shared-memory bank twice.
template <int D, int BITS>
struct Converter {
    static constexpr int row_bytes = D * BITS / 8;
    static constexpr int pieces = D / 16;                   // of a row
    static constexpr int piece_words = BITS / 2;
    static constexpr int warp_rows = 32 / pieces;
    static constexpr int step = 8 * warp_rows;              // rows of one pass of the eight warps
    static constexpr int passes = kKeys / step;
    using Words = uint32_t[passes][piece_words];

    int lane, u, r0;
    bool high;  // r0 is in the second 32 rows of a pass

    __device__ __forceinline__ explicit Converter(int warp) {
        lane = threadIdx.x & 31;
        u = D == 128 ? (lane & 3) | ((lane >> 4) << 2) : lane & 3;
        r0 = warp_rows * warp + (D == 128 ? (lane >> 2) & 3 : lane >> 2);
        high = warp_rows * warp >= 32;
    }

    // Tokens [from, to) of a tile, those that some row sees: the others may lie in pages that
    // were given away and hold any bytes, so they are not read and count for no reference.
    struct Span {
        int from, to;
    };
    static __device__ __forceinline__ Span span(int lo, int hi, int t0) {
        return Span{min(max(lo - t0, 0), kKeys), min(max(hi - t0, 0), kKeys)};
    }
    // The page number and the place in it of the tile's token 16 i, in lane i < 8.
    // row_of makes the cached row of it, when the page number has arrived.
    struct Place {
        int page, in;
    };
    template <class P>
    __device__ __forceinline__ Place place(const P& p, int seq, int t0, Span sp) const {
        Place pl{0, 0};
        if (lane < 8 && 16 * lane < sp.to && 16 * lane + 16 > sp.from) {
            const unsigned per_page = (unsigned)p.page_size / 16u;
            const unsigned gr = (unsigned)(t0 / 16) + lane;
            const unsigned at = gr / per_page;
            pl.page = __ldg(dev::table_of(p, seq) + at);
            pl.in = (int)(gr - at * per_page) * 16;
        }
        return pl;
    }
    static __device__ __forceinline__ uint32_t row_of(const AttentionParams& p, const Place& pl, int head) {
        const int page = min(max(pl.page, 0), p.pages - 1);
        return ((uint32_t)page * p.kv_heads + head) * p.page_size + pl.in;
    }
    __device__ __forceinline__ void load(uint32_t place, Span sp, const uint8_t* values, Words& x) const {
#pragma unroll
        for (int i = 0; i < passes; ++i) {
            const int r = r0 + step * i;
            const uint32_t row = __shfl_sync(kFull, place, r >> 4) + (r & 15);
#pragma unroll
            for (int k = 0; k < piece_words; ++k) x[i][k] = 0;
            if (r >= sp.from && r < sp.to)
                ldg_bytes<4 * piece_words>(values + (uint64_t)row * row_bytes + u * (4 * piece_words), x[i]);
        }
    }
    // Scale bytes of rows lane + 32 i.
    __device__ __forceinline__ void load_scales(uint32_t place, Span sp, const uint8_t* scales, uint32_t (&s)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = lane + 32 * i;
            const uint32_t row = __shfl_sync(kFull, place, r >> 4) + (r & 15);
            s[i] = 0;
            if (r >= sp.from && r < sp.to) {
                if constexpr (D == 128)
                    s[i] = __ldg(reinterpret_cast<const uint32_t*>(scales) + row);
                else
                    s[i] = __ldg(reinterpret_cast<const uint16_t*>(scales) + row);
            }
        }
    }
    static __device__ __forceinline__ unsigned top_byte(uint32_t w) {
        const uint32_t m = max(w & 0xffffu, w >> 16);  // of the high bytes, or
        return max(max(m >> 8, w & 255u), (w >> 16) & 255u);
    }
    static __device__ __forceinline__ int top_scale(const uint32_t (&s)[4]) {
        return (int)__reduce_max_sync(kFull, top_byte(__vmaxu4(__vmaxu4(s[0], s[1]), __vmaxu4(s[2], s[3]))));
    }
    // The smallest scale but 0 (a row that takes no part, or 2^-127); 256 if there is none.
    static __device__ __forceinline__ int low_scale(const uint32_t (&s)[4]) {
        uint32_t up = 0;  // bytewise 255 - (s - 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) up = __vmaxu4(up, ~__vsub4(s[i], 0x01010101u));
        return 256 - (int)__reduce_max_sync(kFull, top_byte(up));
    }
    // The tile's references: keys are lifted to 2^kKeyLift below theirs.
    static __device__ __forceinline__ int key_ref(const uint32_t (&s)[4]) { return max(top_scale(s), 1); }
    static __device__ __forceinline__ bool wide_keys(const uint32_t (&s)[4], int ref) {
        return ref - low_scale(s) > kKeyLift + kExactDown<BITS>;
    }
    // Rare: the references of a tile of keys whose scales differ too much for one.  Zero
    // blocks are left out, and if that is not enough each row gets its own at refs[row] (one
    // warp has to write them), and the scales become relative to it.  Returns the tile's
    // reference or kWide.
    static __device__ __forceinline__ int spread_keys(const uint8_t* values, uint32_t place, Span sp,
                                                      uint32_t (&s)[4], uint8_t* refs, bool write) {
        const uint4 m = magnitude_scales<D, BITS>(values, place, sp.from, sp.to, make_uint4(s[0], s[1], s[2], s[3]));
        s[0] = m.x, s[1] = m.y, s[2] = m.z, s[3] = m.w;
        const int ref = key_ref(s);
        if (!wide_keys(s, ref)) return ref;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int own = max((int)top_byte(s[i]), 1);
            if (write) refs[(threadIdx.x & 31) + 32 * i] = (uint8_t)own;
            uint32_t t = 0;
#pragma unroll
            for (int b = 0; b < D / 32; ++b) {
                const int e = (int)((s[i] >> (8 * b)) & 255u);
                t |= (uint32_t)(e ? max(e - own + kWideRef, 0) : 0) << (8 * b);
            }
            s[i] = t;
        }
        return kWide;
    }
    // What the scales of a tile are stored relative to.
    static __device__ __forceinline__ int key_base(int ref) { return (ref == kWide ? kWideRef : ref) - kKeyLift; }
    static __device__ __forceinline__ int value_ref(const uint32_t (&s)[4]) {
        // top - ref in (kKeyLift - kRefStep, kKeyLift]
        return max(((top_scale(s) - kKeyLift + kRefStep - 1) >> 2) << 2, 1);
    }
    // Whether the scales of a tile of values ask for spread_values: too far apart to be exact
    // relative to one reference or, if some rows see the tile's end but not its beginning
    // (leading) and go on to others, for those rows' references; or perhaps all zeros.
    static __device__ __forceinline__ bool wide_values(const uint32_t (&s)[4], bool leading) {
        const int top = top_scale(s), low = low_scale(s);
        return too_far(top, low, leading) || (top == kScaleOfZeros && low == kScaleOfZeros);
    }
    // (top - value_ref is at least kKeyLift - kRefStep + 1.)
    static __device__ __forceinline__ bool too_far(int top, int low, bool leading) {
        return top - low > (leading ? kMostLift : kKeyLift - kRefStep + 1 + kExactDown<BITS>);
    }
    // Rare: leaves out zero blocks and returns the tile's reference, with kWide if that was not
    // enough and the rows see different parts of the tile.
    static __device__ __forceinline__ int spread_values(const uint8_t* values, uint32_t place, Span sp,
                                                        uint32_t (&s)[4], bool leading, bool trailing) {
        const uint4 m = magnitude_scales<D, BITS>(values, place, sp.from, sp.to, make_uint4(s[0], s[1], s[2], s[3]));
        s[0] = m.x, s[1] = m.y, s[2] = m.z, s[3] = m.w;
        const bool by_hand = (leading || trailing) && too_far(top_scale(s), low_scale(s), leading);
        return value_ref(s) | (by_hand ? kWide : 0);
    }
    // f16 relative to the scale byte `ref` into a SWIZZLE_128B tile image.
    __device__ __forceinline__ void store(const Words& x, const uint32_t (&s)[4], int ref, uint8_t* tile) const {
#pragma unroll
        for (int i = 0; i < passes; ++i) {
            const int r = r0 + step * i;
            uint32_t sw;
            if constexpr (step == 32)
                sw = __shfl_sync(kFull, s[i], r & 31);
            else
                sw = __shfl_sync(kFull, high ? s[2 * i + 1] : s[2 * i], r & 31);
            const int e = (int)((sw >> (8 * (u >> 1))) & 255u) - ref;
            uint32_t h[8];
            convert16<BITS>(x[i], dev::pow2_f16x2(e, e), h);
            uint8_t* row = tile + (u >> 2) * Smem<D>::half + r * 128;
            const int chunk = (u & 3) * 2;
            *reinterpret_cast<uint4*>(row + ((chunk ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ (r & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
        }
    }
    // Zeroes E4M3 NaNs; true if there were any among this thread's.
    static __device__ __forceinline__ bool take_out_nans(Words& x) {
        bool any = false;
        if constexpr (BITS == 8) {
#pragma unroll
            for (int i = 0; i < passes; ++i)
#pragma unroll
                for (int k = 0; k < piece_words; ++k) {
                    const uint32_t bad = __vcmpeq4(x[i][k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                    any |= bad != 0;
                    x[i][k] &= ~bad;
                }
        }
        return any;
    }
};
static_assert(kRefStep == 4, "value_ref rounds to multiples of four");

// The sequence that is the rank-th of those the launch takes, -1 if there is none.  A whole warp.
template <class P>
__device__ __forceinline__ int seq_of_rank(const P& p, int rank) {
    for (int base = 0; base < p.seqs; base += 32) {
        const int i = base + (threadIdx.x & 31);
        const unsigned m = __ballot_sync(kFull, i < p.seqs && dev::taken(p, dev::seq_view(p, min(i, p.seqs - 1))));
        if (rank < __popc(m)) return base + (int)__fns(m, 0, rank + 1);
        rank -= __popc(m);
    }
    return -1;
}

// The other way round: the rank of a sequence, and how many there are.
struct Ranks {
    int rank, all;
};
template <class P>
__device__ __forceinline__ Ranks rank_of_seq(const P& p, int seq) {
    Ranks r{0, 0};
#pragma unroll 4
    for (int base = 0; base < p.seqs; base += 32) {
        const int i = base + (threadIdx.x & 31);
        const unsigned m = __ballot_sync(kFull, i < p.seqs && dev::taken(p, dev::seq_view(p, min(i, p.seqs - 1))));
        const int before = min(max(seq - base, 0), 32);
        r.all += __popc(m);
        r.rank += __popc(before ? m & (0xffffffffu >> (32 - before)) : 0u);
    }
    return r;
}

// Converts the key tiles that some row sees once for all row tiles of a key head.
// Block (x, side): key tile x % max_tiles of (rank of the sequence, head) x / max_tiles, its
// keys or its values; the f16 tiles lie in the workspace as shared memory will hold them, so each
// is built there and leaves as one bulk copy.
template <int D, int BITS, class P>
__global__ void __launch_bounds__(256) attention_unpack_kernel(const P p) {
    using C = Converter<D, BITS>;
    __shared__ __align__(128) uint8_t image[Smem<D>::tile];
    dev::let_next_start();
    const int tile = blockIdx.x % p.max_tiles, sh = blockIdx.x / p.max_tiles;
    const int rank = sh / p.kv_heads, head = sh - rank * p.kv_heads;
    const int seq = p.seqs == 1 ? rank : seq_of_rank(p, rank);
    if (seq < 0) return;
    const auto view = dev::seq_view(p, seq);
    if (!dev::taken(p, view)) return;
    int lo, hi;
    dev::seen_range(p, view, 0, view.n - 1, lo, hi);
    const int t0 = tile * kKeys;
    // rows that see nothing still have a first key tile, of zeros where no token exists
    if (tile != dev::first_token(view) / kKeys && (t0 >= hi || t0 + kKeys <= lo)) return;
    const typename C::Span sp = C::span(lo, hi, t0);
    const bool keys = blockIdx.y == 0;
    const C cv(threadIdx.x >> 5);
    const uint32_t place = C::row_of(p, cv.place(p, seq, t0, sp), head);
    uint32_t s[4];
    typename C::Words x;
    cv.load_scales(place, sp, keys ? p.k_scales : p.v_scales, s);
    cv.load(place, sp, keys ? p.k_values : p.v_values, x);
    int ref = keys ? C::key_ref(s) : C::value_ref(s);
    if (keys && C::wide_keys(s, ref))
        ref = C::spread_keys(p.k_values, place, sp, s, p.ready_key_refs + (int64_t)blockIdx.x * kKeys, threadIdx.x < 32);
    if (!keys) {
        int last_lo, first_hi, other;
        dev::seen_range(p, view, view.n - 1, view.n - 1, last_lo, other);
        dev::seen_range(p, view, 0, 0, other, first_hi);
        const bool leading = max(t0, lo) < last_lo, trailing = min(t0 + kKeys, hi) > first_hi;
        if (C::wide_values(s, leading)) ref = C::spread_values(p.v_values, place, sp, s, leading, trailing);
    }
    const int nans = keys ? 0 : C::take_out_nans(x);
    cv.store(x, s, keys ? C::key_base(ref) : ref & 0xffff, image);
    dev::fence_proxy_async();
    const int any_nans = __syncthreads_or(nans);
    if (threadIdx.x == 0) {
        int* meta = reinterpret_cast<int*>(p.ready_meta + blockIdx.x) + (keys ? 0 : 1);
        *meta = ref | (any_nans ? 1 << 16 : 0);
        dev::bulk_store_wait((keys ? p.ready_k : p.ready_v) + (int64_t)blockIdx.x * Smem<D>::tile, image, Smem<D>::tile);
    }
}

// Converter warps: every key tile of the CTA's share, rows loaded one tile ahead of
// their conversion and page numbers two.
template <int D, int BITS, class P>
__device__ __forceinline__ bool convert_role(const P& p, const Block& b, Cursor<Packed, P> c, int warp) {
    using C = Converter<D, BITS>;
    using L = Smem<D, Packed::row_tiles>;
    const C cv(warp);
    typename C::Words kx, vx;
    uint32_t ks[4], vs[4];
    Cursor<Packed, P> ahead = c;
    int at = 0;  // key tile of `ahead`'s unit
    bool more = true;
    struct Next {
        typename C::Place place;
        int head;
        typename C::Span span;  // to < 0: no such tile
    };
    int lo = 0, hi = 0;  // tokens that some row of `ahead`'s unit sees
    auto here = [&]() -> Next {
        const int t0 = (ahead.w.first + ahead.tile0 + at) * kKeys;
        if (at == 0) {
            const int r0 = ahead.w.rt * Packed::rows;
            dev::seen_range(p, ahead.w.view, r0 / p.group, (r0 + ahead.rows(p) - 1) / p.group, lo, hi);
        }
        const typename C::Span sp = C::span(lo, hi, t0);
        return Next{cv.place(p, ahead.w.seq, t0, sp), ahead.w.head, sp};
    };
    auto advance = [&]() -> Next {
        if (more && ++at == ahead.tiles) at = 0, more = ahead.next(p);
        return more ? here() : Next{{0, 0}, 0, {0, -1}};
    };
    Next then = here();
    uint32_t row = C::row_of(p, then.place, then.head);
    typename C::Span sp = then.span;
    cv.load_scales(row, sp, p.k_scales, ks);
    cv.load_scales(row, sp, p.v_scales, vs);
    cv.load(row, sp, p.k_values, kx);
    cv.load(row, sp, p.v_values, vx);
    then = advance();
    int stage = 0, meta_at = 0;
    uint32_t phase = 1;  // the first pass over the stages finds them empty
    do {
        const Whole whole = whole_tiles(p, c);
        for (int t = 0; t < c.tiles; ++t) {
            int kref = C::key_ref(ks), vref = C::value_ref(vs);
            const bool wide = C::wide_keys(ks, kref), leading = t < whole.from, trailing = t >= whole.to;
            if (C::wide_values(vs, leading)) vref = C::spread_values(p.v_values, row, sp, vs, leading, trailing);
            uint32_t vs_now[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) vs_now[i] = vs[i];

            if (!b.wait(&b.sh->k_empty[stage], phase)) return false;
            if (wide) kref = C::spread_keys(p.k_values, row, sp, ks, b.sh->key_refs[meta_at % kMeta], warp == 0);
            cv.store(kx, ks, C::key_base(kref), b.smem + L::k + stage * L::tile);
            if (warp == 0 && cv.lane == 0) b.sh->meta[meta_at % kMeta] = make_int2(kref, vref);
            dev::fence_proxy_async();
            b.arrive(&b.sh->k_full[stage]);

            // the next key tile is on its way while this one's values are converted
            sp = then.span;
            if (sp.to >= 0) {
                row = C::row_of(p, then.place, then.head);
                cv.load_scales(row, sp, p.k_scales, ks);
                cv.load_scales(row, sp, p.v_scales, vs);
                cv.load(row, sp, p.k_values, kx);
                then = advance();
            }
            // a NaN belongs to the rows that see it: they get it at the end
            if (t < whole.from || t >= whole.to)
                if (C::take_out_nans(vx)) *reinterpret_cast<volatile int*>(&b.sh->nan_unit[c.unit & 3]) = c.unit;
            if (!b.wait(&b.sh->v_empty[stage], phase)) return false;
            cv.store(vx, vs_now, vref & 0xffff, b.smem + L::v + stage * L::tile);
            dev::fence_proxy_async();
            b.arrive(&b.sh->v_full[stage]);
            if (sp.to >= 0) cv.load(row, sp, p.v_values, vx);

            ++meta_at;
            if (++stage == kStages) stage = 0, phase ^= 1;
        }
    } while (c.next(p));
    return true;
}

// Index of a key tile among the converted ones.
template <class Cfg, class P>
__device__ __forceinline__ int64_t ready_at(const P& p, const Cursor<Cfg, P>& c) {
    return ((int64_t)c.w.rank * p.kv_heads + c.w.head) * p.max_tiles + c.w.first + c.tile0;
}

// One warp copying ready-made tiles (its elected lane).
template <int D, class P>
__device__ __forceinline__ void load_role(const P& p, const Block& b, Cursor<Ready, P> c) {
    using L = Smem<D, Ready::row_tiles>;
    constexpr int bytes = L::tile;
    int stage = 0, issued = 0;
    uint32_t phase = 1;
    bool ok = true, values = true;  // values: the last tile's were issued as well
    dev::wait_for_previous();       // the converted tiles
    do {
        const int64_t at = ready_at(p, c);
        for (int t = 0; t < c.tiles && ok; ++t) {
            ok = b.wait_lean(&b.sh->k_empty[stage], phase);
            if (!ok) break;
            if (dev::elect_one()) {
                dev::mbar_arrive_expect_tx(&b.sh->k_full[stage], bytes);
                dev::bulk_load(b.smem + L::k + stage * bytes, p.ready_k + (at + t) * bytes, bytes, &b.sh->k_full[stage]);
            }
            __syncwarp();
            values = ok = b.wait_lean(&b.sh->v_empty[stage], phase);
            if (ok && dev::elect_one()) {
                dev::mbar_arrive_expect_tx(&b.sh->v_full[stage], bytes);
                dev::bulk_load(b.smem + L::v + stage * bytes, p.ready_v + (at + t) * bytes, bytes, &b.sh->v_full[stage]);
            }
            __syncwarp();
            ++issued;
            if (++stage == kStages) stage = 0, phase ^= 1;
        }
    } while (ok && c.next(p));
    // Copies in flight must land before the CTA's memory goes: the last tile of each stage.
    for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
        const uint32_t parity = (uint32_t)(i / kStages) & 1u;
        const long long start = clock64();
        while (!(dev::mbar_try_wait(&b.sh->k_full[i % kStages], parity) &&
                 ((i == issued - 1 && !values) || dev::mbar_try_wait(&b.sh->v_full[i % kStages], parity))))
            if (clock64() - start > dev::kWaitLimitCycles) break;
    }
}

// --------------------------------------------------------------------------- products

template <int D, class Cfg, class P>
__device__ __forceinline__ void product_role(const P& p, const Block& b, Cursor<Cfg, P> c) {
    using L = Smem<D, Cfg::row_tiles>;
    constexpr int kTiles = Cfg::row_tiles;
    constexpr uint32_t idesc_s = dev::f16_idesc(kTileRows, kHalf, false);
    constexpr uint32_t idesc_o = dev::f16_idesc(kTileRows, D, true);
    // The whole warp walks, one elected lane issues: descriptors and addresses stay
    // warp-uniform and are advanced by constants.
    const uint32_t base = dev::smem_addr(b.smem);
    const uint64_t q_desc = dev::smem_desc(base + L::q, 16, 1024, dev::kLayoutSwizzle128);
    const uint64_t k_desc = dev::smem_desc(base + L::k, 16, 1024, dev::kLayoutSwizzle128);
    const uint64_t v_desc = dev::smem_desc(base + L::v, L::half, 1024, dev::kLayoutSwizzle128);
    Shared* sh = b.sh;
    bool ok = true;
    uint32_t k_stage = 0, v_stage = 0, k_phase = 0, v_phase = 0, p_phase[2] = {0, 0}, q_phase[2] = {0, 0};
    // A key tile goes through in two halves of 64 tokens, each with its own columns: while
    // a row tile's softmax works on one, the scores of the next are multiplied.
    auto scores = [&](int w, int half) {
        const uint64_t kd = k_desc + (uint64_t)(k_stage * (L::tile >> 4) + half * (kHalf * 128 >> 4));
        const uint64_t qd = q_desc + (uint64_t)(w * (L::tile >> 4));
        if (dev::elect_one()) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t at = ((i / 4) * L::half + (i % 4) * 32) >> 4;
                dev::tc_mma_f16(b.tmem + w * kKeys + half * kHalf, qd + at, kd + at, idesc_s, i > 0);
            }
            dev::tc_commit(&sh->s_full[w][half]);
        }
        __syncwarp();
    };
    auto release_keys = [&]() {
        if (dev::elect_one()) dev::tc_commit(&sh->k_empty[k_stage]);
        __syncwarp();
        if (++k_stage == kStages) k_stage = 0, k_phase ^= 1;
    };
    do {
        const int nw = kTiles == 1 ? 1 : __shfl_sync(kFull, c.rows(p) > kTileRows ? 2 : 1, 0);
        const int tiles = __shfl_sync(kFull, c.tiles, 0);
        ok = b.wait_lean(&sh->k_full[k_stage], k_phase);
#pragma unroll
        for (int w = 0; w < kTiles; ++w)
            if (w < nw && ok) ok = b.wait_lean(&sh->q_ready[w], q_phase[w]), q_phase[w] ^= 1;
        if (!ok) break;
        dev::tc_fence_after();
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int w = 0; w < kTiles; ++w)
                if (w < nw) scores(w, half);
        release_keys();
        for (int t = 0; t < tiles && ok; ++t) {
            // weighted values of key tile t, scores of key tile t + 1
            ok = b.wait_lean(&sh->v_full[v_stage], v_phase);
            if (ok && t + 1 < tiles) ok = b.wait_lean(&sh->k_full[k_stage], k_phase);
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int w = 0; w < kTiles; ++w) {
                    if (w >= nw || !ok) continue;
                    ok = b.wait_lean(&sh->p_ready[w][half], p_phase[w]);
                    if (!ok) continue;
                    if (half == 1) p_phase[w] ^= 1;
                    dev::tc_fence_after();
                    // the first product of a unit begins the output, unless that holds something
                    const bool more = t > 0 || half > 0 || *reinterpret_cast<volatile int*>(&sh->kept[w]);
                    const uint64_t vd = v_desc + (uint64_t)(v_stage * (L::tile >> 4) + half * (kHalf * 128 >> 4));
                    if (dev::elect_one()) {
#pragma unroll
                        for (int i = 0; i < kHalf / 16; ++i)
                            dev::tc_mma_f16_ta(b.tmem + kTiles * kKeys + w * D, b.tmem + w * kKeys + half * kHalf + 8 * i,
                                               vd + i * (2048 >> 4), idesc_o, i > 0 || more);
                        dev::tc_commit(&sh->o_done[w][half]);
                        if (half == 1 && w == nw - 1) dev::tc_commit(&sh->v_empty[v_stage]);
                    }
                    __syncwarp();
                    if (t + 1 < tiles) scores(w, half);
                }
            if (++v_stage == kStages) v_stage = 0, v_phase ^= 1;
            if (ok && t + 1 < tiles) release_keys();
        }
    } while (ok && c.next(p));
    // Products in flight must not outlive the CTA's memory.
    if (dev::elect_one()) {
        dev::tc_commit(&sh->drain);
        const long long start = clock64();
        while (!dev::mbar_try_wait(&sh->drain, 0))
            if (clock64() - start > dev::kWaitLimitCycles) break;
    }
    __syncwarp();
}

// ---------------------------------------------------------------------------- softmax

__device__ __forceinline__ float max3f(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Folds 32 scores into the running maxima m.
__device__ __forceinline__ void fold_top(const uint32_t (&s)[32], float (&m)[4]) {
#pragma unroll
    for (int i = 0; i < 32; i += 2)
        m[(i / 2) & 3] = max3f(m[(i / 2) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
}

// 2^x of a pair on the FMA pipe, for x below 128: with n the integer nearest to x and
// r = x - n, 2^x = 2^n 2^r, and on [-1/2, 1/2] a polynomial of degree five is within 7.5e-8
// of 2^r (least squares on the relative error, reweighted towards its largest values);
// in float32, whose constant term is 1 + 2^-23, within 2.2e-7.  The weights it makes are
// rounded to f16 afterwards.  Below -127 the result is zero; a NaN stays one.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));  // -127
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
    const float2 magic = make_float2(12582912.0f, 12582912.0f);  // 1.5 * 2^23: sums end in the integer
    const float2 y = __fadd2_rn(x, magic);
    const float2 n = __fadd2_rn(y, make_float2(-12582912.0f, -12582912.0f));
    const float2 r = __fadd2_rn(x, make_float2(-n.x, -n.y));
    auto c = [](float v) { return make_float2(v, v); };
    float2 v = __ffma2_rn(c(1.3276469420750838e-3f), r, c(9.67554164625246e-3f));
    v = __ffma2_rn(v, r, c(5.550713284339852e-2f));
    v = __ffma2_rn(v, r, c(2.4022119718243962e-1f));
    v = __ffma2_rn(v, r, c(6.931469670563168e-1f));
    v = __ffma2_rn(v, r, c(1.000000071655749f));
    const float2 p = make_float2(__uint_as_float(__float_as_uint(y.x) * 0x800000u + 0x3f800000u),
                                 __uint_as_float(__float_as_uint(y.y) * 0x800000u + 0x3f800000u));
    return __fmul2_rn(v, p);
}

// Weights 2^(score * f - base) of 32 scores, added to sum, as f16 pairs.  The exponential
// unit, 16 a cycle and SM, takes as long for them as the tensor core for both products; one
// pair in kFmaEvery is computed on the FMA pipe instead (chunk of 4096 over 16,384 tokens of
// heads of 128: 945 us without, 900 with one in 8, 928 one in 4, 962 one in 2).
constexpr int kFmaEvery = 8;
__device__ __forceinline__ void fold_weights(const uint32_t (&s)[32], float f, float base, float2 (&sum)[2],
                                             uint32_t (&pw)[16]) {
    const float2 f2 = make_float2(f, f), b2 = make_float2(-base, -base);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        float2 t = __ffma2_rn(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), f2, b2);
        if ((i / 2) % kFmaEvery == kFmaEvery - 1)
            t = ex2_fma(t);
        else
            t.x = ex2(t.x), t.y = ex2(t.y);
        sum[(i / 2) & 1] = __fadd2_rn(sum[(i / 2) & 1], t);
        const __half2 u = __float22half2_rn(t);
        pw[i / 2] = *reinterpret_cast<const uint32_t*>(&u);
    }
}

// The rare steps.  Rescaling the output happens inside the loop over the usual halves and is
// kept out of its registers by a call; the others have a place of their own outside it.

// An output row in TMEM times g.
template <int D>
__device__ __noinline__ void scale_output(uint32_t o_col, float g) {
#pragma unroll 1
    for (int h = 0; h < D / 32; ++h) {
        uint32_t o[32];
        dev::tmem_ld_32x32b_x32(o_col + 32 * h, o);
        dev::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * g);
        dev::tmem_st_32x32b_x32(o_col + 32 * h, o);
    }
    dev::tmem_wait_st();
}

// The largest score of a half key tile of which the row sees columns [from, to).
__device__ __forceinline__ float masked_top(uint32_t s_col, int from, int to) {
    float m = __int_as_float(0xff800000);
#pragma unroll 1
    for (int h = 0; h < kHalf / 32; ++h) {
        uint32_t s[32];
        dev::tmem_ld_32x32b_x32(s_col + 32 * h, s);
        dev::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (32 * h + i >= from && 32 * h + i < to) m = fmaxf(m, __uint_as_float(s[i]));
    }
    return m;
}

// Its weights, the f16 ones times `down`; returns their sum.
__device__ __forceinline__ float masked_weights(uint32_t s_col, int from, int to, float f, float base, float down) {
    float sum = 0.0f;
#pragma unroll 1
    for (int h = 0; h < kHalf / 32; ++h) {
        uint32_t s[32], pw[16];
        dev::tmem_ld_32x32b_x32(s_col + 32 * h, s);
        dev::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float a = ex2(fmaf(__uint_as_float(s[i]), f, -base)), b = ex2(fmaf(__uint_as_float(s[i + 1]), f, -base));
            if (32 * h + i < from || 32 * h + i >= to) a = 0.0f;
            if (32 * h + i + 1 < from || 32 * h + i + 1 >= to) b = 0.0f;
            sum += a + b;
            const __half2 u = __floats2half2_rn(a * down, b * down);
            pw[i / 2] = *reinterpret_cast<const uint32_t*>(&u);
        }
        dev::tmem_st_32x32b_x16(s_col + 16 * h, pw);
    }
    dev::tmem_wait_st();
    return sum;
}

// The score of column i in log2 units: f, or f and the token's own reference, times s.
__device__ __forceinline__ float own_score(const uint8_t* refs, int i, float s, float f) {
    return s * (refs ? f * __uint_as_float((uint32_t)refs[i] << 23) : f);
}

// The same as masked_top for a tile whose keys have a reference each, in log2 units.
__device__ __forceinline__ float wide_top(uint32_t s_col, int from, int to, float f, const uint8_t* refs) {
    float m = __int_as_float(0xff800000);
#pragma unroll 1
    for (int i = 0; i < kHalf; ++i) {
        const float s = __uint_as_float(dev::tmem_ld_32x32b_x1(s_col + i));
        dev::tmem_wait_ld();
        if (i >= from && i < to) m = fmaxf(m, own_score(refs, i, s, f));
    }
    return m;
}

// Features of a value row that are NaN (8-bit elements) among the tokens [k0, k1) that
// a row sees, as bits.
template <int D>
__device__ __noinline__ uint4 nan_features(const uint8_t* values, const int* table, int page_size, int pages,
                                           int kv_heads, int head, int k0, int k1) {
    uint32_t bad[4] = {0, 0, 0, 0};
    for (int k = k0; k < k1; ++k) {
        int page = __ldg(table + k / page_size);
        page = page < 0 ? 0 : (page >= pages ? pages - 1 : page);
        const uint32_t* v = reinterpret_cast<const uint32_t*>(
            values + (((int64_t)page * kv_heads + head) * page_size + k % page_size) * D);
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
            const uint32_t b = __vcmpeq4(__ldg(v + i) & 0x7f7f7f7fu, 0x7f7f7f7fu);
            const uint32_t bits = (b & 1u) | ((b >> 7) & 2u) | ((b >> 14) & 4u) | ((b >> 21) & 8u);
            bad[i / 8] |= bits << (4 * (i % 8));
        }
    }
    return make_uint4(bad[0], bad[1], bad[2], bad[3]);
}

// Queries of a row tile into shared memory, each row scaled by a power of two to a largest
// magnitude in [2^12, 2^13); a negative scale of the scores goes into their sign.  Of the
// tile's four warps, warp r0 has rows r0, r0 + 4, ..., so a tile with few rows is loaded by
// all of them.  Lane i names row r0 + 4 i (`at`, elements from p.q; `real`: it exists) and
// returns the factor that makes scores of its products with lifted keys, less the keys'
// reference.  D / 4 lanes load a row together (a thread that loads its own row touches 32
// of them in every access), kBatch such loads at a time; what is needed once a row is done
// by the lane that names it.
template <int D>
__device__ __forceinline__ float put_queries(const AttentionParams& p, int64_t at, bool real, uint8_t* rows, int r0) {
    constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes, kBatch = 8;
    const int lane = threadIdx.x & 31, piece = lane % kLanes, sub = lane / kLanes;
    const unsigned reals = __ballot_sync(kFull, real);
    const bool f16 = p.dtype == MXK_F16;
    auto fetch = [&](int base, uint2 (&x)[kBatch]) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = base + i * kAtOnce + sub;
            const int64_t row = __shfl_sync(kFull, at, r);
            x[i] = make_uint2(0, 0);
            if (reals >> r & 1u) {
                const uint16_t* q = static_cast<const uint16_t*>(p.q) + row + 4 * piece;
                if (p.q_vec)
                    x[i] = __ldg(reinterpret_cast<const uint2*>(q));
                else
                    x[i] = make_uint2(q[0] | ((uint32_t)q[1] << 16), q[2] | ((uint32_t)q[3] << 16));
            }
        }
    };
    // row r0 + 4 r: its swizzle depends on r's lowest bit
    const int chunk = piece / 2;
    uint8_t* const to = rows + (chunk / 8) * Smem<D>::half + r0 * 128 + (piece & 1) * 8;
    const int even = ((chunk % 8) ^ r0) << 4, odd = ((chunk % 8) ^ (r0 + 4)) << 4;
    // Rows past the last real one are left as they are: a row's scores are its own.
    const int rows_here = 32 - __clz(reals);
    unsigned own = 0;  // the largest magnitude of this lane's row, as 16 bits
    float f0 = 0.0f, f1 = 0.0f, factor = 0.0f;
    uint2 next[kBatch];
    if (rows_here) fetch(0, next);
#pragma unroll 1
    for (int base = 0; base < rows_here; base += kBatch * kAtOnce) {
        uint2 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) x[i] = next[i];
        if (base + kBatch * kAtOnce < rows_here) fetch(base + kBatch * kAtOnce, next);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            // 16-bit floats order as their bits (a NaN's row is NaN whatever its scale)
            const unsigned m2 = __vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu);
            const unsigned m = max(m2 & 0xffffu, m2 >> 16);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const unsigned top = __reduce_max_sync(kFull, sub == k ? m : 0u);
                if (lane == base + i * kAtOnce + k) own = top;
            }
        }
        const unsigned amax = f16 ? __float_as_uint(__half2float(__ushort_as_half((unsigned short)own))) : own << 16;
        const int e = amax ? max((int)(amax >> 23) - 127, -126) : 0;
        const int down = (kQueryExp - e) / 2, rest = kQueryExp - e - down;
        f0 = __uint_as_float((uint32_t)(down + 127) << 23);
        f1 = copysignf(__uint_as_float((uint32_t)(rest + 127) << 23), p.scale_log2);
        factor = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 - down - kKeyLift / 2) << 23) *
                 __uint_as_float((uint32_t)(127 - rest - kKeyLift / 2) << 23);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = base + i * kAtOnce + sub;
            const float g0 = __shfl_sync(kFull, f0, r), g1 = __shfl_sync(kFull, f1, r);
            float2 u, v;
            if (f16) {
                u = __half22float2(*reinterpret_cast<const __half2*>(&x[i].x));
                v = __half22float2(*reinterpret_cast<const __half2*>(&x[i].y));
            } else {
                u = make_float2(__uint_as_float(x[i].x << 16), __uint_as_float(x[i].x & 0xffff0000u));
                v = make_float2(__uint_as_float(x[i].y << 16), __uint_as_float(x[i].y & 0xffff0000u));
            }
            const __half2 a = __floats2half2_rn(u.x * g0 * g1, u.y * g0 * g1);
            const __half2 c = __floats2half2_rn(v.x * g0 * g1, v.y * g0 * g1);
            *reinterpret_cast<uint2*>(to + 512 * r + ((i * kAtOnce + sub) & 1 ? odd : even)) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
        }
    }
    return factor;
}

// A warp's 32 output rows from shared memory to where they belong, D / 8 lanes a row:
// columns [col, col + D / 2), four a lane, staged by their owners with the 16-byte chunks
// permuted by row.
template <int D, class P>
__device__ __forceinline__ void put_rows(const P& p, const float4* stage, unsigned reals, int64_t out_at,
                                         float* part, int col) {
    constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
    const int lane = threadIdx.x & 31, piece = lane % kLanes, sub = lane / kLanes;
    const int rows_here = 32 - __clz(reals);
    if (part) {
#pragma unroll 4
        for (int r = sub; r < rows_here; r += kAtOnce)
            *reinterpret_cast<float4*>(part + r * D + col + 4 * piece) = stage[r * kLanes + (piece ^ (r & 7))];
        return;
    }
#pragma unroll 1
    for (int base = 0; base < rows_here; base += 4 * kAtOnce) {
        int64_t at[4];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = base + i * kAtOnce + sub;
            at[i] = __shfl_sync(kFull, out_at, r);
            v[i] = stage[r * kLanes + (piece ^ (r & 7))];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (reals >> (base + i * kAtOnce + sub) & 1u) dev::store4_at(p, at[i] + col + 4 * piece, v[i]);
    }
}

// 32 packed elements as float32.
template <int BITS>
__device__ __forceinline__ void block_values(const uint32_t* w, float (&v)[32]) {
    uint32_t h2[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (BITS == 4) {
            uint32_t x[4];
            dev::e2m1x8_to_f16(w[j], x);
#pragma unroll
            for (int i = 0; i < 4; ++i) h2[4 * j + i] = x[i];
        } else {
            constexpr int kCode = BITS == 4 ? 8 : BITS;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t four = BITS == 8 ? w[2 * j + i] : dev::four6(w, 2 * j + i);
                h2[4 * j + 2 * i] = dev::codes_to_f16x2<kCode>(four);
                h2[4 * j + 2 * i + 1] = dev::codes_to_f16x2<kCode>(four >> 16);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2[j]));
        v[2 * j] = f.x, v[2 * j + 1] = f.y;
    }
}

// 2^(to - from), of scale bytes, up to 2^127 and down to where it is 0.
__device__ __forceinline__ float octaves(int to, int from) {
    return __uint_as_float((uint32_t)min(max(to - from + 127, 0), 254) << 23);
}

// The weights of a half key tile's columns [from, to) where its keys have a reference each
// (refs), or its values are worked through by hand (o_col).  Returns their sum and the
// row's reference of the values.
//
// The weights are left for the product with the values in f16, relative to base and
// lowered from vrun to vref.  By hand, because the tile's value scales are too far apart to be
// held relative to one reference for rows that see different tokens, the weighted values are
// added to the row's output in TMEM in float32 and the weights left for the product are zero.
// The output is relative to 2^(vrun - 127) with a factor g yet to come, or holds nothing
// yet (g = 0); vrun goes up where the row sees a token that asks for it.  A tile takes 115 to
// 140 us this way (chunks of 16 to 512 tokens, one overflowed value), most of it decoding
// that every row repeats.
struct WideHalf {
    uint32_t s_col, o_col;  // scores; output, or 0: weights only
    int t0;                 // its first token
    int seq, head;          // of the unit
    const uint8_t* refs;    // or none: f then holds the tile's
};
struct WideSum {
    float sum;
    int vrun;
};
template <int D, class P>
__device__ __forceinline__ WideSum wide_weights(const P& p, WideHalf half, int from, int to, float f,
                                             float base, int vref, int vrun_at, float g) {
    constexpr int kBlocks = D / 32;
    const uint32_t o_col = half.o_col;
    float sum = 0.0f;
    if (!o_col) {
        // (a row that sees nothing of the tile may be below its reference)
        const float lower = octaves(vref, max(vrun_at, vref));
#pragma unroll 1
        for (int i = 0; i < kHalf / 2; ++i) {
            float w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int t = 2 * i + k;
                const float s = __uint_as_float(dev::tmem_ld_32x32b_x1(half.s_col + t));
                dev::tmem_wait_ld();
                w[k] = t >= from && t < to ? ex2(own_score(half.refs, t, s, f) - base) : 0.0f;
            }
            sum += w[0] + w[1];
            const __half2 u = __floats2half2_rn(w[0] * lower, w[1] * lower);
            __syncwarp();
            dev::tmem_st_32x32b_x1(half.s_col + i, *reinterpret_cast<const uint32_t*>(&u));
        }
        dev::tmem_wait_st();
        return WideSum{sum, vrun_at};
    }
    // The warp goes through the tokens that some lane sees together; lane i fetches what is
    // needed of tokens i and i + 32.
    const int lane = threadIdx.x & 31;
    const int first = (int)__reduce_min_sync(kFull, (unsigned)(from < to ? from : kHalf));
    const int end = (int)__reduce_max_sync(kFull, (unsigned)(from < to ? to : 0));
    int64_t row[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int t = lane + 32 * k, token = half.t0 + t, at = token / p.page_size;
        row[k] = -1;
        if (t >= first && t < end) {
            const int page = min(max(__ldg(dev::table_of(p, half.seq) + at), 0), p.pages - 1);
            row[k] = ((int64_t)page * p.kv_heads + half.head) * p.page_size + (token - at * p.page_size);
        }
    }
    // Block b of a lane's token: its words and scale byte, zeros without a token.
    auto fetch = [&](int k, int b, uint32_t (&w)[8]) -> int {
        const uint32_t* at = reinterpret_cast<const uint32_t*>(p.v_values) + (row[k] * kBlocks + b) * p.bits;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const uint2 x = row[k] >= 0 && i < p.bits ? __ldg(reinterpret_cast<const uint2*>(at + i)) : make_uint2(0, 0);
            w[i] = x.x, w[i + 1] = x.y;
        }
        return row[k] >= 0 ? __ldg(p.v_scales + row[k] * kBlocks + b) : 0;
    };
    auto magnitude = [&](const uint32_t (&w)[8]) -> bool {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            any |= w[i] & (p.bits == 8 ? dev::magnitude_bits<8>(i)
                                       : (p.bits == 6 ? dev::magnitude_bits<6>(i) : dev::magnitude_bits<4>(i)));
        return any != 0;
    };
    int top = 0, vrun = vrun_at;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int own = 0;  // the largest scale of this lane's token, blocks of zeros left out
#pragma unroll 1
        for (int b = 0; b < kBlocks; ++b) {
            uint32_t w[8];
            const int scale = fetch(k, b, w);
            if (magnitude(w)) own = max(own, scale);
        }
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            const int t = 32 * k + i, x = __shfl_sync(kFull, own, i);
            if (t >= from && t < to) top = max(top, x);
        }
    }
    if (top > 0 && (vrun == 0 || top > vrun + kValueMax)) vrun = max(top - kValueLift, 1);
    g *= octaves(vrun_at, vrun);
#pragma unroll 1
    for (int b = 0; b < kBlocks; ++b) {
        uint32_t o[32];
        dev::tmem_ld_32x32b_x32(o_col + 32 * b, o);
        dev::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = g == 0.0f ? 0u : __float_as_uint(__uint_as_float(o[i]) * g);
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            uint32_t w[8];
            const int scale = fetch(k, b, w);
#pragma unroll 1
            for (int i = max(first - 32 * k, 0); i < min(end - 32 * k, 32); ++i) {
                const int t = 32 * k + i;
                const float s = __uint_as_float(dev::tmem_ld_32x32b_x1(half.s_col + t));
                uint32_t x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __shfl_sync(kFull, w[j], i);
                float v[32];
                if (p.bits == 8)
                    block_values<8>(x, v);
                else if (p.bits == 6)
                    block_values<6>(x, v);
                else
                    block_values<4>(x, v);
                const float unit = octaves(__shfl_sync(kFull, scale, i), vrun);
                dev::tmem_wait_ld();
                const bool sees = t >= from && t < to;
                const float weight = sees ? ex2(own_score(half.refs, t, s, f) - base) : 0.0f;
                if (b == 0) sum += weight;
                if (sees) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(fmaf(weight * unit, v[j], __uint_as_float(o[j])));
                }
            }
        }
        __syncwarp();
        dev::tmem_st_32x32b_x32(o_col + 32 * b, o);
    }
    uint32_t none[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) none[i] = 0;
    dev::tmem_st_32x32b_x32(half.s_col, none);
    dev::tmem_wait_st();
    return WideSum{sum, vrun};
}

// READY: tiles were converted beforehand, their references lie in global memory.
template <int D, class Cfg, bool READY, class P>
__device__ __forceinline__ bool softmax_role(const P& p, const Block& b, Cursor<Cfg, P> c, int warp) {
    using L = Smem<D, Cfg::row_tiles>;
    constexpr int kRows = Cfg::rows;
    Shared* sh = b.sh;
    const int w = warp >> 2;                                    // row tile
    const int r = threadIdx.x & (kTileRows - 1);                // row in the tile
    const uint32_t lane_base = b.tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t s_col = lane_base + w * kKeys, o_col = lane_base + Cfg::row_tiles * kKeys + w * D;
    const float neg_inf = __int_as_float(0xff800000);
    // Phases of s_full and o_done; a wait is never more than one completion behind, since
    // the scores of a half follow the products of the half before the last.
    uint32_t s_phase = 0, o_phase[2] = {0, 0};
    int meta_at = 0;
    uint32_t units_out = 0, out_phase = 0;  // units this row tile has put out, phase of the last
    bool open = false;
    do {
        const int rows = c.rows(p);
        if (w * kTileRows < rows) {
            const bool real = w * kTileRows + r < rows;
            const bool warp_real = w * kTileRows + (r & ~31) < rows;
            const int row = c.w.rt * kRows + w * kTileRows + r;
            const int j = row / p.group, head = c.w.head * p.group + (row - j * p.group);
            const Whole whole = whole_tiles(p, c);
            int lo = 0, hi = c.w.view.len;
            if (real) dev::seen_range(p, c.w.view, j, j, lo, hi);
            const int first_key = (c.w.first + c.tile0) * kKeys;
            // A warp's queries go where other warps' output rows of the unit before were.
            if (units_out > 0 && !b.wait(&sh->rows_out[w], out_phase)) return false;
            {
                const int r_load = (warp & 3) + 4 * (r & 31);  // the row this lane names
                const bool here = w * kTileRows + r_load < rows;
                const int row_load = c.w.rt * kRows + w * kTileRows + r_load, j_load = row_load / p.group;
                const int head_load = c.w.head * p.group + (row_load - j_load * p.group);
                const float f = put_queries<D>(
                    p, (int64_t)(c.w.view.row0 + j_load) * p.q_token + (int64_t)head_load * p.q_head, here,
                    b.smem + L::q + w * L::tile, warp & 3);
                sh->row_factor[w][r_load] = f;  // the row's own thread reads it after the first scores
            }
            dev::fence_proxy_async();
            b.arrive(&sh->q_ready[w]);

            float run_max = neg_inf, base = -kExpShift, sum = 0.0f;
            int vrun = 0;  // the output row is held relative to 2^(vrun - 127); 0: it saw nothing yet
            int vleast = 0, vmost = 0;  // the warp's smallest and largest
            bool nans = false;
            const int2* meta = nullptr;
            int2 ref = make_int2(0, 0);
            if constexpr (READY) {
                dev::wait_for_previous();  // the converted tiles' references
                meta = p.ready_meta + ready_at(p, c), ref = *meta;
            }
            // Scores of the half at hand; the next half's are fetched as the registers get free.
            uint32_t s[2][32];
            if (!b.wait(&sh->s_full[w][0], s_phase)) return false;
            dev::tc_fence_after();
            const int halves = 2 * c.tiles;
            // The half t's weights are in place; the next half's scores are waited for unless
            // fetched has been done already.
            auto pass_on = [&](int t, bool fetched) -> bool {
                dev::tc_fence_before();
                b.arrive(&sh->p_ready[w][t & 1]);
                if (t & 1)
                    o_phase[1] ^= 1;
                else
                    o_phase[0] ^= 1;
                if (t + 1 < halves && !fetched) {
                    if (!b.wait(&sh->s_full[w][~t & 1], s_phase ^ (t & 1))) return false;
                    dev::tc_fence_after();
                    if (warp_real) {
                        dev::tmem_ld_32x32b_x32(s_col + (~t & 1) * kHalf, s[0]);
                        dev::tmem_ld_32x32b_x32(s_col + (~t & 1) * kHalf + 32, s[1]);
                    }
                }
                if (t & 1) s_phase ^= 1;
                return true;
            };
            if (!warp_real) {
                for (int t = 0; t < halves; ++t)
                    if (!pass_on(t, false)) return false;
            } else {
                dev::tmem_ld_32x32b_x32(s_col, s[0]);
                dev::tmem_ld_32x32b_x32(s_col + 32, s[1]);
                const float row_factor = *const_cast<volatile float*>(&sh->row_factor[w][r]);
                // The references of half t's tile, from where they lie to `ref`.
                auto fetch_ref = [&](int t) {
                    if (READY)
                        ref = meta[t / 2];
                    else
                        ref = *const_cast<const int2*>(&sh->meta[(meta_at + t / 2) % kMeta]);
                };
                if (!READY) fetch_ref(0);
                // Halves that are out of the ordinary leave the loop below.
                auto partly = [&](int t) -> bool { return t < 2 * whole.from || t >= 2 * whole.to; };
                auto rare = [&](int t) -> bool {
                    return partly(t) || ref.x == kWide || vmost - (ref.y & 0xffff) > kMostDown;
                };
                // Waits for the products before half t, which have added to the output.
                auto output_so_far = [&](int t) -> bool {
                    if (!b.wait(&sh->o_done[w][(t - 1) & 1], (t & 1 ? o_phase[0] : o_phase[1]) ^ 1)) return false;
                    dev::tc_fence_after();
                    return true;
                };
                // Before this warp lets the unit's first product with the values start.
                if ((threadIdx.x & 31) == 0)
                    *reinterpret_cast<volatile int*>(&sh->kept[w]) = partly(0) && (ref.y & kWide) ? 1 : 0;
                for (int t = 0; t < halves;) {
                    while (t < halves && !rare(t)) {
                        const uint32_t s_at = s_col + (t & 1) * kHalf, s_next = s_col + (~t & 1) * kHalf;
                        const float f = row_factor * __uint_as_float((uint32_t)ref.x << 23);
                        const int vref = ref.y & 0xffff;
                        if (READY && (t & 1)) {
                            nans |= ref.y >> 16 & 1;
                            if (t + 1 < halves) fetch_ref(t + 1);
                        }
                        float m[4] = {neg_inf, neg_inf, neg_inf, neg_inf};
                        dev::tmem_wait_ld();
                        fold_top(s[0], m);
                        fold_top(s[1], m);
                        float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
                        if (top != neg_inf) top *= f;

                        // Raise the row's maximum, or the reference of the output, if need be.
                        const bool raise = top > run_max + kMaxSlack;
                        if (__any_sync(kFull, raise) || vref > vleast) {
                            const float x = raise ? top : run_max;
                            float g = x == run_max ? 1.0f : ex2(run_max - x);
                            run_max = x;
                            base = (x == neg_inf ? 0.0f : x) - kExpShift;
                            sum *= g;
                            if (vref > vrun) g *= octaves(vrun, vref), vrun = vref;
                            vleast = (int)__reduce_min_sync(kFull, (unsigned)vrun);
                            vmost = max(vmost, vref);
                            if (t > 0) {
                                if (!output_so_far(t)) return false;
                                scale_output<D>(o_col, g);
                            }
                        }
                        // The weights, over the scores they come from, scaled by 2^(vref - vrun):
                        // up to kMostDown octaves in their exponents, which float32 sums do not notice.
                        const int down = vrun - vref;
                        const float shifted = base + (float)down, back = __uint_as_float((uint32_t)(127 + down) << 23);
                        float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                        uint32_t pw[16];
                        fold_weights(s[0], f, shifted, part, pw);
                        dev::tmem_st_32x32b_x16(s_at, pw);
                        bool fetched = false;
                        if (t + 1 < halves) {
                            fetched = __all_sync(kFull, dev::mbar_test(&sh->s_full[w][~t & 1], s_phase ^ (t & 1)));
                            if (fetched) {
                                dev::tc_fence_after();
                                dev::tmem_ld_32x32b_x32(s_next, s[0]);
                            }
                        }
                        fold_weights(s[1], f, shifted, part, pw);
                        dev::tmem_st_32x32b_x16(s_at + 16, pw);
                        if (fetched) dev::tmem_ld_32x32b_x32(s_next + 32, s[1]);
                        dev::tmem_wait_st();
                        sum += back * ((part[0].x + part[0].y) + (part[1].x + part[1].y));
                        if (!pass_on(t, fetched)) return false;
                        ++t;
                        if (!READY && !(t & 1) && t < halves) fetch_ref(t);
                    }
                    if (t == halves) break;
                    // A half that the rows see different parts of, whose keys have a reference
                    // each, or whose values lie far below those before.
                    dev::tmem_wait_ld();
                    const int t0 = first_key + t * kHalf, vref = ref.y & 0xffff;
                    const bool by_hand = partly(t) && (ref.y & kWide);
                    const int from = min(max(lo - t0, 0), kHalf), to = min(max(hi - t0, 0), kHalf);
                    WideHalf half{s_col + (t & 1) * kHalf, by_hand ? o_col : 0, t0, c.w.seq, c.w.head, nullptr};
                    float f = row_factor, top;
                    if (ref.x == kWide) {
                        half.refs = (READY ? p.ready_key_refs + (meta + t / 2 - p.ready_meta) * kKeys
                                           : sh->key_refs[(meta_at + t / 2) % kMeta]) + (t & 1) * kHalf;
                        top = wide_top(half.s_col, from, to, f, half.refs);
                    } else {
                        f *= __uint_as_float((uint32_t)ref.x << 23);
                        top = masked_top(half.s_col, from, to);
                        if (top != neg_inf) top *= f;
                    }
                    if (READY && (t & 1)) nans |= ref.y >> 16 & 1;
                    const bool raise = top > run_max + kMaxSlack;
                    const bool up = vref > vrun && to > from && !by_hand;  // only rows that see something of it
                    float g = 1.0f;
                    if (__any_sync(kFull, raise || up) || by_hand) {
                        const float x = raise ? top : run_max;
                        g = x == run_max ? 1.0f : ex2(run_max - x);
                        run_max = x;
                        base = (x == neg_inf ? 0.0f : x) - kExpShift;
                        sum *= g;
                        if (up) g *= octaves(vrun, vref), vrun = vref;
                        if (t > 0) {
                            if (!output_so_far(t)) return false;
                            if (!by_hand) scale_output<D>(o_col, g);
                        }
                    }
                    if (by_hand || half.refs) {
                        const WideSum ws = wide_weights<D>(p, half, from, to, f, base, vref, vrun, t > 0 ? g : 0.0f);
                        sum += ws.sum, vrun = ws.vrun;
                    } else {
                        // (a row that sees nothing of the tile may be below its reference)
                        sum += masked_weights(half.s_col, from, to, f, base, octaves(vref, max(vrun, vref)));
                    }
                    vleast = (int)__reduce_min_sync(kFull, (unsigned)vrun);
                    vmost = (int)__reduce_max_sync(kFull, (unsigned)vrun);
                    if (!pass_on(t, false)) return false;
                    ++t;
                    if (!(t & 1) && t < halves) fetch_ref(t);
                }
            }

            // The output row.
            if (!b.wait(&sh->o_done[w][0], o_phase[0] ^ 1) || !b.wait(&sh->o_done[w][1], o_phase[1] ^ 1)) return false;
            dev::tc_fence_after();
            if (warp_real) {
                const bool all = c.whole();
                // NaNs that were taken out of the values, for the rows that see them
                uint32_t bad[4] = {0, 0, 0, 0};
                if constexpr (!READY) nans = *reinterpret_cast<volatile int*>(&sh->nan_unit[c.unit & 3]) == c.unit;
                if (nans && real) {
                    const int end = first_key + c.tiles * kKeys;
                    const uint4 f = nan_features<D>(p.v_values, dev::table_of(p, c.w.seq), p.page_size, p.pages, p.kv_heads,
                                                    c.w.head, max(lo, first_key), min(hi, end));
                    bad[0] = f.x, bad[1] = f.y, bad[2] = f.z, bad[3] = f.w;
                }
                const float vfactor = __uint_as_float((uint32_t)vrun << 23);
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int64_t slot = 2 * (int64_t)blockIdx.x + (c.tile0 == 0 ? 1 : 0);
                const int tile_row = w * kTileRows + r;
                const unsigned reals = __ballot_sync(kFull, real);
                const int64_t out_at = (dev::out_row(p, c.w.view) + j) * p.out_token + (int64_t)head * p.out_head;
                float* part = all ? nullptr : p.part + (slot * kRows + (tile_row & ~31)) * D;
                // The rows leave through the queries' shared memory, which no product reads any
                // more: a warp's quarter of the row tile holds 32 rows of D / 2 floats.
                float4* stage = reinterpret_cast<float4*>(b.smem + L::q + w * L::tile + (warp & 3) * (L::tile / 4));
#pragma unroll
                for (int h = 0; h < D / 32; ++h) {
                    uint32_t o[32];
                    dev::tmem_ld_32x32b_x32(o_col + 32 * h, o);
                    dev::tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 v = make_float4(__uint_as_float(o[i]) * inv * vfactor, __uint_as_float(o[i + 1]) * inv * vfactor,
                                               __uint_as_float(o[i + 2]) * inv * vfactor, __uint_as_float(o[i + 3]) * inv * vfactor);
                        if (sum == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (nans) {
                            const float nan = __int_as_float(0x7fc00000);
                            if (bad[h] >> i & 1u) v.x = nan;
                            if (bad[h] >> (i + 1) & 1u) v.y = nan;
                            if (bad[h] >> (i + 2) & 1u) v.z = nan;
                            if (bad[h] >> (i + 3) & 1u) v.w = nan;
                        }
                        const int chunk = (h % (D / 64)) * 8 + i / 4;
                        stage[(r & 31) * (D / 8) + (chunk ^ (r & 7))] = v;
                    }
                    if ((h + 1) % (D / 64) == 0) {
                        __syncwarp();
                        put_rows<D>(p, stage, reals, out_at, part, (h / (D / 64)) * (D / 2));
                        __syncwarp();
                    }
                }
                if (real) {
                    if (all) {
                        dev::store_stat(p, c.w.view, dev::out_row(p, c.w.view) + j, head, run_max, sum);
                    } else {
                        p.part_stat[slot * kRows + tile_row] = make_float2(run_max, sum);
                        if (std::is_same<P, SharedParams>::value && c.tile0 == 0)
                            dev::store_where(p, c.w.view, dev::out_row(p, c.w.view) + j, head, tile_row,
                                             b.share.followers(b.share.tiles - c.left, c.w.tiles));
                    }
                }
            }
            dev::tc_fence_before();
            b.arrive(&sh->rows_out[w]);
            out_phase = units_out++ & 1u;
        }
        meta_at += c.tiles;
        if (!c.whole() && c.tile0 == 0) {
            open = true;
            if (threadIdx.x == 0)
                p.part_open[blockIdx.x] =
                    make_int4(c.w.seq, c.w.rt, c.w.head, b.share.followers(b.share.tiles - c.left, c.w.tiles));
        }
    } while (c.next(p));
    if (threadIdx.x == 0 && !open) p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0);
    return true;
}

// ---------------------------------------------------------------------------- kernels

// Barriers, TMEM and the cursor; false: the CTA has no share.
constexpr int tmem_columns(int d, int row_tiles) { return row_tiles * (kKeys + d) <= 256 ? 256 : 512; }

template <int D, class Cfg, int FULL_COUNT, class P>
__device__ __forceinline__ bool begin(const P& p, uint8_t* smem_raw, Shared* sh, int* scratch, unsigned* err, Block& b,
                                      Cursor<Cfg, P>& c) {
    constexpr int kRows = Cfg::rows;
    const int tid = threadIdx.x;
    dev::let_next_start();
    const dev::Share share = dev::take_share<kRows, kKeys, Cfg::unit_cost, Cfg::threads>(p, scratch);
    c.left = 0;
    if (share.tiles > 0) {
        c.w = dev::walk_to<kRows, kKeys>(p, share);
        c.left = share.tiles - c.w.skip;
        if (std::is_same<Cfg, Ready>::value && p.seqs > 1) {
            // More than the host made room for can only be sequences whose rows overlap.
            const Ranks r = rank_of_seq(p, share.seq);
            c.w.rank = r.rank;
            if (r.all > p.ready_seqs) c.left = 0;
        }
    }
    if (c.left <= 0) {
        if (tid == 0) p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0);
        dev::wait_for_previous();
        return false;
    }
    if (tid == 0) {
        sh->abort_word = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            dev::mbar_init(&sh->q_ready[i], kTileRows / 32);
            dev::mbar_init(&sh->rows_out[i], kTileRows / 32);
            dev::mbar_init(&sh->s_full[i][0], 1);
            dev::mbar_init(&sh->s_full[i][1], 1);
            dev::mbar_init(&sh->p_ready[i][0], kTileRows / 32);
            dev::mbar_init(&sh->p_ready[i][1], kTileRows / 32);
            dev::mbar_init(&sh->o_done[i][0], 1);
            dev::mbar_init(&sh->o_done[i][1], 1);
        }
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
            dev::mbar_init(&sh->k_full[i], FULL_COUNT);
            dev::mbar_init(&sh->v_full[i], FULL_COUNT);
            dev::mbar_init(&sh->k_empty[i], 1);
            dev::mbar_init(&sh->v_empty[i], 1);
        }
        dev::mbar_init(&sh->drain, 1);
        dev::fence_barrier_init();
    }
    if (tid < 4) sh->nan_unit[tid] = -1;
    if (tid < 32) dev::tmem_alloc(&sh->tmem, tmem_columns(D, Cfg::row_tiles));
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    b.smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    b.sh = sh;
    b.tmem = __shfl_sync(kFull, sh->tmem, 0);
    b.err = err;
    b.share = share;
    c.unit = 0;
    c.cost = share.cost;
    c.take();
    return true;
}

template <int D, class Cfg>
__device__ __forceinline__ void finish(const AttentionParams& p, const Block& b) {
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    if (threadIdx.x < 32) dev::tmem_dealloc(b.tmem, tmem_columns(D, Cfg::row_tiles));
    dev::wait_for_previous();
    // After a wait gave up nothing of this CTA is joined.
    if (threadIdx.x == 0 && *b.abort_flag())
        p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0);
}

template <int D, int BITS, class P>
__global__ void __launch_bounds__(Packed::threads, 1) attention_tiles_kernel(const __grid_constant__ P p, unsigned* err) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) Shared shared;
    __shared__ int scratch[Packed::threads / 16 + 2];
    Block b;
    Cursor<Packed, P> c;
    if (!begin<D, Packed, Packed::convert_warps>(p, smem_raw, &shared, scratch, err, b, c)) return;
    const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0);
    if (warp < Packed::softmax_warps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Packed::softmax_regs));
        softmax_role<D, Packed, false>(p, b, c, warp);
    } else if (warp < Packed::product_warp) {
        convert_role<D, BITS>(p, b, c, warp - Packed::softmax_warps);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Packed::product_regs));
        if (warp == Packed::product_warp) product_role<D, Packed>(p, b, c);
    }
    finish<D, Packed>(p, b);
}

template <int D, class P>
__global__ void __launch_bounds__(Ready::threads, 1) attention_ready_kernel(const __grid_constant__ P p, unsigned* err) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) Shared shared;
    __shared__ int scratch[Ready::threads / 16 + 2];
    Block b;
    Cursor<Ready, P> c;
    if (!begin<D, Ready, 1>(p, smem_raw, &shared, scratch, err, b, c)) return;
    const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0);
    if (warp < Ready::softmax_warps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Ready::softmax_regs));
        softmax_role<D, Ready, true>(p, b, c, warp);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Ready::product_regs));
        if (warp == Ready::product_warp)
            product_role<D, Ready>(p, b, c);
        else if (warp == Ready::load_warp)
            load_role<D>(p, b, c);
    }
    finish<D, Ready>(p, b);
}

// Once per device: shared memory, and that the build has the registers the split assumes.
template <class K>
int prepare_kernel(K kernel, int smem, int regs, int& ready_device) {
    int dev = 0;
    MXK_CUDA(cudaGetDevice(&dev));
    if (ready_device == dev) return MXK_OK;
    MXK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaFuncAttributes attr{};
    MXK_CUDA(cudaFuncGetAttributes(&attr, kernel));
    if (attr.numRegs != regs)
        return fail(MXK_ERR_UNSUPPORTED, "cache_attention: kernel built with " + std::to_string(attr.numRegs) +
                                             " registers, the register split needs " + std::to_string(regs));
    ready_device = dev;
    return MXK_OK;
}

// One CTA an SM, or one a key tile if there cannot be as many.
template <class Cfg, class P>
int grid_size(const P& p, int max_q, int max_rows, int64_t* ctas) {
    const int64_t most = attention_tile_bound(p, max_q, max_rows, Cfg::rows, kKeys);
    MXK_REQUIRE(most <= std::numeric_limits<int>::max() / (1 + Cfg::unit_cost), "cache_attention: too much work for one call");
    static const int sms = sm_count();
    *ctas = most < sms ? most : sms;
    return MXK_OK;
}

template <int D, int BITS, class P>
int launch_packed(P p, int max_q, int max_rows, AttentionCall<P>& call) {
    constexpr int smem = Smem<D, Packed::row_tiles>::total;
    static thread_local int ready_device = -1;
    MXK_CHECK(prepare_kernel(attention_tiles_kernel<D, BITS, P>, smem, Packed::launch_regs, ready_device));
    unsigned* err = device_error_word();
    if (!err) return fail(MXK_ERR_CUDA, "cache_attention: cannot allocate the device error word");
    int64_t ctas;
    MXK_CHECK((grid_size<Packed>(p, max_q, max_rows, &ctas)));
    MXK_CHECK(call.take(p, ctas, Packed::rows, D));
    MXK_CHECK(call.launch("attention_tiles", attention_tiles_kernel<D, BITS, P>, (unsigned)ctas, Packed::threads, smem, p, err));
    call.join_later(p, ctas, Packed::rows, Packed::join_split);
    return MXK_OK;
}

template <int D, int BITS, class P>
int launch_ready(P p, int max_q, int max_rows, AttentionCall<P>& call) {
    constexpr int smem = Smem<D, Ready::row_tiles>::total;
    static thread_local int ready_device = -1;
    MXK_CHECK(prepare_kernel(attention_ready_kernel<D, P>, smem, Ready::launch_regs, ready_device));
    unsigned* err = device_error_word();
    if (!err) return fail(MXK_ERR_CUDA, "cache_attention: cannot allocate the device error word");
    int64_t ctas;
    MXK_CHECK((grid_size<Ready>(p, max_q, max_rows, &ctas)));
    const int64_t tiles = (int64_t)p.ready_seqs * p.kv_heads * p.max_tiles;
    void* extra = nullptr;
    MXK_CHECK(call.take(p, ctas, Ready::rows, D, tiles * (2 * Smem<D>::tile + (int64_t)sizeof(int2) + kKeys), &extra));
    p.ready_k = static_cast<uint8_t*>(extra);
    p.ready_v = p.ready_k + tiles * Smem<D>::tile;
    p.ready_meta = reinterpret_cast<int2*>(p.ready_v + tiles * Smem<D>::tile);
    p.ready_key_refs = reinterpret_cast<uint8_t*>(p.ready_meta + tiles);
    MXK_CHECK(call.launch("attention_unpack", attention_unpack_kernel<D, BITS, P>, dim3((unsigned)tiles, 2), 256, 0, p));
    MXK_CHECK(call.launch("attention_ready", attention_ready_kernel<D, P>, (unsigned)ctas, Ready::threads, smem, p, err));
    call.join_later(p, ctas, Ready::rows, Ready::join_split);
    return MXK_OK;
}

template <int D, int BITS, class P>
int launch(const P& p, bool ready, int max_q, int max_rows, AttentionCall<P>& call) {
    return ready ? launch_ready<D, BITS>(p, max_q, max_rows, call) : launch_packed<D, BITS>(p, max_q, max_rows, call);
}

template <int D, class P>
int launch_bits(int bits, const P& p, bool ready, int max_q, int max_rows, AttentionCall<P>& call) {
    if (bits == 8) return launch<D, 8>(p, ready, max_q, max_rows, call);
    if (bits == 6) return launch<D, 6>(p, ready, max_q, max_rows, call);
    return launch<D, 4>(p, ready, max_q, max_rows, call);
}

// Sequences (parts) that can have more than `rows` rows per key head, and their most tokens.
struct Most {
    int64_t seqs;
    int tokens;
};
[[maybe_unused]] Most most_ready(const AttentionParams& p, int max_q, int, int rows) {
    if ((int64_t)max_q * p.group <= rows) return {0, 0};
    return {p.seqs == 1 ? 1 : std::min<int64_t>(p.seqs, p.tokens * p.group / (rows + 1)), p.max_kv};
}
[[maybe_unused]] Most most_ready(const SharedParams& p, int max_q, int max_rows, int rows) {
    AttentionParams own = p, prefix = p;
    own.seqs = p.seqs - p.groups;
    prefix.seqs = p.groups, prefix.max_kv = p.max_prefix;
    const Most a = own.seqs ? most_ready(own, max_q, 0, rows) : Most{0, 0};
    const Most b = prefix.seqs ? most_ready(prefix, max_rows, 0, rows) : Most{0, 0};
    return {a.seqs + b.seqs, std::max(a.tokens, b.tokens)};
}

}  // namespace

template <class P>
int launch_attention_tiles(int bits, int head_dim, P p, int max_q, int max_rows, AttentionCall<P>& call) {
    // Several row tiles of a key head share its keys: converting those once pays for
    // writing and reading them as f16.  So many sequences can have enough rows for that:
    const int ready_rows = std::is_same<P, SharedParams>::value ? kReadyRowsShared : (p.seqs == 1 ? kReadyRows : kReadyRowsMany);
    const Most most = most_ready(p, max_q, max_rows, ready_rows);
    p.max_tiles = (most.tokens + kKeys - 1) / kKeys;
    p.ready_seqs = (int)most.seqs;
    const int64_t bytes = most.seqs * p.kv_heads * p.max_tiles * 2 * kKeys * head_dim * 2;
    const bool many = most.seqs > 0 && p.max_tiles > 0 && bytes <= kReadyBytes;
    const int few_q = (int)((ready_rows + p.group - 1) / p.group);
    if (many) {
        P q = p;
        if (p.seqs > 1 && q.min_rows <= ready_rows) q.min_rows = ready_rows + 1;
        MXK_CHECK(head_dim == 128 ? launch_bits<128>(bits, q, true, max_q, max_rows, call)
                                  : launch_bits<64>(bits, q, true, max_q, max_rows, call));
        if (p.seqs == 1) return MXK_OK;
        p.max_rows = ready_rows;
        max_q = max_rows = few_q;
    }
    return head_dim == 128 ? launch_bits<128>(bits, p, false, max_q, max_rows, call)
                           : launch_bits<64>(bits, p, false, max_q, max_rows, call);
}

// Compiled for each kind of calls (attention_tiles_shared.cu).
#ifndef MXK_ATTENTION_PARAMS
#define MXK_ATTENTION_PARAMS AttentionParams
#endif
template int launch_attention_tiles(int, int, MXK_ATTENTION_PARAMS, int, int, AttentionCall<MXK_ATTENTION_PARAMS>&);

}  // namespace mxk
