// Shared pieces of the attention kernels over the paged MX cache: parameters,
// the division of the work over CTAs, and the layout of partial sums.
//
// Work is divided without the host knowing the lengths.  A unit is one (sequence,
// row tile, key head): the rows r = j * group + g (query token j, query head g of
// the key head's group) of one tile, over the tokens that any of them sees, in
// key tiles.  Starting and ending a unit takes a CTA as long as COST key tiles (a
// constant of each kernel), so where there are more key tiles than CTAs a unit counts
// as that many more (not more than a CTA's part of the tiles), which come first and
// hold nothing.  All units' tiles, numbered
// one after the other, are split evenly over the CTAs, so every CTA has about the same
// to do whatever the lengths are; a CTA walks its tiles unit by unit.  A unit that one CTA has to itself is
// written out by it; the parts of a unit that spans several go to the workspace
// (at most two per CTA: the end of a unit that an earlier CTA began, and the
// beginning of one that a later CTA goes on with) and attention_join_kernel adds
// them in CTA order, so the result does not depend on timing.  A part holds the weighted
// mean of the values it saw, which is no larger than they are, and the maximum and sum of
// its weights.
#pragma once

#include <algorithm>

#include "cache.cuh"

namespace mxk {

struct AttentionParams {
    // cache
    const uint8_t* k_values;
    const uint8_t* v_values;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
    int bits, kv_heads, page_size, pages;
    // queries and outputs
    const void* q;
    void* out;
    float* lse;
    int64_t q_token, q_head, out_token, out_head;  // strides in elements
    int64_t tokens;
    int dtype, heads, group, seqs, max_q;
    int q_vec, out_vec;  // rows can be moved 8 bytes at a time
    const int* cu_q;
    const int* page_table;
    int64_t table_stride;
    int max_kv;
    const int* kv_lens;
    float scale_log2;  // scale * log2(e)
    int causal, window;
    int min_rows, max_rows;  // this launch takes the sequences with min_rows <= n * group <= max_rows
    // partial sums
    float* part;  // [2 * CTAs][tile rows][head_dim]: means
    float2* part_stat;  // [2 * CTAs][tile rows]: running maximum (log2 units), sum
    int4* part_open;    // [CTAs]: {sequence, row tile, key head, n} of the unit that the CTA began and the n
                        // following ones went on with; n = 0: it left none unfinished
    // keys and values converted beforehand (tiles kernel), [ready_seqs][kv_heads][max_tiles], of
    // this launch's sequences, one after the other
    uint8_t* ready_k;
    uint8_t* ready_v;
    int2* ready_meta;   // reference scales of the keys (or kWide) and values; bit 16 of y: NaNs taken out
    uint8_t* ready_key_refs;  // [tile][token] reference scales of the keys of kWide tiles
    int max_tiles, ready_seqs;
};

// A call whose sequences share prefixes.  Its units belong to parts of the sequences' tokens:
// part g < groups is the prefix of group g, seen by all its sequences' rows, part groups + i
// what sequence i has behind it.  `seqs` counts the parts.  The rows of units that one CTA has to
// itself come out in float32 with their maxima and sums, those of the prefixes before those of
// the rest; for all rows `where` tells attention_merge_kernel (attention_shared.cu), which joins
// what there is of a row, where that lies.
struct SharedParams : AttentionParams {
    float2* row_stat;  // [2][tokens][heads]: as part_stat
    int4* where;       // [2][tokens][heads]: {kernel of the call, or -1: the row is whole, -2: no such row;
                       // CTA that began the unit; CTAs that went on with it; row in its tile, and kHasPrefix}
    int kernel;        // of the call: 0, 1, ...
    const int4* parts;  // two to a part: {first row, rows, tokens end, position of the first row},
                        // {first token, page table row, 0, 0}
    int groups, max_prefix;
    // Parts of single tokens, where attention_solo_kernel takes them (else null): chunks, two int4 each:
    // {sequence, query row, first token, tokens end}, {number of the chunk in its part, chunks of the part,
    // first token of the part, number of its first chunk among those of parts that have several}; and how
    // many there are.
    const int4* solo;
    int* solo_count;  // and of those taken from a counter
};
constexpr int kSoloRows = 8;  // query rows of such a part, at most

constexpr int kHasPrefix = 1 << 30;  // what the row sees of the prefix comes to it

// Key tiles there can be at most when no sequence has more than max_q query and
// p.max_kv cached tokens, and all of them p.tokens query tokens: a window touches at
// most one tile more than it and the row tile's tokens fill.  (One long sequence among
// many short ones has few row tiles, so their number is not seqs times its own.)
inline int64_t attention_tile_bound(const AttentionParams& p, int max_q, int rows, int keys) {
    const int64_t one = ((int64_t)max_q * p.group + rows - 1) / rows;
    const int64_t row_tiles = std::min<int64_t>(p.seqs * one, p.tokens * p.group / rows + std::min<int64_t>(p.seqs, p.tokens));
    int64_t span = p.max_kv;  // below 2^30, as the window
    if (p.window > 0 && p.window + rows < span) span = p.window + rows;
    return p.kv_heads * row_tiles * (span / keys + 2);
}

// The same of a call with prefixes: of the sequences and of the groups, whose rows are those
// of up to max_rows query tokens.
inline int64_t attention_tile_bound(const SharedParams& p, int max_q, int max_rows, int rows, int keys) {
    AttentionParams own = p, prefix = p;
    own.seqs = p.seqs - p.groups;
    prefix.seqs = p.groups, prefix.max_kv = p.max_prefix;
    return attention_tile_bound(own, max_q, rows, keys) + attention_tile_bound(prefix, max_rows, rows, keys);
}
inline int64_t attention_tile_bound(const AttentionParams& p, int max_q, int, int rows, int keys) {
    return attention_tile_bound(p, max_q, rows, keys);
}

namespace dev {

// exp(s - max) is held as 2^(s2 - m2 + kExpShift) with s2, m2 in log2 units: up
// to 2^(kExpShift + kMaxSlack) = 2^15 it fits f16 (whose largest value is below
// 2^16), and values down to 2^-35 of the row's largest keep a nonzero f16.
// The running maximum m2 is only raised when a score exceeds it by more than
// kMaxSlack: below that the sums need no rescaling.
constexpr float kExpShift = 11.0f;
constexpr float kMaxSlack = 4.0f;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Element headroom: codes are at most 448 < 2^9, f16 reaches 2^16, so block
// factors go up to 2^6; keys use it fully, values start at 2^4 and may grow to 2^6
// before their reference moves.
constexpr int kKeyLift = 6;
constexpr int kValueLift = 4, kValueMax = 6;
constexpr int kScaleOfZeros = 127;  // scale byte of a block of zeros, as written
// Octaves that a token which a row does not see may lift the row's reference above what it
// sees, when more tokens follow: its f16 weights then still reach down to 2^-24 of the largest.
constexpr int kMostLift = 8;
// Octaves by which a block's scale may lie below what its f16 factors are relative to, so
// that every element stays a multiple of f16's smallest, 2^-24 (elements are multiples of
// 2^-9, 2^-3 and 2^-1).
template <int BITS>
constexpr int kExactDown = BITS == 8 ? 15 : (BITS == 6 ? 21 : 23);
constexpr int kQueryExp = 12;  // query rows are scaled to a largest magnitude in [2^12, 2^13)

// The magnitude bits of word i of packed elements that begin with word 0.
template <int BITS>
__device__ __forceinline__ uint32_t magnitude_bits(int i) {
    if (BITS == 8) return 0x7f7f7f7fu;
    if (BITS == 4) return 0x77777777u;
    return i % 3 == 0 ? 0xdf7df7dfu : (i % 3 == 1 ? 0xf7df7df7u : 0x7df7df7du);
}

// The j-th group of four 6-bit codes of a packed row, one per byte.
__device__ __forceinline__ uint32_t four6(const uint32_t* w, int j) {
    const int bit = 24 * j, i = bit / 32, s = bit % 32;
    const uint32_t v = s <= 8 ? w[i] >> s : __funnelshift_r(w[i], w[i + 1], s);
    return dev::spread6(v);
}

// f16 pair of 2^(e0), 2^(e1), zero where that is below f16's range (e <= 15).
__device__ __forceinline__ uint32_t pow2_f16x2(int e0, int e1) {
    const float a = __uint_as_float((uint32_t)max(e0 + 127, 0) << 23);
    const float b = __uint_as_float((uint32_t)max(e1 + 127, 0) << 23);
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// One sequence as the host's bounds let it be seen.
struct SeqView {
    int row0;  // first query row
    int n;     // query tokens
    int len;   // cached tokens
};

__device__ __forceinline__ int first_position(const SeqView& s) { return s.len - s.n; }  // of its query tokens
__device__ __forceinline__ int first_token(const SeqView&) { return 0; }

// A part of a call with prefixes, rows and tokens as a sequence's.
struct PartView {
    int row0, n, len;
    int position;  // of its first query token
    int start;     // its tokens begin here; -1: it is a prefix
};
__device__ __forceinline__ int first_position(const PartView& s) { return s.position; }
__device__ __forceinline__ int first_token(const PartView& s) { return max(s.start, 0); }

template <class P>
struct ViewOf { using type = SeqView; };
template <>
struct ViewOf<SharedParams> { using type = PartView; };

// A sequence's page numbers.
__device__ __forceinline__ const int* table_of(const AttentionParams& p, int seq) {
    return p.page_table + (int64_t)seq * p.table_stride;
}
__device__ __forceinline__ const int* table_of(const SharedParams& p, int part) {
    return p.page_table + (int64_t)__ldg(&p.parts[2 * part + 1].y) * p.table_stride;
}

// Where a sequence's rows go.
__device__ __forceinline__ int64_t out_row(const AttentionParams&, const SeqView& s) { return s.row0; }
__device__ __forceinline__ int64_t out_row(const SharedParams& p, const PartView& s) {
    return s.row0 + (s.start < 0 ? 0 : p.tokens);
}

__device__ __forceinline__ PartView seq_view(const SharedParams& p, int part) {
    const int4 a = __ldg(p.parts + 2 * part), b = __ldg(p.parts + 2 * part + 1);
    return PartView{a.x, a.y, a.z, a.w, b.x};
}

__device__ __forceinline__ SeqView seq_view(const AttentionParams& p, int seq) {
    SeqView v;
    const int a = __ldg(p.cu_q + seq), b = __ldg(p.cu_q + seq + 1), len = __ldg(p.kv_lens + seq);
    v.row0 = min(max(a, 0), (int)p.tokens);
    v.n = min(min(max(b, v.row0), (int)p.tokens) - v.row0, p.max_q);
    v.len = min(max(len, 0), p.max_kv);
    return v;
}

// Tokens [lo, hi) that the rows of query tokens j0..j1 see, all of them together
// (empty: hi <= lo).
template <class P, class V>
__device__ __forceinline__ void seen_range(const P& p, const V& s, int j0, int j1, int& lo, int& hi) {
    const int first = first_position(s) + j0, last = first_position(s) + j1;
    hi = p.causal ? min(last + 1, s.len) : s.len;
    lo = p.window > 0 ? max(first - p.window + 1, 0) : first_token(s);
}

// Key tiles of a row tile (at least one: rows that see nothing are written too).
template <int ROWS, int KEYS, class P, class V>
__device__ __forceinline__ int tile_count(const P& p, const V& s, int rt, int* first = nullptr) {
    int lo, hi;
    if (!p.causal) {
        lo = first_token(s), hi = s.len;
    } else {
        const int last = min((rt + 1) * ROWS, s.n * p.group) - 1;
        seen_range(p, s, p.window > 0 ? rt * ROWS / p.group : 0, last / p.group, lo, hi);
    }
    const int t0 = lo / KEYS;
    if (first) *first = t0;
    return hi <= lo ? 1 : (hi + KEYS - 1) / KEYS - t0;
}

// Whether this launch takes a sequence.
__device__ __forceinline__ bool taken(const AttentionParams& p, const SeqView& s) {
    const int rows = s.n * p.group;
    return rows != 0 && rows >= p.min_rows && rows <= p.max_rows;
}

__device__ __forceinline__ bool taken(const SharedParams& p, const PartView& s) {
    const int rows = s.n * p.group;
    return rows != 0 && rows >= p.min_rows && rows <= p.max_rows && !(p.solo && s.start >= 0 && s.n == 1);
}

// Key tiles and units of a sequence.
template <int ROWS, int KEYS, class P, class V>
__device__ __forceinline__ int2 seq_tiles(const P& p, const V& s) {
    const int rows = s.n * p.group;
    if (!taken(p, s)) return make_int2(0, 0);
    const int tiles = (rows + ROWS - 1) / ROWS, units = tiles * p.kv_heads;
    if (!p.causal) return make_int2(units * tile_count<ROWS, KEYS>(p, s, 0), units);
    int total = 0;
    for (int rt = 0; rt < tiles; ++rt) total += tile_count<ROWS, KEYS>(p, s, rt);
    return make_int2(total * p.kv_heads, units);
}

// Where a CTA's share begins, and how many tiles it counts as: `each`, and one more for
// the first `extra` CTAs.
struct Share {
    int tiles;   // of this CTA
    int seq;     // first sequence of the share
    int offset;  // of the share's first tile in that sequence
    int begin;   // the share's first tile among all
    int each, extra;
    int cost;    // tiles that a unit counts as beside its own

    // CTAs after this one that work on a unit of n tiles whose first is `at` of the share.
    __device__ __forceinline__ int followers(int at, int n) const {
        const int last = begin + at + n - 1, longer = extra * (each + 1);
        return (last < longer ? last / (each + 1) : extra + (last - longer) / each) - (int)blockIdx.x;
    }
};

// All threads of the CTA; scratch: THREADS / 16 + 2 words of shared memory.
// CTAs past the number of tiles get none.  Sequences whose rows overlap can have more
// tiles together than the host's bound, which counts every query token once; where that
// is more than can be numbered, nobody gets any.
template <int ROWS, int KEYS, int COST, int THREADS, class P>
__device__ __forceinline__ Share take_share(const P& p, int* scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = THREADS / 32;
    int* found = scratch + 2 * kWarps;  // sequence, offset
    int2 mine = make_int2(0, 0);
    for (int i = tid; i < p.seqs; i += THREADS) {
        const int2 t = seq_tiles<ROWS, KEYS>(p, seq_view(p, i));
        mine.x = (int)min((unsigned)mine.x + (unsigned)t.x, 0x7fffffffu), mine.y += t.y;
    }
    // (the sum of 32 numbers below 2^31, in two halves, at most 2^31 - 1)
    const unsigned low = __reduce_add_sync(0xffffffffu, (unsigned)mine.x & 0xffffu);
    const unsigned high = __reduce_add_sync(0xffffffffu, (unsigned)mine.x >> 16) + (low >> 16);
    const int tiles = high > 0x7fffu ? 0x7fffffff : (int)(high << 16 | (low & 0xffffu));
    const int units = (int)__reduce_add_sync(0xffffffffu, (unsigned)mine.y);
    if (lane == 0) scratch[2 * warp] = tiles, scratch[2 * warp + 1] = units;
    __syncthreads();
    int64_t all = 0;
    int all_units = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all += scratch[2 * w], all_units += scratch[2 * w + 1];
    int total = all <= 0x7fffffff / (1 + COST) ? (int)all : 0;
    // (A CTA that takes up a unit in its middle pays as well, so with little to do for each
    // a high price would only leave CTAs without work.)
    const int cost = total > (int)gridDim.x ? min(COST, total / (int)gridDim.x) : 0;
    total += cost * all_units;
    const int ctas = min(total, (int)gridDim.x);
    Share s{0, 0, 0, 0, 1, 0, cost};
    if ((int)blockIdx.x >= ctas) return s;
    s.each = total / ctas;
    s.extra = total - s.each * ctas;
    s.begin = (int)blockIdx.x * s.each + min((int)blockIdx.x, s.extra);
    s.tiles = s.each + ((int)blockIdx.x < s.extra ? 1 : 0);
    int before = 0;  // tiles of the sequences before these
    for (int base = 0; base < p.seqs; base += THREADS) {
        const int i = base + tid;
        const int2 its = p.seqs <= THREADS ? mine
                                           : (i < p.seqs ? seq_tiles<ROWS, KEYS>(p, seq_view(p, i)) : make_int2(0, 0));
        const int t = its.x + cost * its.y;
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (p.seqs > THREADS) {  // else the warps' sums are there already
            __syncthreads();
            if (lane == 31) scratch[2 * warp] = incl, scratch[2 * warp + 1] = 0;
            __syncthreads();
        }
        int start = before, round = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int v = scratch[2 * w] + cost * scratch[2 * w + 1];
            if (w < warp) start += v;
            round += v;
        }
        start += incl - t;
        if (s.begin >= start && s.begin < start + t) found[0] = i, found[1] = s.begin - start;
        before += round;
        if (s.begin < before) break;
    }
    __syncthreads();
    s.seq = found[0];
    s.offset = found[1];
    return s;
}

// A position in the walk over the units.
template <class P>
struct Walk {
    int seq, rt, head;
    int tile, tiles;  // next key tile of the unit, and how many it has
    int skip;         // empty ones to pass before it
    int first;        // number of the unit's first key tile in the sequence
    int rank;         // of the sequence among those that the launch takes (the ready kernel sets it)
    typename ViewOf<P>::type view;
};

template <int ROWS, int KEYS, class P>
__device__ __forceinline__ Walk<P> walk_to(const P& p, const Share& s) {
    Walk<P> w;
    w.seq = s.seq;
    w.rank = 0;
    w.view = seq_view(p, s.seq);
    int offset = s.offset;
    w.rt = 0;
    while (true) {
        w.tiles = tile_count<ROWS, KEYS>(p, w.view, w.rt, &w.first);
        const int all = (w.tiles + s.cost) * p.kv_heads;
        if (offset < all) break;
        offset -= all;
        ++w.rt;
    }
    w.head = offset / (w.tiles + s.cost);
    offset -= w.head * (w.tiles + s.cost);
    w.tile = max(offset - s.cost, 0);
    w.skip = max(s.cost - offset, 0);
    return w;
}

// To the next unit's first tile; the caller has passed its empty ones and knows that there is one.
template <int ROWS, int KEYS, class P>
__device__ __forceinline__ void walk_on(const P& p, Walk<P>& w) {
    w.tile = 0;
    if (++w.head < p.kv_heads) return;
    w.head = 0;
    ++w.rt;
    if (w.rt * ROWS >= w.view.n * p.group) {
        w.rt = 0;
        ++w.rank;
        do {
            ++w.seq;
            if (w.seq >= p.seqs) return;
            w.view = seq_view(p, w.seq);
        } while (!taken(p, w.view));
    }
    w.tiles = tile_count<ROWS, KEYS>(p, w.view, w.rt, &w.first);
}

// log(sum exp) of a row from its running maximum (log2 units) and sum.
__device__ __forceinline__ float row_lse(float m2, float sum) {
    return sum > 0.0f ? (m2 - kExpShift) * 0.693147180559945f + logf(sum)
                      : (sum == 0.0f ? __int_as_float(0xff800000) : sum);
}

// What is known of the weights of a row that is whole, with its output.
__device__ __forceinline__ void store_stat(const AttentionParams& p, const SeqView&, int64_t row, int head, float top,
                                           float total) {
    if (p.lse) p.lse[row * p.heads + head] = row_lse(top, total);
}
__device__ __forceinline__ void store_stat(const SharedParams& p, const PartView& view, int64_t row, int head, float top,
                                           float total) {
    p.row_stat[row * p.heads + head] = make_float2(top, total);
    p.where[row * p.heads + head] = make_int4(-1, 0, 0, view.start > 0 ? kHasPrefix : 0);
}
// Where the parts of a row are that this CTA began and `followers` went on with.
__device__ __forceinline__ void store_where(const AttentionParams&, const SeqView&, int64_t, int, int, int) {}
__device__ __forceinline__ void store_where(const SharedParams& p, const PartView& view, int64_t row, int head,
                                            int in_tile, int followers) {
    p.where[row * p.heads + head] =
        make_int4(p.kernel, (int)blockIdx.x, followers, in_tile | (view.start > 0 ? kHasPrefix : 0));
}

// Four consecutive features of an output row.
__device__ __forceinline__ void store4_at(const AttentionParams& p, int64_t at, float4 v) {
    uint16_t h[4];
    if (p.dtype == MXK_F16) {
        h[0] = __half_as_ushort(__float2half_rn(v.x)), h[1] = __half_as_ushort(__float2half_rn(v.y));
        h[2] = __half_as_ushort(__float2half_rn(v.z)), h[3] = __half_as_ushort(__float2half_rn(v.w));
    } else {
        h[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v.x)), h[1] = __bfloat16_as_ushort(__float2bfloat16_rn(v.y));
        h[2] = __bfloat16_as_ushort(__float2bfloat16_rn(v.z)), h[3] = __bfloat16_as_ushort(__float2bfloat16_rn(v.w));
    }
    uint16_t* o = static_cast<uint16_t*>(p.out) + at;
    if (p.out_vec) {
        *reinterpret_cast<uint2*>(o) = make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = h[i];
    }
}

__device__ __forceinline__ void store4_at(const SharedParams& p, int64_t at, float4 v) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v;
}

template <class P>
__device__ __forceinline__ void store4(const P& p, int64_t token, int head, int feature, float4 v) {
    store4_at(p, token * p.out_token + (int64_t)head * p.out_head + feature, v);
}

}  // namespace dev

// The partial sums of one kernel's CTAs: as in AttentionParams.
struct Parts {
    const float* part;
    const float2* stat;
    const int4* open;  // null: a row's parts lie in slots one after the other
    int ctas, rows;    // rows: of its row tiles; without `open`, ctas is the number of slots
    int split;         // CTAs that join a unit
};
constexpr int kMostParts = 4;  // kernels of a call

// Rows per key head up to which attention_rows_kernel is taken, one pass over the keys for every 16
// of them.  In us, it and the tiles kernel, over 16,384 tokens (32 heads of 128 on 8): 32
// rows 39, 45; 48 rows 47, 47; 64 rows 56, 47; 24 sequences with 2 to 5 query tokens of 8
// heads a key head and windows 27, 54.
constexpr int kMostFewRows = 32;
// Rows per key head above which its keys are converted beforehand.  In us, packed and
// ready kernel, over 16,384 tokens (32 heads of 128 on 8): 256 rows 72, 94; 384 rows 84,
// 109; 512 rows 99, 111; 1024 rows (eight passes of the packed one) 121 ready.  (Where the
// two cross above 512 was not measured.)  Among several sequences a lower bound, as the two
// kernels run one after the other and the second has little to do: nine sequences with 4
// to 2804 rows 147 us with 512, 132 with 256.
constexpr int kReadyRows = 512, kReadyRowsMany = 256;
// kReadyRowsMany of calls with prefixes.  In us for 256, 384 and 512, one token a sequence but for the
// drafts, 32 heads of 128 on 8: 80 sequences behind 8192 tokens 78, 73, 73; 128: 89, 89, 98; 96
// behind 32,768 tokens 160, 167, 167; 128: 168, 167, 206; 2 groups of 48 behind 8192 103, 95, 96; 8 of
// 12: 150, 144, 144; 17 sequences of 2 to 5 tokens in 3 groups (24 heads of 64 on 4, 4 bits) 38, 35, 35;
// 34: 61, 49, 49.  (Where too few rows are there, the two launches are made for nothing.)
constexpr int kReadyRowsShared = 384;
struct JoinParams {
    AttentionParams p;
    Parts parts[kMostParts];
    int count;
};

// A row of a joined unit; total: the sum of its weights relative to `top`.
__device__ __forceinline__ void store_joined(const AttentionParams& p, const int4& unit, const dev::SeqView& view, int row, int chunk, float4 v, float top, float total) {
    const int j = row / p.group;
    const int head = unit.z * p.group + (row - j * p.group);
    if (total == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int64_t to = dev::out_row(p, view) + j;
    dev::store4(p, to, head, chunk * 4, v);
    if (chunk == 0) dev::store_stat(p, view, to, head, top, total);
}

// Block (x, y) of a set of parts: the unit that CTA x began and did not finish, some of its
// rows.  Its parts are the beginning (slot 2x + 1) and what the following CTAs did first
// (slots 2j); they add up in a fixed order.  Few parts: every D / 4 threads take a row and
// go through its parts.  Many: the block takes a row, every D / 4 of its threads some of the
// parts, so a unit in hundreds of parts has several loads under way.  One launch joins the
// parts of all of a call's kernels: a launch for each took 5 us more a kernel.
template <int D>
__global__ void __launch_bounds__(128) attention_join_kernel(const JoinParams jp) {
    const AttentionParams& p = jp.p;
    constexpr int kLanes = D / 4;            // threads of a row
    constexpr int kSub = 128 / kLanes;       // rows, or parts, at a time
    constexpr int kFew = 8;
    __shared__ float4 sums[kSub][kLanes];
    __shared__ float stats[4], sub_totals[4];
    int local = blockIdx.x;
    Parts set = jp.parts[0];
#pragma unroll
    for (int i = 1; i < kMostParts; ++i)
        if (i < jp.count && local >= set.ctas * set.split) local -= set.ctas * set.split, set = jp.parts[i];
    const int x = local / set.split, y = local - x * set.split;
    dev::wait_for_previous();
    const int4 unit = set.open[x];
    if (!unit.w) return;
    const dev::SeqView view = dev::seq_view(p, unit.x);
    const int rows = min(view.n * p.group - unit.y * set.rows, set.rows);
    const int tid = threadIdx.x, chunk = tid % kLanes, sub = tid / kLanes, parts = unit.w + 1;
    auto slot = [&](int i) -> int64_t { return 2 * (int64_t)(x + i) + (i == 0 ? 1 : 0); };
    if (parts <= kFew) {
        for (int r = y * kSub + sub; r < rows; r += set.split * kSub) {
            float2 st[kFew];
            float4 v_part[kFew];
#pragma unroll
            for (int i = 0; i < kFew; ++i)
                if (i < parts) {
                    st[i] = set.stat[slot(i) * set.rows + r];
                    v_part[i] = reinterpret_cast<const float4*>(set.part + (slot(i) * set.rows + r) * D)[chunk];
                }
            float top = st[0].x;
#pragma unroll
            for (int i = 1; i < kFew; ++i)
                if (i < parts) top = fmaxf(top, st[i].x);
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < kFew; ++i)
                if (i < parts) {
                    st[i].y *= st[i].x == top ? 1.0f : dev::ex2(st[i].x - top);
                    total += st[i].y;
                }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < kFew; ++i)
                if (i < parts) {
                    const float f = st[i].y * inv;
                    v.x += v_part[i].x * f, v.y += v_part[i].y * f, v.z += v_part[i].z * f, v.w += v_part[i].w * f;
                }
            store_joined(p, unit, view, unit.y * set.rows + r, chunk, v, top, total);
        }
        return;
    }
    for (int r = y; r < rows; r += set.split) {
        // the common maximum
        float top = __int_as_float(0xff800000);
        for (int i = tid; i < parts; i += 128) top = fmaxf(top, set.stat[slot(i) * set.rows + r].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((tid & 31) == 0) stats[tid >> 5] = top;
        __syncthreads();
        top = fmaxf(fmaxf(stats[0], stats[1]), fmaxf(stats[2], stats[3]));
        // the sum of the weights
        float total = 0.0f;
        for (int i = tid; i < parts; i += 128) {
            const float2 st = set.stat[slot(i) * set.rows + r];
            total += st.y * (st.x == top ? 1.0f : dev::ex2(st.x - top));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if ((tid & 31) == 0) sub_totals[tid >> 5] = total;
        __syncthreads();
        total = (sub_totals[0] + sub_totals[1]) + (sub_totals[2] + sub_totals[3]);
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int i = sub; i < parts; i += kSub) {
            const float2 st = set.stat[slot(i) * set.rows + r];
            const float4 o = reinterpret_cast<const float4*>(set.part + (slot(i) * set.rows + r) * D)[chunk];
            const float f = st.y * (st.x == top ? 1.0f : dev::ex2(st.x - top)) * inv;
            v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
        }
        sums[sub][chunk] = v;
        __syncthreads();
        if (tid < kLanes) {
            v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < kSub; ++i) {
                const float4 o = sums[i][chunk];
                v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
            }
            store_joined(p, unit, view, unit.y * set.rows + r, chunk, v, top, total);
        }
        __syncthreads();  // before the shared sums are written again
    }
}

// The launches of one call and the memory of their partial sums, which goes back to the
// pool, in stream order, at its end.  Kernels for sequences of different sizes write
// different outputs, so each is launched as soon as the one before has started everywhere;
// every one ends only when its predecessor has, so the join, launched last, finds all done.
template <class P>
class AttentionCall {
public:
    explicit AttentionCall(cudaStream_t s) : stream_(s) {}
    ~AttentionCall() {
        for (int i = 0; i < blocks_; ++i) cudaFreeAsync(block_[i], stream_);
    }
    AttentionCall(const AttentionCall&) = delete;
    AttentionCall& operator=(const AttentionCall&) = delete;

    // Partial sums of `ctas` CTAs with tiles of `rows` rows, and extra_bytes more at *extra
    // (256-byte aligned).
    int take(P& p, int64_t ctas, int rows, int d, int64_t extra_bytes = 0, void** extra = nullptr) {
        const size_t part = (size_t)(2 * ctas * rows) * d * 4, stat = (size_t)(2 * ctas * rows) * 8;
        const size_t own = (part + stat + (size_t)ctas * 16 + 255) / 256 * 256;
        cudaMemPool_t pool = workspace_pool();
        if (!pool) return fail(MXK_ERR_CUDA, "cache_attention: cannot create the workspace pool");
        void* ptr = nullptr;
        MXK_CUDA(cudaMallocFromPoolAsync(&ptr, own + (size_t)extra_bytes, pool, stream_));
        block_[blocks_++] = ptr;
        if (extra) *extra = static_cast<char*>(ptr) + own;
        number(p, join_.count);
        p.part = static_cast<float*>(ptr);
        p.part_stat = reinterpret_cast<float2*>(static_cast<char*>(ptr) + part);
        p.part_open = reinterpret_cast<int4*>(static_cast<char*>(ptr) + part + stat);
        return MXK_OK;
    }

    // Partial sums that lie one after the other: `slots` of them with `rows` rows each.
    int take_slots(P& p, int64_t slots, int rows, int d) {
        void* ptr = nullptr;
        const size_t part = (size_t)(slots * rows) * d * 4;
        MXK_CHECK(room(part + (size_t)(slots * rows) * 8, &ptr));
        number(p, join_.count);
        p.part = static_cast<float*>(ptr);
        p.part_stat = reinterpret_cast<float2*>(static_cast<char*>(ptr) + part);
        return MXK_OK;
    }
    void slots_later(const P& p, int64_t slots, int rows) {
        join_.parts[join_.count++] = Parts{p.part, p.part_stat, nullptr, (int)slots, rows, 0};
    }

    // Room for something else of the call.
    int room(size_t bytes, void** ptr) {
        cudaMemPool_t pool = workspace_pool();
        if (!pool) return fail(MXK_ERR_CUDA, "cache_attention: cannot create the workspace pool");
        MXK_CUDA(cudaMallocFromPoolAsync(ptr, bytes, pool, stream_));
        block_[blocks_++] = *ptr;
        return MXK_OK;
    }

    template <class K, class... Args>
    int launch(const char* name, K kernel, unsigned ctas, unsigned threads, size_t smem, const Args&... args) {
        return launch(name, kernel, dim3(ctas), threads, smem, args...);
    }
    template <class K, class... Args>
    int launch(const char* name, K kernel, dim3 grid, unsigned threads, size_t smem, const Args&... args) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream_;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = first_ ? 0 : 1;  // the call's first kernel waits for all that the stream held before
        first_ = false;
        LaunchScope scope(name, stream_);
        MXK_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
        return MXK_OK;
    }

    // Joins the parts of a kernel's CTAs, `split` blocks to a unit, when all are launched.
    void join_later(const P& p, int64_t ctas, int rows, int64_t split) {
        join_.p = p;
        join_.parts[join_.count++] = Parts{p.part, p.part_stat, p.part_open, (int)ctas, rows, (int)split};
    }
    const Parts* parts() const { return join_.parts; }
    int join_all(int d) {
        if (!join_.count) return MXK_OK;
        int64_t blocks = 0;
        for (int i = 0; i < join_.count; ++i) blocks += (int64_t)join_.parts[i].ctas * join_.parts[i].split;
        return launch("attention_join", d == 128 ? attention_join_kernel<128> : attention_join_kernel<64>,
                      (unsigned)blocks, 128, 0, join_);
    }

private:
    static void number(AttentionParams&, int) {}
    static void number(SharedParams& p, int kernel) { p.kernel = kernel; }
    cudaStream_t stream_;
    bool first_ = true;
    void* block_[kMostParts + 1] = {};
    JoinParams join_{};
    int blocks_ = 0;
};

// attention_tiles.cu: many query rows per key head (max_rows: of query tokens that a part of a
// call with prefixes can have).
template <class P>
int launch_attention_tiles(int bits, int head_dim, P p, int max_q, int max_rows, AttentionCall<P>& call);

// attention.cu: few query rows, and all of a call's kernels but the join; max_rows as above.
template <class P>
int launch_attention(const mxk_cache& cache, P p, int max_rows, AttentionCall<P>& call);

// attention_solo.cu: parts of single tokens.
int launch_attention_solo(int bits, int head_dim, SharedParams p, int64_t slots, AttentionCall<SharedParams>& call);

// Checks of a call's arguments, and the kernels' parameters; p.tokens = 0: nothing to do.
int check_attention(const char* who, const mxk_cache* cache, const mxk_attention* a, AttentionParams& p);

}  // namespace mxk
