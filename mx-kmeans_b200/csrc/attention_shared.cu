// Attention of a batch whose sequences share prefixes (no counterpart in the reference).
//
// The softmax over a sequence's tokens falls into that over the prefix, which all rows of a
// group see whole, and that over the rest: with their means o1, o2 and log-sums l1, l2 and
// m = max(l1, l2),
//     out = (e^(l1 - m) o1 + e^(l2 - m) o2) / (e^(l1 - m) + e^(l2 - m)).
// So a group's prefix is attended over once by the rows of all its sequences together, as one
// sequence of that many query tokens, and only the rest sequence by sequence.  Both are units
// of the same division of work in the same kernels (attention.cu, attention_tiles.cu), which
// take a prefix with few rows or many as they take a sequence's.  Prefixes are cut to whole key
// tiles of 128 tokens: a sequence's own part begins with a tile then, and no tile is partly
// seen by a prefix's rows.
//
//   attention_parts_kernel   lengths to parts, on the device: graphs replay as they grow
//   attention_solo_kernel    what sequences with one query token have behind the prefix (attention_solo.cu)
//   the attention kernels    everything else; rows in float32 with their maxima and sums, whole or in parts, prefixes'
//                            and own, and where they are
//   attention_merge_kernel   everything there is of a row, by the formula above
//
// With many rows the products bound it; short calls are a chain of launches and dependent loads.
// Measured at 32 heads of 128 on 8, 8 bits: 64 sequences with 1 to 512 own tokens behind 8192 60 us (each
// by itself 244), of which the prefix 35, the own tokens 10 behind it and the merge 5; 256 with 10 to
// 300 behind 32,768 225 us (each by itself 3335): 137 GFLOP in 150 us, tiles converted before in 40, own
// tokens in 30.
#include <algorithm>
#include <limits>

#include "attention.cuh"

namespace mxk {
namespace {

constexpr int kTile = 128;  // tokens that prefixes are multiples of: a key tile
// Rows (query tokens times heads) up to which a block of the merge takes one row, its four warps
// the parts of it, instead of a warp a row.  In us with one row and with four: 4 sequences of 32 heads
// behind 1024 tokens 17.5, 19.7, 16 behind 8192 43, 49, 64 60.6, 61.6, 256 134, 133.
constexpr int64_t kFewRows = 2048;
// Sequences times key heads from which on single tokens' parts go to attention_solo_kernel: fewer are
// done sooner by four warps each, and the prefix's few rows by attention_rows_kernel beside them.  In
// us with it and without, on 8 key heads: 4 sequences 28.6, 17.5, 8 38.3, 27.8, 16 42.9, 43.0, 32 45, 51, 64 60,
// 70, 256 132, 170.
constexpr int kManyParts = 128;
// Chunks of single tokens' parts that a warp is to have.  In us for 1, 2, 3 and 4 (before, with one and
// no counter): 256 sequences with 10 to 300 own tokens 232, 225, 224, 224 (229), 128 with 1 to 2000
// 159, 134, 134, 134 (142), 40 with 1 to 8000 156, 122, 126, 126 (141), 512 with 1 to 1000 265, 258, 249, 246
// (281), 64 with 1 to 512 60, 60, 60, 60 (61).  More take more memory.
constexpr int kSoloShares = 2;

// What a call has to save to share, in passes over a token of 128 features by a key head that wait
// for its bytes (some 45 ps each).  A prefix's rows take one kernel's CTAs for themselves, the parts, single
// tokens and the merge have kernels of their own (5 to 30 us), and every row is written twice in float32
// and read again by the merge.  In us, each sequence by itself and shared, 32 heads of 128 on 8, 8 bits:
//   up to 32 rows a prefix: 2 sequences of one token behind 16,384 (128 K saved) 28.7, 33.1, behind 32,768 (256 K)
//     43, 39; 4 behind 4096 (96 K) 21.7, 22.7; 8 behind 4096 (192 K) 28.9, 25.0
//   more: 16 of one token behind 1024 (120 K) 22, 33, behind 4096 (480 K) 43, 37; 64 behind 512 (248 K) 41, 40,
//     behind 1024 (496 K) 54, 40
//   of which the rows' way takes 1638 K: 64 with 32 tokens behind 1024 (1000 K) 154, 193, behind 4096 (4000 K) 340,
//     277; 16 with 128 behind 1024 (360 K) 126, 150, behind 4096 (1440 K) 258, 246
//   6554 K: 64 with 128 behind 1024 (1512 K) 360, 517, behind 4096 (6048 K) 869, 884; 4 with 2048 behind 4096
//     (288 K) 684, 897
// Over 1437 sizes (1 to 16 key heads, 2 to 128 sequences of 1 to 2048 tokens in 1 to 4 groups, 4 to 8 bits, prefixes
// of 256 to 32,768) 24 calls took over 5 % longer than the ordinary one, most of them of single tokens and one
// or two key heads (up to 1.75 of it), whose prefixes come in a hundred parts; 415 were faster, at 0.57 of it.
constexpr int64_t kWorthFew = 160 << 10, kWorth = 300 << 10, kWorthReady = 50 << 10;
constexpr int kWayCost = 5;  // elements of rows whose way takes as long as such a pass
// A pass of 128 rows of a sequence by the tiles kernel, of a prefix, whose tiles all CTAs share, and keys that are
// converted beforehand.
constexpr double kTilePass = 2.0, kPrefixPass = 1.0, kReadyPass = 3.0;
// Sequences that fill a row tile by themselves multiply as many tiles together as apart, unless there
// are rows for several of the ready kernel's: 4 with 32 tokens (512 rows) behind 16,384 94, 110; 8 (1024)
// 166, 138; 8 with 16 (64 rows each) 159, 109.
constexpr int64_t kFullRows = 96, kEnoughRows = 1024;

struct PartsParams {
    const int* cu_q;
    const int* kv_lens;
    const int* cu_groups;
    const int* prefix_lens;
    int4* parts;
    int4* where;  // the sequences' side
    int64_t rows;
    int tokens, seqs, groups, max_q, max_kv, max_prefix;
    int4* solo;  // as SharedParams
    int* solo_count;
    int solo_warps;  // a key head's work is cut into about as many chunks
    int solo_most;   // entries of the list
};

// Block 0: the sequences' parts, a thread each, then the groups', a warp each.  The others: no row
// is anywhere yet (a row behind the last sequence stays so).
constexpr int kClear = 4096;  // rows of a block: four a thread
constexpr int kPartsThreads = 1024;
__global__ void __launch_bounds__(kPartsThreads) attention_parts_kernel(const PartsParams p) {
    if (blockIdx.x > 0) {
        const int64_t first = (int64_t)(blockIdx.x - 1) * kClear, end = min(first + kClear, p.rows);
        for (int64_t i = first + threadIdx.x; i < end; i += blockDim.x) p.where[i] = make_int4(-2, 0, 0, 0);
        return;
    }
    AttentionParams a{};  // (for seq_view)
    a.cu_q = p.cu_q, a.kv_lens = p.kv_lens, a.tokens = p.tokens, a.max_q = p.max_q, a.max_kv = p.max_kv;
    // (of the first sequences, which are mostly all, what comes below is not read back)
    __shared__ int starts[kPartsThreads];
    dev::SeqView first_view{};
    starts[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < p.seqs; i += kPartsThreads) {
        const dev::SeqView s = dev::seq_view(a, i);
        if (i < kPartsThreads) first_view = s;
        p.parts[2 * (p.groups + i)] = make_int4(s.row0, s.n, s.len, s.len - s.n);
        p.parts[2 * (p.groups + i) + 1] = make_int4(0, i, 0, 0);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < p.groups; g += blockDim.x >> 5) {
        const int first = min(max(__ldg(p.cu_groups + g), 0), p.seqs), end = min(max(__ldg(p.cu_groups + g + 1), first), p.seqs);
        // The prefix ends before any of the group's query tokens.  (Sequences without any do
        // not count.)
        int least = 0x7fffffff, count = 0, lead = 0x7fffffff, row0 = 0x7fffffff, row_end = 0;
        for (int i = first + lane; i < end; i += 32) {
            const dev::SeqView s = dev::seq_view(a, i);
            if (s.n <= 0) continue;
            least = min(least, s.len - s.n), lead = min(lead, i), ++count;
            row0 = min(row0, s.row0), row_end = max(row_end, s.row0 + s.n);
        }
        least = __reduce_min_sync(0xffffffffu, least), lead = __reduce_min_sync(0xffffffffu, lead);
        count = __reduce_add_sync(0xffffffffu, count);
        row0 = __reduce_min_sync(0xffffffffu, row0), row_end = __reduce_max_sync(0xffffffffu, row_end);
        const int prefix = count < 2 ? 0 : max(min(min(least, __ldg(p.prefix_lens + g)), p.max_prefix), 0) / kTile * kTile;
        if (lane == 0) {
            p.parts[2 * g] = make_int4(prefix ? row0 : 0, prefix ? row_end - row0 : 0, prefix, prefix);
            p.parts[2 * g + 1] = make_int4(-1, prefix ? lead : 0, 0, 0);
        }
        for (int i = first + lane; i < end && prefix; i += 32) {
            p.parts[2 * (p.groups + i) + 1].x = prefix;
            if (i < kPartsThreads) starts[i] = prefix;
        }
    }
    if (!p.solo) return;
    // The chunks of single tokens' parts: as long that there are as many as warps, in multiples of a
    // key tile, and at least one a part.  As a part in several chunks is longer than one, and
    // solo_warps chunks are longer than everything, such parts have at most 2 solo_warps chunks.
    __shared__ uint64_t sums[32];
    const int warp = threadIdx.x >> 5;
    __syncthreads();
    auto tokens_of = [&](int i, int& row, int& start, int& end) -> int {  // behind the prefix; -1: no such part
        if (i >= p.seqs) return -1;
        if (i < kPartsThreads) {
            row = first_view.row0, start = starts[i], end = first_view.len;
            return first_view.n == 1 ? max(end - start, 0) : -1;
        }
        const int4 view = p.parts[2 * (p.groups + i)];
        row = view.x, start = p.parts[2 * (p.groups + i) + 1].x, end = view.z;
        return view.y == 1 ? max(end - start, 0) : -1;
    };
    // Of the block's threads: the sum of x, and that of the threads up to this one.
    auto scan = [&](uint64_t x, uint64_t& all) -> uint64_t {
        uint64_t incl = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        uint64_t warps = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t v = __shfl_up_sync(0xffffffffu, warps, o);
            if (lane >= o) warps += v;
        }
        all = __shfl_sync(0xffffffffu, warps, 31);
        return incl + (warp ? __shfl_sync(0xffffffffu, warps, warp - 1) : 0);
    };
    int row, start, end;
    uint64_t mine = 0, all;
    for (int i = threadIdx.x; i < p.seqs; i += kPartsThreads) mine += max(tokens_of(i, row, start, end), 0);
    scan(mine, all);
    // (From a cu_q that does not ascend there can be more than fits; nothing is longer than that.)
    constexpr uint64_t kMost = 0x7fffffff / kTile * kTile - kTile;
    const int chunk = (int)((min(all / p.solo_warps, kMost) + kTile) / kTile * kTile);
    uint64_t before = 0;  // chunks so far, and from bit 32 on those of parts that have several
    for (int base = 0; base < p.seqs; base += kPartsThreads) {
        const int i = base + threadIdx.x, tokens = tokens_of(i, row, start, end);
        const int chunks = tokens < 0 ? 0 : max(tokens / chunk + (tokens % chunk != 0), 1);
        const uint64_t own = (uint64_t)chunks | (uint64_t)(chunks > 1 ? chunks : 0) << 32;
        const uint64_t at = before + scan(own, all) - own;
        before += all;
        // (More sequences of one token than tokens, from a cu_q that does not ascend: not followed.)
        for (int k = 0; k < chunks && (int)at + k < p.solo_most; ++k) {
            int4* to = p.solo + 2 * ((int)at + k);
            const int from = start + k * chunk;
            to[0] = make_int4(i, row, from, from + min(end - from, chunk));
            to[1] = make_int4(k, chunks, start, (int)(at >> 32));
        }
    }
    if (threadIdx.x == 0) p.solo_count[0] = min((int)before, p.solo_most), p.solo_count[1] = 0;
}

struct MergeParams {
    AttentionParams p;    // the caller's queries and outputs
    const float* rows;    // [2][tokens][heads][D]
    const float2* stat;   // [2][tokens][heads]
    const int4* where;    // [2][tokens][heads]
    Parts parts[kMostParts];
};

// What there is of a row: means, maxima and sums from one slot of the workspace to the next.
template <int D>
struct Found {
    const float* mean;
    const float2* stat;
    int count, rows;  // rows: of a slot; 0: the row is whole
    bool pairs = false;  // a CTA has two slots
    __device__ __forceinline__ Found(const MergeParams& m, const int4& w, int64_t at) {
        // (What a wait that gave up left unwritten is not followed out of the workspace.)
        const Parts& set = m.parts[min(max(w.x, 0), kMostParts - 1)];
        if (w.x < 0 || !set.part) {
            mean = m.rows + at * D, stat = m.stat + at, count = w.x == -2 ? 0 : 1, rows = 0;
        } else {
            const int x = min(max(w.y, 0), set.ctas - 1), r = min(w.w & (kHasPrefix - 1), set.rows - 1);
            const int64_t at = (int64_t)(set.open ? 2 * x : x) * set.rows + r;
            mean = set.part + at * D, stat = set.stat + at;
            count = min(max(w.z, 0), set.ctas - 1 - x) + 1, rows = set.rows, pairs = set.open != nullptr;
        }
    }
    // Its i-th part: the beginning in the second slot of its CTA, the others in the first of theirs, or
    // one after the other.
    __device__ __forceinline__ int64_t slot(int i) const { return (int64_t)(pairs ? 2 * i + (i == 0 ? 1 : 0) : i) * rows; }
};

// A row of the output, by SPLIT warps, every D / 4 threads of which take some of its parts.  They
// add up in a fixed order.
template <int D, int SPLIT>
__global__ void __launch_bounds__(128) attention_merge_kernel(const MergeParams m) {
    const AttentionParams& p = m.p;
    constexpr int kLanes = D / 4, kSub = 32 * SPLIT / kLanes, kAtOnce = 4 / SPLIT;  // parts, rows at a time
    __shared__ float4 sums[kAtOnce][kSub][kLanes];
    const int tid = threadIdx.x % (32 * SPLIT), lane = threadIdx.x & 31, chunk = tid % kLanes, sub = tid / kLanes;
    const int64_t all = p.tokens * p.heads, row = (int64_t)blockIdx.x * kAtOnce + threadIdx.x / (32 * SPLIT);
    dev::wait_for_previous();
    if (row >= all) return;
    const int4 at_own = m.where[all + row], at_prefix = m.where[row];
    if (at_own.x == -2) return;
    const Found<D> own(m, at_own, all + row);
    Found<D> prefix(m, at_prefix, row);
    if (!(at_own.w & kHasPrefix)) prefix.count = 0;
    const int count = prefix.count + own.count;
    auto stat_of = [&](int i) -> float2 {
        return i < prefix.count ? prefix.stat[prefix.slot(i)] : own.stat[own.slot(i - prefix.count)];
    };
    // the common maximum and the sum of the weights (every warp, all parts)
    const float neg_inf = __int_as_float(0xff800000);
    const float2 mine = lane < count ? stat_of(lane) : make_float2(neg_inf, 0.0f);
    float top = mine.x;
    for (int i = lane + 32; i < count; i += 32) top = fmaxf(top, stat_of(i).x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    auto weight = [&](float2 st) { return st.y * (st.x == top ? 1.0f : dev::ex2(st.x - top)); };
    const float first = weight(mine);
    float total = first;
    for (int i = lane + 32; i < count; i += 32) total += weight(stat_of(i));
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int base = 0; base < count; base += kSub) {
        const int i = base + sub;
        float f = __shfl_sync(0xffffffffu, first, i & 31);
        if (i >= count) f = 0.0f;
        if (i >= 32 && i < count) f = weight(stat_of(i));
        if (f == 0.0f) continue;  // a part that weighs nothing has no say, whatever it holds
        const float* at = i < prefix.count ? prefix.mean + prefix.slot(i) * D : own.mean + own.slot(i - prefix.count) * D;
        const float4 o = reinterpret_cast<const float4*>(at)[chunk];
        f *= inv;
        v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
    }
    if (kSub > 1) {
        float4 (*all_sums)[kLanes] = sums[threadIdx.x / (32 * SPLIT)];
        all_sums[sub][chunk] = v;
        if (SPLIT == 1)
            __syncwarp();
        else
            __syncthreads();
        if (sub > 0) return;
#pragma unroll
        for (int i = 1; i < kSub; ++i) {
            const float4 o = all_sums[i][chunk];
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
    }
    const int token = (int)(row / p.heads), head = (int)(row - (int64_t)token * p.heads);
    dev::store4(p, token, head, chunk * 4, v);
    if (p.lse && chunk == 0) p.lse[row] = dev::row_lse(top, total);
}

// Whether the call shares anything, by what the host knows.
bool worth_sharing(const AttentionParams& p, int groups, int64_t max_prefix, int head_dim) {
    const int64_t seqs = std::min<int64_t>(p.seqs, p.tokens);  // that can have query tokens
    if (groups == 0 || seqs <= groups || max_prefix == 0) return false;
    const int64_t rows = p.tokens * p.group, each = rows / seqs, together = rows / groups;
    if (each >= kFullRows && rows < kEnoughRows) return false;
    const double width = head_dim / 128.0;
    auto passes = [&](int64_t rows, int most_tiles, double tile) -> double {
        if (rows <= kMostFewRows) return (double)((rows + 15) / 16) * width;  // of attention_rows_kernel
        return rows <= most_tiles ? (double)((rows + 127) / 128) * tile : kReadyPass * width;
    };
    const double saved = seqs * passes(each, kReadyRowsMany, kTilePass) - groups * passes(together, kReadyRowsShared, kPrefixPass);
    const int64_t worth = together <= kMostFewRows ? kWorthFew : (each > kReadyRowsMany ? kWorthReady : kWorth);
    return saved * max_prefix * p.kv_heads >= worth + (double)(p.tokens * p.heads * head_dim) / kWayCost;
}

}  // namespace
}  // namespace mxk

extern "C" int mxk_cache_attention_shared(const mxk_cache* cache, const mxk_attention* args, const mxk_prefixes* prefixes,
                                          void* stream) {
    using namespace mxk;
    AttentionParams p{};
    MXK_CHECK(check_attention("cache_attention_shared", cache, args, p));
    MXK_REQUIRE(prefixes, "cache_attention_shared: prefixes is null");
    MXK_REQUIRE(args->window == 0, "cache_attention_shared: there may be no window");
    MXK_REQUIRE(prefixes->groups >= 0 && prefixes->groups <= std::numeric_limits<int>::max() / 4 && args->seqs <= std::numeric_limits<int>::max() / 4,
                "cache_attention_shared: groups must not be negative, groups and seqs at most 2^29");
    MXK_REQUIRE(prefixes->max_prefix >= 0, "cache_attention_shared: max_prefix must not be negative");
    MXK_REQUIRE(args->tokens * args->heads <= std::numeric_limits<int>::max() / 2,
                "cache_attention_shared: tokens * heads must be below 2^30");
    if (p.tokens == 0) return MXK_OK;
    MXK_REQUIRE(prefixes->groups == 0 || (prefixes->cu_groups && prefixes->prefix_lens),
                "cache_attention_shared: cu_groups and prefix_lens must be non-null");
    MXK_REQUIRE((reinterpret_cast<uintptr_t>(prefixes->cu_groups) | reinterpret_cast<uintptr_t>(prefixes->prefix_lens)) % 4 == 0,
                "cache_attention_shared: pointers must be aligned to their elements");
    const int64_t max_prefix = std::min<int64_t>(prefixes->max_prefix, p.max_kv) / kTile * kTile;
    if (!worth_sharing(p, prefixes->groups, max_prefix, cache->head_dim)) {
        AttentionCall<AttentionParams> call(as_stream(stream));
        MXK_CHECK(launch_attention(*cache, p, 0, call));
        return call.join_all(cache->head_dim);
    }

    AttentionCall<SharedParams> call(as_stream(stream));
    const int64_t rows = p.tokens * p.heads, parts = (int64_t)prefixes->groups + p.seqs;
    const size_t out_bytes = (size_t)rows * 2 * cache->head_dim * 4;
    void* room = nullptr;
    // Parts of one token are cut into about as many chunks as there are warps for them, key heads counted.
    static const int solo_warps = 12 * sm_count();
    const int64_t per_head = std::max(kSoloShares * solo_warps / p.kv_heads, 1), most = std::min<int64_t>(p.seqs, p.tokens);
    const bool solo = cache->bits != 6 && p.group <= kSoloRows && (int64_t)p.seqs * p.kv_heads >= kManyParts &&
                      most * p.max_kv / per_head < std::numeric_limits<int>::max() - 2 * kTile;
    const int64_t chunks = solo ? per_head + most + 1 : 0;
    MXK_CHECK(call.room(out_bytes + (size_t)rows * 48 + (size_t)(parts + chunks) * 32 + 16, &room));
    SharedParams s;
    static_cast<AttentionParams&>(s) = p;
    s.out = room;
    int4* list = reinterpret_cast<int4*>(static_cast<char*>(room) + out_bytes);
    s.parts = list;
    int4* solo_list = list + 2 * parts;
    int* solo_count = reinterpret_cast<int*>(solo_list + 2 * chunks);
    s.solo = solo ? solo_list : nullptr, s.solo_count = solo_count;
    s.where = solo_list + 2 * chunks + 1;
    s.row_stat = reinterpret_cast<float2*>(s.where + 2 * rows);
    s.out_token = (int64_t)p.heads * cache->head_dim, s.out_head = cache->head_dim;
    s.groups = prefixes->groups, s.max_prefix = (int)max_prefix;
    s.seqs = (int)parts;
    const PartsParams pp{p.cu_q, p.kv_lens, prefixes->cu_groups, prefixes->prefix_lens, list, s.where + rows, rows,
                         (int)p.tokens, p.seqs, s.groups, p.max_q, p.max_kv, s.max_prefix,
                         solo ? solo_list : nullptr, solo_count, (int)per_head, (int)chunks};
    {
        LaunchScope scope("attention_parts", as_stream(stream));
        attention_parts_kernel<<<(unsigned)(1 + (rows + kClear - 1) / kClear), kPartsThreads, 0, as_stream(stream)>>>(pp);
        MXK_CUDA(cudaGetLastError());
    }
    MXK_CHECK(launch_attention(*cache, s, (int)p.tokens, call));
    if (solo) MXK_CHECK(launch_attention_solo(cache->bits, cache->head_dim, s, 2 * per_head * p.kv_heads, call));
    MergeParams m{p, static_cast<const float*>(room), s.row_stat, s.where, {}};
    std::copy(call.parts(), call.parts() + kMostParts, m.parts);
    // With few rows all four warps of a block take parts of one, else one each.
    const bool few = rows <= kFewRows;
    const int at_once = few ? 1 : 4;
    return call.launch("attention_merge",
                       cache->head_dim == 128 ? (few ? attention_merge_kernel<128, 4> : attention_merge_kernel<128, 1>)
                                              : (few ? attention_merge_kernel<64, 4> : attention_merge_kernel<64, 1>),
                       (unsigned)((rows + at_once - 1) / at_once), 128, 0, m);
}
