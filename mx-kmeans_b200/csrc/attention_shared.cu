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
//   the attention kernels    rows in float32 with their log-sums, prefixes' and own
//   attention_merge_kernel   the formula above, a row by D / 4 threads
#include <limits>

#include "attention.cuh"

namespace mxk {
namespace {

constexpr int kTile = 128;  // tokens that prefixes are multiples of: a key tile

struct PartsParams {
    const int* cu_q;
    const int* kv_lens;
    const int* cu_groups;
    const int* prefix_lens;
    int4* parts;
    int tokens, seqs, groups, max_q, max_kv, max_prefix;
};

// One block: the sequences' parts, a thread each, then the groups', a warp each.
__global__ void __launch_bounds__(1024) attention_parts_kernel(const PartsParams p) {
    AttentionParams a{};  // (for seq_view)
    a.cu_q = p.cu_q, a.kv_lens = p.kv_lens, a.tokens = p.tokens, a.max_q = p.max_q, a.max_kv = p.max_kv;
    for (int i = threadIdx.x; i < p.seqs; i += blockDim.x) {
        const dev::SeqView s = dev::seq_view(a, i);
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
        for (int i = first + lane; i < end && prefix; i += 32) p.parts[2 * (p.groups + i) + 1].x = prefix;
    }
}

struct MergeParams {
    AttentionParams p;  // the caller's queries and outputs
    const float* rows;  // [2][tokens][heads][D]
    const float* lse;   // [2][tokens][heads]
    const int4* parts;
    int groups;
};

template <int D>
__global__ void __launch_bounds__(128) attention_merge_kernel(const MergeParams m) {
    const AttentionParams& p = m.p;
    constexpr int kLanes = D / 4;
    const int64_t all = p.tokens * p.heads, row = (int64_t)blockIdx.x * (128 / kLanes) + threadIdx.x / kLanes;
    if (row >= all) return;
    const int chunk = threadIdx.x % kLanes, token = (int)(row / p.heads), head = (int)(row - (int64_t)token * p.heads);
    // the token's sequence: the last that begins at it or before
    int seq = -1, after = p.seqs;
    while (after - seq > 1) {
        const int mid = (seq + after) / 2;
        (__ldg(p.cu_q + mid) <= token ? seq : after) = mid;
    }
    if (seq < 0) return;
    const int first = max(__ldg(p.cu_q + seq), 0);
    if (token >= __ldg(p.cu_q + seq + 1) || token - first >= p.max_q) return;
    dev::wait_for_previous();
    float4 v = reinterpret_cast<const float4*>(m.rows + (all + row) * D)[chunk];
    float lse = m.lse[all + row];
    if (m.parts[2 * (m.groups + seq) + 1].x > 0) {
        const float4 u = reinterpret_cast<const float4*>(m.rows + row * D)[chunk];
        const float other = m.lse[row], top = fmaxf(lse, other);
        if (top > __int_as_float(0xff800000)) {
            const float f = expf(lse - top), g = expf(other - top), sum = f + g, inv = 1.0f / sum;
            // (a part that weighs nothing has no say, whatever it holds)
            const float a = f * inv, b = g * inv;
            v.x = (a == 0.0f ? 0.0f : a * v.x) + (b == 0.0f ? 0.0f : b * u.x);
            v.y = (a == 0.0f ? 0.0f : a * v.y) + (b == 0.0f ? 0.0f : b * u.y);
            v.z = (a == 0.0f ? 0.0f : a * v.z) + (b == 0.0f ? 0.0f : b * u.z);
            v.w = (a == 0.0f ? 0.0f : a * v.w) + (b == 0.0f ? 0.0f : b * u.w);
            lse = top + logf(sum);
        } else if (other != other || lse != lse) {
            lse = other + lse;
            v = make_float4(lse, lse, lse, lse);
        }
    }
    dev::store4(p, token, head, chunk * 4, v);
    if (p.lse && chunk == 0) p.lse[row] = lse;
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
    if (prefixes->groups == 0 || p.seqs < 2 || max_prefix == 0) {  // nothing to share
        AttentionCall<AttentionParams> call(as_stream(stream));
        return launch_attention(*cache, p, 0, call);
    }

    AttentionCall<SharedParams> call(as_stream(stream));
    const int64_t rows = p.tokens * p.heads, parts = (int64_t)prefixes->groups + p.seqs;
    const size_t out_bytes = (size_t)rows * 2 * cache->head_dim * 4, lse_bytes = ((size_t)rows * 8 + 15) / 16 * 16;
    void* room = nullptr;
    MXK_CHECK(call.room(out_bytes + lse_bytes + (size_t)parts * 32, &room));
    SharedParams s;
    static_cast<AttentionParams&>(s) = p;
    s.out = room;
    s.lse = reinterpret_cast<float*>(static_cast<char*>(room) + out_bytes);
    int4* list = reinterpret_cast<int4*>(static_cast<char*>(room) + out_bytes + lse_bytes);
    s.parts = list;
    s.out_token = (int64_t)p.heads * cache->head_dim, s.out_head = cache->head_dim;
    s.groups = prefixes->groups, s.max_prefix = (int)max_prefix;
    s.seqs = (int)parts;
    const PartsParams pp{p.cu_q, p.kv_lens, prefixes->cu_groups, prefixes->prefix_lens, list,
                         (int)p.tokens, p.seqs, s.groups, p.max_q, p.max_kv, s.max_prefix};
    {
        LaunchScope scope("attention_parts", as_stream(stream));
        attention_parts_kernel<<<1, 1024, 0, as_stream(stream)>>>(pp);
        MXK_CUDA(cudaGetLastError());
    }
    MXK_CHECK(launch_attention(*cache, s, (int)p.tokens, call));
    const int at_once = 128 / (cache->head_dim / 4);
    const MergeParams m{p, static_cast<const float*>(room), s.lse, list, s.groups};
    return call.launch("attention_merge", cache->head_dim == 128 ? attention_merge_kernel<128> : attention_merge_kernel<64>,
                       (unsigned)((rows + at_once - 1) / at_once), 128, 0, m);
}
