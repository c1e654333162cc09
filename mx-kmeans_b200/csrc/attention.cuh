// Shared pieces of the attention kernels over the paged MX cache: parameters,
// the division of the work over CTAs, and the layout of partial sums.
//
// Work is divided without the host knowing the lengths.  A unit is one (sequence,
// row tile, key head): the rows r = j * group + g (query token j, query head g of
// the key head's group) of one tile, over the tokens that any of them sees, in
// key tiles.  All units' key tiles, numbered one after the other, are split
// evenly over the CTAs, so every CTA gets the same number whatever the lengths
// are; a CTA walks its tiles unit by unit.  A unit that one CTA has to itself is
// written out by it; the parts of a unit that spans several go to the workspace
// (at most two per CTA: the end of a unit that an earlier CTA began, and the
// beginning of one that a later CTA goes on with) and attention_join_kernel adds
// them in CTA order, so the result does not depend on timing.
#pragma once

#include "cache.cuh"

namespace mxk {

struct AttentionParams {
    // cache
    const uint8_t* k_values;
    const uint8_t* v_values;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
    int kv_heads, page_size, pages;
    // queries and outputs
    const void* q;
    void* out;
    float* lse;
    int64_t q_token, q_head, out_token, out_head;  // strides in elements
    int64_t tokens;
    int dtype, heads, group, seqs;
    int q_vec, out_vec;  // rows can be moved 8 bytes at a time
    const int* cu_q;
    const int* page_table;
    int64_t table_stride;
    int64_t max_kv;
    const int* kv_lens;
    float scale_log2;  // scale * log2(e)
    int causal;
    int64_t window;
    int min_rows, max_rows;  // this launch takes the sequences with min_rows <= n * group <= max_rows
    // partial sums
    float* part;  // [2 * CTAs][tile rows][head_dim]
    float2* part_stat;  // [2 * CTAs][tile rows]: running maximum (log2 units), sum
    int4* part_open;    // [CTAs]: {sequence, row tile, key head, n} of the unit that the CTA began and the n
                        // following ones went on with; n = 0: it left none unfinished
    // keys and values converted beforehand (tiles kernel), [seqs][kv_heads][max_tiles]
    uint8_t* ready_k;
    uint8_t* ready_v;
    int2* ready_meta;   // reference scales of the keys and values; bit 16 of y: NaNs taken out
    int max_tiles;
};

// Key tiles there can be at most when no sequence has more than max_q query and
// p.max_kv cached tokens: a window touches at most one tile more than it and the
// row tile's tokens fill.
inline int64_t attention_tile_bound(const AttentionParams& p, int max_q, int rows, int keys) {
    const int64_t row_tiles = ((int64_t)max_q * p.group + rows - 1) / rows;
    int64_t span = p.max_kv;
    if (p.window > 0 && p.window + rows < span) span = p.window + rows;
    return (int64_t)p.seqs * p.kv_heads * row_tiles * (span / keys + 2);
}

// attention_tiles.cu: many query rows per key head.
int launch_attention_tiles(int bits, int head_dim, AttentionParams p, int max_q, cudaStream_t stream);

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
constexpr int kQueryExp = 12;  // query rows are scaled to a largest magnitude in [2^12, 2^13)

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
    int row0;     // first query row
    int n;        // query tokens
    int64_t len;  // cached tokens
};

__device__ __forceinline__ SeqView seq_view(const AttentionParams& p, int seq) {
    SeqView v;
    const int64_t a = __ldg(p.cu_q + seq), b = __ldg(p.cu_q + seq + 1);
    const int64_t lo = a < 0 ? 0 : (a > p.tokens ? p.tokens : a);
    const int64_t hi = b < lo ? lo : (b > p.tokens ? p.tokens : b);
    v.row0 = (int)lo;
    v.n = (int)(hi - lo);
    const int64_t len = __ldg(p.kv_lens + seq);
    v.len = len < 0 ? 0 : (len > p.max_kv ? p.max_kv : len);
    return v;
}

// Tokens [lo, hi) that the rows of query tokens j0..j1 see, all of them together
// (empty: hi <= lo).
__device__ __forceinline__ void seen_range(const AttentionParams& p, const SeqView& s, int j0, int j1, int64_t& lo,
                                           int64_t& hi) {
    const int64_t first = s.len - s.n + j0, last = s.len - s.n + j1;
    hi = p.causal && last + 1 < s.len ? last + 1 : s.len;
    lo = p.window > 0 && first - p.window + 1 > 0 ? first - p.window + 1 : 0;
}

// Key tiles of a row tile (at least one: rows that see nothing are written too).
template <int ROWS, int KEYS>
__device__ __forceinline__ int tile_count(const AttentionParams& p, const SeqView& s, int rt, int64_t* first = nullptr) {
    const int rows = s.n * p.group;
    const int j0 = rt * ROWS / p.group;
    const int last = (rt + 1) * ROWS < rows ? (rt + 1) * ROWS - 1 : rows - 1;
    int64_t lo, hi;
    seen_range(p, s, j0, last / p.group, lo, hi);
    const int64_t t0 = lo / KEYS;
    if (first) *first = t0;
    if (hi <= lo) return 1;
    return (int)((hi + KEYS - 1) / KEYS - t0);
}

template <int ROWS, int KEYS>
__device__ __forceinline__ int64_t seq_tiles(const AttentionParams& p, const SeqView& s) {
    const int64_t rows = (int64_t)s.n * p.group;
    if (rows < p.min_rows || rows > p.max_rows || rows == 0) return 0;
    int64_t total = 0;
    const int tiles = (int)((rows + ROWS - 1) / ROWS);
    if (!p.causal && p.window == 0) return (int64_t)tiles * p.kv_heads * tile_count<ROWS, KEYS>(p, s, 0);
    for (int rt = 0; rt < tiles; ++rt) total += tile_count<ROWS, KEYS>(p, s, rt);
    return total * p.kv_heads;
}

// Where a CTA's share begins, and how many tiles it has.
struct Share {
    int64_t tiles;   // of this CTA
    int seq;         // first sequence of the share
    int64_t offset;  // of the share's first tile in that sequence
    int64_t begin;   // the share's first tile among all,
    int64_t total;   // of so many,
    int64_t ctas;    // for so many CTAs

    // CTAs after this one that work on a unit of n tiles whose first is `at` of the share.
    __device__ __forceinline__ int followers(int64_t at, int64_t n) const {
        const int64_t last = begin + at + n - 1;  // tile x belongs to CTA ceil((x + 1) ctas / total) - 1
        return (int)(((last + 1) * ctas + total - 1) / total - 1 - blockIdx.x);
    }
};

// All threads of the CTA; scratch: THREADS / 32 + 4 words of shared memory.
// CTAs past the number of tiles get none.
template <int ROWS, int KEYS, int THREADS>
__device__ __forceinline__ Share take_share(const AttentionParams& p, int64_t* scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = THREADS / 32;
    int64_t* found = scratch + kWarps;  // sequence, offset
    int64_t sum = 0;
    for (int i = tid; i < p.seqs; i += THREADS) sum += seq_tiles<ROWS, KEYS>(p, seq_view(p, i));
    const int64_t mine = sum;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) scratch[warp] = sum;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += scratch[w];
    const int64_t ctas = total < gridDim.x ? total : gridDim.x;
    Share s{0, 0, 0, 0, total, ctas};
    if ((int64_t)blockIdx.x >= ctas) return s;
    const int64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
    s.tiles = end - begin;
    s.begin = begin;
    int64_t before = 0;  // tiles of the sequences before this round's
    for (int base = 0; base < p.seqs; base += THREADS) {
        const int i = base + tid;
        int64_t t = p.seqs <= THREADS ? mine : (i < p.seqs ? seq_tiles<ROWS, KEYS>(p, seq_view(p, i)) : 0);
        int64_t incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        __syncthreads();
        if (lane == 31) scratch[warp] = incl;
        __syncthreads();
        int64_t start = before, round = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) start += scratch[w];
            round += scratch[w];
        }
        start += incl - t;
        if (begin >= start && begin < start + t) found[0] = i, found[1] = begin - start;
        before += round;
        if (begin < before) break;
    }
    __syncthreads();
    s.seq = (int)found[0];
    s.offset = found[1];
    __syncthreads();
    return s;
}

// A position in the walk over the units.
struct Walk {
    int seq, rt, head;
    int tile, tiles;   // next key tile of the unit, and how many it has
    int64_t first;     // number of the unit's first key tile in the sequence
    SeqView view;
};

template <int ROWS, int KEYS>
__device__ __forceinline__ Walk walk_to(const AttentionParams& p, int seq, int64_t offset) {
    Walk w;
    w.seq = seq;
    w.view = seq_view(p, seq);
    w.rt = 0;
    while (true) {
        w.tiles = tile_count<ROWS, KEYS>(p, w.view, w.rt, &w.first);
        const int64_t all = (int64_t)w.tiles * p.kv_heads;
        if (offset < all) break;
        offset -= all;
        ++w.rt;
    }
    w.head = (int)(offset / w.tiles);
    w.tile = (int)(offset - (int64_t)w.head * w.tiles);
    return w;
}

// To the next unit; the caller knows that there is one.
template <int ROWS, int KEYS>
__device__ __forceinline__ void walk_on(const AttentionParams& p, Walk& w) {
    w.tile = 0;
    if (++w.head < p.kv_heads) return;
    w.head = 0;
    ++w.rt;
    if ((int64_t)w.rt * ROWS >= (int64_t)w.view.n * p.group) {
        w.rt = 0;
        int64_t rows;
        do {
            ++w.seq;
            if (w.seq >= p.seqs) return;
            w.view = seq_view(p, w.seq);
            rows = (int64_t)w.view.n * p.group;
        } while (rows == 0 || rows < p.min_rows || rows > p.max_rows);
    }
    w.tiles = tile_count<ROWS, KEYS>(p, w.view, w.rt, &w.first);
}

// Four consecutive features of an output row.
__device__ __forceinline__ void store4(const AttentionParams& p, int64_t token, int head, int feature, float4 v) {
    const int64_t at = token * p.out_token + (int64_t)head * p.out_head + feature;
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

// log(sum exp) of a row from its running maximum (log2 units) and sum.
__device__ __forceinline__ float row_lse(float m2, float sum) {
    return sum > 0.0f ? (m2 - kExpShift) * 0.693147180559945f + logf(sum)
                      : (sum == 0.0f ? __int_as_float(0xff800000) : sum);
}

}  // namespace dev

// Block (x, y): the unit that CTA x began and did not finish, rows y, y + gridDim.y, ...
// Its parts are the beginning (slot 2x + 1) and what the following CTAs did first (slots
// 2j).  The four warps take every fourth part (with D = 64 every half-warp every eighth),
// so a unit in hundreds of parts has several rows of loads under way, and add up in a
// fixed order.
template <int ROWS, int D>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttentionParams p) {
    constexpr int kLanes = D / 4;            // threads of a row
    constexpr int kSub = 128 / kLanes;       // parts at a time
    __shared__ float4 sums[kSub][kLanes];
    __shared__ float stats[4], sub_totals[kSub];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 unit = p.part_open[blockIdx.x];
    if (!unit.w) return;
    const dev::SeqView view = dev::seq_view(p, unit.x);
    const int rows = view.n * p.group - unit.y * ROWS < ROWS ? view.n * p.group - unit.y * ROWS : ROWS;
    const int tid = threadIdx.x, chunk = tid % kLanes, sub = tid / kLanes, parts = unit.w + 1;
    auto slot = [&](int i) -> int64_t { return 2 * (int64_t)(blockIdx.x + i) + (i == 0 ? 1 : 0); };
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        // the common maximum and the sum
        float top = __int_as_float(0xff800000);
        for (int i = tid; i < parts; i += 128) top = fmaxf(top, p.part_stat[slot(i) * ROWS + r].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((tid & 31) == 0) stats[tid >> 5] = top;
        __syncthreads();
        top = fmaxf(fmaxf(stats[0], stats[1]), fmaxf(stats[2], stats[3]));
        float total = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int i = sub; i < parts; i += kSub) {
            const float2 st = p.part_stat[slot(i) * ROWS + r];
            const float4 x = reinterpret_cast<const float4*>(p.part + (slot(i) * ROWS + r) * D)[chunk];
            const float f = st.x == top ? 1.0f : dev::ex2(st.x - top);
            total += st.y * f;
            v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
        }
        sums[sub][chunk] = v;
        // every thread of a sub has the same total
        if (chunk == 0) sub_totals[sub] = total;
        __syncthreads();
        if (tid < kLanes) {
            total = 0.0f;
            v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < kSub; ++i) {
                const float4 x = sums[i][chunk];
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                total += sub_totals[i];
            }
            const int row = unit.y * ROWS + r, j = row / p.group;
            const int head = unit.z * p.group + (row - j * p.group);
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            if (total == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            dev::store4(p, view.row0 + j, head, chunk * 4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            if (p.lse && chunk == 0) p.lse[(int64_t)(view.row0 + j) * p.heads + head] = dev::row_lse(top, total);
        }
        __syncthreads();  // before the shared sums are written again
    }
}

// Memory of a launch's partial sums.
struct Workspace {
    void* ptr = nullptr;
    void* extra = nullptr;
    cudaStream_t stream;
    explicit Workspace(cudaStream_t s) : stream(s) {}
    ~Workspace() {
        if (ptr) cudaFreeAsync(ptr, stream);
    }
    Workspace(const Workspace&) = delete;
    Workspace& operator=(const Workspace&) = delete;
    // extra: bytes at `extra`, 256-byte aligned.
    int take(AttentionParams& p, int64_t ctas, int rows, int d, int64_t extra_bytes = 0) {
        const size_t part = (size_t)(2 * ctas * rows) * d * 4, stat = (size_t)(2 * ctas * rows) * 8;
        const size_t own = (part + stat + (size_t)ctas * 16 + 255) / 256 * 256;
        cudaMemPool_t pool = workspace_pool();
        if (!pool) return fail(MXK_ERR_CUDA, "cache_attention: cannot create the workspace pool");
        MXK_CUDA(cudaMallocFromPoolAsync(&ptr, own + (size_t)extra_bytes, pool, stream));
        extra = static_cast<char*>(ptr) + own;
        p.part = static_cast<float*>(ptr);
        p.part_stat = reinterpret_cast<float2*>(static_cast<char*>(ptr) + part);
        p.part_open = reinterpret_cast<int4*>(static_cast<char*>(ptr) + part + stat);
        return MXK_OK;
    }
};

template <int ROWS, int D>
inline int join_parts(const AttentionParams& p, int ctas, int grid_y, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas, (unsigned)grid_y);
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    LaunchScope scope("attention_join", stream);
    MXK_CUDA(cudaLaunchKernelEx(&cfg, attention_join_kernel<ROWS, D>, p));
    return MXK_OK;
}

}  // namespace mxk
