// Attention of new tokens over the paged MX cache: the kernel for many query rows
// per key head (no counterpart in the reference).
//
// With many rows the two products bound it (4 * rows * keys * D operations), with
// the exponentials close behind: one per row and key, 16 a cycle and SM, against
// 4 * D / 8192 cycles of tensor time.  A CTA works on 256 rows as two tiles of
// 128, each with its scores and its output in TMEM, so the tensor core multiplies
// for one tile while the other one is in its softmax.
//
//   warps 0-3, 4-7   softmax of row tile 0, 1: a thread owns one row -- its query,
//                    running maximum and sum, its weights and its output row
//   warps 8-11       converters: packed keys and values from the cache's pages to
//                    f16 tiles in shared memory (SWIZZLE_128B), two stages each
//   warp 12          the only thread that issues products (warps 13-15 idle):
//                    S = Q K^T from shared memory, O += P V with P from TMEM
//
// P (f16) overwrites the S it came from, so TMEM holds S0 S1 O0 O1, 512 columns at
// D = 128.  Values are the right operand as they lie in the cache (one row per
// token), read by the tensor core as an N-major operand, so nothing is transposed.
//
// Scales: the keys of a 128-token tile are converted relative to the tile's
// largest scale, which goes into the factor of the scores (per tile and row);
// values relative to a reference that moves up with the data (attention_rows_kernel
// does the same), on which the output rows are rescaled together with the running
// maximum, both rarely.
#include "attention.cuh"

namespace mxk {
namespace {

using dev::ex2;
using dev::kExpShift;
using dev::kKeyLift;
using dev::kMaxSlack;
using dev::kQueryExp;
using dev::kValueLift;
using dev::kValueMax;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kTileRows = 128;           // M of one product
constexpr int kRows = 2 * kTileRows;     // rows of a unit
constexpr int kKeys = 128;               // tokens of a key tile
constexpr int kSoftmaxWarps = 8;
constexpr int kConvertWarps = 4;
constexpr int kThreads = 512;            // whole warpgroups, for the register split
// Registers a thread: the kernel is launched with 128, warps 12-15 give theirs up.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 160, kConvertRegs = 144, kProductRegs = 48;
static_assert(256 * kSoftmaxRegs + 128 * (kConvertRegs + kProductRegs) <= kThreads * kLaunchRegs,
              "the split draws on what the block was launched with");
constexpr int kStages = 2;
constexpr int kMeta = 4;                 // key tiles whose references are kept

template <int D>
struct Smem {
    static constexpr int half = kKeys * 128;        // 128 rows x 64 features
    static constexpr int tile = (D / 64) * half;    // 128 rows x D features
    static constexpr int q = 0;                     // two row tiles
    static constexpr int k = 2 * tile;
    static constexpr int v = k + kStages * tile;
    static constexpr int total = v + kStages * tile + 1024;  // 1024: alignment
};

struct Bars {
    uint64_t q_ready[2];       // the tile's queries are in shared memory
    uint64_t k_full[kStages], v_full[kStages], k_empty[kStages], v_empty[kStages];
    uint64_t s_full[2];        // scores are in TMEM
    uint64_t p_ready[2];       // weights are in TMEM, the output may be added to
    uint64_t o_done[2];        // the tile's product with the values has finished
    uint64_t drain;
};

// A pass over the CTA's share: every role makes the same one.
struct Cursor {
    dev::Walk w;
    int64_t left;
    int tile0, tiles;  // key tiles of the current unit that are this CTA's
    int unit;          // units begun so far

    __device__ __forceinline__ void take() {
        tile0 = w.tile;
        tiles = (int)(left < w.tiles - tile0 ? left : w.tiles - tile0);
    }
    __device__ __forceinline__ bool next(const AttentionParams& p) {
        left -= tiles;
        if (left <= 0) return false;
        dev::walk_on<kRows, kKeys>(p, w);
        ++unit;
        take();
        return true;
    }
    __device__ __forceinline__ int rows(const AttentionParams& p) const {
        const int r = w.view.n * p.group - w.rt * kRows;
        return r < kRows ? r : kRows;
    }
};

// Tokens seen by some and by all rows of a unit.
struct UnitRange {
    int64_t any_lo, any_hi, all_lo, all_hi;
};
__device__ __forceinline__ UnitRange unit_range(const AttentionParams& p, const Cursor& c) {
    UnitRange u;
    const int r0 = c.w.rt * kRows, j0 = r0 / p.group, j1 = (r0 + c.rows(p) - 1) / p.group;
    int64_t x;
    dev::seen_range(p, c.w.view, j0, j1, u.any_lo, u.any_hi);
    dev::seen_range(p, c.w.view, j0, j0, x, u.all_hi);
    dev::seen_range(p, c.w.view, j1, j1, u.all_lo, x);
    return u;
}

__device__ __forceinline__ int2 lds_int2(uint32_t at) {
    int2 v;
    asm volatile("ld.shared.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}

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

template <int D, int BITS>
__global__ void __launch_bounds__(kThreads, 1) attention_tiles_kernel(const AttentionParams p, unsigned* err) {
    using L = Smem<D>;
    constexpr int kRowBytes = D * BITS / 8;
    constexpr int kUnits = D / 16;      // 16-element pieces of a row; a converter thread has as many of a tile
    constexpr int kUnitBytes = 2 * BITS;
    constexpr int kScales = D / 32;     // scale bytes of a row
    constexpr uint32_t kO = 2 * kKeys;  // first TMEM column of the outputs
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) Bars bars;
    __shared__ int64_t scratch[kThreads / 32 + 2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ int2 meta[kMeta];        // per key tile: the keys' and the values' reference scales
    __shared__ int nan_unit[4];         // unit whose values had a NaN taken out of a partly seen tile
    volatile int* abort_flag = &abort_word;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    const dev::Share share = dev::take_share<kRows, kKeys, kThreads>(p, scratch);
    if (share.tiles == 0) {
        if (tid == 0) p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0), p.part_ends[blockIdx.x] = 0;
        return;
    }
    if (tid == 0) {
        abort_word = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            dev::mbar_init(&bars.q_ready[i], kTileRows);
            dev::mbar_init(&bars.s_full[i], 1);
            dev::mbar_init(&bars.p_ready[i], kTileRows);
            dev::mbar_init(&bars.o_done[i], 1);
        }
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
            dev::mbar_init(&bars.k_full[i], 32 * kConvertWarps);
            dev::mbar_init(&bars.v_full[i], 32 * kConvertWarps);
            dev::mbar_init(&bars.k_empty[i], 1);
            dev::mbar_init(&bars.v_empty[i], 1);
        }
        dev::mbar_init(&bars.drain, 1);
        dev::fence_barrier_init();
    }
    if (tid < 4) nan_unit[tid] = -1;
    if (warp == 0) dev::tmem_alloc(&tmem_slot, 512);
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    const uint32_t tmem = tmem_slot;

    Cursor c;
    c.w = dev::walk_to<kRows, kKeys>(p, share.seq, share.offset);
    c.left = share.tiles;
    c.unit = 0;
    c.take();

    // Every wait is bounded; a wait that gives up raises the CTA's abort flag and the
    // roles leave for the end, warp by warp.
#define MXK_WAIT(bar, parity)                                                                  \
    do {                                                                                       \
        const bool ok_ = dev::mbar_wait((bar), (parity), abort_flag, err);                     \
        if (!__all_sync(kFull, ok_)) goto done;                                                \
    } while (0)

    if (warp < kSoftmaxWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ------------------------------------------------------------ softmax
        const int w = warp >> 2;                        // row tile
        const int r = tid & (kTileRows - 1);            // row in the tile
        const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t s_col = lane_base + w * kKeys, o_col = lane_base + kO + w * D;
        const float neg_inf = __int_as_float(0xff800000);
        uint32_t s_phase = 0, o_phase = 0;
        int meta_at = 0;
        bool open = false, went_on = false, ended = false;
        do {
            const int rows = c.rows(p);
            if (w * kTileRows < rows) {
                const bool real = w * kTileRows + r < rows;
                const bool warp_real = w * kTileRows + (r & ~31) < rows;
                const int row = c.w.rt * kRows + w * kTileRows + r;
                const int j = row / p.group, head = c.w.head * p.group + (row - j * p.group);
                const UnitRange range = unit_range(p, c);
                int64_t lo = 0, hi = c.w.view.len;
                if (real) dev::seen_range(p, c.w.view, j, j, lo, hi);

                // This row's query into shared memory, scaled by a power of two to a largest
                // magnitude in [2^12, 2^13); a negative scale of the scores goes into its sign.
                float row_factor;
                {
                    const int64_t at = (int64_t)(c.w.view.row0 + j) * p.q_token + (int64_t)head * p.q_head;
                    const uint16_t* q = static_cast<const uint16_t*>(p.q) + at;
                    uint32_t x[D / 2];
#pragma unroll
                    for (int i = 0; i < D / 4; ++i) {
                        x[2 * i] = x[2 * i + 1] = 0;
                        if (real) {
                            if (p.q_vec) {
                                const uint2 v = __ldg(reinterpret_cast<const uint2*>(q) + i);
                                x[2 * i] = v.x, x[2 * i + 1] = v.y;
                            } else {
                                x[2 * i] = q[4 * i] | ((uint32_t)q[4 * i + 1] << 16);
                                x[2 * i + 1] = q[4 * i + 2] | ((uint32_t)q[4 * i + 3] << 16);
                            }
                        }
                    }
                    const bool f16 = p.dtype == MXK_F16;
                    auto pair = [&](uint32_t v) -> float2 {
                        if (f16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
                        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
                    };
                    float amax = 0.0f;
#pragma unroll
                    for (int i = 0; i < D / 2; ++i) {
                        const float2 v = pair(x[i]);
                        amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
                    }
                    int e = amax > 0.0f ? (int)(__float_as_uint(amax) >> 23) - 127 : 0;
                    e = max(e, -126);
                    const int down = (kQueryExp - e) / 2, rest = kQueryExp - e - down;
                    const float f0 = __uint_as_float((uint32_t)(down + 127) << 23);
                    const float f1 = copysignf(__uint_as_float((uint32_t)(rest + 127) << 23), p.scale_log2);
                    row_factor = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 - down - kKeyLift / 2) << 23) *
                                 __uint_as_float((uint32_t)(127 - rest - kKeyLift / 2) << 23);
                    uint8_t* dst = smem + L::q + w * L::tile + r * 128;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        uint32_t h[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float2 v = pair(x[4 * i + k]);
                            const __half2 u = __floats2half2_rn(v.x * f0 * f1, v.y * f0 * f1);
                            h[k] = *reinterpret_cast<const uint32_t*>(&u);
                        }
                        *reinterpret_cast<uint4*>(dst + (i / 8) * L::half + (((i % 8) ^ (r & 7)) << 4)) =
                            make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
                dev::fence_proxy_async();
                dev::mbar_arrive(&bars.q_ready[w]);

                float run_max = neg_inf, base = -kExpShift, sum = 0.0f;
                int vref = 0;
                for (int t = 0; t < c.tiles; ++t) {
                    MXK_WAIT(&bars.s_full[w], s_phase);
                    s_phase ^= 1;
                    dev::tc_fence_after();
                    const int2 ref = lds_int2(dev::smem_addr(&meta[(meta_at + t) % kMeta]));
                    if (warp_real) {
                        const float f = row_factor * __uint_as_float((uint32_t)ref.x << 23);
                        const int64_t t0 = (c.w.first + c.tile0 + t) * kKeys;
                        const bool partly = t0 < range.all_lo || t0 + kKeys > range.all_hi;
                        int from = 0, to = kKeys;  // columns that take part
                        if (partly) {
                            from = lo > t0 ? (lo - t0 < kKeys ? (int)(lo - t0) : kKeys) : 0;
                            to = hi < t0 ? 0 : (hi - t0 < kKeys ? (int)(hi - t0) : kKeys);
                        }
                        // the largest score
                        float top = neg_inf;
#pragma unroll
                        for (int h = 0; h < kKeys / 32; ++h) {
                            uint32_t s[32];
                            dev::tmem_ld_32x32b_x32(s_col + 32 * h, s);
                            dev::tmem_wait_ld();
                            if (partly) {
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (32 * h + i < from || 32 * h + i >= to) s[i] = 0xff800000u;
                            }
                            float m[4] = {neg_inf, neg_inf, neg_inf, neg_inf};
#pragma unroll
                            for (int i = 0; i < 32; ++i) m[i & 3] = fmaxf(m[i & 3], __uint_as_float(s[i]));
                            top = fmaxf(top, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
                        }
                        if (top != neg_inf) top *= f;
                        const bool raise = top > run_max + kMaxSlack;
                        const bool shift = ref.y != vref;
                        if (__any_sync(kFull, raise) || shift) {
                            const float m = raise ? top : run_max;
                            float g = m == run_max ? 1.0f : ex2(run_max - m);
                            run_max = m;
                            base = (m == neg_inf ? 0.0f : m) - kExpShift;
                            sum *= g;
                            if (t > 0) {  // the output so far, once the products before have finished
                                if (shift) g *= __uint_as_float((uint32_t)max(vref - ref.y + 127, 0) << 23);
                                MXK_WAIT(&bars.o_done[w], o_phase ^ 1);
                                dev::tc_fence_after();
#pragma unroll
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
                            vref = ref.y;
                        }
                        // the weights, over the scores they come from
                        float part[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int h = 0; h < kKeys / 32; ++h) {
                            uint32_t s[32];
                            dev::tmem_ld_32x32b_x32(s_col + 32 * h, s);
                            dev::tmem_wait_ld();
                            uint32_t pw[16];
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                float a = ex2(fmaf(__uint_as_float(s[i]), f, -base));
                                float b = ex2(fmaf(__uint_as_float(s[i + 1]), f, -base));
                                if (partly) {
                                    if (32 * h + i < from || 32 * h + i >= to) a = 0.0f;
                                    if (32 * h + i + 1 < from || 32 * h + i + 1 >= to) b = 0.0f;
                                }
                                part[0] += a, part[1] += b;
                                const __half2 u = __floats2half2_rn(a, b);
                                pw[i / 2] = *reinterpret_cast<const uint32_t*>(&u);
                            }
                            dev::tmem_st_32x32b_x16(s_col + 16 * h, pw);
                        }
                        dev::tmem_wait_st();
                        sum += part[0] + part[1];
                    }
                    dev::tc_fence_before();
                    dev::mbar_arrive(&bars.p_ready[w]);
                    o_phase ^= 1;
                }
                meta_at += c.tiles;

                // The output row.
                MXK_WAIT(&bars.o_done[w], o_phase ^ 1);
                dev::tc_fence_after();
                if (warp_real) {
                    const bool whole = c.tile0 == 0 && c.tiles == c.w.tiles;
                    // NaNs that were taken out of the values, for the rows that see them
                    uint32_t bad[D / 32] = {};
                    if constexpr (BITS == 8) {
                        if (*reinterpret_cast<volatile int*>(&nan_unit[c.unit & 3]) == c.unit && real) {
                            for (int t = 0; t < c.tiles; ++t) {
                                const int64_t t0 = (c.w.first + c.tile0 + t) * kKeys;
                                if (!(t0 < range.all_lo || t0 + kKeys > range.all_hi)) continue;
                                for (int64_t k = t0 > lo ? t0 : lo; k < hi && k < t0 + kKeys; ++k) {
                                    int page = __ldg(p.page_table + (int64_t)c.w.seq * p.table_stride + k / p.page_size);
                                    page = page < 0 ? 0 : (page >= p.pages ? p.pages - 1 : page);
                                    const uint8_t* v = p.v_values + (((int64_t)page * p.kv_heads + c.w.head) * p.page_size +
                                                                     k % p.page_size) * kRowBytes;
#pragma unroll 1
                                    for (int i = 0; i < D; ++i)
                                        if ((v[i] & 0x7fu) == 0x7fu) {
#pragma unroll
                                            for (int b = 0; b < D / 32; ++b)
                                                if (b == i / 32) bad[b] |= 1u << (i & 31);
                                        }
                                }
                            }
                        }
                    }
                    const float vfactor = __uint_as_float((uint32_t)vref << 23);
                    const float inv = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
                    const int64_t slot = 2 * (int64_t)blockIdx.x + (c.tile0 == 0 ? 1 : 0);
                    const int tile_row = w * kTileRows + r;
#pragma unroll
                    for (int h = 0; h < D / 32; ++h) {
                        uint32_t o[32];
                        dev::tmem_ld_32x32b_x32(o_col + 32 * h, o);
                        dev::tmem_wait_ld();
                        if (real) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                float v = __uint_as_float(o[i]) * inv * vfactor;
                                if (sum == 0.0f) v = 0.0f;
                                if (BITS == 8 && (bad[h] >> i & 1u)) v = __int_as_float(0x7fc00000);
                                o[i] = __float_as_uint(v);
                            }
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 v = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]),
                                                             __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                                if (whole)
                                    dev::store4(p, c.w.view.row0 + j, head, 32 * h + i, v);
                                else
                                    *reinterpret_cast<float4*>(p.part + (slot * kRows + tile_row) * D + 32 * h + i) = v;
                            }
                        }
                    }
                    if (real) {
                        if (!whole)
                            p.part_stat[slot * kRows + tile_row] = make_float2(run_max, sum);
                        else if (p.lse)
                            p.lse[(int64_t)(c.w.view.row0 + j) * p.heads + head] = dev::row_lse(run_max, sum);
                    }
                }
                dev::tc_fence_before();
            } else {
                meta_at += c.tiles;
            }
            if (!(c.tile0 == 0 && c.tiles == c.w.tiles)) {
                if (c.tile0 == 0) {
                    open = true;
                    if (tid == 0) p.part_open[blockIdx.x] = make_int4(c.w.seq, c.w.rt, c.w.head, 1);
                } else {
                    went_on = true;
                    ended = c.tile0 + c.tiles == c.w.tiles;
                }
            }
        } while (c.next(p));
        if (tid == 0) {
            if (!open) p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0);
            p.part_ends[blockIdx.x] = went_on && ended ? 1 : 0;
        }
    } else if (warp < kSoftmaxWarps + kConvertWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
        // --------------------------------------------------------- converters
        // A thread converts piece u of kUnits rows: eight neighbouring lanes cover the
        // 16-byte chunks of two rows, so the swizzled stores meet no bank twice.
        const int cw = warp - kSoftmaxWarps;
        const int u = D == 128 ? (lane & 3) | ((lane >> 4) << 2) : lane & 3;
        const int r0 = D == 128 ? 4 * cw + ((lane >> 2) & 3) : 8 * cw + (lane >> 2);  // and every kStep-th row
        constexpr int kStep = kKeys / kUnits;
        const unsigned per_page = (unsigned)p.page_size / 16u;

        uint32_t kx[kUnits][kUnitBytes / 4], vx[kUnits][kUnitBytes / 4];
        uint32_t ks[4], vs[4];  // scale bytes of rows lane + 32 i

        // Where the key tile `t` of the cursor's unit lies: lane i < 8 has granule i's first row.
        struct Place {
            uint32_t row;
            int valid;
        };
        auto place = [&](const Cursor& at, int t) -> Place {
            Place pl{0, 0};
            const int64_t t0 = (at.w.first + at.tile0 + t) * kKeys;
            const int64_t rest = at.w.view.len - t0;
            pl.valid = rest < 0 ? 0 : (rest < kKeys ? (int)rest : kKeys);
            if (lane < 8 && 16 * lane < pl.valid) {
                const unsigned gr = (unsigned)(t0 / 16) + lane;
                int page = __ldg(p.page_table + (int64_t)at.w.seq * p.table_stride + gr / per_page);
                page = page < 0 ? 0 : (page >= p.pages ? p.pages - 1 : page);
                pl.row = ((uint32_t)page * p.kv_heads + at.w.head) * p.page_size + (gr % per_page) * 16u;
            }
            return pl;
        };
        auto load = [&](const Place& pl, const uint8_t* values, uint32_t (&x)[kUnits][kUnitBytes / 4]) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = r0 + kStep * i;
                const uint32_t row = __shfl_sync(kFull, pl.row, r >> 4) + (r & 15);
#pragma unroll
                for (int k = 0; k < kUnitBytes / 4; ++k) x[i][k] = 0;
                if (r < pl.valid) ldg_bytes<kUnitBytes>(values + (uint64_t)row * kRowBytes + u * kUnitBytes, x[i]);
            }
        };
        auto load_scales = [&](const Place& pl, const uint8_t* scales, uint32_t (&s)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = lane + 32 * i;
                const uint32_t row = __shfl_sync(kFull, pl.row, r >> 4) + (r & 15);
                s[i] = 0;
                if (r < pl.valid) {
                    if constexpr (D == 128)
                        s[i] = __ldg(reinterpret_cast<const uint32_t*>(scales) + row);
                    else
                        s[i] = __ldg(reinterpret_cast<const uint16_t*>(scales) + row);
                }
            }
        };
        auto top_scale = [&](const uint32_t (&s)[4]) -> int {
            unsigned m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < kScales; ++b) m = max(m, (s[i] >> (8 * b)) & 255u);
            return (int)__reduce_max_sync(kFull, m);
        };
        // f16 of x relative to the scale byte `ref`, into a shared-memory tile
        auto store = [&](const uint32_t (&x)[kUnits][kUnitBytes / 4], const uint32_t (&s)[4], int ref, uint8_t* tile) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = r0 + kStep * i;
                const uint32_t sw = __shfl_sync(kFull, s[kStep * i / 32], r & 31);
                const int e = (int)((sw >> (8 * (u >> 1))) & 255u) - ref;
                uint32_t h[8];
                convert16<BITS>(x[i], dev::pow2_f16x2(e, e), h);
                uint8_t* row = tile + (u >> 2) * L::half + r * 128;
                const int chunk = (u & 3) * 2;
                *reinterpret_cast<uint4*>(row + ((chunk ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(row + (((chunk + 1) ^ (r & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
            }
        };

        Cursor ahead = c;  // one key tile ahead of c
        int at = 0;        // key tile of `ahead`'s unit
        bool more = true;
        Place pl = place(ahead, 0);
        load_scales(pl, p.k_scales, ks);
        load_scales(pl, p.v_scales, vs);
        load(pl, p.k_values, kx);
        load(pl, p.v_values, vx);
        int vref = 0, stage = 0, meta_at = 0;
        uint32_t phase = 1;  // the first pass over the stages finds them empty
        do {
            const UnitRange range = unit_range(p, c);
            vref = 0;
            for (int t = 0; t < c.tiles; ++t) {
                const int64_t t0 = (c.w.first + c.tile0 + t) * kKeys;
                const bool partly = t0 < range.all_lo || t0 + kKeys > range.all_hi;
                const int kref = max(top_scale(ks), 1), vtop = top_scale(vs);
                if (vref == 0 || vtop > vref + kValueMax) vref = max(vtop - kValueLift, 1);
                uint32_t vs_now[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) vs_now[i] = vs[i];

                MXK_WAIT(&bars.k_empty[stage], phase);
                store(kx, ks, kref - kKeyLift, smem + L::k + stage * L::tile);
                if (cw == 0 && lane == 0) meta[meta_at % kMeta] = make_int2(kref, vref);
                dev::fence_proxy_async();
                dev::mbar_arrive(&bars.k_full[stage]);

                // the next key tile is on its way while this one's values are converted
                if (more) {
                    if (++at == ahead.tiles) at = 0, more = ahead.next(p);
                }
                if (more) {
                    pl = place(ahead, at);
                    load_scales(pl, p.k_scales, ks);
                    load_scales(pl, p.v_scales, vs);
                    load(pl, p.k_values, kx);
                }
                if constexpr (BITS == 8) {
                    if (partly) {  // a NaN belongs to the rows that see it: they get it at the end
                        bool nans = false;
#pragma unroll
                        for (int i = 0; i < kUnits; ++i)
#pragma unroll
                            for (int k = 0; k < kUnitBytes / 4; ++k) {
                                const uint32_t b = __vcmpeq4(vx[i][k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                                nans |= b != 0;
                                vx[i][k] &= ~b;
                            }
                        if (nans) *reinterpret_cast<volatile int*>(&nan_unit[c.unit & 3]) = c.unit;
                    }
                }
                MXK_WAIT(&bars.v_empty[stage], phase);
                store(vx, vs_now, vref, smem + L::v + stage * L::tile);
                dev::fence_proxy_async();
                dev::mbar_arrive(&bars.v_full[stage]);
                if (more) load(pl, p.v_values, vx);

                ++meta_at;
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
        } while (c.next(p));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProductRegs));
        // ----------------------------------------------------------- products
        constexpr uint32_t idesc_s = dev::f16_idesc(kTileRows, kKeys, false);
        constexpr uint32_t idesc_o = dev::f16_idesc(kTileRows, D, true);
        const uint32_t base = dev::smem_addr(smem);
        if (warp == kSoftmaxWarps + kConvertWarps && lane == 0) {
            bool ok = true;
            int k_stage = 0, v_stage = 0;
            uint32_t k_phase = 0, v_phase = 0, p_phase[2] = {0, 0}, q_phase[2] = {0, 0};
            auto scores = [&](int w) {  // S_w = Q_w K^T
                dev::tc_fence_after();
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint32_t at = (i / 4) * L::half + (i % 4) * 32;
                    dev::tc_mma_f16(tmem + w * kKeys,
                                    dev::smem_desc(base + L::q + w * L::tile + at, 16, 1024, dev::kLayoutSwizzle128),
                                    dev::smem_desc(base + L::k + k_stage * L::tile + at, 16, 1024, dev::kLayoutSwizzle128),
                                    idesc_s, i > 0);
                }
                dev::tc_commit(&bars.s_full[w]);
            };
            do {
                const int nw = c.rows(p) > kTileRows ? 2 : 1;
                for (int t = 0; t <= c.tiles && ok; ++t) {
                    // scores of key tile t, weighted values of key tile t - 1
                    for (int w = 0; w < nw && ok; ++w) {
                        if (t > 0) {
                            ok = dev::mbar_wait_lean(&bars.p_ready[w], p_phase[w], abort_flag, err);
                            if (ok && w == 0) ok = dev::mbar_wait_lean(&bars.v_full[v_stage], v_phase, abort_flag, err);
                            if (!ok) break;
                            p_phase[w] ^= 1;
                            dev::tc_fence_after();
#pragma unroll
                            for (int i = 0; i < kKeys / 16; ++i)
                                dev::tc_mma_f16_ta(
                                    tmem + kO + w * D, tmem + w * kKeys + 8 * i,
                                    dev::smem_desc(base + L::v + v_stage * L::tile + i * 2048, L::half, 1024,
                                                   dev::kLayoutSwizzle128),
                                    idesc_o, t > 1 || i > 0);
                            dev::tc_commit(&bars.o_done[w]);
                            if (w == nw - 1) dev::tc_commit(&bars.v_empty[v_stage]);
                        }
                        if (t < c.tiles) {
                            if (w == 0) ok = dev::mbar_wait_lean(&bars.k_full[k_stage], k_phase, abort_flag, err);
                            if (ok && t == 0) {
                                ok = dev::mbar_wait_lean(&bars.q_ready[w], q_phase[w], abort_flag, err);
                                q_phase[w] ^= 1;
                            }
                            if (!ok) break;
                            scores(w);
                        }
                    }
                    if (!ok) break;
                    if (t > 0) {
                        if (++v_stage == kStages) v_stage = 0, v_phase ^= 1;
                    }
                    if (t < c.tiles) {
                        dev::tc_commit(&bars.k_empty[k_stage]);
                        if (++k_stage == kStages) k_stage = 0, k_phase ^= 1;
                    }
                }
            } while (ok && c.next(p));
            // Products in flight must not outlive the CTA's memory.
            dev::tc_commit(&bars.drain);
            const long long start = clock64();
            while (!dev::mbar_try_wait(&bars.drain, 0))
                if (clock64() - start > dev::kWaitLimitCycles) break;
        }
        __syncwarp();
    }
#undef MXK_WAIT
done:
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    if (warp == 0) dev::tmem_dealloc(tmem, 512);
    // After a wait gave up nothing of this CTA is joined.
    if (tid == 0 && *abort_flag) p.part_open[blockIdx.x] = make_int4(0, 0, 0, 0), p.part_ends[blockIdx.x] = 1;
}

template <int D, int BITS>
int launch(AttentionParams p, int64_t most_tiles, cudaStream_t stream) {
    constexpr int smem = Smem<D>::total;
    static thread_local int ready_device = -1;
    int dev = 0;
    MXK_CUDA(cudaGetDevice(&dev));
    if (ready_device != dev) {
        MXK_CUDA(cudaFuncSetAttribute(attention_tiles_kernel<D, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        cudaFuncAttributes attr{};
        MXK_CUDA(cudaFuncGetAttributes(&attr, attention_tiles_kernel<D, BITS>));
        if (attr.numRegs != kLaunchRegs)
            return fail(MXK_ERR_CUDA, "cache_attention: the build does not have the registers its split assumes");
        ready_device = dev;
    }
    unsigned* err = device_error_word();
    if (!err) return fail(MXK_ERR_CUDA, "cache_attention: cannot allocate the device error word");
    static const int sms = sm_count();
    const int64_t ctas = most_tiles < sms ? most_tiles : sms;
    Workspace ws(stream);
    MXK_CHECK(ws.take(p, ctas, kRows, D));
    {
        LaunchScope scope("attention_tiles", stream);
        attention_tiles_kernel<D, BITS><<<(unsigned)ctas, kThreads, smem, stream>>>(p, err);
        MXK_CUDA(cudaGetLastError());
    }
    return join_parts<kRows, D>(p, (int)ctas, 32, stream);
}

template <int D>
int launch_bits(int bits, const AttentionParams& p, int64_t most_tiles, cudaStream_t stream) {
    if (bits == 8) return launch<D, 8>(p, most_tiles, stream);
    if (bits == 6) return launch<D, 6>(p, most_tiles, stream);
    return launch<D, 4>(p, most_tiles, stream);
}

}  // namespace

int launch_attention_tiles(int bits, int head_dim, const AttentionParams& p, int max_q, cudaStream_t stream) {
    const int64_t most = attention_tile_bound(p, max_q, kRows, kKeys);
    return head_dim == 128 ? launch_bits<128>(bits, p, most, stream) : launch_bits<64>(bits, p, most, stream);
}

}  // namespace mxk
