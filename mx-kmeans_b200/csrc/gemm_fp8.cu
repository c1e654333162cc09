// E4M3 products with a float32 scale per block of 128 (no counterpart in the reference,
// whose products have MX scales, src/kernels/gemm.cu:348-363).
//
//     out[i][j] = sum_b sa[i][b] sb[j / 128][b] sum_{k in block b} a[i][k] b[j][k]
//
// The tensor core sums the 128 products of a block in float32 (tcgen05.mma kind::f8f6f4,
// TMEM accumulators); threads take each block's sums from TMEM, one row a thread, and add
// them to float32 registers with the factor sa sb, which is one number per thread and block.
// Two TMEM buffers let the tensor core multiply the next block meanwhile.
//
// With few rows the weights' bytes over HBM bound it, so all SMs have to stream: a tile's
// blocks are split over the CTAs of a cluster, which add their sums through distributed
// shared memory in rank order, so results do not depend on timing.
//
// Large ones (pair::) are bound by the sums' way and by the power cap: every block's products leave TMEM once,
// 128 KB a CTA (128 rows of 256 columns) for 512 cycles of products, and go through two multiply-adds an
// instruction.  A wait for TMEM is for all loads that a warp has under way, so a load of 16 columns is covered by
// the sums of the 16 before it and no more; with issue slots at 44 % and FMA at 35 % the tensor pipe is busy for 60 %.
// Measured: 8192^3 460 to 500 us on an idle card (2.2 to 2.4 Pflop/s; a library product of E4M3 with one scale
// a matrix, which leaves TMEM once at the end, 350), 550 under the cap; 2048 x 14,336 x 4096 105 us, 777 x 1003 x
// 1040 9, one row through 4096 x 4096 9.6 to 10.5 (1.7 TB/s), 64 rows through 6144 x 4096 11 (2.3 TB/s): these
// are a launch, an empty pipeline, eight steps and the cluster's sums.
#include <algorithm>
#include <limits>

#include "gemm_fp8.cuh"

namespace mxk {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kBlock = 128;  // features of a scale

// Rows that the kernel quantises itself.
struct RowsToQuantize {
    const void* x;
    int64_t stride;  // elements
    int dtype, wide; // wide: 16 features can be loaded 16 bytes at a time
    int k;
};

struct GemmFp8Params {
    int m, n, blocks;        // blocks: of k
    int tiles_m;
    const float* a_scales;   // [m][blocks]
    const float* b_scales;   // [n / 128][blocks]
    char* out;
    int64_t out_stride;      // elements
    int dtype;
    int out_vec, out_wide;   // four elements, or 16 bytes, can be stored at once
    int copied;              // columns that fill whole 16-byte pieces
    int a_wide, b_wide;      // rows of scales can be loaded four at a time
    int beside;              // the kernel before writes nothing that this one reads
    unsigned* err;
};

// Four 16-bit elements.
__device__ __forceinline__ uint2 pack4(int dtype, float2 a, float2 b) {
    if (dtype == MXK_F16) {
        const __half2 u = __float22half2_rn(a), v = __float22half2_rn(b);
        return make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
    }
    const __nv_bfloat162 u = __float22bfloat162_rn(a), v = __float22bfloat162_rn(b);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
}

// Up to four elements of an output row.
__device__ __forceinline__ void store_out(const GemmFp8Params& p, int row, int col, float4 v) {
    const int64_t at = (int64_t)row * p.out_stride + col;
    const float x[4] = {v.x, v.y, v.z, v.w};
    if (p.dtype == MXK_F32) {
        float* o = reinterpret_cast<float*>(p.out) + at;
        if (p.out_vec && col + 4 <= p.n)
            *reinterpret_cast<float4*>(o) = v;
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < p.n) o[i] = x[i];
        return;
    }
    const uint2 h = pack4(p.dtype, make_float2(v.x, v.y), make_float2(v.z, v.w));
    uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + at;
    if (p.out_vec && col + 4 <= p.n)
        *reinterpret_cast<uint2*>(o) = h;
    else
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < p.n) o[i] = (uint16_t)((i < 2 ? h.x : h.y) >> (16 * (i & 1)));
}

// Scales i .. i + 3 of `count`, zeros past them.  They are asked for four blocks ahead: every
// lane has a row of scales of its own, and while tiles stream past they take their time.
__device__ __forceinline__ void load_scales(const float* p, int i, int count, bool wide, float (&v)[4]) {
    if (wide && i < count) {
        const float4 x = *reinterpret_cast<const float4*>(p + i);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = i + k < count ? p[i + k] : 0.0f;
    }
}

// 32 rows of 128 elements, a row a lane, to the output, by way of 8 KB of shared memory.  Where
// the output is aligned they leave as asynchronous copies and the warp goes on; the next call
// waits until they have been read.  (With stores the warps of all CTAs wait at about the same time:
// 4500 cycles of 50,000.  So they do for a copy from each lane, which are issued one by one.)
// The copies write whole 16-byte pieces, whatever the output's width is, so a row's last elements that fill
// none are stored by themselves.
// 16-byte pieces of a row are permuted by row, so that eight lanes write to different banks.
__device__ __forceinline__ void store_rows(const GemmFp8Params& p, const CUtensorMap* map, uint8_t* stage, int row0,
                                           int col, const float2 (&x)[64]) {
    constexpr int kPart = 32 * 128;  // bytes of 32 rows' 128 bytes each
    const int lane = threadIdx.x & 31, size = p.dtype == MXK_F32 ? 4 : 2, part = 128 / size;
    auto piece = [&](int row, int i) { return stage + i / 8 * kPart + row * 128 + (((i ^ row) & 7) << 4); };
    auto wait_for_copies = [&]() {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
    };
    auto send = [&](int at) {  // two parts, which begin with element `at` of the row
        if (p.out_wide) dev::fence_proxy_async();
        __syncwarp();
        if (row0 >= p.m) return;
        if (p.out_wide) {
            if (lane == 0) {
                for (int i = 0; i < 2; ++i)
                    if (at + i * part < p.copied)
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map),
                                     "r"(at + i * part), "r"(row0), "r"(dev::smem_addr(stage + i * kPart))
                                     : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            if (p.copied >= at && p.copied < at + 2 * part && row0 + lane < p.m) {
                for (int c = p.copied; c < p.n; ++c) {
                    const uint8_t* from = piece(lane, (c - at) * size / 16) + (c - at) * size % 16;
                    char* to = p.out + ((int64_t)(row0 + lane) * p.out_stride + c) * size;
                    if (size == 4)
                        *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
                    else
                        *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
                }
            }
            return;
        }
        const int rows = min(p.m - row0, 32), count = min(p.n - at, 2 * part);
        for (int r = 0; r < rows; ++r)
            for (int c = lane; c < count; c += 32) {
                const uint8_t* from = piece(r, c * size / 16) + c * size % 16;
                char* to = p.out + ((int64_t)(row0 + r) * p.out_stride + at + c) * size;
                if (size == 4)
                    *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
                else
                    *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
            }
    };
    wait_for_copies();
    if (size == 4) {  // two halves
#pragma unroll
        for (int i = 0; i < 16; ++i)
            *reinterpret_cast<float4*>(piece(lane, i)) = make_float4(x[2 * i].x, x[2 * i].y, x[2 * i + 1].x, x[2 * i + 1].y);
        send(col);
        wait_for_copies();
#pragma unroll
        for (int i = 0; i < 16; ++i)
            *reinterpret_cast<float4*>(piece(lane, i)) =
                make_float4(x[32 + 2 * i].x, x[32 + 2 * i].y, x[33 + 2 * i].x, x[33 + 2 * i].y);
        send(col + 64);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint2 u = pack4(p.dtype, x[4 * i], x[4 * i + 1]), v = pack4(p.dtype, x[4 * i + 2], x[4 * i + 3]);
            *reinterpret_cast<uint4*>(piece(lane, i)) = make_uint4(u.x, u.y, v.x, v.y);
        }
        send(col);
    }
}

// A wait that goes on after an abort: for copies and products in flight.
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity) {
    const long long start = clock64();
    while (!dev::mbar_try_wait(bar, parity))
        if (clock64() - start > dev::kWaitLimitCycles) break;
}

// ------------------------------------------------------------------ one tile a cluster

namespace tile {

constexpr int kM = 128, kN = 128;
constexpr int kStages = 3, kBuffers = 2;
constexpr int kSide = kM * kBlock;            // bytes of an operand's tile
constexpr int kStage = 2 * kSide;
constexpr int kSumWarps = 8, kLoadWarp = 8, kProductWarp = 9, kThreads = 320;
constexpr int kCols = kN / 2;                 // columns of a warp: four lane quarters, two halves
constexpr int kSmem = kStages * kStage + 1024;  // 1024: alignment
static_assert(kN * kM * 4 <= kStages * kStage, "the sums go out through the operands' memory");

// With few rows, and no more than kOwnBytes of them, a CTA quantises its part of them itself: they
// lie before the operands' stages, which then hold B alone.
constexpr int kOwnRows = 16, kOwnBytes = 32768, kOwnStages = 4;
constexpr int kOwnSmem = kOwnBytes + kOwnStages * kSide + kOwnBytes / kBlock * 4 + 1024;
static_assert(kN * kOwnRows * 4 <= kOwnStages * kSide, "");

struct Shared {
    uint64_t full[kOwnStages], done[kOwnStages];  // loaded; multiplied, so the sums are in TMEM
    uint64_t taken[kBuffers];               // a buffer's sums have been read
    uint64_t rows_ready;                    // the CTA's own rows are quantised
    uint64_t drain;
    int abort_word;
    uint32_t tmem;
};

// 16 features of a row of any type.
__device__ __forceinline__ void load16(const RowsToQuantize& q, int64_t at, float (&v)[16]) {
    if (q.dtype == MXK_F32) {
        dev::Raw16<float, 16> wide;
        dev::Raw16<float, 0> any;
        const float* from = static_cast<const float*>(q.x) + at;
        if (q.wide) wide.load(from), wide.to_float(v);
        else any.load(from), any.to_float(v);
    } else {
        dev::Raw16<__half, 16> raw;
        if (q.wide) {
            raw.load(static_cast<const __half*>(q.x) + at);
        } else {
            dev::Raw16<__half, 0> any;
            any.load(static_cast<const __half*>(q.x) + at);
            raw.w[0] = any.w[0], raw.w[1] = any.w[1];
        }
        if (q.dtype == MXK_F16) {
            raw.to_float(v);
        } else {
            dev::Raw16<__nv_bfloat16, 16> b;
            b.w[0] = raw.w[0], b.w[1] = raw.w[1];
            b.to_float(v);
        }
    }
}

template <bool OWN>
__global__ void __launch_bounds__(kThreads, 2)
    gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                         const GemmFp8Params p, const RowsToQuantize q, int split, int rows_loaded) {
    constexpr int kDepth = OWN ? kOwnStages : kStages, kStep = OWN ? kSide : kStage;  // stages, and bytes of one
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) Shared sh;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(kFull, tid >> 5, 0);
    const int tile = blockIdx.x / split, rank = blockIdx.x - tile * split;
    const int tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const int first = (int)((int64_t)rank * p.blocks / split), last = (int)((int64_t)(rank + 1) * p.blocks / split);
    const int count = last - first;
    volatile int* abort = &sh.abort_word;
    uint8_t* stages = OWN ? smem + kOwnBytes : smem;  // of operands, or B alone
    const int row_bytes = rows_loaded * kBlock;       // of a block's own rows
    float* own_scales = reinterpret_cast<float*>(smem + kOwnBytes + kOwnStages * kSide);  // [block][row]
    const int sum_warps = OWN ? 2 : kSumWarps;        // own rows lie in the first quarter of the lanes

    if (tid == 0) {
        sh.abort_word = 0;
        for (int i = 0; i < kDepth; ++i) dev::mbar_init(&sh.full[i], 1), dev::mbar_init(&sh.done[i], 1);
        for (int i = 0; i < kBuffers; ++i) dev::mbar_init(&sh.taken[i], sum_warps);
        dev::mbar_init(&sh.rows_ready, kSumWarps);
        dev::mbar_init(&sh.drain, 1);
        dev::fence_barrier_init();
    }
    if (warp == kProductWarp) dev::tmem_alloc(&sh.tmem, kBuffers * kN);
    if (warp == kLoadWarp && lane == 0) {
        if (!OWN) dev::prefetch_tensor_map(&map_a);
        dev::prefetch_tensor_map(&map_b);
    }
    dev::tc_fence_before();
    __syncthreads();
    dev::tc_fence_after();
    const uint32_t tmem = __shfl_sync(kFull, sh.tmem, 0);
    dev::let_next_start();

    float acc[kCols];
#pragma unroll
    for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;

    if (warp == kLoadWarp) {
        if (dev::elect_one()) {
            // The weights are no output of the kernel before (which may be the quantiser).
            const int early = min(count, kDepth);
            const uint32_t bytes = kSide + (OWN ? 0 : row_bytes);
            auto load_b = [&](int i, int stage) {
                dev::mbar_arrive_expect_tx(&sh.full[stage], bytes);
                dev::tma_load_2d(stages + stage * kStep + kStep - kSide, &map_b, (first + i) * kBlock, tn * kN, &sh.full[stage]);
            };
            auto load_a = [&](int i, int stage) {
                if (!OWN) dev::tma_load_2d(stages + stage * kStep, &map_a, (first + i) * kBlock, tm * kM, &sh.full[stage]);
            };
            for (int i = 0; i < early; ++i) load_b(i, i);
            if (!p.beside) dev::wait_for_previous();
            for (int i = 0; i < early; ++i) load_a(i, i);
            int i = early, stage = 0;
            uint32_t phase = 0;
            for (; i < count; ++i) {
                if (!dev::mbar_wait(&sh.done[stage], phase, abort, p.err)) break;
                load_b(i, stage), load_a(i, stage);
                if (++stage == kDepth) stage = 0, phase ^= 1;
            }
            if (*abort)
                for (int k = max(i - kDepth, 0); k < i; ++k) settle(&sh.full[k % kDepth], (uint32_t)(k / kDepth) & 1u);
        }
        __syncwarp();
    } else if (warp == kProductWarp) {
        constexpr uint32_t idesc = dev::f16_idesc(kM, kN, false);
        const uint64_t a_desc = dev::smem_desc(dev::smem_addr(smem), 16, 1024, dev::kLayoutSwizzle128);
        const uint64_t b_desc = dev::smem_desc(dev::smem_addr(stages + kStep - kSide), 16, 1024, dev::kLayoutSwizzle128);
        int stage = 0, buffer = 0;
        uint32_t phase = 0, taken_phase = 1;
        bool ok = !OWN || __all_sync(kFull, dev::mbar_wait(&sh.rows_ready, 0, abort, p.err));
        for (int i = 0; i < count && ok; ++i) {
            ok = __all_sync(kFull, dev::mbar_wait(&sh.taken[buffer], taken_phase, abort, p.err)) &&
                 __all_sync(kFull, dev::mbar_wait(&sh.full[stage], phase, abort, p.err));
            if (!ok) break;
            dev::tc_fence_after();
            if (dev::elect_one()) {
                const uint64_t a = a_desc + (uint64_t)(OWN ? i * (row_bytes >> 4) : stage * (kStep >> 4));
                const uint64_t b = b_desc + (uint64_t)(stage * (kStep >> 4));
#pragma unroll
                for (int k = 0; k < kBlock / 32; ++k)
                    dev::tc_mma_f8(tmem + buffer * kN, a + 2 * k, b + 2 * k, idesc, k > 0);
                dev::tc_commit(&sh.done[stage]);
            }
            __syncwarp();
            if (++stage == kDepth) stage = 0, phase ^= 1;
            if (++buffer == kBuffers) buffer = 0, taken_phase ^= 1;
        }
        if (!ok && dev::elect_one()) {  // products in flight must not outlive the CTA's memory
            dev::tc_commit(&sh.drain);
            settle(&sh.drain, 0);
        }
        __syncwarp();
    } else {
        const int row = tm * kM + (warp & 3) * 32 + lane;
        const bool real = row < p.m;
        const float* sa = OWN ? nullptr : p.a_scales + (int64_t)(real ? row : 0) * p.blocks + first;
        const float* sb = p.b_scales + (int64_t)tn * p.blocks + first;
        const uint32_t column = tmem + ((uint32_t)(warp & 3) << 21) + (warp >> 2) * kCols;
        if (!p.beside) dev::wait_for_previous();
        if constexpr (OWN) {
            // Eight threads to a row of a block, 16 features each, which are one 16-byte piece of the
            // swizzled tile.
            const int items = count * rows_loaded;
            for (int base = 0; base < items; base += kSumWarps * 4) {
                const int item = base + (tid >> 3), sub = tid & 7;
                const int block = item / rows_loaded, r = item - block * rows_loaded, f = (first + block) * kBlock + sub * 16;
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0.0f;
                if (item < items && r < p.m && f < q.k) load16(q, r * q.stride + f, v);
                float amax = dev::largest16(v);
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, o));
                const float s = dev::fp8_scale(amax);
                if (item < items) {
                    *reinterpret_cast<uint4*>(smem + block * row_bytes + r * kBlock + ((sub ^ (r & 7)) << 4)) =
                        q.dtype == MXK_F32 ? dev::fp8_codes16(v, s, amax) : dev::fp8_codes16_narrow(v, s, amax);
                    if (sub == 0) own_scales[item] = s;
                }
            }
            dev::fence_proxy_async();
            __syncwarp();
            if (lane == 0) dev::mbar_arrive(&sh.rows_ready);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kSumWarps) : "memory");  // all rows' scales are there
        }
        float fa[4], fb[4];
        auto scales_of = [&](int i) {
            if constexpr (OWN) {
#pragma unroll
                for (int k = 0; k < 4; ++k) fa[k] = real && i + k < count ? own_scales[(i + k) * rows_loaded + row] : 0.0f;
            } else {
                load_scales(sa, i, count, false, fa);
            }
            load_scales(sb, i, count, false, fb);
        };
        scales_of(0);
        int stage = 0, buffer = 0;
        uint32_t phase = 0;
        bool ok = !OWN || (warp & 3) == 0;  // (no rows of its own: nothing to add up)
        for (int i0 = 0; i0 < count && ok; i0 += 4) {
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = fa[k] * fb[k];
            scales_of(i0 + 4);
#pragma unroll
            for (int at = 0; at < 4; ++at) {
                if (i0 + at >= count) break;
                ok = __all_sync(kFull, dev::mbar_wait(&sh.done[stage], phase, abort, p.err));
                if (!ok) break;
                dev::tc_fence_after();
#pragma unroll
                for (int c = 0; c < kCols; c += 16) {
                    uint32_t v[16];
                    dev::tmem_ld_32x32b_x16(column + buffer * kN + c, v);
                    dev::tmem_wait_ld();
                    if (c + 16 == kCols) {
                        dev::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) dev::mbar_arrive(&sh.taken[buffer]);
                    }
#pragma unroll
                    for (int k = 0; k < 16; ++k) acc[c + k] = fmaf(__uint_as_float(v[k]), f[at], acc[c + k]);
                }
                if (++stage == kDepth) stage = 0, phase ^= 1;
                if (++buffer == kBuffers) buffer = 0;
            }
        }
        // All products have read their operands: the sums take that memory, a row's 16-byte
        // chunks permuted so that eight rows' chunks lie in different banks.
        const int r = (warp & 3) * 32 + lane;
        if (real) {
#pragma unroll
            for (int c = 0; c < kCols / 4; ++c)
                *reinterpret_cast<float4*>(stages + r * (kN * 4) + ((((warp >> 2) * (kCols / 4) + c) ^ (r & 7)) << 4)) =
                    make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
        }
    }
    if (split > 1)
        dev::cluster_arrive(), dev::cluster_wait();
    else
        __syncthreads();
    // The cluster's sums, each CTA its part of the tile's rows and chunks.
    const int rows = min(p.m - tm * kM, kM), total = rows * (kN / 4);
    const uint32_t sums = dev::smem_addr(stages);
    const int end = (int)((int64_t)(rank + 1) * total / split);
    for (int i = (int)((int64_t)rank * total / split) + tid; i < end; i += kThreads) {
        const int r = i >> 5, c = i & 31;
        if (tn * kN + 4 * c >= p.n) continue;
        const uint32_t at = sums + r * (kN * 4) + ((c ^ (r & 7)) << 4);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < split; ++k) {
            const float4 x = dev::cluster_ld4(dev::in_cta(at, k));
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        store_out(p, tm * kM + r, tn * kN + 4 * c, v);
    }
    dev::tc_fence_before();
    if (split > 1)
        dev::cluster_arrive(), dev::cluster_wait();  // nobody leaves while its sums are read
    else
        __syncthreads();
    dev::tc_fence_after();
    if (warp == kProductWarp) dev::tmem_dealloc(tmem, kBuffers * kN);
    if (p.beside) dev::wait_for_previous();  // what comes after this kernel comes after both
}

// Parts of k, as long as there are not many more CTAs than SMs and a part has two blocks.  In us
// for 1, 2, 4 and 8: one row through 4096 x 4096 (32 tiles) 15.3, 10.6, 8.5, 8.8, through
// 14,336 x 4096 (112) 17.4, 15.9, 19.2, 27.4; 64 rows through 6144 x 4096 (48) 17.5, 13.0, 12.0,
// 18.0; 16 through 1024 x 4096 (8) 14.8, 10.1, 7.6, 6.6.
int split_of(int64_t tiles, int blocks) {
    static const int sms = sm_count();
    int split = 1;
    while (split < 8 && tiles * split * 10 <= 8 * sms && blocks >= 4 * split) split *= 2;
    return split;
}

int64_t tiles_of(const GemmFp8& g) { return (g.m + kM - 1) / kM * ((g.n + kN - 1) / kN); }

// Whether the CTAs quantise the rows themselves, which saves a launch and a workspace but holds the
// products up by the rows' way through registers.  In us on the device alone, in a graph (in a loop of
// calls), with and without, the weights of several layers in turn:
//   1 row: 2048 x 2048 7.2, 7.6 (10.0, 11.6), 4096 x 2048 7.7, 7.3 (10.3, 11.6), 4096 x 4096 10.1, 10.1 (12.4, 12.5),
//     6144 x 4096 11.0, 11.9 (12.9, 14.3), 5120 x 5120 13.0, 12.3 (15.2, 14.5), 8192 x 4096 15.4, 14.3 (17.0, 16.5)
//   8 rows: 4096 x 4096 10.5, 10.5 (12.4, 12.5), 6144 x 4096 11.9, 12.2 (14.4, 14.5), 8192 x 4096 16.1, 14.4 (18.5, 16.5)
//   16 rows: 2048 x 2048 8.2, 8.2 (10.3, 11.9), 2048 x 4096 9.8, 9.2 (12.4, 11.8), 4096 x 4096 12.9, 10.7 (14.6, 12.6),
//     8192 x 4096 19.8, 14.7 (21.8, 16.5)
constexpr int64_t kOwnWeights = 24 << 20, kOwnWeightsMore = 4 << 20;  // up to 8 rows; more
bool own_rows(const GemmFp8& g, int blocks) {
    const int split = split_of(tiles_of(g), blocks);
    return g.m <= kOwnRows && g.n * g.k <= (g.m <= 8 ? kOwnWeights : kOwnWeightsMore) &&
           (g.m + 7) / 8 * 8 * kBlock * ((blocks + split - 1) / split) <= kOwnBytes;
}

template <bool OWN>
int launch(const GemmFp8& g, GemmFp8Params p, const RowsToQuantize& q, bool follows, cudaStream_t stream) {
    CUtensorMap map_a{}, map_b;
    // With few rows only those are loaded (in multiples of 8): the products of the others' memory,
    // whatever it holds, go to rows that nobody stores.  (Rows past the end as zeros: one row
    // through 14,336 x 4096 took 22 us instead of 13.)
    const int rows_loaded = (int)std::min<int64_t>((g.m + 7) / 8 * 8, kM);
    if (!OWN)
        MXK_CHECK(encode_tensor_map_2d(&map_a, g.a, (uint64_t)g.k, (uint64_t)g.m, (uint64_t)g.k, kBlock, rows_loaded,
                                       CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B));
    MXK_CHECK(encode_tensor_map_2d(&map_b, g.b, (uint64_t)g.k, (uint64_t)g.n, (uint64_t)g.k, kBlock, kN,
                                   CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B));
    constexpr int smem = OWN ? kOwnSmem : kSmem;
    static thread_local int ready_device = -1;
    int dev = 0;
    MXK_CUDA(cudaGetDevice(&dev));
    if (ready_device != dev) {
        MXK_CUDA(cudaFuncSetAttribute(gemm_fp8_tile_kernel<OWN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ready_device = dev;
    }
    p.tiles_m = (p.m + kM - 1) / kM;
    const int64_t tiles = tiles_of(g);
    const int split = split_of(tiles, p.blocks);
    MXK_REQUIRE(tiles * split <= std::numeric_limits<int>::max(), "gemm_fp8: too much work for one call");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * split));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = follows ? 2 : 1;
    LaunchScope scope(OWN ? "linear_fp8" : "gemm_fp8", stream);
    MXK_CUDA(cudaLaunchKernelEx(&cfg, gemm_fp8_tile_kernel<OWN>, map_a, map_b, p, q, split, rows_loaded));
    return MXK_OK;
}

}  // namespace tile

// ------------------------------------------------------------------ large products

namespace pair {

// A pair of CTAs holds 256 rows and 256 columns: each loads its 128 rows of A and 128 of the 256
// rows of B, which the pair's products read from both.  The pairs stay and go from tile to tile.
// Eight warps add up (16 at half the registers were slower), the scales' factors come from
// warps of their own (loaded by the adding ones they held them up: 8192^3 483 us instead of 459).
constexpr int kM = 256, kN = 256;
constexpr int kStages = 4, kBuffers = 2;
constexpr int kSide = 128 * kBlock;  // bytes of an operand's tile in one CTA
constexpr int kStage = 2 * kSide;
constexpr int kSumWarps = 8, kLoadWarp = 8, kProductWarp = 9, kThreads = 384;
constexpr int kLaunchRegs = 168, kSumRegs = 216, kOtherRegs = 72;
static_assert(256 * kSumRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "");
constexpr int kCols = kN / 2;        // columns of a warp: four lane quarters, two halves
constexpr int kGroup = 4, kGroups = 4;  // blocks whose scales come together; groups at hand
constexpr int kScales = kGroups * kGroup * 2 * 128 * 4;  // bytes
constexpr int kSmem = kStages * kStage + kScales + kSumWarps * 8192 + 1024;  // 1024: alignment
constexpr int kScaleWarps = 2;          // the last two
constexpr int kRaster = 8;           // row tiles that are gone through side by side

struct Shared {
    uint64_t full[kStages];   // (even CTA) both CTAs' tiles are loaded
    uint64_t done[kStages];   // multiplied, so the sums are in TMEM
    uint64_t taken[kBuffers]; // (even CTA) a buffer's sums have been read by both CTAs
    uint64_t scales_full[kGroups], scales_free[kGroups];
    uint64_t drain;
    int abort_word;
    uint32_t tmem;
};

// Tiles are numbered so that those at hand at a time share operands: kRaster row tiles, column
// tile by column tile.
__device__ __forceinline__ void place_of(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int band = tile / (kRaster * tiles_n), first = band * kRaster, high = min(kRaster, tiles_m - first);
    const int in = tile - first * tiles_n;
    tn = in / high;
    tm = first + in - tn * high;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                         const __grid_constant__ CUtensorMap map_out, const GemmFp8Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) Shared sh;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(kFull, tid >> 5, 0);
    const int rank = blockIdx.x & 1, pairs = gridDim.x >> 1;
    const int tiles_n = (p.n + kN - 1) / kN, tiles = p.tiles_m * tiles_n;
    volatile int* abort = &sh.abort_word;
    // a[row] b[half of the columns] of the groups' blocks: [group][block][half][row]
    float* scales = reinterpret_cast<float*>(smem + kStages * kStage);
    uint8_t* out_stage = smem + kStages * kStage + kScales;

    if (tid == 0) {
        sh.abort_word = 0;
        for (int i = 0; i < kStages; ++i) dev::mbar_init(&sh.full[i], 1), dev::mbar_init(&sh.done[i], 1);
        for (int i = 0; i < kBuffers; ++i) dev::mbar_init(&sh.taken[i], 2 * kSumWarps);
        for (int i = 0; i < kGroups; ++i) dev::mbar_init(&sh.scales_full[i], 1), dev::mbar_init(&sh.scales_free[i], kSumWarps);
        dev::mbar_init(&sh.drain, 1);
        dev::fence_barrier_init();
    }
    if (warp == kProductWarp) dev::tmem_alloc_pair(&sh.tmem, kBuffers * kN);
    if (warp == kLoadWarp && lane == 0) dev::prefetch_tensor_map(&map_a), dev::prefetch_tensor_map(&map_b);
    dev::tc_fence_before();
    __syncthreads();
    dev::cluster_arrive(), dev::cluster_wait();  // the other CTA's barriers are there
    dev::tc_fence_after();
    const uint32_t tmem = __shfl_sync(kFull, sh.tmem, 0);

    if (warp < kSumWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        const int half = warp >> 2;
        const uint32_t column = tmem + ((uint32_t)(warp & 3) << 21) + half * kCols;
        const uint32_t taken = dev::in_cta(dev::smem_addr(&sh.taken[0]), 0);
        const float* my_scales = scales + half * 128 + (warp & 3) * 32 + lane;
        dev::wait_for_previous();
        int stage = 0, buffer = 0, group = 0;
        uint32_t phase = 0, group_phase = 0;
        bool ok = true;
        for (int tile = blockIdx.x >> 1; tile < tiles && ok; tile += pairs) {
            int tm, tn;
            place_of(tile, p.tiles_m, tiles_n, tm, tn);
            const int row0 = tm * kM + rank * 128 + (warp & 3) * 32, col = tn * kN + half * kCols;
            float2 acc[kCols / 2];
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
            for (int i = 0; i < p.blocks; ++i) {
                if (i % kGroup == 0) ok = __all_sync(kFull, dev::mbar_wait(&sh.scales_full[group], group_phase, abort, p.err));
                if (!ok) break;
                const float f = my_scales[(group * kGroup + i % kGroup) * 256];
                ok = __all_sync(kFull, dev::mbar_wait(&sh.done[stage], phase, abort, p.err));
                if (!ok) break;
                dev::tc_fence_after();
                uint32_t v[2][16];
                dev::tmem_ld_32x32b_x16(column + buffer * kN, v[0]);
#pragma unroll
                for (int c = 0; c < kCols / 16; ++c) {
                    dev::tmem_wait_ld();
                    if (c + 1 < kCols / 16) {
                        dev::tmem_ld_32x32b_x16(column + buffer * kN + 16 * (c + 1), v[(c + 1) & 1]);
                    } else {
                        dev::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) dev::cluster_mbar_arrive(taken + 8 * buffer);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        acc[8 * c + k] =
                            __ffma2_rn(make_float2(__uint_as_float(v[c & 1][2 * k]), __uint_as_float(v[c & 1][2 * k + 1])),
                                       make_float2(f, f), acc[8 * c + k]);
                }
                if (++stage == kStages) stage = 0, phase ^= 1;
                if (++buffer == kBuffers) buffer = 0;
                if (i % kGroup == kGroup - 1 || i + 1 == p.blocks) {
                    __syncwarp();
                    if (lane == 0) dev::mbar_arrive(&sh.scales_free[group]);
                    if (++group == kGroups) group = 0, group_phase ^= 1;
                }
            }
            if (ok) store_rows(p, &map_out, out_stage + warp * 8192, row0, col, acc);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kLoadWarp) {
            if (dev::elect_one()) {
                const uint32_t full = dev::in_cta(dev::smem_addr(&sh.full[0]), 0);
                int stage = 0;
                int64_t issued = 0;
                uint32_t phase = 1;  // the first pass over the stages finds them free
                bool ok = true;
                dev::wait_for_previous();
                dev::let_next_start();  // a kernel beside this one reads the same rows, which are there now
                for (int tile = blockIdx.x >> 1; tile < tiles && ok; tile += pairs) {
                    int tm, tn;
                    place_of(tile, p.tiles_m, tiles_n, tm, tn);
                    for (int i = 0; i < p.blocks; ++i) {
                        ok = dev::mbar_wait(&sh.done[stage], phase, abort, p.err);
                        if (!ok) break;
                        if (rank == 0) dev::mbar_arrive_expect_tx(&sh.full[stage], 2 * kStage);
                        uint8_t* at = smem + stage * kStage;
                        dev::tma_load_2d_pair(at, &map_a, i * kBlock, tm * kM + rank * 128, full + 8 * stage);
                        dev::tma_load_2d_pair(at + kSide, &map_b, i * kBlock, tn * kN + rank * 128, full + 8 * stage);
                        ++issued;
                        if (++stage == kStages) stage = 0, phase ^= 1;
                    }
                }
                if (!ok && rank == 0)  // copies in flight must not outlive the CTAs' memory
                    for (int64_t k = issued > kStages ? issued - kStages : 0; k < issued; ++k)
                        settle(&sh.full[k % kStages], (uint32_t)(k / kStages) & 1u);
            }
            __syncwarp();
        } else if (warp >= kThreads / 32 - kScaleWarps) {
            // Each of these warps takes every other group, four rows a lane: under way while tiles
            // stream past, such a load takes up to 2000 cycles.
            dev::wait_for_previous();
            int count = 0;
            bool ok = true;
            for (int tile = blockIdx.x >> 1; tile < tiles && ok; tile += pairs) {
                int tm, tn;
                place_of(tile, p.tiles_m, tiles_n, tm, tn);
                const int row = tm * kM + rank * 128 + lane, block_n = tn * (kN / kBlock), last_n = (p.n - 1) / kBlock;
                const float* sb = p.b_scales + (int64_t)block_n * p.blocks;
                const float* sb1 = p.b_scales + (int64_t)min(block_n + 1, last_n) * p.blocks;
                for (int i = 0; i < p.blocks; i += kGroup, ++count) {
                    if (count % kScaleWarps != kThreads / 32 - 1 - warp) continue;
                    float a[4][kGroup], b0[kGroup], b1[kGroup];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        load_scales(p.a_scales + (int64_t)min(row + 32 * r, p.m - 1) * p.blocks, i, p.blocks, p.a_wide, a[r]);
                    load_scales(sb, i, p.blocks, p.b_wide, b0), load_scales(sb1, i, p.blocks, p.b_wide, b1);
                    const int group = count % kGroups;
                    ok = __all_sync(kFull, dev::mbar_wait(&sh.scales_free[group], ~(count / kGroups) & 1u, abort, p.err));
                    if (!ok) break;
                    float* to = scales + group * kGroup * 256 + lane;
#pragma unroll
                    for (int k = 0; k < kGroup; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            to[k * 256 + 32 * r] = a[r][k] * b0[k], to[k * 256 + 128 + 32 * r] = a[r][k] * b1[k];
                    __syncwarp();
                    if (lane == 0) dev::mbar_arrive(&sh.scales_full[group]);
                }
            }
        } else if (warp == kProductWarp && rank == 0) {
            constexpr uint32_t idesc = dev::f16_idesc(kM, kN, false);
            const uint64_t a_desc = dev::smem_desc(dev::smem_addr(smem), 16, 1024, dev::kLayoutSwizzle128);
            int stage = 0, buffer = 0;
            uint32_t phase = 0, taken_phase = 1;
            bool ok = true;
            for (int tile = blockIdx.x >> 1; tile < tiles && ok; tile += pairs) {
                for (int i = 0; i < p.blocks; ++i) {
                    ok = __all_sync(kFull, dev::mbar_wait_lean(&sh.full[stage], phase, abort, p.err)) &&
                         __all_sync(kFull, dev::mbar_wait_lean(&sh.taken[buffer], taken_phase, abort, p.err));
                    if (!ok) break;
                    dev::tc_fence_after();
                    if (dev::elect_one()) {
                        const uint64_t a = a_desc + (uint64_t)(stage * (kStage >> 4)), b = a + (kSide >> 4);
#pragma unroll
                        for (int k = 0; k < kBlock / 32; ++k)
                            dev::tc_mma_f8_pair(tmem + buffer * kN, a + 2 * k, b + 2 * k, idesc, k > 0);
                        dev::tc_commit_pair(&sh.done[stage]);
                    }
                    __syncwarp();
                    if (++stage == kStages) stage = 0, phase ^= 1;
                    if (++buffer == kBuffers) buffer = 0, taken_phase ^= 1;
                }
            }
            if (!ok && dev::elect_one()) {
                dev::tc_commit_pair(&sh.drain);
                settle(&sh.drain, 0);
            }
            __syncwarp();
        }
    }
    dev::tc_fence_before();
    __syncthreads();
    dev::cluster_arrive(), dev::cluster_wait();  // nobody leaves while the other CTA arrives or multiplies
    dev::tc_fence_after();
    if (warp == kProductWarp) dev::tmem_dealloc_pair(tmem, kBuffers * kN);
}

// Sets the kernel up on the current device; how many pairs it holds at a time.
int prepare(int* pairs) {
    static thread_local int ready_device = -1, most_pairs = 0;
    int dev = 0;
    MXK_CUDA(cudaGetDevice(&dev));
    if (ready_device != dev) {
        MXK_CUDA(cudaFuncSetAttribute(gemm_fp8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        cudaFuncAttributes attr{};
        MXK_CUDA(cudaFuncGetAttributes(&attr, gemm_fp8_pair_kernel));
        if (attr.numRegs != kLaunchRegs)
            return fail(MXK_ERR_UNSUPPORTED, "gemm_fp8: kernel built with " + std::to_string(attr.numRegs) +
                                                 " registers, the register split needs " + std::to_string(kLaunchRegs));
        // Pairs lie in one GPC each, so there can be fewer than half the SMs.
        cudaLaunchConfig_t all{};
        all.gridDim = dim3((unsigned)sm_count() / 2 * 2), all.blockDim = dim3(kThreads), all.dynamicSmemBytes = kSmem;
        MXK_CUDA(cudaOccupancyMaxActiveClusters(&most_pairs, gemm_fp8_pair_kernel, &all));
        MXK_REQUIRE(most_pairs > 0, "gemm_fp8: the device holds no pair of CTAs");
        ready_device = dev;
    }
    *pairs = most_pairs;
    return MXK_OK;
}

int launch(const GemmFp8& g, GemmFp8Params p, int most_pairs, bool follows, cudaStream_t stream) {
    CUtensorMap map_a, map_b;
    MXK_CHECK(encode_tensor_map_2d(&map_a, g.a, (uint64_t)g.k, (uint64_t)g.m, (uint64_t)g.k, kBlock, 128,
                                   CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B));
    MXK_CHECK(encode_tensor_map_2d(&map_b, g.b, (uint64_t)g.k, (uint64_t)g.n, (uint64_t)g.k, kBlock, 128,
                                   CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B));
    p.tiles_m = (p.m + kM - 1) / kM;
    const int64_t tiles = (int64_t)p.tiles_m * ((p.n + kN - 1) / kN);
    MXK_REQUIRE(tiles <= std::numeric_limits<int>::max() / 2, "gemm_fp8: too much work for one call");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, most_pairs)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    CUtensorMap map_out{};
    if (p.out_wide) {
        const bool full = p.dtype == MXK_F32;
        MXK_CHECK(encode_tensor_map_2d(&map_out, g.out, (uint64_t)p.copied, (uint64_t)g.m, (uint64_t)g.out_stride * (full ? 4 : 2),
                                       full ? 32 : 64, 32, full ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                                       CU_TENSOR_MAP_SWIZZLE_128B));
    }
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = follows ? 1 : 0;
    LaunchScope scope("gemm_fp8_pair", stream);
    MXK_CUDA(cudaLaunchKernelEx(&cfg, gemm_fp8_pair_kernel, map_a, map_b, map_out, p));
    return MXK_OK;
}

}  // namespace pair

int check_product(const char* who, int dtype, int64_t m, int64_t n, int64_t k, const void* b, const float* b_scales,
                  const void* out) {
    const std::string w(who);
    MXK_REQUIRE(dtype == MXK_F32 || dtype == MXK_F16 || dtype == MXK_BF16, w + ": unknown dtype");
    MXK_REQUIRE(m >= 0 && n >= 0 && k >= 0 && k % 16 == 0, w + ": k must be a multiple of 16, sizes not negative");
    MXK_REQUIRE(m < (1ll << 30) && n < (1ll << 30) && k < (1ll << 30), w + ": sizes must be below 2^30");
    if (m == 0 || n == 0) return MXK_OK;
    MXK_REQUIRE(out, w + ": out must be non-null");
    MXK_REQUIRE(reinterpret_cast<uintptr_t>(out) % (dtype == MXK_F32 ? 4 : 2) == 0, w + ": out must be aligned to its elements");
    if (k == 0) return MXK_OK;
    MXK_REQUIRE(b && b_scales, w + ": an operand is null");
    MXK_REQUIRE(reinterpret_cast<uintptr_t>(b) % 16 == 0 && reinterpret_cast<uintptr_t>(b_scales) % 4 == 0,
                w + ": operands must be aligned to 16 bytes, scales to 4");
    return MXK_OK;
}

// At most pairs / kLastTiles tiles are such, of kLastK features at least.  us without and with: 512 x 9728 x
// 4096 (76 tiles) 34.5, 28.5, 512 x 9984 x 8192 (78) 62, 48, 2560 x 2048 x 14,336 (80) 112, 85, 1280 x 4096 x 4096
// (80) 38.0, 36.1, 1024 x 19,200 x 4096 (300) 91, 80, 2048 x 14,336 x 4096 (448) 110.4, 110.2 (power); with
// fewer features 2048 x 2560 x 2048 (80) 21.5, 22.1, 1280 x 4096 x 1024 16, 21.
constexpr int kLastTiles = 2, kLastK = 4096;

GemmFp8Params params_of(const GemmFp8& g, unsigned* err) {
    const int size = g.dtype == MXK_F32 ? 4 : 2;
    GemmFp8Params p{};
    p.m = (int)g.m, p.n = (int)g.n;
    p.blocks = (int)((g.k + kBlock - 1) / kBlock);
    p.a_scales = g.a_scales, p.b_scales = g.b_scales;
    p.out = static_cast<char*>(g.out);
    p.out_stride = g.out_stride;
    p.dtype = g.dtype;
    p.out_vec = (reinterpret_cast<uintptr_t>(g.out) | (uint64_t)(g.out_stride * size)) % (4 * size) == 0;
    p.copied = (int)(g.n * size / 16 * 16 / size);
    p.out_wide = (reinterpret_cast<uintptr_t>(g.out) | (uint64_t)(g.out_stride * size)) % 16 == 0 && p.copied > 0;
    p.a_wide = p.blocks % 4 == 0 && reinterpret_cast<uintptr_t>(g.a_scales) % 16 == 0;
    p.b_wide = p.blocks % 4 == 0 && reinterpret_cast<uintptr_t>(g.b_scales) % 16 == 0;
    p.err = err;
    return p;
}

// Large products: the pairs, but where the last few tiles would keep all waiting for a whole
// tile's time, the columns that they lie in go to the other kernel, whose CTAs start as pairs end.
int gemm_fp8_large(const GemmFp8& g, unsigned* err, bool follows, cudaStream_t stream) {
    int pairs;
    MXK_CHECK(pair::prepare(&pairs));
    const int64_t tiles_m = (g.m + pair::kM - 1) / pair::kM, tiles = tiles_m * ((g.n + pair::kN - 1) / pair::kN);
    const int64_t rest = tiles % pairs, columns = (rest + tiles_m - 1) / tiles_m;  // of tiles
    GemmFp8 first = g, last = g;
    const bool split = rest > 0 && tiles > pairs && columns * tiles_m * kLastTiles <= pairs && g.k >= kLastK;
    if (split) {
        first.n = g.n / pair::kN * pair::kN - (columns - (g.n % pair::kN != 0)) * pair::kN;
        last.n = g.n - first.n;
        last.b = g.b + first.n * g.k;
        last.b_scales = g.b_scales + first.n / kBlock * ((g.k + kBlock - 1) / kBlock);
        last.out = static_cast<char*>(g.out) + first.n * (g.dtype == MXK_F32 ? 4 : 2);
    }
    MXK_CHECK(pair::launch(first, params_of(first, err), pairs, follows, stream));
    if (!split) return MXK_OK;
    GemmFp8Params p = params_of(last, err);
    p.beside = 1;
    return tile::launch<false>(last, p, RowsToQuantize{}, true, stream);
}

// q: rows to quantise on the way, which tile::own_rows allows, in place of g.a.
int gemm_fp8(const GemmFp8& g, const RowsToQuantize* q, bool follows, cudaStream_t stream) {
    unsigned* err = device_error_word();
    if (!err) return fail(MXK_ERR_CUDA, "gemm_fp8: cannot allocate the device error word");
    if (q) return tile::launch<true>(g, params_of(g, err), *q, false, stream);
    // Pairs from 28 tiles on: fewer leave SMs idle that the split of K puts to work.  us, pairs | tiles:
    //   512 x 4096 x 4096 (32) 18.8 | 20.9, 512 x 8192 x 8192 (64) 33.7 | 51.0, 2048 x 4096 x 4096 (128) 34.9 | 54.5,
    //   512 x 4096 x 512 (32) 7.5 | 8.3, 256 x 7168 x 4096 (28) 18.7 | 19.2, 640 x 2048 x 4096 (24) 18.6 | 18.5,
    //   256 x 6144 x 16,384 (24) 57.3 | 50.4, 256 x 4096 x 4096 (16) 18.2 | 14.3.
    // Rows of one of the smaller tiles leave half a pair without work: 129 x 8192 x 4096 18.6 | 20.7.
    if (g.m > tile::kM && (g.m + pair::kM - 1) / pair::kM * ((g.n + pair::kN - 1) / pair::kN) >= 28)
        return gemm_fp8_large(g, err, follows, stream);
    return tile::launch<false>(g, params_of(g, err), RowsToQuantize{}, follows, stream);
}

// Products of no features.
int zero_out(const GemmFp8& g, cudaStream_t stream) {
    const size_t size = g.dtype == MXK_F32 ? 4 : 2;
    MXK_CUDA(cudaMemset2DAsync(g.out, (size_t)g.out_stride * size, 0, (size_t)g.n * size, (size_t)g.m, stream));
    return MXK_OK;
}

}  // namespace
}  // namespace mxk

extern "C" {

int mxk_gemm_fp8(int dtype, int64_t m, int64_t n, int64_t k, const uint8_t* a, const float* a_scales, const uint8_t* b,
                 const float* b_scales, void* out, int64_t out_stride, void* stream) {
    using namespace mxk;
    MXK_CHECK(check_product("gemm_fp8", dtype, m, n, k, b, b_scales, out));
    MXK_REQUIRE(out_stride >= n, "gemm_fp8: out_stride must be at least n");
    if (m == 0 || n == 0) return MXK_OK;
    const GemmFp8 g{dtype, m, n, k, a, a_scales, b, b_scales, out, out_stride};
    if (k == 0) return zero_out(g, as_stream(stream));
    MXK_REQUIRE(a && a_scales, "gemm_fp8: an operand is null");
    MXK_REQUIRE(reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(a_scales) % 4 == 0,
                "gemm_fp8: operands must be aligned to 16 bytes, scales to 4");
    return gemm_fp8(g, nullptr, false, as_stream(stream));
}

int mxk_linear_fp8(int dtype, int64_t m, int64_t n, int64_t k, const void* x, int64_t x_stride, const uint8_t* b,
                   const float* b_scales, void* out, int64_t out_stride, void* stream) {
    using namespace mxk;
    MXK_CHECK(check_product("linear_fp8", dtype, m, n, k, b, b_scales, out));
    MXK_REQUIRE(out_stride >= n, "linear_fp8: out_stride must be at least n");
    if (m == 0 || n == 0) return MXK_OK;
    GemmFp8 g{dtype, m, n, k, nullptr, nullptr, b, b_scales, out, out_stride};
    const cudaStream_t st = as_stream(stream);
    if (k == 0) return zero_out(g, st);
    MXK_REQUIRE(x && reinterpret_cast<uintptr_t>(x) % (dtype == MXK_F32 ? 4 : 2) == 0,
                "linear_fp8: x must be non-null and aligned to its elements");
    const int64_t blocks = (k + kBlock - 1) / kBlock;
    if (tile::own_rows(g, (int)blocks)) {
        const int size = dtype == MXK_F32 ? 4 : 2;
        const bool wide = (reinterpret_cast<uintptr_t>(x) | (uint64_t)(x_stride * size)) % 16 == 0;
        const RowsToQuantize q{x, x_stride, dtype, wide, (int)k};
        return gemm_fp8(g, &q, false, st);
    }
    const size_t values = ((size_t)m * k + 255) / 256 * 256;
    cudaMemPool_t pool = workspace_pool();
    if (!pool) return fail(MXK_ERR_CUDA, "linear_fp8: cannot create the workspace pool");
    void* work = nullptr;
    MXK_CUDA(cudaMallocFromPoolAsync(&work, values + (size_t)m * blocks * 4, pool, st));
    uint8_t* a = static_cast<uint8_t*>(work);
    float* scales = reinterpret_cast<float*>(a + values);
    g.a = a, g.a_scales = scales;
    int status = launch_quantize_fp8({dtype, 1, m, k, x, x_stride, a, scales}, st);
    if (status == MXK_OK) status = gemm_fp8(g, nullptr, true, st);
    const cudaError_t freed = cudaFreeAsync(work, st);
    MXK_CHECK(status);
    MXK_CUDA(freed);
    return MXK_OK;
}

}  // extern "C"
