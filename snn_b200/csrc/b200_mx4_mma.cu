// The product of two packed 4-bit matrices on the tensor cores.
//
// tcgen05.mma kind::mxf4 multiplies 4-bit operands with a scale byte for every
// 32 of them and adds in 32 bits in tensor memory, 64 of k an instruction. The
// weights are the operand of 128 rows, x the one of BN rows, so an accumulator
// lane is an output feature and a column a row of x: a warp reads 32
// neighbouring features of a column at a time and writes them as one run, and
// few rows of x cost a narrow instruction, not a padded one.
//
// A stage holds 256 of k: 128 bytes a row for both operands (TMA, 128-byte
// swizzle) and their scales, which lie in memory as the 512-byte tiles that
// tcgen05.cp spreads over the lanes (row r of a 128-row tile: lane r % 32,
// column r / 32, a byte for each of 4 blocks). Rows and columns behind the
// matrices are zero (TMA's fill, and the packer's for scales); a scale tile
// that is not loaded belongs to k or rows that no instruction or store uses.
//
// One warp issues the loads, one the instructions; the others read the
// accumulators and write. Two forms share this:
//  * pairs: two CTAs on two SMs share 256 x 256 tiles, one after another; the
//    accumulators are moved to registers and given back before they are
//    written, so that the writes of a tile overlap the next one's instructions.
//  * skinny: one tile a CTA and BN down to 16, the k of a tile split over the
//    CTAs of a cluster, which add their parts through shared memory in the
//    order of their ranks. Up to 16 rows of x are packed on the way: four more
//    warps write their codes and scales where the copies would have put them.
// Every wait is bounded; one that gives up makes its tile NaN.
#include "b200_mx4.cuh"
#include "b200_tma.h"

#include <algorithm>
#include <type_traits>

namespace b200 {
namespace mx4 {
namespace {

constexpr uint32_t kRows = 128;        // weight rows of a tile
constexpr uint32_t kStageK = 256;      // k of a stage
constexpr uint32_t kStageBytes = 128;  // of a row
constexpr uint32_t kScaleTile = 512;

using tma::bar_arrive;
using tma::bar_expect;
using tma::bar_init;
using tma::bar_wait;
using tma::load_box;
using tma::load_run;
using tma::smem_of;

// ---- tensor memory and instructions ----
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_of(slot)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_of(bar))
                 : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect() {
    uint32_t on;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(on));
    return on != 0;
}
// Descriptors of shared memory, of which only the low word changes: operands
// are rows of 128 bytes in 8-row groups of 1024, swizzled by 128 bytes; scales
// 32 rows of 16 bytes, one behind the other.
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29, kScaleHigh = 128 >> 4 | 1u << 14;
__device__ __forceinline__ uint32_t desc_low(uint32_t smem) { return (smem & 0x3ffffu) >> 4 | 1u << 16; }

template <bool Pair>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t low) {
    if constexpr (Pair)
        asm volatile("{\n .reg .b64 d;\n mov.b64 d, {%1, %2};\n tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n}" ::"r"(tmem),
                     "r"(low), "n"(kScaleHigh)
                     : "memory");
    else
        asm volatile("{\n .reg .b64 d;\n mov.b64 d, {%1, %2};\n tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n}" ::"r"(tmem),
                     "r"(low), "n"(kScaleHigh)
                     : "memory");
}
// Both operands e2m1, K-major; scales ue8m0; m x n. The scale bytes of 64 of
// k are the low or the high half of a scale column's word.
constexpr uint32_t instruction(uint32_t m, uint32_t n, uint32_t half) {
    return (half * 2u) << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | 1u << 23 | (m >> 7) << 27 | (half * 2u) << 29;
}
template <bool Pair>
__device__ __forceinline__ void multiply(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t add) {
    if constexpr (Pair)
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.u32 p, %6, 0;\n mov.b64 a, {%1, %7};\n mov.b64 b, {%2, %7};\n"
            " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(add), "n"(kOperandHigh)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.u32 p, %6, 0;\n mov.b64 a, {%1, %7};\n mov.b64 b, {%2, %7};\n"
            " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(add), "n"(kOperandHigh)
            : "memory");
}
// A loaded stage's instructions, by one thread: weights at w, BN rows of x at x
// (of which this CTA may hold half), their scales at ws and xs; d the accumulators,
// sf the stage's tensor memory columns for scales; pieces of 64 of k. What changes
// from stage to stage is few additions, as the issuing thread has to keep ahead.
template <bool Pair, uint32_t BN>
__device__ __forceinline__ void issue_stage(uint32_t w, uint32_t x, uint32_t ws, uint32_t xs, uint32_t d, uint32_t sf,
                                            uint32_t pieces, uint32_t add) {
    constexpr uint32_t kM = Pair ? 256 : 128, kR = (BN + 127) / 128;
    const uint32_t a = desc_low(w), b = desc_low(x), cs = desc_low(ws), cx = desc_low(xs);
    // The second half's scales behind the first half's products, which they overlap.
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) {
        if (t * 2 >= pieces) return;
        copy_scales<Pair>(sf + 4 * t, cs + t * (512 >> 4));
#pragma unroll
        for (uint32_t r = 0; r < kR; ++r)
            copy_scales<Pair>(sf + 8 + 4 * (t * kR + r), cx + (r * 2 + t) * (512 >> 4));
#pragma unroll
        for (uint32_t q = 2 * t; q < 2 * t + 2; ++q)
            if (q < pieces)
                multiply<Pair>(d, a + q * 2, b + q * 2, instruction(kM, BN, q & 1), sf + 4 * (q / 2),
                               sf + 8 + 4 * kR * (q / 2), q ? 1u : add);
    }
}
// 16 accumulator columns of the warp's 32 lanes.
__device__ __forceinline__ void read_columns(uint32_t at, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void read_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Behind read_done: nothing that uses the columns moves before it.
__device__ __forceinline__ void settle(float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(v[i]));
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
// ---- a tile's k loop ----
template <uint32_t BN>
struct Shape {
    static constexpr uint32_t kScaleRows = (BN + 127) / 128;  // scale tiles across x's rows
    static constexpr uint32_t kW = kRows * kStageBytes, kX = BN * kStageBytes;
    static constexpr uint32_t kWScales = 2 * kScaleTile, kXScales = 2 * kScaleTile * kScaleRows;
    static constexpr uint32_t kStage = kW + kX + kWScales + kXScales;  // a multiple of 1024
    static constexpr uint32_t kScaleColumns = 8 + 8 * kScaleRows;      // tensor memory columns of a stage's scales
    // Offsets of a stage's parts.
    static constexpr uint32_t kAtX = kW, kAtWScales = kW + kX, kAtXScales = kW + kX + kWScales;
};

struct Problem {
    const void *x;  // plain x, rows of x_stride elements
    int64_t x_stride;
    const uint8_t *x_scales, *w_scales;
    uint32_t m, n, k, scale_tiles;  // scale tiles along k
    const float *bias;
    void *out;
    int64_t row_stride;
    uint32_t tiles_n, tiles_m, splits, stages;  // stages along k
};

// Loads stage `at` (of k) of a tile into slot memory; Plain x is packed there by others.
template <uint32_t BN, bool Plain = false>
__device__ __forceinline__ void load_stage(const Problem &p, const CUtensorMap *wm, const CUtensorMap *xm,
                                           uint32_t slot, uint64_t *full, uint32_t at, uint32_t j0, uint32_t i0) {
    using S = Shape<BN>;
    const uint32_t tile = at * 2, bytes = kScaleTile * min(2u, p.scale_tiles - tile);
    const uint32_t row_tiles = min(S::kScaleRows, (p.m + 127) / 128 - i0 / 128);
    bar_expect(full, S::kW + bytes + (Plain ? 0 : S::kX + bytes * row_tiles));
    load_box(slot, wm, (int32_t)(at * kStageBytes), (int32_t)j0, full);
    load_run(slot + S::kAtWScales, p.w_scales + ((uint64_t)(j0 / 128) * p.scale_tiles + tile) * kScaleTile, bytes, full);
    if (Plain) return;
    load_box(slot + S::kAtX, xm, (int32_t)(at * kStageBytes), (int32_t)i0, full);
    for (uint32_t r = 0; r < row_tiles; ++r)
        load_run(slot + S::kAtXScales + r * 2 * kScaleTile,
                 p.x_scales + ((uint64_t)(i0 / 128 + r) * p.scale_tiles + tile) * kScaleTile, bytes, full);
}

template <typename T>
__device__ __forceinline__ void put(const Problem &p, uint32_t i, uint32_t j, float v) {
    ((T *)p.out)[(int64_t)i * p.row_stride + j] = from_float<T>(v);
}

constexpr uint32_t kNoValue = 0x7fffffffu;

// ---- pairs ----
// A pair of CTAs (cta_group::2) works on 256 weight rows and 256 rows of x: each
// CTA holds 128 of both in shared memory and the accumulators of its weight
// rows, and the instructions read x from both, so an SM loads 35 KB for 256 of k
// where a CTA of its own with 256 rows of x would load 52.
//
// 8192 x 8192 x 8192: 193 us, 5.7 PFLOP/s, the tensor pipe active 72% of the
// time. The bound was the issue (347 us while one lane of a divergent warp put
// the descriptors together; leaving out the loads or the stores changed nothing,
// leaving out the scale copies gave 277). 50000 x 784 x 1000 to f32: 49 us, of
// which the writes of 200 MB are 30; 16 warps read the accumulators there, as
// with 8 (43 against 33 us at 768 of k to bf16) a tile's writes took longer than
// its instructions.
constexpr uint32_t kPairN = 256, kPairStages = 6;
constexpr uint32_t kReaders = 16;  // warps that read and write accumulators: four share the lanes, kReaders / 4 the columns
constexpr uint32_t kPairThreads = 128 + kReaders * 32, kReadN = kPairN / (kReaders / 4);
constexpr uint32_t kPairX = 128 * kStageBytes, kPairW = kRows * kStageBytes;
// A stage: weights, x, the scales of the CTA's weights, of all of x's rows.
constexpr uint32_t kPairAtX = kPairW, kPairAtWScales = kPairW + kPairX, kPairAtXScales = kPairAtWScales + 2 * kScaleTile;
constexpr uint32_t kPairStage = kPairAtXScales + 4 * kScaleTile;
constexpr uint32_t kPairSmem = 1024 + kPairStages * kPairStage;
constexpr uint32_t kPairColumns = 24;  // tensor memory columns of a stage's scales
static_assert(kPairN + kPairStages * kPairColumns <= 512, "tensor memory");

struct PairMaps {
    CUtensorMap w, x, w_scales, x_scales;
};

// An address of this CTA's shared memory, in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(uint32_t smem, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem), "r"(rank));
    return at;
}
// Into this CTA's memory, counted by a barrier of either CTA of the pair.
__device__ __forceinline__ void load_pair(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_of(bar)),
        "h"((uint16_t)3)
        : "memory");
}
template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ Problem p) {
    extern __shared__ uint8_t s_raw[];
    __shared__ uint64_t s_full[kPairStages], s_empty[kPairStages], s_ready, s_free;
    __shared__ uint32_t s_tmem;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x & 31, rank = cluster_rank();
    const uint32_t base = (smem_of(s_raw) + 1023) & ~1023u;  // the same in both CTAs
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kPairStages; ++s) bar_init(&s_full[s], 1), bar_init(&s_empty[s], 1);
        bar_init(&s_ready, 1);
        bar_init(&s_free, 2 * kReaders);  // of both CTAs
        tma::bar_init_done();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_of(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    after_previous();
    const uint32_t tmem = s_tmem, tiles = p.tiles_n * p.tiles_m, pairs = gridDim.x / 2, pair = blockIdx.x / 2;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            uint32_t n = 0;  // stages so far
            for (uint32_t tile = pair; ok && tile < tiles; tile += pairs) {
                const uint32_t j0 = tile % p.tiles_n * 256 + rank * 128, i0 = tile / p.tiles_n * kPairN;
                for (uint32_t at = 0; at < p.stages; ++at, ++n) {
                    const uint32_t s = n % kPairStages, turn = n / kPairStages, slot = base + s * kPairStage;
                    ok = turn == 0 || bar_wait(&s_empty[s], (turn - 1) & 1);
                    if (!ok) break;
                    // Both CTAs' bytes are counted by the first one's barrier.
                    if (rank == 0) bar_expect(&s_full[s], 2 * kPairStage);
                    const uint32_t full = in_cta(smem_of(&s_full[s]), 0);
                    load_pair(slot, &maps.w, at * kStageBytes, j0, full);
                    load_pair(slot + kPairAtX, &maps.x, at * kStageBytes, i0 + rank * 128, full);
                    load_pair(slot + kPairAtWScales, &maps.w_scales, at * 256, j0 / 128, full);
                    load_pair(slot + kPairAtXScales, &maps.x_scales, at * 256, i0 / 128, full);
                }
            }
            // Let the last copies land before the CTAs may end.
            if (rank == 0)
                for (uint32_t d = 1; d <= kPairStages && d <= n; ++d)
                    bar_wait(&s_full[(n - d) % kPairStages], ((n - d) / kPairStages) & 1);
        }
    } else if (warp == 1) {
        // The whole warp keeps the count, so that what it issues lies in uniform registers.
        if (rank == 0) {
            const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0);
            uint32_t n = 0, count = 0, s = 0, parity = 0;
            for (uint32_t tile = pair; ok && tile < tiles; tile += pairs, ++count) {
                // Lanes give up one by one, and the warp goes on as a whole.
                ok = __all_sync(0xffffffffu, count == 0 || bar_wait(&s_free, (count - 1) & 1));
                fence_after();
                for (uint32_t at = 0; ok && at < p.stages; ++at, ++n) {
                    ok = __all_sync(0xffffffffu, bar_wait(&s_full[s], parity));
                    fence_after();
                    if (!ok) break;
                    const uint32_t slot = base + s * kPairStage;
                    if (elect()) {
                        issue_stage<true, kPairN>(slot, slot + kPairAtX, slot + kPairAtWScales, slot + kPairAtXScales, acc,
                                                  acc + kPairN + s * kPairColumns,
                                                  min(kStageK / 64, (p.k - at * kStageK + 63) / 64), at);
                        commit_pair(&s_empty[s]);
                    }
                    __syncwarp();
                    if (++s == kPairStages) s = 0, parity ^= 1;
                }
                if (ok && elect()) commit_pair(&s_ready);
                __syncwarp();
            }
        }
    } else if (warp >= 4) {
        const uint32_t quarter = warp & 3, part = (warp - 4) / 4;
        const uint32_t free = in_cta(smem_of(&s_free), 0);
        uint32_t count = 0;
        for (uint32_t tile = pair; tile < tiles; tile += pairs, ++count) {
            const uint32_t j = tile % p.tiles_n * 256 + rank * 128 + quarter * 32 + lane;
            const uint32_t i0 = tile / p.tiles_n * kPairN + part * kReadN;
            const float bias = p.bias && j < p.n ? p.bias[j] : 0.0f;
            ok = ok && bar_wait(&s_ready, count & 1);
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
            float v[kReadN / 16][16];
#pragma unroll
            for (uint32_t c = 0; c < kReadN / 16; ++c)
                read_columns(tmem + (quarter * 32 << 16) + part * kReadN + c * 16, v[c]);
            read_done();
#pragma unroll
            for (uint32_t c = 0; c < kReadN / 16; ++c) settle(v[c]);
            fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(free) : "memory");
            if (j < p.n) {
                T *to = (T *)p.out + (int64_t)i0 * p.row_stride + j;
                const uint32_t rows = i0 < p.m ? min(p.m - i0, kReadN) : 0;
#pragma unroll
                for (uint32_t c = 0; c < kReadN / 16; ++c)
#pragma unroll
                    for (uint32_t q = 0; q < 16; ++q) {
                        if (c * 16 + q < rows)
                            __stcs(to, from_float<T>(ok ? __fadd_rn(v[c][q], bias) : __uint_as_float(kNoValue)));
                        to += p.row_stride;
                    }
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA's memory is used any more
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// ---- skinny form ----
// Four parts of k of 4 x 8192 x 8192 are one wave of 256 CTAs, two an SM: 8 to 10 us
// a launch among others, of which the 36 MB of weights are 5.5; the rest is set-up
// and the joining of the parts. Packing x on the way takes 16 rows in 13.1 us where
// a packing kernel before it makes 15.6 of 17 rows (the product itself 11.0); 32 rows
// took 22.7 on the way, 15.9 that way, so 16 rows are the most.
constexpr uint32_t kMostSplits = 8;
template <uint32_t BN>
struct Skinny {
    static constexpr uint32_t kStages = BN >= 128 ? 3 : BN >= 64 ? 4 : 5;  // two CTAs an SM
    static constexpr uint32_t kSmem = 1024 + kStages * Shape<BN>::kStage;
    static constexpr uint32_t kColumns = BN + kStages * Shape<BN>::kScaleColumns <= 128 ? 128 : 256;
    static_assert(BN + kStages * Shape<BN>::kScaleColumns <= kColumns, "tensor memory");
    static_assert(BN * kRows * 4 <= kStages * Shape<BN>::kStage, "the parts lie where the stages were");
};

__device__ __forceinline__ float4 read_remote(uint32_t smem, uint32_t rank) {
    const uint32_t at = in_cta(smem, rank);
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
}

// Packs a stage of plain x (rows of 16-byte pieces) into a slot: a lane a block of 32.
template <typename X, uint32_t BN>
__device__ __forceinline__ void pack_stage(const Problem &p, uint32_t slot, uint32_t at) {
    using S = Shape<BN>;
    constexpr uint32_t kPieces = kBlock / Piece<X>::kOwn, kRounds = BN * 8 / 32;
    constexpr uint32_t kHeld = kPieces * kRounds <= 16 ? kRounds : 16 / kPieces;  // rounds whose loads are under way
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (uint32_t round = 0; round < kRounds; round += kHeld) {
        Piece<X> v[kHeld][kPieces];
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h) {
            const uint32_t n = (round + h) * 32 + lane, r = n / 8, c = at * kStageK + n % 8 * kBlock;
#pragma unroll
            for (uint32_t q = 0; q < kPieces; ++q) {
                const uint32_t e = c + q * Piece<X>::kOwn;
                v[h][q] = r < p.m && e < p.k ? load_piece<true, true>((const X *)p.x + r * p.x_stride + e, p.k - e) : Piece<X>{};
            }
        }
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h) {
            const uint32_t n = (round + h) * 32 + lane, r = n / 8, b = n % 8;
            if (r >= p.m) continue;
            uint32_t top = 0, w[4];
#pragma unroll
            for (uint32_t q = 0; q < kPieces; ++q) top = max(top, v[h][q].largest());
            const uint32_t s = scale_byte(top);
            pack_block(v[h], s, w);
            // Chunk b of the row, where the 128-byte swizzle puts it.
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot + S::kAtX + r * kStageBytes + ((b ^ r % 8) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
            asm volatile("st.shared.u8 [%0], %1;" ::"r"(slot + S::kAtXScales + b / 4 * kScaleTile + scale_slot(r, b % 4)),
                         "r"(s)
                         : "memory");
        }
    }
}

struct None {};  // x is packed already

template <typename T, uint32_t BN, typename X>
__global__ void __launch_bounds__(std::is_same<X, None>::value ? 128 : 256)
    skinny_kernel(const __grid_constant__ CUtensorMap wm, const __grid_constant__ CUtensorMap xm, Problem p) {
    constexpr bool kPlain = !std::is_same<X, None>::value;
    constexpr uint32_t kSkinnyWarps = kPlain ? 8 : 4;
    using S = Shape<BN>;
    using K = Skinny<BN>;
    extern __shared__ uint8_t s_raw[];
    __shared__ uint64_t s_full[K::kStages], s_empty[K::kStages], s_ready;
    __shared__ uint32_t s_tmem;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
    const uint32_t base = (smem_of(s_raw) + 1023) & ~1023u;
    const uint32_t rank = p.splits > 1 ? cluster_rank() : 0;
    const uint32_t tile = blockIdx.x / p.splits;
    const uint32_t j0 = tile % p.tiles_n * kRows, i0 = tile / p.tiles_n * BN;
    // This CTA's stages along k.
    const uint32_t first = (uint32_t)((uint64_t)p.stages * rank / p.splits);
    const uint32_t count = (uint32_t)((uint64_t)p.stages * (rank + 1) / p.splits) - first;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < K::kStages; ++s) bar_init(&s_full[s], kPlain ? 33 : 1), bar_init(&s_empty[s], 1);
        bar_init(&s_ready, 1);
        tma::bar_init_done();
    }
    if (warp == 0) tmem_alloc(&s_tmem, K::kColumns);
    fence_before();
    __syncthreads();
    fence_after();
    // Only now that this CTA has its tensor memory: one of the next kernel's, which
    // ends after it, could hold what it waits for.
    allow_next();
    after_previous();
    const uint32_t tmem = s_tmem;
    bool ok = true;
    if (warp == 0 && lane == 0) {
        uint32_t n = 0;
        for (; ok && n < count; ++n) {
            const uint32_t s = n % K::kStages, turn = n / K::kStages;
            ok = turn == 0 || bar_wait(&s_empty[s], (turn - 1) & 1);
            if (!ok) break;
            load_stage<BN, kPlain>(p, &wm, &xm, base + s * S::kStage, &s_full[s], first + n, j0, i0);
        }
        for (uint32_t d = 1; d <= K::kStages && d <= n; ++d)
            bar_wait(&s_full[(n - d) % K::kStages], ((n - d) / K::kStages) & 1);
    } else if (warp == 1) {
        const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0);
        for (uint32_t n = 0; ok && n < count; ++n) {
            const uint32_t s = n % K::kStages;
            ok = __all_sync(0xffffffffu, bar_wait(&s_full[s], (n / K::kStages) & 1));
            fence_after();
            if (!ok) break;
            const uint32_t slot = base + s * S::kStage;
            if (elect()) {
                issue_stage<false, BN>(slot, slot + S::kAtX, slot + S::kAtWScales, slot + S::kAtXScales, acc,
                                       acc + BN + s * S::kScaleColumns,
                                       min(kStageK / 64, (p.k - (first + n) * kStageK + 63) / 64), n);
                commit(&s_empty[s]);
            }
            __syncwarp();
        }
        if (ok && elect()) commit(&s_ready);
    } else if (kPlain && warp >= 4) {
        // A stage a warp: the loads of four stages are under way at a time.
        if constexpr (kPlain)
            for (uint32_t n = warp - 4; ok && n < count; n += 4) {
                const uint32_t s = n % K::kStages, turn = n / K::kStages;
                ok = turn == 0 || bar_wait(&s_empty[s], (turn - 1) & 1);
                if (!ok) break;
                pack_stage<X, BN>(p, base + s * S::kStage, first + n);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(&s_full[s]);
            }
    }
    __syncwarp();
    const uint32_t feature = warp * 32 + lane, j = j0 + feature;
    const float bias = warp < 4 && p.bias && j < p.n ? p.bias[j] : 0.0f;
    ok = bar_wait(&s_ready, 0);
    ok = __all_sync(0xffffffffu, ok);
    fence_after();
    // All instructions are done, so the stages' memory is free.
#pragma unroll 1
    for (uint32_t c = 0; warp < 4 && c < BN; c += 16) {
        float v[16];
        read_columns(tmem + (warp * 32 << 16) + c, v);
        read_done();
        settle(v);
#pragma unroll
        for (uint32_t q = 0; q < 16; ++q) {
            const float part = ok ? v[q] : __uint_as_float(kNoValue);
            if (p.splits > 1)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + ((c + q) * kRows + feature) * 4), "f"(part) : "memory");
            else if (j < p.n && i0 + c + q < p.m)
                put<T>(p, i0 + c + q, j, __fadd_rn(part, bias));
        }
    }
    if (p.splits > 1) {
        // The ranks share the rows of x; a warp takes one at a time, a lane four features of it.
        cluster_sync();
        const uint32_t f = lane * 4;
        for (uint32_t c = rank * kSkinnyWarps + warp; c < BN && i0 + c < p.m; c += p.splits * kSkinnyWarps) {
            float4 part[kMostSplits];
#pragma unroll
            for (uint32_t r = 0; r < kMostSplits; ++r)
                if (r < p.splits) part[r] = read_remote(base + (c * kRows + f) * 4, r);
            float sum[4] = {};
#pragma unroll
            for (uint32_t r = 0; r < kMostSplits; ++r)
                if (r < p.splits) {
                    sum[0] = __fadd_rn(sum[0], part[r].x), sum[1] = __fadd_rn(sum[1], part[r].y);
                    sum[2] = __fadd_rn(sum[2], part[r].z), sum[3] = __fadd_rn(sum[3], part[r].w);
                }
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q)
                if (j0 + f + q < p.n)
                    put<T>(p, i0 + c, j0 + f + q, p.bias ? __fadd_rn(sum[q], p.bias[j0 + f + q]) : sum[q]);
        }
        cluster_sync();
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        tmem_free(tmem, K::kColumns);
    }
}

// ---- host side ----
// Boxes of `box` rows and 128 bytes of a packed matrix.
cudaError_t map_of(CUtensorMap *map, const Packed &q, uint64_t k, uint32_t box) {
    const cuuint64_t dims[2] = {blocks_of(k) * 16, q.rows}, strides[1] = {blocks_of(k) * 16};
    const cuuint32_t boxes[2] = {kStageBytes, box};
    return tma::encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, q.codes, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The scales of a packed matrix as rows of 512-byte tiles, two of them wide and `high` rows high.
cudaError_t scale_map_of(CUtensorMap *map, const Packed &q, uint64_t k, uint32_t high) {
    const cuuint64_t dims[2] = {scale_tiles(k) * 128, (q.rows + 127) / 128}, strides[1] = {scale_tiles(k) * 512};
    const cuuint32_t boxes[2] = {256, high};
    return tma::encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, q.scales, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <typename T>
cudaError_t launch_pairs(int device, cudaStream_t s, const Packed &x, const Packed &w, uint64_t k, const Problem &p) {
    PairMaps m;
    cudaError_t e = map_of(&m.w, w, k, 128);
    if (e == cudaSuccess) e = map_of(&m.x, x, k, 128);
    if (e == cudaSuccess) e = scale_map_of(&m.w_scales, w, k, 1);
    if (e == cudaSuccess) e = scale_map_of(&m.x_scales, x, k, 2);
    if (e == cudaSuccess) e = allow_smem<pair_kernel<T>>(kPairSmem);
    if (e != cudaSuccess) return e;
    const uint64_t tiles = (uint64_t)p.tiles_n * p.tiles_m, most = (uint64_t)sm_count(device) / 2;
    return launch_early(pair_kernel<T>, 2 * (uint32_t)std::min(tiles, most), kPairThreads, kPairSmem, s, 2, m, p);
}

template <typename T, uint32_t BN, typename X>
cudaError_t launch_skinny(cudaStream_t s, const CUtensorMap &wm, const CUtensorMap &xm, const Problem &p) {
    using K = Skinny<BN>;
    constexpr auto kernel = skinny_kernel<T, BN, X>;
    const cudaError_t e = allow_smem<kernel>(K::kSmem);
    if (e != cudaSuccess) return e;
    const uint32_t threads = std::is_same<X, None>::value ? 128 : 256;
    return launch_early(kernel, p.tiles_n * p.tiles_m * p.splits, threads, K::kSmem, s, p.splits, wm, xm, p);
}

Problem problem_of(uint64_t m, const Packed &w, uint64_t k, const float *bias, void *out, int64_t row_stride) {
    Problem p = {};
    p.w_scales = w.scales;
    p.m = (uint32_t)m, p.n = (uint32_t)w.rows, p.k = (uint32_t)k;
    p.scale_tiles = (uint32_t)scale_tiles(k);
    p.bias = bias, p.out = out, p.row_stride = row_stride;
    p.stages = (uint32_t)((k + kStageK - 1) / kStageK);
    p.tiles_n = (uint32_t)((w.rows + kRows - 1) / kRows);
    return p;
}
// As many parts of k (of two stages at least) as two CTAs an SM hold at once.
void split_k(int device, Problem &p) {
    const uint64_t tiles = (uint64_t)p.tiles_n * p.tiles_m, most = (uint64_t)sm_count(device) * 2;
    p.splits = 1;
    while (p.splits < kMostSplits && tiles * p.splits * 2 <= most && p.stages >= p.splits * 4) p.splits *= 2;
}

template <typename T>
cudaError_t run(int device, cudaStream_t s, const Packed &x, const Packed &w, uint64_t k, Problem &p) {
    p.x_scales = x.scales;
    // Pairs of CTAs for more than 64 rows of x, except where a long k and few
    // tiles gain by splitting it. Measured in us, pairs and split tiles (rows of x,
    // k, rows of w): 128 x 784 x 1000: 7.0, 12.1; 1024 x 2048 x 2048: 8.2, 14.4;
    // 256 x 8192 x 8192: 16.0, 19.3; but 128 x 8192 x 8192: 15.9, 13.9;
    // 300 x 8192 x 256: 15.8, 9.5; 64 x 2048 x 2048: 7.5, 6.6.
    constexpr uint32_t kShortStages = 12;
    const uint64_t across = (w.rows + 255) / 256, high = (x.rows + kPairN - 1) / kPairN;
    if (x.rows > 64 && (p.stages <= kShortStages || (x.rows > 128 && across * high * 8 >= (uint64_t)sm_count(device)))) {
        p.tiles_n = (uint32_t)across, p.tiles_m = (uint32_t)high, p.splits = 1;
        return launch_pairs<T>(device, s, x, w, k, p);
    }
    CUtensorMap wm, xm;
    cudaError_t e = map_of(&wm, w, k, kRows);
    if (e != cudaSuccess) return e;
    const uint32_t bn = x.rows <= 16 ? 16 : x.rows <= 32 ? 32 : x.rows <= 64 ? 64 : 128;
    p.tiles_m = (uint32_t)((x.rows + bn - 1) / bn);
    split_k(device, p);
    e = map_of(&xm, x, k, bn);
    if (e != cudaSuccess) return e;
    switch (bn) {
        case 16: return launch_skinny<T, 16, None>(s, wm, xm, p);
        case 32: return launch_skinny<T, 32, None>(s, wm, xm, p);
        case 64: return launch_skinny<T, 64, None>(s, wm, xm, p);
        default: return launch_skinny<T, 128, None>(s, wm, xm, p);
    }
}

template <typename T, typename X>
cudaError_t run_plain(int device, cudaStream_t s, const Packed &w, uint64_t k, Problem &p) {
    CUtensorMap wm;
    const cudaError_t e = map_of(&wm, w, k, kRows);
    if (e != cudaSuccess) return e;
    p.tiles_m = 1;
    split_k(device, p);
    return launch_skinny<T, 16, X>(s, wm, wm, p);
}
template <typename T>
cudaError_t run_plain_as(int device, cudaStream_t s, int x_dtype, const Packed &w, uint64_t k, Problem &p) {
    switch (x_dtype) {
        case SNN_B200_F32: return run_plain<T, float>(device, s, w, k, p);
        case SNN_B200_F16: return run_plain<T, __half>(device, s, w, k, p);
        case SNN_B200_BF16: return run_plain<T, __nv_bfloat16>(device, s, w, k, p);
        default: return run_plain<T, Spike>(device, s, w, k, p);
    }
}

}  // namespace

bool packs_on_the_way(const void *x, int x_dtype, uint64_t m, int64_t row_stride, int64_t col_stride) {
    return m <= 16 && col_stride == 1 && aligned_to(x, 16) && row_stride * dtype_bytes(x_dtype) % 16 == 0;
}

cudaError_t linear(int device, cudaStream_t s, const void *x, int x_dtype, uint64_t m, int64_t x_stride, const Packed &w,
                   uint64_t k, const float *bias, void *out, int dtype, int64_t row_stride) {
    Problem p = problem_of(m, w, k, bias, out, row_stride);
    p.x = x, p.x_stride = x_stride;
    switch (dtype) {
        case SNN_B200_F32: return run_plain_as<float>(device, s, x_dtype, w, k, p);
        case SNN_B200_F16: return run_plain_as<__half>(device, s, x_dtype, w, k, p);
        default: return run_plain_as<__nv_bfloat16>(device, s, x_dtype, w, k, p);
    }
}

cudaError_t matmul(int device, cudaStream_t s, const Packed &x, const Packed &w, uint64_t k, const float *bias,
                   void *out, int dtype, int64_t row_stride) {
    Problem p = problem_of(x.rows, w, k, bias, out, row_stride);
    switch (dtype) {
        case SNN_B200_F32: return run<float>(device, s, x, w, k, p);
        case SNN_B200_F16: return run<__half>(device, s, x, w, k, p);
        default: return run<__nv_bfloat16>(device, s, x, w, k, p);
    }
}

}  // namespace mx4
}  // namespace b200
