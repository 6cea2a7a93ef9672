// Tensor maps and the barrier and copy instructions of TMA.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace b200 {
namespace tma {

// A map of `rank` dimensions (the first one contiguous; strides in bytes of
// the others, multiples of 16), boxes of `box` elements. What lies behind the
// dimensions reads as zero.
cudaError_t encode(CUtensorMap *map, CUtensorMapDataType type, uint32_t rank, const void *base, const cuuint64_t *dims,
                   const cuuint64_t *strides, const cuuint32_t *box, CUtensorMapSwizzle swizzle);

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t smem_of(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint64_t *b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_of(b)), "r"(count) : "memory");
}
// Makes initialised barriers visible to the copies (before a __syncthreads).
__device__ __forceinline__ void bar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_expect(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_of(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_of(b)) : "memory");
}
// Waits for the phase of that parity to end; false when it gave up, after about
// two seconds of the SM's clock.
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity) {
    constexpr long long kMostCycles = 1ll << 32;
    const uint32_t at = smem_of(b);
    const long long start = clock64();
    do {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(at), "r"(parity)
            : "memory");
        if (done) return true;
    } while (clock64() - start < kMostCycles);
    return false;
}

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
            "r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_of(bar))
        : "memory");
}
// Both addresses and the size are multiples of 16.
__device__ __forceinline__ void load_run(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_of(bar))
                 : "memory");
}
#endif

}  // namespace tma
}  // namespace b200
