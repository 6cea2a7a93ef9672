// Shared by the sequence operators (b200_mx4*.cu, b200_leaky*.cu): element
// types, argument checks and the device a call runs on.
#pragma once

#include "snn_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace b200 {

// Records the text of snn_b200_last_error (snn_cuda_b200.cu).
snn_status_t op_status(cudaError_t e, const char *where);

// Number of SMs of a device (b200_kernels.cu).
int sm_count(int device);

// Makes `device` current for the scope and puts the caller's device back.
class DeviceScope {
  public:
    explicit DeviceScope(int device) {
        err_ = cudaGetDevice(&prev_);
        if (err_ == cudaSuccess && prev_ != device) err_ = cudaSetDevice(device);
        moved_ = err_ == cudaSuccess && prev_ != device;
    }
    ~DeviceScope() {
        if (moved_) cudaSetDevice(prev_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    cudaError_t error() const { return err_; }

  private:
    int prev_ = -1;
    bool moved_ = false;
    cudaError_t err_ = cudaSuccess;
};

constexpr snn_size_t kMaxCount = 0x7fffffffull;

inline bool is_dtype(int t) { return t >= SNN_B200_F32 && t <= SNN_B200_SPIKES; }
inline bool is_float_dtype(int t) { return t >= SNN_B200_F32 && t <= SNN_B200_BF16; }
inline uint32_t dtype_bytes(int t) { return t == SNN_B200_F32 ? 4u : t == SNN_B200_SPIKES ? 1u : 2u; }
inline bool aligned_to(const void *p, uintptr_t a) { return ((uintptr_t)p % a) == 0; }

// (count - 1) * stride summed over the dimensions stays below 2^60, so that
// byte offsets fit 64 bits.
inline bool offset_fits(snn_size_t count, int64_t stride) {
    return stride >= 0 && (count <= 1 || (unsigned __int128)(count - 1) * (uint64_t)stride < ((unsigned __int128)1 << 60));
}

// Two strides under which no two of na x nb runs of `run` elements overlap.
inline bool disjoint_runs(snn_size_t na, int64_t sa, snn_size_t nb, int64_t sb, snn_size_t run) {
    if (na <= 1 && nb <= 1) return true;
    if (na <= 1) return (uint64_t)sb >= run;
    if (nb <= 1) return (uint64_t)sa >= run;
    const uint64_t inner = (uint64_t)(sa < sb ? sa : sb), outer = (uint64_t)(sa < sb ? sb : sa);
    const snn_size_t n = sa < sb ? na : nb;
    return inner >= run && (unsigned __int128)(n - 1) * inner + run <= outer;
}

// Launches that may start while the kernel before them in the stream ends: their
// set-up overlaps its last CTAs. Every kernel launched so calls after_previous()
// before it reads or writes global memory, which waits for all of that kernel.
// allow_next() lets its own successor start before its CTAs have ended; only the
// skinny product, a single wave of CTAs, gains by it (4x8192x8192: 10.4 against
// 11.2 us; a step of 2000 rows lost by it: 11.6 against 8.1 us).
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, uint32_t cluster,
                         A &&...args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid, c.blockDim = block, c.dynamicSmemBytes = smem, c.stream = stream;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}
// Lets a kernel have that much dynamic shared memory on the current device;
// asked for once a device.
template <auto Kernel>
cudaError_t allow_smem(uint32_t bytes) {
    static std::atomic<uint64_t> asked{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && asked.load(std::memory_order_acquire) >> device & 1)) return e;
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && device < 64) asked.fetch_or(1ull << device, std::memory_order_release);
    return e;
}
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;"); }

// Element types: a spike byte counts as one when it is not zero.
struct Spike {
    uint8_t byte;
};
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(Spike v) { return v.byte ? 1.0f : 0.0f; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace b200
