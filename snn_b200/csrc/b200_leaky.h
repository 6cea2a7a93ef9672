// Host side of the leaky recurrence: the plan of a call and the launchers of
// the kernels, one translation unit for each type of x.
#pragma once

#include "b200_ops.h"

namespace b200 {
namespace leaky {

constexpr uint32_t kSteps = SNN_B200_LEAKY_BLOCK;  // steps worked on at a time, and of a saved state
constexpr uint32_t kWarps = 4;                     // of a CTA
constexpr uint32_t kDepth = 4;                     // blocks of steps under way or at hand

struct Args {
    uint64_t flat;  // batch * channels
    uint32_t batch, steps, channels;
    const void *x, *gate, *dy;
    void *y, *dx, *dgate;
    const float *h0, *dh_last;
    float *h_last, *dh0, *saved;
    const uint32_t *lengths;
    int64_t xb, xt, gb, gt, yb, yt, dyb, dyt, dxb, dxt, dgb, dgt;
    float decay, scale;
    int logit, complement;
    int wide;                          // rows of x, gate and dy can be read in pieces of 16 bytes
    uint32_t columns;                  // warps' widths across the channels
    uint32_t segments, segment_steps;  // along the steps
    uint32_t crew;                     // a CTA of 16 or 8 warps a column, 0: none
    float2 *maps;                      // [segments][flat], (A, H) of h -> A h + H
    float *states;                     // [segments][flat], before each (backward: behind each)
    float *partial;                    // backward: sums of a shared gate's gradient, [segments, or warps of a crew][flat]
};

// Maps hold products of gates. One that has become zero although no gate is zero
// stays at the smallest magnitude, with its sign: times zero, an infinite state
// would turn into NaN, where step by step it stays infinite. It adds at most 2^-149
// of a finite state, which is what the rounding of a product so small may add too.
__device__ __forceinline__ float kept(float product, bool zero) {
    return product == 0.0f && !zero ? copysignf(__uint_as_float(1u), product) : product;
}

// x's type is the translation unit's; g and y are snn_b200_dtype_t, `every`
// says that the gate has a value for every step. width: channels a thread
// holds.
struct Form {
    int gate_dtype, y_dtype;
    bool every;
    uint32_t width;
};

// The states between segments from their maps.
cudaError_t carry(cudaStream_t s, const Args &a, bool back);

cudaError_t forward_f32(cudaStream_t s, const Form &f, const Args &a);
cudaError_t forward_f16(cudaStream_t s, const Form &f, const Args &a);
cudaError_t forward_bf16(cudaStream_t s, const Form &f, const Args &a);
cudaError_t forward_spikes(cudaStream_t s, const Form &f, const Args &a);
cudaError_t backward_f32(cudaStream_t s, const Form &f, const Args &a);
cudaError_t backward_f16(cudaStream_t s, const Form &f, const Args &a);
cudaError_t backward_bf16(cudaStream_t s, const Form &f, const Args &a);
cudaError_t backward_spikes(cudaStream_t s, const Form &f, const Args &a);

// The single step. rows: rows of a CTA of 256 threads (8 or 1).
struct StepArgs {
    uint32_t batch, slot_count, channels;
    const void *x, *gate;
    int64_t xs, gs, ps, ys;
    int logit, complement;
    float decay, scale;
    float *pool;
    const int32_t *slots;
    void *y;
    uint32_t rows;
};
cudaError_t step_f32(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid);
cudaError_t step_f16(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid);
cudaError_t step_bf16(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid);
cudaError_t step_spikes(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid);

}  // namespace leaky
}  // namespace b200
