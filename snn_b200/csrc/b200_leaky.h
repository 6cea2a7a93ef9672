// Host side of the leaky recurrence: the plan of a call and the launchers of
// the kernels, one translation unit for each type of x.
#pragma once

#include "b200_ops.h"

namespace b200 {
namespace leaky {

constexpr uint32_t kSteps = SNN_B200_LEAKY_BLOCK;  // steps a thread holds in registers
constexpr uint32_t kScanWarps = 16, kBackWarps = 8;  // warps of a tile (one CTA), kSteps of the steps each
constexpr uint32_t kSuper = 16;              // tiles between two published states

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
    // Work split along the steps: a ticket, flags and what tiles publish.
    uint32_t tiles, columns;  // tiles along the steps, warps' widths across the channels
    uint32_t *ticket, *tile_flags, *state_flags;
    float2 *aggregates;  // [tiles][columns * width]
    float *states;       // [tiles / kSuper][columns * width]
    float *partial;      // backward: sums of a shared gate's gradient, [tiles (1 unsplit)][flat]
};

// x's type is the translation unit's; g and y are snn_b200_dtype_t, `every`
// says that the gate has a value for every step. width: channels a thread
// holds. split: tiles along the steps.
struct Form {
    int gate_dtype, y_dtype;
    bool every, split;
    uint32_t width;
};

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
