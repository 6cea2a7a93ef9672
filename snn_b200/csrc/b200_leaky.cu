// The leaky recurrence over device arrays: the calls, their checks and how the
// work is split, the sum of a shared gate's gradient, and the single step.
#include "b200_leaky.h"

#include <algorithm>

namespace b200 {
namespace leaky {
namespace {

// ---- states between segments ----
// states[s] = the state before segment s, folded in order from `first` (or
// zero) and the maps of the segments before it (backward: behind it). A CTA takes
// 32 channels; each of its warps composes the maps of one run of segments, folds
// those of the runs before onto the first state, and walks its run again. Runs of
// up to kHeld maps stay in registers, all of them under way at once (with 8 under
// way and two passes over them it took 10 us for 444 segments of 1024 channels).
constexpr uint32_t kCarryWarps = 32, kHeld = 16;
__global__ void __launch_bounds__(kCarryWarps * 32) carry_kernel(const float2 *maps, uint32_t segments, uint64_t flat,
                                                                 const float *first, float *states, bool back) {
    __shared__ float2 s_run[kCarryWarps][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint64_t i = (uint64_t)blockIdx.x * 32 + lane;
    const uint32_t run = (segments + kCarryWarps - 1) / kCarryWarps;
    const uint32_t from = min(segments, warp * run), to = i < flat ? min(segments, from + run) : from;
    const auto at = [&](uint32_t n) { return (uint64_t)(back ? segments - 1 - n : n) * flat + i; };
    after_previous();
    float2 m = make_float2(1.0f, 0.0f), held[kHeld];
    for (uint32_t n0 = from; n0 < to; n0 += kHeld) {
#pragma unroll
        for (uint32_t n = 0; n < kHeld; ++n) held[n] = n0 + n < to ? maps[at(n0 + n)] : make_float2(1.0f, 0.0f);
        float x = m.x;
#pragma unroll
        for (uint32_t n = 0; n < kHeld; ++n) {
            x = __fmul_rn(held[n].x, x);
            m.y = __fmaf_rn(held[n].x, m.y, held[n].y);
        }
        if (x == 0.0f) {
            bool zero = m.x == 0.0f;
#pragma unroll
            for (uint32_t n = 0; n < kHeld; ++n) zero |= held[n].x == 0.0f;
            x = kept(x, zero);
        }
        m.x = x;
    }
    s_run[warp][lane] = m;
    float h = i < flat && first ? first[i] : 0.0f;
    __syncthreads();
    if (i >= flat) return;
    for (uint32_t w = 0; w < warp; ++w) h = __fmaf_rn(s_run[w][lane].x, h, s_run[w][lane].y);
    for (uint32_t n0 = from; n0 < to; n0 += kHeld) {
        if (run > kHeld)
#pragma unroll
            for (uint32_t n = 0; n < kHeld; ++n) held[n] = n0 + n < to ? maps[at(n0 + n)] : make_float2(1.0f, 0.0f);
#pragma unroll
        for (uint32_t n = 0; n < kHeld; ++n)
            if (n0 + n < to) {
                states[at(n0 + n)] = h;
                h = __fmaf_rn(held[n].x, h, held[n].y);
            }
    }
}

// ---- a shared gate's gradient ----
// out[r][c] = the sum of partial[t][b][c] over the segments and, where the gate
// is shared over the sequences (rows of out: 1), over b. A CTA takes 32
// channels of a row; its warps share the terms, in an order that depends on
// the counts only. Terms are few (one a segment), so they are summed in 64 bits.
constexpr uint32_t kSumWarps = 16;
__global__ void __launch_bounds__(kSumWarps * 32) gate_sum_kernel(const float *partial, uint32_t segments, uint32_t batch,
                                                                  uint32_t channels, float *out, int64_t row_stride) {
    __shared__ double s_sum[kSumWarps][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t c = blockIdx.x * 32 + lane;
    const uint64_t flat = (uint64_t)batch * channels;
    after_previous();
    for (uint32_t r = blockIdx.y; r < (row_stride ? batch : 1u); r += gridDim.y) {
        const uint64_t terms = row_stride ? segments : (uint64_t)segments * batch;
        // Term n of row r: segment n, sequence r; or n-th of all [segments][batch].
        const float *p = partial + (row_stride ? (uint64_t)r * channels : 0) + c;
        const uint64_t step = row_stride ? flat : channels;
        double sum = 0.0;
        if (c < channels)
#pragma unroll 4
            for (uint64_t n = warp; n < terms; n += kSumWarps) sum += (double)p[n * step];
        s_sum[warp][lane] = sum;
        __syncthreads();
        if (warp == 0 && c < channels) {
            for (uint32_t w = 1; w < kSumWarps; ++w) sum += s_sum[w][lane];
            out[(int64_t)r * row_stride + c] = (float)sum;
        }
        __syncthreads();
    }
}

// Every CTA of a step looks through all slots, eight rows to a CTA: 131,072 rows take 3.1
// ms, so this many about three seconds, and as many as other counts may be days.
constexpr snn_size_t kMostNamedRows = 1ull << 22;

// The listed combinations of types. Without a gate array its type is not looked at.
bool types_listed(int x, bool has_gate, int gate, int y, bool gate_every_step) {
    if (x == SNN_B200_SPIKES || x == SNN_B200_F32)
        return y == SNN_B200_F32 && (!has_gate || gate == SNN_B200_F32);
    return (y == x || y == SNN_B200_F32) &&
           (!has_gate || gate == SNN_B200_F32 || (gate == x && gate_every_step));
}

bool array_ok(const void *p, int dtype, snn_size_t batch, int64_t sb, snn_size_t steps, int64_t st) {
    return p && aligned_to(p, dtype_bytes(dtype)) && offset_fits(batch, sb) && offset_fits(steps, st);
}
bool output_ok(const void *p, int dtype, const snn_b200_leaky_t &q, int64_t sb, int64_t st) {
    return array_ok(p, dtype, q.batch, sb, q.steps, st) && disjoint_runs(q.batch, sb, q.steps, st, q.channels);
}
bool floats_ok(const void *p) { return aligned_to(p, 4); }

snn_status_t check_common(int device, const snn_b200_leaky_t *q, const void *x, const void *gate,
                          const uint32_t *lengths) {
    if (q == nullptr || device < 0) return SNN_ERR_INVALID_ARGUMENT;
    if (q->batch > kMaxCount || q->steps > kMaxCount || q->channels > kMaxCount) return SNN_ERR_OVERFLOW;
    if (!is_dtype(q->x_dtype) || !is_float_dtype(q->y_dtype) || (gate && !is_float_dtype(q->gate_dtype)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (!types_listed(q->x_dtype, gate != nullptr, q->gate_dtype, q->y_dtype, q->gate_step_stride != 0))
        return SNN_ERR_UNSUPPORTED;
    if (!floats_ok(lengths)) return SNN_ERR_INVALID_ARGUMENT;
    if (q->batch == 0 || q->steps == 0 || q->channels == 0) return SNN_OK;
    if (!array_ok(x, q->x_dtype, q->batch, q->x_batch_stride, q->steps, q->x_step_stride) ||
        (gate && !array_ok(gate, q->gate_dtype, q->batch, q->gate_batch_stride, q->steps, q->gate_step_stride)))
        return SNN_ERR_INVALID_ARGUMENT;
    return SNN_OK;
}

// How a call is cut and where its parts lie in the workspace.
struct Plan {
    uint64_t flat, columns;
    uint32_t segments, segment_steps, partials;  // partials: sums of a shared gate's gradient a channel
    uint32_t crew;
    uint64_t maps, states, partial, bytes;
};
// Warps that walk whole sequences; where those would be too few to keep the loads
// of 148 SMs under way, crews; where even crews are too few and the sequences
// long, segments (64 steps at least), which cost three launches.
// Measured in us, forward and gradient (f32 with a leak a channel):
//   512 channels:   32 steps  128        512         1024        2048
//     whole         3.1, 5.5  7.4, 11.7  23.9, 36.0  45.6, 68.4
//     crews                   3.1, 5.5   6.4, 10.0   11.1, 16.2  20.4, 28.8
//     segments                11.2, 14.1 11.5, 14.7  12.0, 15.3  12.6, 16.2
//   8192 steps of 64 columns: crews 102, segments about 70 (bf16), of 128: 104, 140;
//   of 1024 steps (bf16): 768 columns in crews 76, whole 109, 1024 columns 89, 108,
//   1600 columns 135, 129; 64 steps of 1024 columns: crews 11.1, whole 9.2.
// A crew has 16 warps where it has an SM to itself, else 8 (8192 steps, bf16, 128
// columns: 104 against 127 us, 256 columns of 4096: 105 against 90 us).
// Walks are counted two channels a thread, also of the rasters that four are walked of
// (1000 channels, a leak each, whole and in segments: 64 sequences of 200 steps 15, 51 us,
// 128 of 400 steps 49, 124 us).
constexpr uint64_t kFewWalks = 148 * 8, kFewShortWalks = 148 * 5, kFewCrews = 104, kManyWalks = 148 * 48;
constexpr uint32_t kVeryShort = 256, kShort = 1024, kLeastSegment = 64;
Plan plan_of(const snn_b200_leaky_t &q, uint32_t width, bool back) {
    Plan p = {};
    p.flat = q.batch * q.channels;
    p.columns = (p.flat + 32 * width - 1) / (32 * width);
    p.segments = 1, p.segment_steps = (uint32_t)q.steps;
    const uint64_t walks = width == 4 ? (p.flat + 63) / 64 : p.columns;
    if (walks && walks < (q.steps > kVeryShort ? kFewWalks : kFewShortWalks) && q.steps > 2 * kSteps) {
        if (walks >= kFewCrews || q.steps <= kShort) {
            p.crew = p.columns <= 148 ? 16 : 8;
        } else if (q.steps >= 2 * kLeastSegment) {
            const uint64_t want = std::max<uint64_t>(kLeastSegment, q.steps * p.columns / kManyWalks);
            p.segment_steps = (uint32_t)((want + kSteps - 1) / kSteps * kSteps);
            p.segments = (uint32_t)((q.steps + p.segment_steps - 1) / p.segment_steps);
        }
    }
    p.partials = p.crew ? p.crew : p.segments;
    const auto round = [](uint64_t v) { return (v + 255) / 256 * 256; };
    const uint64_t cut = p.segments > 1 ? p.segments * p.flat : 0;
    p.maps = 0;
    p.states = p.maps + round(cut * 8);
    p.partial = p.states + round(cut * 4);
    p.bytes = p.partial + (back && !q.gate_step_stride ? round(p.partials * p.flat * 4) : 0);
    // Crews need no workspace of their own, but a call of so many steps that they walk is
    // refused without one all the same: it stays so, with the least there is.
    if (p.crew && q.steps >= 2 * kLeastSegment) p.bytes = std::max<uint64_t>(p.bytes, 256);
    return p;
}

void fill(Args &g, const snn_b200_leaky_t &q, const Plan &p, void *workspace) {
    g.flat = p.flat;
    g.batch = (uint32_t)q.batch, g.steps = (uint32_t)q.steps, g.channels = (uint32_t)q.channels;
    g.xb = q.x_batch_stride, g.xt = q.x_step_stride, g.gb = q.gate_batch_stride, g.gt = q.gate_step_stride;
    g.yb = q.y_batch_stride, g.yt = q.y_step_stride, g.dyb = q.dy_batch_stride, g.dyt = q.dy_step_stride;
    g.dxb = q.dx_batch_stride, g.dxt = q.dx_step_stride, g.dgb = q.dgate_batch_stride, g.dgt = q.dgate_step_stride;
    g.decay = q.decay, g.scale = q.input_scale, g.logit = q.logit, g.complement = q.complement;
    g.columns = (uint32_t)p.columns, g.segments = p.segments, g.segment_steps = p.segment_steps, g.crew = p.crew;
    char *w = (char *)workspace;
    g.maps = (float2 *)(w + p.maps);
    g.states = (float *)(w + p.states);
}

// May a thread hold n channels of an array?
bool pieces(uint32_t n, const void *p, uint32_t bytes, int64_t sb, int64_t st) {
    return !p || (aligned_to(p, n * bytes) && sb % n == 0 && st % n == 0);
}
bool float_pieces(uint32_t n, const float *p) { return aligned_to(p, 4 * n); }

// 16 bytes of a row at a time, from one sequence each.
bool wide_rows(const void *p, int dtype, uint64_t channels, int64_t sb, int64_t st) {
    const uint32_t n = 16 / dtype_bytes(dtype);
    return channels % n == 0 && pieces(n, p, dtype_bytes(dtype), sb, st);
}

// Of x, of a gate for every step and, backward, of dy.
bool wide_rows(const snn_b200_leaky_t &q, const Args &g, bool back) {
    return wide_rows(g.x, q.x_dtype, q.channels, q.x_batch_stride, q.x_step_stride) &&
           (!(g.gate && q.gate_step_stride) ||
            wide_rows(g.gate, q.gate_dtype, q.channels, q.gate_batch_stride, q.gate_step_stride)) &&
           (!back || wide_rows(g.dy, q.y_dtype, q.channels, q.dy_batch_stride, q.dy_step_stride));
}

cudaError_t run(cudaStream_t s, const snn_b200_leaky_t &q, Args &g, const Plan &p, uint32_t width, bool back,
                void *workspace) {
    fill(g, q, p, workspace);
    g.wide = wide_rows(q, g, back);
    const Form f = {q.gate_dtype, q.y_dtype, g.gate && q.gate_step_stride, width};
    switch (q.x_dtype) {
        case SNN_B200_F32: return back ? backward_f32(s, f, g) : forward_f32(s, f, g);
        case SNN_B200_F16: return back ? backward_f16(s, f, g) : forward_f16(s, f, g);
        case SNN_B200_BF16: return back ? backward_bf16(s, f, g) : forward_bf16(s, f, g);
        default: return back ? backward_spikes(s, f, g) : forward_spikes(s, f, g);
    }
}

}  // namespace

cudaError_t carry(cudaStream_t s, const Args &a, bool back) {
    return launch_early(carry_kernel, (uint32_t)((a.flat + 31) / 32), kCarryWarps * 32, 0, s, 1, a.maps, a.segments, a.flat,
                        back ? a.dh_last : a.h0, a.states, back);
}

}  // namespace leaky
}  // namespace b200

using namespace b200;
using namespace b200::leaky;

extern "C" {

snn_size_t snn_b200_leaky_saved_floats(snn_size_t batch, snn_size_t steps, snn_size_t channels) {
    if (batch > kMaxCount || steps > kMaxCount || channels > kMaxCount) return 0;
    return batch * ((steps + kSteps - 1) / kSteps) * channels;
}

snn_size_t snn_b200_leaky_workspace(const snn_b200_leaky_t *q, int backward) {
    if (q == nullptr || q->batch > kMaxCount || q->steps > kMaxCount || q->channels > kMaxCount) return 0;
    const uint64_t need = std::max(plan_of(*q, 1, backward).bytes, plan_of(*q, 2, backward).bytes);
    // Four channels a thread walk rasters only, and forward only.
    return q->x_dtype == SNN_B200_SPIKES && !backward ? std::max(need, plan_of(*q, 4, false).bytes) : need;
}

snn_status_t snn_b200_leaky_scan_async(int device, void *stream, const snn_b200_leaky_t *leaky, const void *x,
                                       const void *gate, const float *h0, const uint32_t *lengths, void *y,
                                       float *h_last, float *saved, void *workspace, snn_size_t workspace_bytes) {
    const snn_status_t st = check_common(device, leaky, x, gate, lengths);
    if (st != SNN_OK) return st;
    const snn_b200_leaky_t &q = *leaky;
    if (!floats_ok(h0) || !floats_ok(h_last) || !floats_ok(saved)) return SNN_ERR_INVALID_ARGUMENT;
    if (q.batch == 0 || q.channels == 0) return SNN_OK;
    if (q.steps && !output_ok(y, q.y_dtype, q, q.y_batch_stride, q.y_step_stride)) return SNN_ERR_INVALID_ARGUMENT;
    const uint64_t need = snn_b200_leaky_workspace(leaky, 0);
    if (need && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (q.batch * q.channels > kMaxCount) return SNN_ERR_OVERFLOW;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    const cudaStream_t s = (cudaStream_t)stream;
    if (q.steps == 0) {  // the state passes through
        if (!h_last) return SNN_OK;
        const cudaError_t e = h0 ? cudaMemcpyAsync(h_last, h0, q.batch * q.channels * 4, cudaMemcpyDeviceToDevice, s)
                                 : cudaMemsetAsync(h_last, 0, q.batch * q.channels * 4, s);
        return op_status(e, __func__);
    }
    Args g = {};
    g.x = x, g.gate = gate, g.h0 = h0, g.lengths = lengths, g.y = y, g.h_last = h_last, g.saved = saved;
    // Two channels a thread where every array can be read so; four of a raster that no
    // crew walks, as two of them are too few bytes to be copied ahead (2000 x 25 x 1000: 46
    // against 82 us). Not with a gate for every step where rows are copied in pieces of 16
    // bytes anyway (762 x 200 x 1008: 311 against 229 us; of 1000 channels 348, 345).
    const auto holds = [&](uint32_t n) {
        return q.channels % n == 0 && pieces(n, x, dtype_bytes(q.x_dtype), q.x_batch_stride, q.x_step_stride) &&
               pieces(n, gate, dtype_bytes(q.gate_dtype), q.gate_batch_stride, q.gate_step_stride) &&
               pieces(n, y, dtype_bytes(q.y_dtype), q.y_batch_stride, q.y_step_stride) && float_pieces(n, h0) &&
               float_pieces(n, h_last) && float_pieces(n, saved);
    };
    const bool four = q.x_dtype == SNN_B200_SPIKES && !plan_of(q, 2, false).crew &&
                      !(gate && q.gate_step_stride && wide_rows(q, g, false)) && holds(4);
    const uint32_t width = four ? 4 : holds(2) ? 2 : 1;
    const cudaError_t e = run(s, q, g, plan_of(q, width, false), width, false, workspace);
    return op_status(e, __func__);
}

snn_status_t snn_b200_leaky_scan_backward_async(int device, void *stream, const snn_b200_leaky_t *leaky,
                                                const void *x, const void *gate, const uint32_t *lengths,
                                                const float *saved, const void *dy, const float *dh_last, void *dx,
                                                void *dgate, float *dh0, void *workspace,
                                                snn_size_t workspace_bytes) {
    const snn_status_t st = check_common(device, leaky, x, gate, lengths);
    if (st != SNN_OK) return st;
    const snn_b200_leaky_t &q = *leaky;
    if (!floats_ok(saved) || !floats_ok(dh_last) || !floats_ok(dh0) || (dgate && !gate))
        return SNN_ERR_INVALID_ARGUMENT;
    const bool every = gate && q.gate_step_stride != 0, shared = gate && !every && q.gate_batch_stride == 0;
    if (dgate && every && q.gate_batch_stride == 0 && q.batch > 1) return SNN_ERR_UNSUPPORTED;
    if (dgate && !every && !floats_ok(dgate)) return SNN_ERR_INVALID_ARGUMENT;
    if (q.channels == 0 || (q.batch == 0 && !(dgate && shared))) return SNN_OK;
    const int dx_type = q.x_dtype == SNN_B200_SPIKES ? SNN_B200_F32 : q.x_dtype;
    if (q.steps && q.batch &&
        (saved == nullptr || !array_ok(dy, q.y_dtype, q.batch, q.dy_batch_stride, q.steps, q.dy_step_stride) ||
         (dx && !output_ok(dx, dx_type, q, q.dx_batch_stride, q.dx_step_stride)) ||
         (dgate && every && !output_ok(dgate, q.gate_dtype, q, q.dgate_batch_stride, q.dgate_step_stride))))
        return SNN_ERR_INVALID_ARGUMENT;
    if (dgate && !every && !shared &&
        (!offset_fits(q.batch, q.dgate_batch_stride) || !disjoint_runs(q.batch, q.dgate_batch_stride, 1, 0, q.channels)))
        return SNN_ERR_INVALID_ARGUMENT;
    const uint64_t need = snn_b200_leaky_workspace(leaky, 1);
    if (need && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (q.batch * q.channels > kMaxCount) return SNN_ERR_OVERFLOW;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    const cudaStream_t s = (cudaStream_t)stream;
    const bool sums = dgate && !every;
    if (q.steps == 0 || q.batch == 0) {  // no steps: the state's gradient passes through, the gate's is zero
        cudaError_t e = cudaSuccess;
        if (dh0 && q.batch)
            e = dh_last ? cudaMemcpyAsync(dh0, dh_last, q.batch * q.channels * 4, cudaMemcpyDeviceToDevice, s)
                        : cudaMemsetAsync(dh0, 0, q.batch * q.channels * 4, s);
        if (e == cudaSuccess && sums)
            e = shared ? cudaMemsetAsync(dgate, 0, q.channels * 4, s)
                       : cudaMemset2DAsync(dgate, 4 * std::max<size_t>(q.dgate_batch_stride, q.channels), 0, q.channels * 4, q.batch, s);
        return op_status(e, __func__);
    }
    const bool even = q.channels % 2 == 0 && pieces(2, x, dtype_bytes(q.x_dtype), q.x_batch_stride, q.x_step_stride) &&
                      pieces(2, gate, dtype_bytes(q.gate_dtype), q.gate_batch_stride, q.gate_step_stride) &&
                      pieces(2, dy, dtype_bytes(q.y_dtype), q.dy_batch_stride, q.dy_step_stride) &&
                      pieces(2, dx, dtype_bytes(dx_type), q.dx_batch_stride, q.dx_step_stride) &&
                      (!every || pieces(2, dgate, dtype_bytes(q.gate_dtype), q.dgate_batch_stride, q.dgate_step_stride)) &&
                      float_pieces(2, dh_last) && float_pieces(2, dh0) && float_pieces(2, saved);
    Args g = {};
    g.x = x, g.gate = gate, g.lengths = lengths, g.saved = const_cast<float *>(saved), g.dy = dy;
    g.dh_last = dh_last, g.dx = dx, g.dgate = every ? dgate : nullptr, g.dh0 = dh0;
    const uint32_t width = even ? 2 : 1;
    const Plan p = plan_of(q, width, true);
    g.partial = sums ? (float *)((char *)workspace + p.partial) : nullptr;
    cudaError_t e = run(s, q, g, p, width, true, workspace);
    if (e == cudaSuccess && sums) {
        const uint32_t rows = shared ? 1u : (uint32_t)(q.batch < 65535 ? q.batch : 65535);
        e = launch_early(gate_sum_kernel, dim3((uint32_t)((q.channels + 31) / 32), rows), kSumWarps * 32, 0, s, 1, g.partial,
                         p.partials, q.batch, q.channels, (float *)dgate, shared ? 0 : q.dgate_batch_stride);
    }
    return op_status(e, __func__);
}

snn_status_t snn_b200_leaky_step_async(int device, void *stream, snn_size_t batch, snn_size_t slot_count,
                                       snn_size_t channels, const void *x, int x_dtype, int64_t x_row_stride,
                                       const void *gate, int gate_dtype, int64_t gate_row_stride, int logit,
                                       int complement, float decay, float input_scale, float *pool,
                                       int64_t pool_row_stride, const int32_t *slots, void *y, int y_dtype,
                                       int64_t y_row_stride) {
    if (device < 0) return SNN_ERR_INVALID_ARGUMENT;
    if (batch > kMaxCount || slot_count > kMaxCount || channels > kMaxCount) return SNN_ERR_OVERFLOW;
    if (slots && batch > kMostNamedRows) return SNN_ERR_OVERFLOW;
    if (!is_dtype(x_dtype) || !is_float_dtype(y_dtype) || (gate && !is_float_dtype(gate_dtype)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (!types_listed(x_dtype, gate != nullptr, gate_dtype, y_dtype, gate_row_stride != 0)) return SNN_ERR_UNSUPPORTED;
    if (batch == 0 || channels == 0) return SNN_OK;
    if (!array_ok(x, x_dtype, batch, x_row_stride, 1, 0) ||
        (gate && !array_ok(gate, gate_dtype, batch, gate_row_stride, 1, 0)) ||
        !array_ok(y, y_dtype, batch, y_row_stride, 1, 0) || !disjoint_runs(batch, y_row_stride, 1, 0, channels) ||
        !floats_ok(slots) || (!slots && batch > slot_count))
        return SNN_ERR_INVALID_ARGUMENT;
    if (slot_count && (!array_ok(pool, SNN_B200_F32, slot_count, pool_row_stride, 1, 0) ||
                       !disjoint_runs(slot_count, pool_row_stride, 1, 0, channels)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (batch * channels > kMaxCount) return SNN_ERR_OVERFLOW;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    StepArgs g = {(uint32_t)batch, (uint32_t)slot_count, (uint32_t)channels, x, gate, x_row_stride, gate_row_stride,
                  pool_row_stride, y_row_stride, logit, complement, decay, input_scale, pool, slots, y, 0};
    // Four channels a thread where every array can be read in fours.
    const auto fours = [&](const void *p, uint32_t bytes, int64_t stride) {
        return !p || (aligned_to(p, 4 * bytes) && stride % 4 == 0);
    };
    const bool wide = channels % 4 == 0 && fours(x, dtype_bytes(x_dtype), x_row_stride) &&
                      fours(gate, dtype_bytes(gate_dtype), gate_row_stride) && fours(pool, 4, pool_row_stride) &&
                      fours(y, dtype_bytes(y_dtype), y_row_stride);
    const Form f = {gate ? gate_dtype : SNN_B200_F32, y_dtype, true, wide ? 4u : 1u};
    const uint32_t pieces = (uint32_t)((channels + f.width - 1) / f.width);  // thread-sized pieces of a row
    // A warp a row, or the whole CTA where that would leave SMs without work.
    const bool many = batch >= (snn_size_t)sm_count(device) * 4;
    g.rows = many ? 8 : 1;
    const uint32_t across = 256 / g.rows;
    const dim3 grid((uint32_t)((batch + g.rows - 1) / g.rows), std::min(many ? 2u : 64u, (pieces + across - 1) / across));
    cudaError_t e;
    switch (x_dtype) {
        case SNN_B200_F32: e = step_f32((cudaStream_t)stream, f, g, grid); break;
        case SNN_B200_F16: e = step_f16((cudaStream_t)stream, f, g, grid); break;
        case SNN_B200_BF16: e = step_bf16((cudaStream_t)stream, f, g, grid); break;
        default: e = step_spikes((cudaStream_t)stream, f, g, grid); break;
    }
    return op_status(e, __func__);
}

}  // extern "C"
