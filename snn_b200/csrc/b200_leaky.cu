// The leaky recurrence over device arrays: scan, gradient and single step.
#include "b200_ops.h"

namespace b200 {
namespace {

constexpr uint32_t kBlockSteps = SNN_B200_LEAKY_BLOCK;

__device__ __forceinline__ float load_any(const void *p, int dtype, int64_t i) {
    switch (dtype) {
        case SNN_B200_F32: return ((const float *)p)[i];
        case SNN_B200_F16: return to_float(((const __half *)p)[i]);
        case SNN_B200_BF16: return to_float(((const __nv_bfloat16 *)p)[i]);
        default: return to_float(((const Spike *)p)[i]);
    }
}
__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, float v) {
    switch (dtype) {
        case SNN_B200_F32: ((float *)p)[i] = v; break;
        case SNN_B200_F16: ((__half *)p)[i] = from_float<__half>(v); break;
        default: ((__nv_bfloat16 *)p)[i] = from_float<__nv_bfloat16>(v); break;
    }
}

struct Leak {
    float a, rest;  // the gate and one minus it
};
// Both from one exponential of a non-positive number, so that neither is a
// difference of nearly equal values.
__device__ __forceinline__ Leak leak_of(float z, int logit) {
    if (!logit) return {z, __fsub_rn(1.0f, z)};
    const float t = expf(-fabsf(z));
    const float r = __fdividef(1.0f, __fadd_rn(1.0f, t)), q = __fmul_rn(t, r);
    return z >= 0.0f ? Leak{r, q} : Leak{q, r};
}

struct Args {
    snn_b200_leaky_t p;
    const void *x, *gate;
    const float *h0;
    const uint32_t *lengths;
    void *y;
    float *h_last, *saved;
    const void *dy;
    const float *dh_last;
    void *dx, *dgate;
    float *dh0;
    float *partial;  // [batch, channels] sums of a shared gate's gradient
};

__device__ __forceinline__ uint64_t length_of(const Args &g, uint64_t b) {
    return g.lengths ? min((uint64_t)g.lengths[b], (uint64_t)g.p.steps) : g.p.steps;
}
__device__ __forceinline__ Leak leak_at(const Args &g, uint64_t b, uint64_t t, uint64_t c) {
    if (!g.gate) return {g.p.decay, __fsub_rn(1.0f, g.p.decay)};
    return leak_of(load_any(g.gate, g.p.gate_dtype,
                            (int64_t)b * g.p.gate_batch_stride + (int64_t)t * g.p.gate_step_stride + (int64_t)c),
                   g.p.logit);
}

// One thread a channel, step by step.
__global__ void leaky_scan_kernel(Args g) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= g.p.batch * g.p.channels) return;
    const uint64_t b = i / g.p.channels, c = i % g.p.channels, len = length_of(g, b);
    const uint64_t blocks = (g.p.steps + kBlockSteps - 1) / kBlockSteps;
    float h = g.h0 ? g.h0[i] : 0.0f;
    for (uint64_t t = 0; t < g.p.steps; ++t) {
        if (g.saved && t % kBlockSteps == 0) g.saved[(b * blocks + t / kBlockSteps) * g.p.channels + c] = h;
        float y = 0.0f;
        if (t < len) {
            const Leak l = leak_at(g, b, t, c);
            float u = __fmul_rn(g.p.input_scale,
                                load_any(g.x, g.p.x_dtype,
                                         (int64_t)b * g.p.x_batch_stride + (int64_t)t * g.p.x_step_stride + (int64_t)c));
            if (g.p.complement) u = __fmul_rn(u, l.rest);
            y = h = __fmaf_rn(l.a, h, u);
        }
        store_any(g.y, g.p.y_dtype, (int64_t)b * g.p.y_batch_stride + (int64_t)t * g.p.y_step_stride + (int64_t)c, y);
    }
    if (g.h_last) g.h_last[i] = h;
}

__global__ void leaky_backward_kernel(Args g) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= g.p.batch * g.p.channels) return;
    const uint64_t b = i / g.p.channels, c = i % g.p.channels, len = length_of(g, b);
    const uint64_t blocks = (g.p.steps + kBlockSteps - 1) / kBlockSteps;
    const int dx_type = g.p.x_dtype == SNN_B200_SPIKES ? SNN_B200_F32 : g.p.x_dtype;
    float e = g.dh_last ? g.dh_last[i] : 0.0f, total = 0.0f;
    for (uint64_t k = blocks; k-- > 0;) {
        float before[kBlockSteps], u[kBlockSteps];
        float h = g.saved[(b * blocks + k) * g.p.channels + c], sum = 0.0f;
        const uint64_t t0 = k * kBlockSteps;
        for (uint32_t j = 0; j < kBlockSteps && t0 + j < len; ++j) {
            const Leak l = leak_at(g, b, t0 + j, c);
            before[j] = h;
            u[j] = __fmul_rn(g.p.input_scale, load_any(g.x, g.p.x_dtype, (int64_t)b * g.p.x_batch_stride +
                                                                               (int64_t)(t0 + j) * g.p.x_step_stride +
                                                                               (int64_t)c));
            h = __fmaf_rn(l.a, h, g.p.complement ? __fmul_rn(u[j], l.rest) : u[j]);
        }
        for (uint32_t j = kBlockSteps; j-- > 0;) {
            const uint64_t t = t0 + j;
            if (t >= g.p.steps) continue;
            float dx = 0.0f, dz = 0.0f;
            if (t < len) {
                const Leak l = leak_at(g, b, t, c);
                const float d = __fadd_rn(
                    load_any(g.dy, g.p.y_dtype,
                             (int64_t)b * g.p.dy_batch_stride + (int64_t)t * g.p.dy_step_stride + (int64_t)c),
                    e);
                e = __fmul_rn(l.a, d);
                dx = __fmul_rn(g.p.input_scale, g.p.complement ? __fmul_rn(d, l.rest) : d);
                dz = __fmul_rn(d, g.p.complement ? __fsub_rn(before[j], u[j]) : before[j]);
                if (g.p.logit) dz = __fmul_rn(dz, __fmul_rn(l.a, l.rest));
                sum = __fadd_rn(sum, dz);
            }
            if (g.dx)
                store_any(g.dx, dx_type,
                          (int64_t)b * g.p.dx_batch_stride + (int64_t)t * g.p.dx_step_stride + (int64_t)c, dx);
            if (g.dgate && g.p.gate_step_stride)
                store_any(g.dgate, g.p.gate_dtype,
                          (int64_t)b * g.p.dgate_batch_stride + (int64_t)t * g.p.dgate_step_stride + (int64_t)c, dz);
        }
        total = __fadd_rn(total, sum);
    }
    if (g.dh0) g.dh0[i] = e;
    if (g.dgate && !g.p.gate_step_stride) {
        if (g.p.gate_batch_stride) ((float *)g.dgate)[(int64_t)b * g.p.dgate_batch_stride + (int64_t)c] = total;
        else g.partial[i] = total;
    }
}

// A gate shared over the sequences: their sums, added in order.
__global__ void leaky_gate_sum_kernel(const float *partial, uint64_t batch, uint64_t channels, float *dgate) {
    const uint64_t c = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= channels) return;
    float sum = 0.0f;
    for (uint64_t b = 0; b < batch; ++b) sum = __fadd_rn(sum, partial[b * channels + c]);
    dgate[c] = sum;
}

struct StepArgs {
    uint64_t batch, slot_count, channels;
    const void *x, *gate;
    int x_dtype, gate_dtype, y_dtype, logit, complement;
    int64_t x_stride, gate_stride, pool_stride, y_stride;
    float decay, input_scale;
    float *pool;
    const int32_t *slots;
    void *y;
};

// A thread does the row that names a slot first, and in order the later
// rows that name it too.
__global__ void leaky_step_kernel(StepArgs g) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= g.batch * g.channels) return;
    const uint64_t row = i / g.channels, c = i % g.channels;
    const int64_t slot = g.slots ? (int64_t)g.slots[row] : (int64_t)row;
    if (slot < 0 || (uint64_t)slot >= g.slot_count) {
        store_any(g.y, g.y_dtype, (int64_t)row * g.y_stride + (int64_t)c, 0.0f);
        return;
    }
    if (g.slots)
        for (uint64_t r = 0; r < row; ++r)
            if (g.slots[r] == (int32_t)slot) return;
    float h = g.pool[slot * g.pool_stride + (int64_t)c];
    for (uint64_t r = row; r < g.batch; ++r) {
        if (r != row && (!g.slots || g.slots[r] != (int32_t)slot)) continue;
        const Leak l = g.gate ? leak_of(load_any(g.gate, g.gate_dtype, (int64_t)r * g.gate_stride + (int64_t)c), g.logit)
                              : Leak{g.decay, __fsub_rn(1.0f, g.decay)};
        float u = __fmul_rn(g.input_scale, load_any(g.x, g.x_dtype, (int64_t)r * g.x_stride + (int64_t)c));
        if (g.complement) u = __fmul_rn(u, l.rest);
        h = __fmaf_rn(l.a, h, u);
        store_any(g.y, g.y_dtype, (int64_t)r * g.y_stride + (int64_t)c, h);
    }
    g.pool[slot * g.pool_stride + (int64_t)c] = h;
}

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

uint32_t grid_of(uint64_t threads) { return (uint32_t)((threads + 127) / 128); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

snn_size_t snn_b200_leaky_saved_floats(snn_size_t batch, snn_size_t steps, snn_size_t channels) {
    if (batch > kMaxCount || steps > kMaxCount || channels > kMaxCount) return 0;
    return batch * ((steps + kBlockSteps - 1) / kBlockSteps) * channels;
}

snn_size_t snn_b200_leaky_workspace(const snn_b200_leaky_t *q) {
    if (q == nullptr || q->batch > kMaxCount || q->steps > kMaxCount || q->channels > kMaxCount) return 0;
    return q->batch * q->channels * 4;
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
    const uint64_t need = snn_b200_leaky_workspace(leaky);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)) return SNN_ERR_INVALID_ARGUMENT;
    if (q.batch * q.channels > kMaxCount) return SNN_ERR_OVERFLOW;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    Args g = {};
    g.p = q, g.x = x, g.gate = gate, g.h0 = h0, g.lengths = lengths, g.y = y, g.h_last = h_last, g.saved = saved;
    leaky_scan_kernel<<<grid_of(q.batch * q.channels), 128, 0, (cudaStream_t)stream>>>(g);
    return op_status(cudaGetLastError(), __func__);
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
    const uint64_t need = snn_b200_leaky_workspace(leaky);
    if (need && (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16)))
        return SNN_ERR_INVALID_ARGUMENT;
    if (q.batch * q.channels > kMaxCount) return SNN_ERR_OVERFLOW;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return op_status(scope.error(), __func__);
    Args g = {};
    g.p = q, g.x = x, g.gate = gate, g.lengths = lengths, g.saved = const_cast<float *>(saved), g.dy = dy;
    g.dh_last = dh_last, g.dx = dx, g.dgate = dgate, g.dh0 = dh0, g.partial = (float *)workspace;
    const cudaStream_t s = (cudaStream_t)stream;
    if (q.batch) leaky_backward_kernel<<<grid_of(q.batch * q.channels), 128, 0, s>>>(g);
    if (dgate && shared)
        leaky_gate_sum_kernel<<<grid_of(q.channels), 128, 0, s>>>(g.partial, q.batch, q.channels, (float *)dgate);
    return op_status(cudaGetLastError(), __func__);
}

snn_status_t snn_b200_leaky_step_async(int device, void *stream, snn_size_t batch, snn_size_t slot_count,
                                       snn_size_t channels, const void *x, int x_dtype, int64_t x_row_stride,
                                       const void *gate, int gate_dtype, int64_t gate_row_stride, int logit,
                                       int complement, float decay, float input_scale, float *pool,
                                       int64_t pool_row_stride, const int32_t *slots, void *y, int y_dtype,
                                       int64_t y_row_stride) {
    if (device < 0) return SNN_ERR_INVALID_ARGUMENT;
    if (batch > kMaxCount || slot_count > kMaxCount || channels > kMaxCount) return SNN_ERR_OVERFLOW;
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
    const StepArgs g = {batch, slot_count, channels, x, gate, x_dtype, gate_dtype, y_dtype, logit, complement,
                        x_row_stride, gate_row_stride, pool_row_stride, y_row_stride, decay, input_scale, pool, slots, y};
    leaky_step_kernel<<<grid_of(batch * channels), 128, 0, (cudaStream_t)stream>>>(g);
    return op_status(cudaGetLastError(), __func__);
}

}  // extern "C"
