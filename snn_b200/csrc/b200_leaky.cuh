// Kernels of the leaky recurrence h[t] = a[t] h[t-1] + u[t] and of its
// gradient, instantiated once for each type of x.
//
// Two forms. A thread always holds kSteps consecutive steps of `V`
// neighbouring channels in registers, and the threads of a warp lie side by
// side across (batch, channel), so every access is one run of 32 V elements.
//
//  * whole: a warp walks through all steps of its channels, kSteps at a time,
//    with the state in registers.
//  * split: a CTA takes one tile of kTile steps (its warps one block of kSteps
//    each). Steps compose as affine maps h -> A h + H, so each tile publishes
//    its (A, H) at once and then folds the maps of the tiles before it onto
//    the last published state. States are published every kSuper tiles, so a
//    tile waits for fewer than kSuper neighbours and one state, always in the
//    same order: the result does not depend on timing.
//    Tiles are handed out by a ticket, all channels of a tile before the next
//    tile, so whatever a tile waits for has started already.
#pragma once

#include "b200_leaky.h"

#include <type_traits>

namespace b200 {
namespace leaky {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr uint32_t kPollLimit = 1u << 22;  // polls of 32+ ns each before a wait gives up

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

// No gate array, or one without a step stride: the gate is a constant of the thread.
struct Fixed {};

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

__device__ __forceinline__ uint32_t load_acquire(const uint32_t *p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void store_release(uint32_t *p, uint32_t v) {
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// Waits until a flag is set; false when it gave up.
__device__ __forceinline__ bool wait_flag(const uint32_t *p) {
    for (uint32_t i = 0; i < kPollLimit; ++i) {
        if (load_acquire(p)) return true;
        __nanosleep(32);
    }
    return false;
}

// A thread's place: V channels of one sequence. Lanes behind the last
// channel take part in the shuffles and waits with a length of zero.
struct Place {
    uint64_t i;  // first of its (batch, channel) numbers
    int64_t b, c;
    uint32_t len;
    bool on;
};
template <int V>
__device__ __forceinline__ Place place_of(const Args &g, uint64_t column) {
    Place p;
    p.i = (column * 32 + (threadIdx.x & 31)) * V;
    p.on = p.i < g.flat;
    p.b = p.on ? (int64_t)(p.i / g.channels) : 0;
    p.c = p.on ? (int64_t)(p.i - (uint64_t)p.b * g.channels) : 0;
    p.len = !p.on ? 0u : g.lengths ? min(g.lengths[p.b], g.steps) : g.steps;
    return p;
}
__device__ __forceinline__ int live_steps(uint32_t len, uint32_t t0) {
    return len <= t0 ? 0 : (int)min(len - t0, kSteps);
}

template <typename T, int V>
__device__ __forceinline__ void load_steps(Vec<T, V> (&r)[kSteps], const T *p, int64_t stride, int live) {
#pragma unroll
    for (int j = 0; j < (int)kSteps; ++j)
        if (j < live) r[j] = *reinterpret_cast<const Vec<T, V> *>(p + j * stride);
        else r[j] = Vec<T, V>{};
}

// The gates of a thread's steps. Fixed gates are kept once.
template <typename G, int V>
struct Gates {
    Vec<G, V> raw[kSteps];
    __device__ __forceinline__ void load(const Args &g, const Place &p, uint32_t t0, int live) {
        load_steps<G, V>(raw, (const G *)g.gate + p.b * g.gb + (int64_t)t0 * g.gt + p.c, g.gt, live);
    }
    __device__ __forceinline__ Leak at(const Args &g, int j, int q) const {
        return leak_of(to_float(raw[j].v[q]), g.logit);
    }
};
template <int V>
struct Gates<Fixed, V> {
    Leak leak[V];
    __device__ __forceinline__ void init(const Args &g, const Place &p) {
#pragma unroll
        for (int q = 0; q < V; ++q)
            leak[q] = !g.gate ? Leak{g.decay, __fsub_rn(1.0f, g.decay)}
                              : p.on ? leak_of(((const float *)g.gate)[p.b * g.gb + p.c + q], g.logit) : Leak{1.0f, 0.0f};
    }
    __device__ __forceinline__ void load(const Args &, const Place &, uint32_t, int) {}
    __device__ __forceinline__ Leak at(const Args &, int, int q) const { return leak[q]; }
};
template <typename G, int V>
__device__ __forceinline__ void init_gates(Gates<G, V> &, const Args &, const Place &) {}
template <int V>
__device__ __forceinline__ void init_gates(Gates<Fixed, V> &k, const Args &g, const Place &p) {
    k.init(g, p);
}

template <int V>
__device__ __forceinline__ Vec<float, V> load_state(const float *p, uint64_t i, bool on) {
    return on && p ? *reinterpret_cast<const Vec<float, V> *>(p + i) : Vec<float, V>{};
}

// The state before a block of steps, kept for the backward pass.
template <int V>
__device__ __forceinline__ float *saved_at(const Args &g, const Place &p, uint32_t t0) {
    const uint32_t blocks = (g.steps + kSteps - 1) / kSteps;
    return g.saved + ((uint64_t)p.b * blocks + t0 / kSteps) * g.channels + p.c;
}

// Walks a thread's steps from state h on, writing y.
template <typename Y, int V>
__device__ __forceinline__ void emit(const Args &g, const Place &p, uint32_t t0, int live,
                                     const float (&a)[kSteps][V], const float (&u)[kSteps][V], Vec<float, V> &h) {
    if (!p.on) return;
    if (g.saved) *reinterpret_cast<Vec<float, V> *>(saved_at<V>(g, p, t0)) = h;
    Y *y = (Y *)g.y + p.b * g.yb + (int64_t)t0 * g.yt + p.c;
    const int rows = (int)min(g.steps - t0, kSteps);
#pragma unroll
    for (int j = 0; j < (int)kSteps; ++j) {
        Vec<Y, V> o;
#pragma unroll
        for (int q = 0; q < V; ++q) {
            h.v[q] = __fmaf_rn(a[j][q], h.v[q], u[j][q]);
            o.v[q] = from_float<Y>(j < live ? h.v[q] : 0.0f);
        }
        if (j < rows) *reinterpret_cast<Vec<Y, V> *>(y + j * g.yt) = o;
    }
}

// Gates and inputs of a thread's steps; rows behind the sequence keep the state (a = 1, u = 0).
template <typename X, typename G, int V>
__device__ __forceinline__ void gather(const Args &g, const Place &p, uint32_t t0, int live, Gates<G, V> &gates,
                                       float (&a)[kSteps][V], float (&u)[kSteps][V]) {
    Vec<X, V> x[kSteps];
    gates.load(g, p, t0, live);
    load_steps<X, V>(x, (const X *)g.x + p.b * g.xb + (int64_t)t0 * g.xt + p.c, g.xt, live);
#pragma unroll
    for (int j = 0; j < (int)kSteps; ++j)
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const Leak l = gates.at(g, j, q);
            float v = __fmul_rn(g.scale, to_float(x[j].v[q]));
            if (g.complement) v = __fmul_rn(v, l.rest);
            a[j][q] = j < live ? l.a : 1.0f;
            u[j][q] = j < live ? v : 0.0f;
        }
}

template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(128) scan_whole_kernel(Args g) {
    const Place p = place_of<V>(g, (uint64_t)blockIdx.x * 4 + threadIdx.x / 32);
    if (!p.on) return;
    Gates<G, V> gates;
    init_gates(gates, g, p);
    Vec<float, V> h = load_state<V>(g.h0, p.i, true);
    for (uint32_t t0 = 0; t0 < g.steps; t0 += kSteps) {
        float a[kSteps][V], u[kSteps][V];
        const int live = live_steps(p.len, t0);
        gather<X, G, V>(g, p, t0, live, gates, a, u);
        emit<Y, V>(g, p, t0, live, a, u, h);
    }
    if (g.h_last) *reinterpret_cast<Vec<float, V> *>(g.h_last + p.i) = h;
}

// ---- split form ----
struct Tile {
    uint32_t k;       // along the steps (in the direction of the walk)
    uint64_t column;  // across the channels
};
__device__ __forceinline__ Tile take_tile(const Args &g) {
    __shared__ uint32_t s_ticket;
    if (threadIdx.x == 0) s_ticket = atomicAdd(g.ticket, 1u);
    __syncthreads();
    return {s_ticket / g.columns, s_ticket % g.columns};
}

template <int V>
struct Exchange {
    float2 map[kWarps][32 * V];  // each warp's (A, H)
    float state[32 * V];         // the state that enters the tile
};

// Publishes the tile's map and finds the state that enters it; `first` is
// the state that enters tile 0. Warp w's own map is in ex.map[w]; `order`
// gives the warps in the direction of the walk. On return (after a barrier)
// ex.state is set.
template <int V, bool Reverse>
__device__ __forceinline__ void link_tiles(const Args &g, const Tile &tile, Exchange<V> &ex, const float *first,
                                           bool on, uint64_t i) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint64_t width = (uint64_t)g.columns * 32 * V, at = tile.column * 32 * V + lane * V;
    const bool last = tile.k + 1 == g.tiles;
    const bool keeps = !last && (tile.k + 1) % kSuper == 0;  // publishes a state
    if (warp < 2 && (warp == 1 || !last)) {
        // Both warps need the tile's map (warp 1 only to publish a state).
        float2 m[V];
#pragma unroll
        for (int q = 0; q < V; ++q) {
            m[q] = make_float2(1.0f, 0.0f);
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                const float2 n = ex.map[Reverse ? kWarps - 1 - w : w][lane * V + q];
                m[q] = make_float2(__fmul_rn(n.x, m[q].x), __fmaf_rn(n.x, m[q].y, n.y));
            }
        }
        if (warp == 0) {
#pragma unroll
            for (int q = 0; q < V; ++q) g.aggregates[tile.k * width + at + q] = m[q];
            __threadfence();
            __syncwarp();
            if (lane == 0) store_release(g.tile_flags + (uint64_t)tile.k * g.columns + tile.column, 1u);
        } else {
            const uint32_t super = tile.k / kSuper, before = tile.k % kSuper;
            bool ok = true;
            if (lane < before)
                ok = wait_flag(g.tile_flags + (uint64_t)(super * kSuper + lane) * g.columns + tile.column);
            else if (lane == 31 && super)
                ok = wait_flag(g.state_flags + (uint64_t)(super - 1) * g.columns + tile.column);
            ok = __all_sync(kAll, ok);
            float h[V];
#pragma unroll
            for (int q = 0; q < V; ++q)
                h[q] = super ? __ldcg(g.states + (super - 1) * width + at + q) : on && first ? first[i + q] : 0.0f;
            const float2 *maps = g.aggregates + (uint64_t)super * kSuper * width + at;
#pragma unroll 4
            for (uint32_t k = 0; k < before; ++k)
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    const float2 n = __ldcg(maps + k * width + q);
                    h[q] = __fmaf_rn(n.x, h[q], n.y);
                }
#pragma unroll
            for (int q = 0; q < V; ++q) {
                if (!ok) h[q] = __uint_as_float(0x7fffffffu);  // a wait gave up: let the result say so
                ex.state[lane * V + q] = h[q];
                if (keeps) g.states[super * width + at + q] = __fmaf_rn(m[q].x, h[q], m[q].y);
            }
            if (keeps) {
                __threadfence();
                __syncwarp();
                if (lane == 0) store_release(g.state_flags + (uint64_t)super * g.columns + tile.column, 1u);
            }
        }
    }
    __syncthreads();
}

template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(kWarps * 32, 2) scan_split_kernel(Args g) {
    __shared__ Exchange<V> ex;
    const Tile tile = take_tile(g);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const Place p = place_of<V>(g, tile.column);
    const uint32_t t0 = tile.k * kTile + warp * kSteps;
    Gates<G, V> gates;
    init_gates(gates, g, p);
    float a[kSteps][V], u[kSteps][V];
    const int live = live_steps(p.len, t0);
    gather<X, G, V>(g, p, t0, live, gates, a, u);
#pragma unroll
    for (int q = 0; q < V; ++q) {
        float2 m = make_float2(1.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j)
            m = make_float2(__fmul_rn(a[j][q], m.x), __fmaf_rn(a[j][q], m.y, u[j][q]));
        ex.map[warp][lane * V + q] = m;
    }
    __syncthreads();
    link_tiles<V, false>(g, tile, ex, g.h0, p.on, p.i);
    Vec<float, V> h;
#pragma unroll
    for (int q = 0; q < V; ++q) {
        h.v[q] = ex.state[lane * V + q];
        for (uint32_t w = 0; w < warp; ++w) {
            const float2 n = ex.map[w][lane * V + q];
            h.v[q] = __fmaf_rn(n.x, h.v[q], n.y);
        }
    }
    if (t0 < g.steps) emit<Y, V>(g, p, t0, live, a, u, h);
    if (g.h_last && p.on && tile.k + 1 == g.tiles && warp + 1 == kWarps)
        *reinterpret_cast<Vec<float, V> *>(g.h_last + p.i) = h;
}

// ---- gradient ----
// With d[t] = dy[t] + e[t+1] and e[t] = a[t] d[t] (e behind the last step:
// dh_last), the walk goes back through the steps as the map e -> a (dy + e):
//   dx = scale d (1 - a if complement),  da = d (h[t-1] - scale x if complement).
// The states come from the one before each block of kSteps, kept by the scan.
template <typename X>
struct GradientOf {
    using type = X;
};
template <>
struct GradientOf<Spike> {
    using type = float;
};

template <typename X, typename G, typename Y, int V>
struct Back {
    Gates<G, V> gates;
    float a[kSteps][V], rest[kSteps][V], dy[kSteps][V], k[kSteps][V];  // k: what d is multiplied with

    __device__ __forceinline__ void gather(const Args &g, const Place &p, uint32_t t0, int live) {
        Vec<X, V> x[kSteps];
        Vec<Y, V> d[kSteps];
        gates.load(g, p, t0, live);
        load_steps<X, V>(x, (const X *)g.x + p.b * g.xb + (int64_t)t0 * g.xt + p.c, g.xt, live);
        load_steps<Y, V>(d, (const Y *)g.dy + p.b * g.dyb + (int64_t)t0 * g.dyt + p.c, g.dyt, live);
        Vec<float, V> h = live ? *reinterpret_cast<const Vec<float, V> *>(saved_at<V>(g, p, t0)) : Vec<float, V>{};
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j)
#pragma unroll
            for (int q = 0; q < V; ++q) {
                const Leak l = gates.at(g, j, q);
                const float v = __fmul_rn(g.scale, to_float(x[j].v[q]));
                k[j][q] = g.complement ? __fsub_rn(h.v[q], v) : h.v[q];
                h.v[q] = __fmaf_rn(l.a, h.v[q], g.complement ? __fmul_rn(v, l.rest) : v);
                a[j][q] = j < live ? l.a : 1.0f;
                rest[j][q] = l.rest;
                dy[j][q] = to_float(d[j].v[q]);
            }
    }
    // Walks back from e, writes dx and the gradient of a gate with a value
    // for every step, and returns the block's sum of da in sum.
    __device__ __forceinline__ void emit(const Args &g, const Place &p, uint32_t t0, int live, Vec<float, V> &e,
                                         float (&sum)[V]) {
        using D = typename GradientOf<X>::type;
        constexpr bool every = !std::is_same<G, Fixed>::value;
        D *dx = (D *)g.dx + p.b * g.dxb + (int64_t)t0 * g.dxt + p.c;
        const int rows = t0 < g.steps ? (int)min(g.steps - t0, kSteps) : 0;
#pragma unroll
        for (int q = 0; q < V; ++q) sum[q] = 0.0f;
#pragma unroll
        for (int j = (int)kSteps - 1; j >= 0; --j) {
            Vec<D, V> ox;
            Vec<float, V> oz;
#pragma unroll
            for (int q = 0; q < V; ++q) {
                const bool on = j < live;
                const float d = __fadd_rn(dy[j][q], e.v[q]);
                e.v[q] = __fmul_rn(a[j][q], on ? d : e.v[q]);
                const float f = g.complement ? __fmul_rn(d, rest[j][q]) : d;
                ox.v[q] = from_float<D>(on ? __fmul_rn(g.scale, f) : 0.0f);
                const float z = on ? __fmul_rn(d, k[j][q]) : 0.0f;
                if (every) oz.v[q] = g.logit && on ? __fmul_rn(z, __fmul_rn(a[j][q], rest[j][q])) : z;
                else sum[q] = __fadd_rn(sum[q], z);
            }
            if (p.on && j < rows) {
                if (g.dx) *reinterpret_cast<Vec<D, V> *>(dx + j * g.dxt) = ox;
                if constexpr (every) {
                    if (g.dgate) {
                        Vec<G, V> o;
#pragma unroll
                        for (int q = 0; q < V; ++q) o.v[q] = from_float<G>(oz.v[q]);
                        *reinterpret_cast<Vec<G, V> *>((G *)g.dgate + p.b * g.dgb + (int64_t)(t0 + j) * g.dgt + p.c) = o;
                    }
                }
            }
        }
    }
};

// A shared gate's sum for one thread: of logits, the gate's own slope is a common factor.
template <int V>
__device__ __forceinline__ void put_partial(const Args &g, const Place &p, const Gates<Fixed, V> &gates, uint32_t tile,
                                            const float (&sum)[V]) {
#pragma unroll
    for (int q = 0; q < V; ++q)
        g.partial[tile * g.flat + p.i + q] =
            g.logit && g.gate ? __fmul_rn(sum[q], __fmul_rn(gates.leak[q].a, gates.leak[q].rest)) : sum[q];
}
template <typename G, int V>
__device__ __forceinline__ void put_partial(const Args &, const Place &, const Gates<G, V> &, uint32_t,
                                            const float (&)[V]) {}

template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(128) back_whole_kernel(Args g) {
    const Place p = place_of<V>(g, (uint64_t)blockIdx.x * 4 + threadIdx.x / 32);
    if (!p.on) return;
    Back<X, G, Y, V> w;
    init_gates(w.gates, g, p);
    Vec<float, V> e = load_state<V>(g.dh_last, p.i, true);
    double total[V] = {};
    for (uint32_t n = (g.steps + kSteps - 1) / kSteps; n-- > 0;) {
        const uint32_t t0 = n * kSteps;
        const int live = live_steps(p.len, t0);
        float sum[V];
        w.gather(g, p, t0, live);
        w.emit(g, p, t0, live, e, sum);
        if (std::is_same<G, Fixed>::value)
#pragma unroll
            for (int q = 0; q < V; ++q) total[q] += (double)sum[q];
    }
    if (g.dh0) *reinterpret_cast<Vec<float, V> *>(g.dh0 + p.i) = e;
    if (g.partial) {
        float sum[V];
#pragma unroll
        for (int q = 0; q < V; ++q) sum[q] = (float)total[q];
        put_partial(g, p, w.gates, 0, sum);
    }
}

template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(kWarps * 32) back_split_kernel(Args g) {
    __shared__ Exchange<V> ex;
    const Tile tile = take_tile(g);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const Place p = place_of<V>(g, tile.column);
    const uint32_t t0 = (g.tiles - 1 - tile.k) * kTile + warp * kSteps;
    Back<X, G, Y, V> w;
    init_gates(w.gates, g, p);
    const int live = live_steps(p.len, t0);
    w.gather(g, p, t0, live);
#pragma unroll
    for (int q = 0; q < V; ++q) {
        float2 m = make_float2(1.0f, 0.0f);
#pragma unroll
        for (int j = (int)kSteps - 1; j >= 0; --j)
            m = make_float2(__fmul_rn(w.a[j][q], m.x),
                            __fmul_rn(w.a[j][q], j < live ? __fadd_rn(m.y, w.dy[j][q]) : m.y));
        ex.map[warp][lane * V + q] = m;
    }
    __syncthreads();
    link_tiles<V, true>(g, tile, ex, g.dh_last, p.on, p.i);
    Vec<float, V> e;
#pragma unroll
    for (int q = 0; q < V; ++q) {
        e.v[q] = ex.state[lane * V + q];
        for (uint32_t n = kWarps - 1; n > warp; --n) {
            const float2 m = ex.map[n][lane * V + q];
            e.v[q] = __fmaf_rn(m.x, e.v[q], m.y);
        }
    }
    float sum[V];
    w.emit(g, p, t0, live, e, sum);
    if (g.dh0 && p.on && tile.k + 1 == g.tiles && warp == 0) *reinterpret_cast<Vec<float, V> *>(g.dh0 + p.i) = e;
    if (std::is_same<G, Fixed>::value && g.partial) {
        __syncthreads();  // ex.map is read above
#pragma unroll
        for (int q = 0; q < V; ++q) ex.map[warp][lane * V + q].x = sum[q];
        __syncthreads();
        if (warp == 0 && p.on) {
#pragma unroll
            for (int q = 0; q < V; ++q) {
                double s = 0.0;
                for (uint32_t n = 0; n < kWarps; ++n) s += (double)ex.map[n][lane * V + q].x;
                sum[q] = (float)s;
            }
            put_partial(g, p, w.gates, tile.k, sum);
        }
    }
}

// ---- single step ----
// A row of the pool is updated by the threads of the first row that names
// it, which also do the later rows that name it, in order. To know, every CTA
// looks through the slots once, for all of its rows at a time.
template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(256) step_kernel(StepArgs g) {
    __shared__ uint32_t s_before[8], s_after[8];  // rows named before, rows named again
    const uint32_t across = 256 / g.rows, mine = threadIdx.x / across;
    const uint32_t row = blockIdx.x * g.rows + mine;
    if (g.slots && g.batch > 1) {
        if (threadIdx.x < 8) s_before[threadIdx.x] = s_after[threadIdx.x] = 0u;
        __syncthreads();
        int32_t named[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r) {
            const uint32_t n = blockIdx.x * g.rows + r;
            named[r] = r < g.rows && n < g.batch ? g.slots[n] : -1;
        }
        for (uint32_t n = threadIdx.x; n < g.batch; n += 256) {
            const int32_t s = g.slots[n];
            if (s < 0) continue;
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {
                const uint32_t of = blockIdx.x * g.rows + r;
                if (s == named[r] && n != of) (n < of ? s_before : s_after)[r] = 1u;
            }
        }
        __syncthreads();
        if (s_before[mine]) return;
    }
    if (row >= g.batch) return;
    const bool again = g.slots && g.batch > 1 && s_after[mine];
    const int64_t slot = g.slots ? (int64_t)g.slots[row] : (int64_t)row;
    const bool padding = slot < 0 || slot >= (int64_t)g.slot_count;
    for (uint64_t c = ((uint64_t)blockIdx.y * across + threadIdx.x % across) * V; c < g.channels;
         c += (uint64_t)gridDim.y * across * V) {
        Vec<Y, V> o = {};
        if (padding) {
            *reinterpret_cast<Vec<Y, V> *>((Y *)g.y + row * g.ys + c) = o;
            continue;
        }
        Vec<float, V> *state = reinterpret_cast<Vec<float, V> *>(g.pool + slot * g.ps + c);
        Vec<float, V> h = *state;
        for (uint32_t r = row; r < g.batch; ++r) {
            if (r != row && g.slots[r] != (int32_t)slot) continue;
            const Vec<X, V> x = *reinterpret_cast<const Vec<X, V> *>((const X *)g.x + r * g.xs + c);
            Vec<G, V> z = {};
            if (g.gate) z = *reinterpret_cast<const Vec<G, V> *>((const G *)g.gate + r * g.gs + c);
#pragma unroll
            for (int q = 0; q < V; ++q) {
                const Leak l = g.gate ? leak_of(to_float(z.v[q]), g.logit) : Leak{g.decay, __fsub_rn(1.0f, g.decay)};
                float u = __fmul_rn(g.scale, to_float(x.v[q]));
                if (g.complement) u = __fmul_rn(u, l.rest);
                h.v[q] = __fmaf_rn(l.a, h.v[q], u);
                o.v[q] = from_float<Y>(h.v[q]);
            }
            *reinterpret_cast<Vec<Y, V> *>((Y *)g.y + r * g.ys + c) = o;
            if (!again) break;
        }
        *state = h;
    }
}

template <typename X, typename G, typename Y>
cudaError_t launch_step(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    if (f.width == 4) step_kernel<X, G, Y, 4><<<grid, 256, 0, s>>>(a);
    else step_kernel<X, G, Y, 1><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}
template <typename X>
cudaError_t step_wide(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    return launch_step<X, float, float>(s, f, a, grid);
}
template <typename X>
cudaError_t step_narrow(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    const bool wide = f.y_dtype == SNN_B200_F32;
    if (f.gate_dtype == SNN_B200_F32)
        return wide ? launch_step<X, float, float>(s, f, a, grid) : launch_step<X, float, X>(s, f, a, grid);
    return wide ? launch_step<X, X, float>(s, f, a, grid) : launch_step<X, X, X>(s, f, a, grid);
}

template <typename X, typename G, typename Y, int V>
void launch_forward(cudaStream_t s, const Form &f, const Args &a) {
    if (f.split) scan_split_kernel<X, G, Y, V><<<a.tiles * a.columns, kWarps * 32, 0, s>>>(a);
    else scan_whole_kernel<X, G, Y, V><<<(a.columns + 3) / 4, 128, 0, s>>>(a);
}
template <typename X, typename G, typename Y, int V>
void launch_backward(cudaStream_t s, const Form &f, const Args &a) {
    if (f.split) back_split_kernel<X, G, Y, V><<<a.tiles * a.columns, kWarps * 32, 0, s>>>(a);
    else back_whole_kernel<X, G, Y, V><<<(a.columns + 3) / 4, 128, 0, s>>>(a);
}

template <typename X, typename G, typename Y>
cudaError_t launch(cudaStream_t s, const Form &f, const Args &a, bool back) {
    if (back) {
        if (f.width == 2) launch_backward<X, G, Y, 2>(s, f, a);
        else launch_backward<X, G, Y, 1>(s, f, a);
    } else {
        if (f.width == 2) launch_forward<X, G, Y, 2>(s, f, a);
        else launch_forward<X, G, Y, 1>(s, f, a);
    }
    return cudaGetLastError();
}

// The combinations of types for 32-bit and spike inputs, and for 16-bit ones.
template <typename X>
cudaError_t launch_wide(cudaStream_t s, const Form &f, const Args &a, bool back) {
    return f.every ? launch<X, float, float>(s, f, a, back) : launch<X, Fixed, float>(s, f, a, back);
}
template <typename X>
cudaError_t launch_narrow(cudaStream_t s, const Form &f, const Args &a, bool back) {
    const bool wide = f.y_dtype == SNN_B200_F32;
    if (!f.every) return wide ? launch<X, Fixed, float>(s, f, a, back) : launch<X, Fixed, X>(s, f, a, back);
    if (f.gate_dtype == SNN_B200_F32)
        return wide ? launch<X, float, float>(s, f, a, back) : launch<X, float, X>(s, f, a, back);
    return wide ? launch<X, X, float>(s, f, a, back) : launch<X, X, X>(s, f, a, back);
}

}  // namespace
}  // namespace leaky
}  // namespace b200
