// Kernels of the leaky recurrence h[t] = a[t] h[t-1] + u[t] and of its
// gradient, instantiated once for each type of x.
//
// Two forms. A thread always holds kSteps consecutive steps of `V`
// neighbouring channels in registers, and the threads of a warp lie side by
// side across (batch, channel), so every access is one run of 32 V elements.
//
//  * whole: a warp walks through all steps of its channels, kSteps at a time,
//    with the state in registers.
//  * split: a CTA takes one tile of steps (its warps one block of kSteps each). Steps compose as affine maps h -> A h + H, so each tile publishes
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

// Arithmetic on a thread's channels, two at a time where there are two: the
// kernels' instruction count, not their arithmetic, is what is scarce.
template <int V>
using Row = Vec<float, V>;
template <int V>
__device__ __forceinline__ uint64_t two(const Row<V> &a, int q) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.v[q]), "f"(a.v[q + 1]));
    return r;
}
template <int V>
__device__ __forceinline__ void split(uint64_t r, Row<V> &o, int q) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.v[q]), "=f"(o.v[q + 1]) : "l"(r));
}
template <int V>
__device__ __forceinline__ Row<V> fma(const Row<V> &a, const Row<V> &b, const Row<V> &c) {
    Row<V> o;
    if constexpr (V == 1) {
        o.v[0] = __fmaf_rn(a.v[0], b.v[0], c.v[0]);
    } else {
#pragma unroll
        for (int q = 0; q < V; q += 2) {
            uint64_t r;
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(two(a, q)), "l"(two(b, q)), "l"(two(c, q)));
            split(r, o, q);
        }
    }
    return o;
}
template <int V>
__device__ __forceinline__ Row<V> mul(const Row<V> &a, const Row<V> &b) {
    Row<V> o;
    if constexpr (V == 1) {
        o.v[0] = __fmul_rn(a.v[0], b.v[0]);
    } else {
#pragma unroll
        for (int q = 0; q < V; q += 2) {
            uint64_t r;
            asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(a, q)), "l"(two(b, q)));
            split(r, o, q);
        }
    }
    return o;
}
template <int V>
__device__ __forceinline__ Row<V> add(const Row<V> &a, const Row<V> &b) {
    Row<V> o;
    if constexpr (V == 1) {
        o.v[0] = __fadd_rn(a.v[0], b.v[0]);
    } else {
#pragma unroll
        for (int q = 0; q < V; q += 2) {
            uint64_t r;
            asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(a, q)), "l"(two(b, q)));
            split(r, o, q);
        }
    }
    return o;
}
template <int V>
__device__ __forceinline__ Row<V> all(float f) {
    Row<V> o;
#pragma unroll
    for (int q = 0; q < V; ++q) o.v[q] = f;
    return o;
}
template <typename T, int V>
__device__ __forceinline__ Row<V> widen(const Vec<T, V> &a) {
    Row<V> o;
#pragma unroll
    for (int q = 0; q < V; ++q) o.v[q] = to_float(a.v[q]);
    return o;
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const Row<V> &a) {
    Vec<T, V> o;
    if constexpr (V > 1 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int q = 0; q < V; q += 2)
            *reinterpret_cast<__nv_bfloat162 *>(&o.v[q]) = __floats2bfloat162_rn(a.v[q], a.v[q + 1]);
    } else if constexpr (V > 1 && std::is_same<T, __half>::value) {
#pragma unroll
        for (int q = 0; q < V; q += 2)
            *reinterpret_cast<__half2 *>(&o.v[q]) = __floats2half2_rn(a.v[q], a.v[q + 1]);
    } else {
#pragma unroll
        for (int q = 0; q < V; ++q) o.v[q] = from_float<T>(a.v[q]);
    }
    return o;
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T *p) {
    return *reinterpret_cast<const Vec<T, V> *>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store(T *p, const Vec<T, V> &v) {
    *reinterpret_cast<Vec<T, V> *>(p) = v;
}

// No gate array, or one without a step stride: the gate is a constant of the thread.
struct Fixed {};

struct Leak {
    float a, rest;  // the gate and one minus it
};
// Both from one exponential of a non-positive number, so that neither is a
// difference of nearly equal values. A 16-bit logit has a rounding of 2^-9 of
// itself, so for it the product with log2(e) is rounded once to 32 bits (2^-20
// of the exponential up to logits of 22).
template <bool Narrow>
__device__ __forceinline__ Leak leak_of(float z, int logit) {
    if (!logit) return {z, __fsub_rn(1.0f, z)};
    float t;
    if (Narrow) {
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(__fmul_rn(-fabsf(z), 1.44269504f)));
    } else {
        t = expf(-fabsf(z));
    }
    const float r = __fdividef(1.0f, __fadd_rn(1.0f, t)), q = __fmul_rn(t, r);
    return z >= 0.0f ? Leak{r, q} : Leak{q, r};
}
template <typename G>
__device__ __forceinline__ Leak leak_from(G z, int logit) {
    return leak_of<sizeof(G) == 2>(to_float(z), logit);
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

// kSteps rows, all of them wanted by most threads.
template <typename T, int V>
__device__ __forceinline__ void load_steps(Vec<T, V> (&r)[kSteps], const T *p, int64_t stride, int live) {
    if (live == (int)kSteps) {
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j) r[j] = load<T, V>(p + j * stride);
    } else {
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j) r[j] = j < live ? load<T, V>(p + j * stride) : Vec<T, V>{};
    }
}

// The gates of a thread's steps. Fixed gates are kept once.
template <typename G, int V>
struct Gates {
    Vec<G, V> raw[kSteps];
    __device__ __forceinline__ void init(const Args &, const Place &) {}
    __device__ __forceinline__ void load(const Args &g, const Place &p, uint32_t t0, int live) {
        load_steps<G, V>(raw, (const G *)g.gate + p.b * g.gb + (int64_t)t0 * g.gt + p.c, g.gt, live);
    }
    __device__ __forceinline__ void at(const Args &g, int j, Row<V> &a, Row<V> &rest) const {
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const Leak l = leak_from(raw[j].v[q], g.logit);
            a.v[q] = l.a, rest.v[q] = l.rest;
        }
    }
};
template <int V>
struct Gates<Fixed, V> {
    Row<V> a_, rest_;
    __device__ __forceinline__ void init(const Args &g, const Place &p) {
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const Leak l = !g.gate ? Leak{g.decay, __fsub_rn(1.0f, g.decay)}
                           : p.on  ? leak_from(((const float *)g.gate)[p.b * g.gb + p.c + q], g.logit)
                                   : Leak{1.0f, 0.0f};
            a_.v[q] = l.a, rest_.v[q] = l.rest;
        }
    }
    __device__ __forceinline__ void load(const Args &, const Place &, uint32_t, int) {}
    __device__ __forceinline__ void at(const Args &, int, Row<V> &a, Row<V> &rest) const { a = a_, rest = rest_; }
};

template <int V>
__device__ __forceinline__ Row<V> load_state(const float *p, uint64_t i, bool on) {
    return on && p ? load<float, V>(p + i) : Row<V>{};
}

// The state before a block of steps, kept for the backward pass.
__device__ __forceinline__ float *saved_at(const Args &g, const Place &p, uint32_t t0) {
    const uint32_t blocks = (g.steps + kSteps - 1) / kSteps;
    return g.saved + ((uint64_t)p.b * blocks + t0 / kSteps) * g.channels + p.c;
}

// Walks a thread's steps from state h on, writing y.
template <typename Y, int V>
__device__ __forceinline__ void emit(const Args &g, const Place &p, uint32_t t0, int live, const Row<V> (&a)[kSteps],
                                     const Row<V> (&u)[kSteps], Row<V> &h) {
    if (!p.on) return;
    if (g.saved) store<float, V>(saved_at(g, p, t0), h);
    Y *y = (Y *)g.y + p.b * g.yb + (int64_t)t0 * g.yt + p.c;
    if (live == (int)kSteps) {
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j) {
            h = fma(a[j], h, u[j]);
            store<Y, V>(y + j * g.yt, narrow<Y, V>(h));
        }
    } else {
        const int rows = (int)min(g.steps - t0, kSteps);
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j) {
            h = fma(a[j], h, u[j]);
            if (j < rows) store<Y, V>(y + j * g.yt, j < live ? narrow<Y, V>(h) : Vec<Y, V>{});
        }
    }
}

// What a block reads, before it is worked on.
template <typename X, typename G, int V>
struct Inputs {
    Gates<G, V> gates;
    Vec<X, V> x[kSteps];
    __device__ __forceinline__ void load(const Args &g, const Place &p, uint32_t t0, int live) {
        gates.load(g, p, t0, live);
        load_steps<X, V>(x, (const X *)g.x + p.b * g.xb + (int64_t)t0 * g.xt + p.c, g.xt, live);
    }
    // Gates and inputs of the steps; rows behind the sequence keep the state (a = 1, u = 0).
    __device__ __forceinline__ void maps(const Args &g, int live, Row<V> (&a)[kSteps], Row<V> (&u)[kSteps]) const {
        const Row<V> scale = all<V>(g.scale);
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j) {
            Row<V> rest;
            gates.at(g, j, a[j], rest);
            u[j] = mul(scale, widen(x[j]));
            if (g.complement) u[j] = mul(u[j], rest);
        }
        if (live < (int)kSteps) {
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j)
                if (j >= live) a[j] = all<V>(1.0f), u[j] = all<V>(0.0f);
        }
    }
};

template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(128) scan_whole_kernel(Args g) {
    const Place p = place_of<V>(g, (uint64_t)blockIdx.x * 4 + threadIdx.x / 32);
    if (!p.on) return;
    Inputs<X, G, V> in;
    in.gates.init(g, p);
    Row<V> h = load_state<V>(g.h0, p.i, true);
    in.load(g, p, 0, live_steps(p.len, 0));
    for (uint32_t t0 = 0; t0 < g.steps; t0 += kSteps) {
        Row<V> a[kSteps], u[kSteps];
        const int live = live_steps(p.len, t0);
        in.maps(g, live, a, u);
        if (t0 + kSteps < g.steps) in.load(g, p, t0 + kSteps, live_steps(p.len, t0 + kSteps));  // on the way while this block is written
        emit<Y, V>(g, p, t0, live, a, u, h);
    }
    if (g.h_last) store<float, V>(g.h_last + p.i, h);
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

template <int V, uint32_t W>
struct Exchange {
    float2 map[W][32 * V];  // each warp's (A, H)
    float state[32 * V];         // the state that enters the tile
};

// Publishes the tile's map and finds the state that enters it; `first` is
// the state that enters tile 0. Warp w's own map is in ex.map[w]; `order`
// gives the warps in the direction of the walk. On return (after a barrier)
// ex.state is set.
template <int V, uint32_t W, bool Reverse>
__device__ __forceinline__ void link_tiles(const Args &g, const Tile &tile, Exchange<V, W> &ex, const float *first,
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
            for (uint32_t w = 0; w < W; ++w) {
                const float2 n = ex.map[Reverse ? W - 1 - w : w][lane * V + q];
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
__global__ void __launch_bounds__(kScanWarps * 32) scan_split_kernel(Args g) {
    __shared__ Exchange<V, kScanWarps> ex;
    const Tile tile = take_tile(g);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const Place p = place_of<V>(g, tile.column);
    const uint32_t t0 = (tile.k * kScanWarps + warp) * kSteps;
    Row<V> a[kSteps], u[kSteps];
    const int live = live_steps(p.len, t0);
    {
        Inputs<X, G, V> in;
        in.gates.init(g, p);
        in.load(g, p, t0, live);
        in.maps(g, live, a, u);
    }
    Row<V> A = all<V>(1.0f), H = all<V>(0.0f);
#pragma unroll
    for (int j = 0; j < (int)kSteps; ++j) A = mul(a[j], A), H = fma(a[j], H, u[j]);
#pragma unroll
    for (int q = 0; q < V; ++q) ex.map[warp][lane * V + q] = make_float2(A.v[q], H.v[q]);
    __syncthreads();
    link_tiles<V, kScanWarps, false>(g, tile, ex, g.h0, p.on, p.i);
    Row<V> h;
#pragma unroll
    for (int q = 0; q < V; ++q) {
        h.v[q] = ex.state[lane * V + q];
        for (uint32_t w = 0; w < warp; ++w) {
            const float2 n = ex.map[w][lane * V + q];
            h.v[q] = __fmaf_rn(n.x, h.v[q], n.y);
        }
    }
    if (t0 < g.steps) emit<Y, V>(g, p, t0, live, a, u, h);
    if (g.h_last && p.on && tile.k + 1 == g.tiles && warp + 1 == kScanWarps) store<float, V>(g.h_last + p.i, h);
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
    Inputs<X, G, V> in;
    Vec<Y, V> dy[kSteps];
    Row<V> h;
    Row<V> a[kSteps], rest[kSteps], k[kSteps];  // k: what d is multiplied with

    __device__ __forceinline__ void load(const Args &g, const Place &p, uint32_t t0, int live) {
        in.load(g, p, t0, live);
        load_steps<Y, V>(dy, (const Y *)g.dy + p.b * g.dyb + (int64_t)t0 * g.dyt + p.c, g.dyt, live);
        h = live ? leaky::load<float, V>(saved_at(g, p, t0)) : Row<V>{};
    }
    __device__ __forceinline__ void maps(const Args &g, int live) {
        const Row<V> scale = all<V>(g.scale);
#pragma unroll
        for (int j = 0; j < (int)kSteps; ++j) {
            in.gates.at(g, j, a[j], rest[j]);
            const Row<V> v = mul(scale, widen(in.x[j]));
            if (g.complement) {
                k[j] = add(h, mul(all<V>(-1.0f), v));
                h = fma(a[j], h, mul(v, rest[j]));
            } else {
                k[j] = h;
                h = fma(a[j], h, v);
            }
        }
        if (live < (int)kSteps) {
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j)
                if (j >= live) a[j] = all<V>(1.0f);
        }
    }
    // One step back: d and e before it.
    __device__ __forceinline__ Row<V> step(int j, int live, Row<V> &e) const {
        const Row<V> d = add(widen(dy[j]), e);
        if (j < live) e = mul(a[j], d);
        return d;
    }
    // Walks back from e, writes dx and the gradient of a gate with a value
    // for every step, and returns the block's sum of da in sum.
    __device__ __forceinline__ void emit(const Args &g, const Place &p, uint32_t t0, int live, Row<V> &e,
                                         Row<V> &sum) {
        using D = typename GradientOf<X>::type;
        constexpr bool every = !std::is_same<G, Fixed>::value;
        D *dx = (D *)g.dx + p.b * g.dxb + (int64_t)t0 * g.dxt + p.c;
        const int rows = !p.on || t0 >= g.steps ? 0 : (int)min(g.steps - t0, kSteps);
        const Row<V> scale = all<V>(g.scale);
        sum = all<V>(0.0f);
#pragma unroll
        for (int j = (int)kSteps - 1; j >= 0; --j) {
            const bool on = j < live;
            const Row<V> d = step(j, live, e);
            Row<V> z = mul(d, k[j]);
            if (!every && on) sum = add(sum, z);
            if (j >= rows) continue;
            if (g.dx) {
                Row<V> f = mul(scale, d);
                if (g.complement) f = mul(f, rest[j]);
                store<D, V>(dx + j * g.dxt, on ? narrow<D, V>(f) : Vec<D, V>{});
            }
            if constexpr (every) {
                if (g.dgate) {
                    if (g.logit) z = mul(z, mul(a[j], rest[j]));
                    store<G, V>((G *)g.dgate + p.b * g.dgb + (int64_t)(t0 + j) * g.dgt + p.c,
                                on ? narrow<G, V>(z) : Vec<G, V>{});
                }
            }
        }
    }
};

// A shared gate's sum for one thread: of logits, the gate's own slope is a common factor.
template <int V>
__device__ __forceinline__ void put_partial(const Args &g, const Place &p, const Gates<Fixed, V> &gates, uint32_t tile,
                                            const Row<V> &sum) {
    store<float, V>(g.partial + tile * g.flat + p.i, g.logit ? mul(sum, mul(gates.a_, gates.rest_)) : sum);
}
template <typename G, int V>
__device__ __forceinline__ void put_partial(const Args &, const Place &, const Gates<G, V> &, uint32_t,
                                            const Row<V> &) {}

template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(128) back_whole_kernel(Args g) {
    const Place p = place_of<V>(g, (uint64_t)blockIdx.x * 4 + threadIdx.x / 32);
    if (!p.on) return;
    Back<X, G, Y, V> w;
    w.in.gates.init(g, p);
    Row<V> e = load_state<V>(g.dh_last, p.i, true);
    double total[V] = {};
    for (uint32_t n = (g.steps + kSteps - 1) / kSteps; n-- > 0;) {
        const uint32_t t0 = n * kSteps;
        const int live = live_steps(p.len, t0);
        Row<V> sum;
        w.load(g, p, t0, live);
        w.maps(g, live);
        w.emit(g, p, t0, live, e, sum);
        if (std::is_same<G, Fixed>::value)
#pragma unroll
            for (int q = 0; q < V; ++q) total[q] += (double)sum.v[q];
    }
    if (g.dh0) store<float, V>(g.dh0 + p.i, e);
    if (g.partial) {
        Row<V> sum;
#pragma unroll
        for (int q = 0; q < V; ++q) sum.v[q] = (float)total[q];
        put_partial(g, p, w.in.gates, 0, sum);
    }
}

template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(kBackWarps * 32) back_split_kernel(Args g) {
    __shared__ Exchange<V, kBackWarps> ex;
    const Tile tile = take_tile(g);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const Place p = place_of<V>(g, tile.column);
    const uint32_t t0 = ((g.tiles - 1 - tile.k) * kBackWarps + warp) * kSteps;
    Back<X, G, Y, V> w;
    w.in.gates.init(g, p);
    const int live = live_steps(p.len, t0);
    w.load(g, p, t0, live);
    w.maps(g, live);
    Row<V> A = all<V>(1.0f), E = all<V>(0.0f);
#pragma unroll
    for (int j = (int)kSteps - 1; j >= 0; --j) A = mul(w.a[j], A), w.step(j, live, E);
#pragma unroll
    for (int q = 0; q < V; ++q) ex.map[warp][lane * V + q] = make_float2(A.v[q], E.v[q]);
    __syncthreads();
    link_tiles<V, kBackWarps, true>(g, tile, ex, g.dh_last, p.on, p.i);
    Row<V> e;
#pragma unroll
    for (int q = 0; q < V; ++q) {
        e.v[q] = ex.state[lane * V + q];
        for (uint32_t n = kBackWarps - 1; n > warp; --n) {
            const float2 m = ex.map[n][lane * V + q];
            e.v[q] = __fmaf_rn(m.x, e.v[q], m.y);
        }
    }
    Row<V> sum;
    w.emit(g, p, t0, live, e, sum);
    if (g.dh0 && p.on && tile.k + 1 == g.tiles && warp == 0) store<float, V>(g.dh0 + p.i, e);
    if (std::is_same<G, Fixed>::value && g.partial) {
        __syncthreads();  // ex.map is read above
#pragma unroll
        for (int q = 0; q < V; ++q) ex.map[warp][lane * V + q].x = sum.v[q];
        __syncthreads();
        if (warp == 0 && p.on) {
#pragma unroll
            for (int q = 0; q < V; ++q) {
                double s = 0.0;
                for (uint32_t n = 0; n < kBackWarps; ++n) s += (double)ex.map[n][lane * V + q].x;
                sum.v[q] = (float)s;
            }
            put_partial(g, p, w.in.gates, tile.k, sum);
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
                const Leak l = g.gate ? leak_from(z.v[q], g.logit) : Leak{g.decay, __fsub_rn(1.0f, g.decay)};
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
cudaError_t launch_whole(cudaStream_t s, const Args &a, bool back) {
    const uint32_t grid = (a.columns + 3) / 4;
    if (back) back_whole_kernel<X, G, Y, V><<<grid, 128, 0, s>>>(a);
    else scan_whole_kernel<X, G, Y, V><<<grid, 128, 0, s>>>(a);
    return cudaGetLastError();
}
template <typename X, typename G, typename Y, int V>
cudaError_t launch_split(cudaStream_t s, const Args &a, bool back) {
    const uint32_t grid = a.tiles * a.columns;
    if (back) back_split_kernel<X, G, Y, V><<<grid, kBackWarps * 32, 0, s>>>(a);
    else scan_split_kernel<X, G, Y, V><<<grid, kScanWarps * 32, 0, s>>>(a);
    return cudaGetLastError();
}
template <typename X, typename G, typename Y>
cudaError_t launch(cudaStream_t s, const Form &f, const Args &a, bool back) {
    if (f.split) return f.width == 2 ? launch_split<X, G, Y, 2>(s, a, back) : launch_split<X, G, Y, 1>(s, a, back);
    return f.width == 2 ? launch_whole<X, G, Y, 2>(s, a, back) : launch_whole<X, G, Y, 1>(s, a, back);
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
