// Kernels of the leaky recurrence h[t] = a[t] h[t-1] + u[t] and of its
// gradient, instantiated once for each type of x.
//
// A warp walks along the steps of 32 V neighbouring (batch, channel) numbers, a
// thread each V of them, with the state in registers, so every access is one
// run of 32 V elements. What limits it is how much it keeps under way: the next
// blocks of kSteps steps are copied to shared memory (cp.async) while one is
// worked on. 1024 sequences of 64 steps and 1024 channels, bf16 with logits: 69 us
// (5.8 TB/s), the gradient 112 us (6.3 TB/s).
//
// Fewer channels than keep the GPU busy that way are walked by crews: the warps
// of a CTA take the next blocks of one column side by side. Steps compose as
// affine maps h -> A h + H; each warp shares its block's map, folds those before
// its own onto the state, and then walks its block. 4 x 8192 x 2048 (128 columns):
// 109 us, the gradient 165 us, of a floor of 62 and 105. No one thing is the bound: 20 SMs
// have no column, the others' schedulers issue (30 and 49 instructions an element) in 62
// and 63 of 100 cycles, and of the 6.4 cycles a warp takes for an instruction 1.4 are
// fixed latencies, 0.9 to 1.2 shared memory, 0.4 to 0.7 the barrier of a round, 0.5 to
// 1.0 a busy arithmetic pipe.
//
// Where even crews are too few, the steps are cut into segments: one kernel
// walks each segment for its map, one folds them in order into the state before
// each segment, and the walk itself then starts everywhere at once. The inputs
// are read twice. 1 x 65536 x 1024: 133 to 144 us, the gradient 180 us. (One pass
// whose tiles publish maps and wait for the ones before them took 370 to 450 us
// there: the tiles under way are too few to cover the waits.)
#pragma once

#include "b200_leaky.h"

#include <type_traits>

namespace b200 {
namespace leaky {
namespace {

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

// A thread's channels of one step, in 32 bits. Two of them share a register pair
// and an instruction: the instructions, not the arithmetic, are what is scarce.
template <int V>
struct Row {
    uint64_t r[V / 2];
    __device__ __forceinline__ float lo(int i) const {
        float f;
        asm("{\n .reg .b32 h;\n mov.b64 {%0, h}, %1;\n}" : "=f"(f) : "l"(r[i]));
        return f;
    }
    __device__ __forceinline__ float hi(int i) const {
        float f;
        asm("{\n .reg .b32 l;\n mov.b64 {l, %0}, %1;\n}" : "=f"(f) : "l"(r[i]));
        return f;
    }
    __device__ __forceinline__ float operator[](int q) const { return q % 2 ? hi(q / 2) : lo(q / 2); }
    // Element q is f(q).
    template <typename F>
    static __device__ __forceinline__ Row of(F f) {
        Row o;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float l = f(2 * i), h = f(2 * i + 1);
            asm("mov.b64 %0, {%1, %2};" : "=l"(o.r[i]) : "f"(l), "f"(h));
        }
        return o;
    }
};
template <>
struct Row<1> {
    float f;
    __device__ __forceinline__ float operator[](int) const { return f; }
    template <typename F>
    static __device__ __forceinline__ Row of(F g) {
        return {g(0)};
    }
};
template <int V>
__device__ __forceinline__ Row<V> fma(const Row<V> &a, const Row<V> &b, const Row<V> &c) {
    if constexpr (V == 1) {
        return {__fmaf_rn(a.f, b.f, c.f)};
    } else {
        Row<V> o;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(o.r[i]) : "l"(a.r[i]), "l"(b.r[i]), "l"(c.r[i]));
        return o;
    }
}
template <int V>
__device__ __forceinline__ Row<V> mul(const Row<V> &a, const Row<V> &b) {
    if constexpr (V == 1) {
        return {__fmul_rn(a.f, b.f)};
    } else {
        Row<V> o;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(o.r[i]) : "l"(a.r[i]), "l"(b.r[i]));
        return o;
    }
}
template <int V>
__device__ __forceinline__ Row<V> add(const Row<V> &a, const Row<V> &b) {
    if constexpr (V == 1) {
        return {__fadd_rn(a.f, b.f)};
    } else {
        Row<V> o;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) asm("add.rn.f32x2 %0, %1, %2;" : "=l"(o.r[i]) : "l"(a.r[i]), "l"(b.r[i]));
        return o;
    }
}
template <int V>
__device__ __forceinline__ Row<V> all(float f) {
    return Row<V>::of([&](int) { return f; });
}
template <typename T, int V>
__device__ __forceinline__ Row<V> widen(const Vec<T, V> &a) {
    if constexpr (V > 1 && std::is_same<T, __nv_bfloat16>::value) {  // the halves of a word, without taking them apart
        return Row<V>::of([&](int q) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(&a)[q / 2];
            return __uint_as_float(q % 2 ? w & 0xffff0000u : w << 16);
        });
    }
    return Row<V>::of([&](int q) { return to_float(a.v[q]); });
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const Row<V> &a) {
    Vec<T, V> o;
    if constexpr (V > 1 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int q = 0; q < V; q += 2) *reinterpret_cast<__nv_bfloat162 *>(&o.v[q]) = __floats2bfloat162_rn(a[q], a[q + 1]);
    } else if constexpr (V > 1 && std::is_same<T, __half>::value) {
#pragma unroll
        for (int q = 0; q < V; q += 2) *reinterpret_cast<__half2 *>(&o.v[q]) = __floats2half2_rn(a[q], a[q + 1]);
    } else {
#pragma unroll
        for (int q = 0; q < V; ++q) o.v[q] = from_float<T>(a[q]);
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

// The gate and one minus it from gates z. Of logits, both come from one
// exponential of a non-positive number, so that neither is a difference of
// nearly equal values. For a 16-bit logit the product with log2(e) is rounded
// once to 32 bits: half a unit of it is a share of 2^-19.8 of the exponential up to
// logits of 22 and of 2^-17.9 up to 87, the hardware exponential's own 2^-22.5 with it. The
// logit's own rounding, 2^-9 of itself in bf16 and 2^-12 in f16, moves the exponential of
// such logits by shares of 2^-5 and 2^-8; the low part of the product would cost every
// element two to four instructions of about thirty.
template <typename G, bool Logit, int V>
__device__ __forceinline__ void leak_of(const Vec<G, V> &z, Row<V> &a, Row<V> &rest) {
    if constexpr (!Logit) {
        a = widen(z);
        rest = fma(a, all<V>(-1.0f), all<V>(1.0f));
    } else {
        const Row<V> f = widen(z);
        const Row<V> m = sizeof(G) == 2 ? mul(f, all<V>(1.44269504f)) : f;
        const Row<V> t = Row<V>::of([&](int q) {
            if constexpr (sizeof(G) == 2) {
                float e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-fabsf(m[q])));
                return e;
            } else {
                return expf(-fabsf(m[q]));
            }
        });
        const Row<V> one = add(t, all<V>(1.0f));
        const Row<V> near = Row<V>::of([&](int q) {
            float i;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(i) : "f"(one[q]));
            return i;
        });
        // A step of Newton's, as an error of the gate grows by 1 / (1 - a) on its way into the state.
        const Row<V> r = fma(near, fma(mul(one, all<V>(-1.0f)), near, all<V>(1.0f)), near);
        const Row<V> s = mul(t, r);
        a = Row<V>::of([&](int q) { return f[q] >= 0.0f ? r[q] : s[q]; });
        rest = Row<V>::of([&](int q) { return f[q] >= 0.0f ? s[q] : r[q]; });
    }
}

// f(logit, complement) with the call's flags as constants: a test for every
// step would cost more than the step.
template <bool B>
using Flag = std::integral_constant<bool, B>;
template <typename F>
__device__ __forceinline__ void with_flags(const Args &g, F f) {
    if (g.logit) {
        if (g.complement) f(Flag<true>(), Flag<true>());
        else f(Flag<true>(), Flag<false>());
    } else {
        if (g.complement) f(Flag<false>(), Flag<true>());
        else f(Flag<false>(), Flag<false>());
    }
}

// A thread's place: V channels of one sequence.
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
// The warp's segment and column; the second walk takes the segments from the other end.
struct Part {
    uint64_t column;
    uint32_t segment, t0, t1;  // steps t0 .. t1-1
    bool on;
};
__device__ __forceinline__ Part part_of(const Args &g, bool ascending) {
    const uint64_t n = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    Part w;
    w.segment = (uint32_t)(n / g.columns);
    w.column = n - (uint64_t)w.segment * g.columns;
    w.on = w.segment < g.segments;
    if (!ascending) w.segment = g.segments - 1 - w.segment;
    w.t0 = w.segment * g.segment_steps;
    w.t1 = min(g.steps, w.t0 + g.segment_steps);
    return w;
}
// How many of the steps from t0 on lie within the sequence.
__device__ __forceinline__ int live_steps(uint32_t len, uint32_t t0) {
    return len <= t0 ? 0 : (int)min(len - t0, kSteps);
}

// A block's rows of an array: copied ahead to the warp's shared memory, in
// pieces of 16 bytes that the lanes share where every row allows it (g.wide),
// in the thread's own pieces where those are 4 bytes or more, else loaded when
// the block is worked on.
template <typename T, int V>
struct Feed {
    static constexpr uint32_t kOwn = (uint32_t)sizeof(T) * V;           // bytes of a thread's piece of a row
    static constexpr uint32_t kRow = 32 * kOwn, kBytes = kRow * kSteps;  // of a row, of a block
    static constexpr uint32_t kAcross = kRow / 16, kAtOnce = 32 / kAcross;  // lanes on a row, rows of a copy
    const T *p, *q;  // the thread's piece, the first one it copies
    int64_t stride;
    uint32_t len;  // of the sequence it copies from
    bool wide;

    __device__ __forceinline__ void init(const Args &g, const void *base, const Place &at, uint64_t column, int64_t sb,
                                         int64_t st) {
        p = (const T *)base + at.b * sb + at.c;
        stride = st;
        wide = g.wide;
        if (wide) {
            const uint64_t i = column * 32 * V + (threadIdx.x & 31) % kAcross * (16 / sizeof(T));
            const int64_t b = i < g.flat ? (int64_t)(i / g.channels) : 0;
            q = (const T *)base + b * sb + (int64_t)(i - (uint64_t)b * g.channels) +
                (int64_t)((threadIdx.x & 31) / kAcross) * st;
            len = i >= g.flat ? 0u : g.lengths ? min(g.lengths[b], g.steps) : g.steps;
        } else {
            q = p;
            len = at.len;
        }
    }
    template <uint32_t N>
    static __device__ __forceinline__ void copy(uint32_t to, const void *from) {
        if constexpr (N == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(N) : "memory");
    }
    // slot: the warp's memory for the block.
    __device__ __forceinline__ void fetch(uint8_t *slot, uint32_t t0) const {
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(slot), lane = threadIdx.x & 31;
        const int live = live_steps(len, t0);
        const T *row = q + (int64_t)t0 * stride;
        if (wide) {
            const int left = live - (int)(lane / kAcross);  // of the rows from this lane's first on
#pragma unroll
            for (uint32_t j = 0; j < kSteps; j += kAtOnce, row += kAtOnce * stride)
                if ((int)j < left) copy<16>(at + (j * kAcross + lane) * 16, row);
        } else if constexpr (kOwn >= 4) {
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j, row += stride)
                if (j < live) copy<kOwn>(at + j * kRow + lane * kOwn, row);
        }
    }
    // The block's rows; those behind the live ones are anything.
    __device__ __forceinline__ void take(const uint8_t *slot, uint32_t t0, int live, Vec<T, V> (&r)[kSteps]) const {
        if (kOwn >= 4 || wide) {
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j)
                r[j] = *reinterpret_cast<const Vec<T, V> *>(slot + j * kRow + (threadIdx.x & 31) * kOwn);
        } else {
            const T *row = p + (int64_t)t0 * stride;
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j, row += stride) r[j] = j < live ? load<T, V>(row) : Vec<T, V>{};
        }
    }
};
template <int V>
struct Feed<Fixed, V> {
    static constexpr uint32_t kBytes = 0;
    __device__ __forceinline__ void init(const Args &, const void *, const Place &, uint64_t, int64_t, int64_t) {}
    __device__ __forceinline__ void fetch(uint8_t *, uint32_t) const {}
};
__device__ __forceinline__ void fetched() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void await() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Walks the blocks of [t0, t1) in either direction: fetch(t0, slot) starts a
// block's copies, work(t0, slot) uses them. Those of kDepth - 1 blocks are under way.
template <bool Reverse, typename Fetch, typename Work>
__device__ __forceinline__ void walk_blocks(uint32_t t0, uint32_t t1, Fetch fetch, Work work) {
    const uint32_t blocks = (t1 - t0 + kSteps - 1) / kSteps;
    const auto at = [&](uint32_t n) { return t0 + (Reverse ? blocks - 1 - n : n) * kSteps; };
#pragma unroll
    for (uint32_t n = 0; n < kDepth - 1; ++n) {
        if (n < blocks) fetch(at(n), n);
        fetched();
    }
    uint32_t slot = 0;
    for (uint32_t n = 0; n < blocks; ++n) {
        const uint32_t to = slot ? slot - 1 : kDepth - 1;
        if (n + kDepth - 1 < blocks) fetch(at(n + kDepth - 1), to);
        fetched();
        await<kDepth - 1>();
        __syncwarp();
        work(at(n), slot);
        __syncwarp();  // the slot may be copied to again
        slot = slot + 1 == kDepth ? 0 : slot + 1;
    }
}

// The gates of a thread's steps. Fixed gates are kept once, and so is their
// product over a block: each block's map has the same one, so its error acts as
// another decay would and adds up over a long memory. Rounded once from 64 bits
// it is at most half a step off (a shared gate's gradient over 5281 steps of 2619
// channels is 5.4e-7 from the one in 64 bits; with seven products of 32 bits it
// was 1.2e-6). It costs no time: 84 us for 256 x 100 x 1000 either way.
template <typename G, int V>
struct Gates {
    Vec<G, V> raw[kSteps];
    __device__ __forceinline__ void init(const Args &, const Place &) {}
    __device__ __forceinline__ void take(const Feed<G, V> &feed, const uint8_t *slot, uint32_t t0, int live) {
        feed.take(slot, t0, live, raw);
    }
    template <bool Logit>
    __device__ __forceinline__ void at(int j, Row<V> &a, Row<V> &rest) const {
        leak_of<G, Logit, V>(raw[j], a, rest);
    }
    // A map's gate over a block's live steps: one's factor, and the whole block's.
    __device__ __forceinline__ void step_into(Row<V> &A, const Row<V> &a, int) const { A = mul(a, A); }
    __device__ __forceinline__ void block_into(Row<V> &, int) const {}
};
template <int V>
struct Gates<Fixed, V> {
    Row<V> a_, rest_, block_;
    __device__ __forceinline__ void init(const Args &g, const Place &p) {
        if (!g.gate) {
            a_ = all<V>(g.decay), rest_ = all<V>(__fsub_rn(1.0f, g.decay));
        } else {
            const Vec<float, V> z = p.on ? load<float, V>((const float *)g.gate + p.b * g.gb + p.c) : Vec<float, V>{};
            if (g.logit) leak_of<float, true, V>(z, a_, rest_);
            else leak_of<float, false, V>(z, a_, rest_);
        }
        static_assert(kSteps == 8, "a block's product is three squares");
        block_ = Row<V>::of([&](int q) {
            const double two = (double)a_[q] * a_[q], four = two * two;
            return kept((float)(four * four), a_[q] == 0.0f);
        });
    }
    __device__ __forceinline__ void step_into(Row<V> &A, const Row<V> &a, int live) const {
        if (live < (int)kSteps) A = mul(a, A);
    }
    __device__ __forceinline__ void block_into(Row<V> &A, int live) const {
        if (live == (int)kSteps) A = mul(block_, A);
    }
    __device__ __forceinline__ void take(const Feed<Fixed, V> &, const uint8_t *, uint32_t, int) {}
    template <bool Logit>
    __device__ __forceinline__ void at(int, Row<V> &a, Row<V> &rest) const {
        a = a_, rest = rest_;
    }
};

template <int V>
__device__ __forceinline__ bool any_zero(const Row<V> &A) {
    bool any = false;
#pragma unroll
    for (int q = 0; q < V; ++q) any |= A[q] == 0.0f;
    return any;
}
// The product P of a block's `live` gates gate(j).
template <int V, typename Gate>
__device__ __forceinline__ void keep(Row<V> &P, int live, Gate gate) {
    if (!any_zero(P)) return;
    uint32_t zero = 0;
#pragma unroll
    for (int j = 0; j < (int)kSteps; ++j) {
        const Row<V> a = gate(j);
#pragma unroll
        for (int q = 0; q < V; ++q)
            if (j < live && a[q] == 0.0f) zero |= 1u << q;
    }
    P = Row<V>::of([&](int q) { return kept(P[q], zero >> q & 1u); });
}
// A map's product A joined with that of a block, whose gates are looked at again where it matters.
template <typename G, int V>
__device__ __forceinline__ void join(const Args &g, const Gates<G, V> &gates, Row<V> &A, Row<V> P, int live) {
    const Row<V> both = mul(P, A);
    if constexpr (std::is_same<G, Fixed>::value) {
        A = Row<V>::of([&](int q) { return kept(both[q], gates.a_[q] == 0.0f); });
    } else if (any_zero(both)) {
        keep<V>(P, live, [&](int j) {
            Row<V> a, rest;
            if (g.logit) gates.template at<true>(j, a, rest);
            else gates.template at<false>(j, a, rest);
            return a;
        });
        A = Row<V>::of([&](int q) { return kept(__fmul_rn(P[q], A[q]), P[q] == 0.0f || A[q] == 0.0f); });
    } else {
        A = both;
    }
}

template <int V>
__device__ __forceinline__ Row<V> load_row(const float *p) {
    return widen(load<float, V>(p));
}
template <int V>
__device__ __forceinline__ void store_row(float *p, const Row<V> &a) {
    store<float, V>(p, narrow<float, V>(a));
}
template <int V>
__device__ __forceinline__ Row<V> load_state(const float *p, uint64_t i) {
    return p ? load_row<V>(p + i) : all<V>(0.0f);
}
template <int V>
__device__ __forceinline__ void store_map(float2 *p, const Row<V> &A, const Row<V> &H) {
#pragma unroll
    for (int q = 0; q < V; q += 2) {
        if constexpr (V == 1) *p = make_float2(A[0], H[0]);
        else *reinterpret_cast<float4 *>(p + q) = make_float4(A[q], H[q], A[q + 1], H[q + 1]);
    }
}

// The state before a block of kSteps steps, kept for the backward pass.
__device__ __forceinline__ float *saved_at(const Args &g, const Place &p, uint32_t t0) {
    const uint32_t blocks = (g.steps + kSteps - 1) / kSteps;
    return g.saved + ((uint64_t)p.b * blocks + t0 / kSteps) * g.channels + p.c;
}

// A block's steps from its gates and inputs: step(j, a, u) for each of the
// `live` ones, with the call's flags as constants.
template <typename X, typename G, int V, typename Step>
__device__ __forceinline__ void each_step(const Args &g, const Gates<G, V> &gates, const Vec<X, V> (&x)[kSteps], int live,
                                          Step step) {
    with_flags(g, [&](auto logit, auto complement) {
        const auto one = [&](int j) {
            Row<V> a, rest;
            gates.template at<logit.value>(j, a, rest);
            Row<V> u = mul(all<V>(g.scale), widen(x[j]));
            if (complement.value) u = mul(u, rest);
            step(j, a, u);
        };
        if (live == (int)kSteps) {
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j) one(j);
        } else {
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j)
                if (j < live) one(j);
        }
    });
}

// Maps: only each segment's map is wanted; else y, from h0 or the segments' states.
template <typename X, typename G, typename Y, int V, bool Maps>
__global__ void __launch_bounds__(kWarps * 32, 6) scan_kernel(const __grid_constant__ Args g) {
    extern __shared__ __align__(16) uint8_t s_feed[];
    const Part w = part_of(g, Maps);
    after_previous();
    if (!w.on) return;
    const Place p = place_of<V>(g, w.column);  // lanes behind the last channel only help to copy
    constexpr uint32_t kX = Feed<X, V>::kBytes, kSlot = kX + Feed<G, V>::kBytes;
    uint8_t *mine = s_feed + threadIdx.x / 32 * (kDepth * kSlot);
    Feed<X, V> fx;
    Feed<G, V> fz;
    Gates<G, V> gates;
    gates.init(g, p);
    fx.init(g, g.x, p, w.column, g.xb, g.xt);
    fz.init(g, g.gate, p, w.column, g.gb, g.gt);
    Row<V> h = all<V>(0.0f), A = all<V>(1.0f);
    if (!Maps && p.on) h = load_state<V>(g.segments > 1 ? g.states + w.segment * g.flat : g.h0, p.i);
    walk_blocks<false>(
        w.t0, w.t1,
        [&](uint32_t t0, uint32_t slot) {
            fz.fetch(mine + slot * kSlot + kX, t0);
            fx.fetch(mine + slot * kSlot, t0);
        },
        [&](uint32_t t0, uint32_t slot) {
            const int live = live_steps(p.len, t0);
            Vec<X, V> x[kSteps];
            gates.take(fz, mine + slot * kSlot + kX, t0, live);
            fx.take(mine + slot * kSlot, t0, live, x);
            if constexpr (Maps) {
                Row<V> P = all<V>(1.0f);
                each_step<X, G, V>(g, gates, x, live, [&](int, const Row<V> &a, const Row<V> &u) {
                    gates.step_into(P, a, live);
                    h = fma(a, h, u);
                });
                gates.block_into(P, live);
                join(g, gates, A, P, live);
            } else if (p.on) {
                if (g.saved) store_row<V>(saved_at(g, p, t0), h);
                Y *y = (Y *)g.y + p.b * g.yb + (int64_t)t0 * g.yt + p.c;
                each_step<X, G, V>(g, gates, x, live, [&](int, const Row<V> &a, const Row<V> &u) {
                    h = fma(a, h, u);
                    store<Y, V>(y, narrow<Y, V>(h));
                    y += g.yt;
                });
                if (live < (int)kSteps)
                    for (int j = live; j < (int)min(w.t1 - t0, kSteps); ++j, y += g.yt) store<Y, V>(y, Vec<Y, V>{});
            }
        });
    if (!p.on) return;
    if constexpr (Maps) {
        store_map<V>(g.maps + w.segment * g.flat + p.i, A, h);
    } else {
        if (g.h_last && w.segment + 1 == g.segments) store_row<V>(g.h_last + p.i, h);
    }
}

// ---- crews ----
template <int V>
struct alignas(2 * sizeof(Row<V>)) Map {
    Row<V> A, H;
};
template <int V, uint32_t N>
struct Crew {
    Map<V> map[2][N][32];      // of this round and the one before
    Row<V> state[2][32];       // behind a round
};
// Blocks under way or at hand for each warp, as shared memory allows.
template <int V, uint32_t N>
constexpr uint32_t crew_depth(uint32_t slot) {
    return 3 * N * slot + (uint32_t)sizeof(Crew<V, N>) <= 227 * 1024 ? 3 : 2;
}
// The next rounds of a crew's warp: fetch(t0, slot) and work(n, t0, slot) of
// its block in each; a block behind the last one is only worked on (on = false).
template <bool Reverse, uint32_t N, uint32_t Depth, typename Fetch, typename Work>
__device__ __forceinline__ void walk_rounds(uint32_t steps, Fetch fetch, Work work) {
    const uint32_t warp = threadIdx.x / 32, blocks = (steps + kSteps - 1) / kSteps;
    const uint32_t rounds = (blocks + N - 1) / N;
    const auto at = [&](uint32_t n) { return (Reverse ? blocks - 1 - (n * N + warp) : n * N + warp) * kSteps; };
    const auto on = [&](uint32_t n) { return n * N + warp < blocks; };
#pragma unroll
    for (uint32_t n = 0; n < Depth - 1; ++n) {
        if (on(n)) fetch(at(n), n);
        fetched();
    }
    uint32_t slot = 0;
    for (uint32_t n = 0; n < rounds; ++n) {
        const uint32_t next = n + Depth - 1;
        if (on(next)) fetch(at(next), slot ? slot - 1 : Depth - 1);
        fetched();
        await<Depth - 1>();
        __syncwarp();
        work(n, on(n), at(n), slot);
        slot = slot + 1 == Depth ? 0 : slot + 1;
    }
}
// Shares a block's map and folds the state before it. The last warp's walk of the
// round before has left the state there.
template <int V, uint32_t N>
__device__ __forceinline__ Row<V> crew_state(Crew<V, N> &c, uint32_t n, const Row<V> &A, const Row<V> &H, const Row<V> &first) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, turn = n & 1;
    c.map[turn][warp][lane] = {A, H};
    __syncthreads();
    Row<V> h = n ? c.state[turn ^ 1][lane] : first;
    const Map<V> *m = &c.map[turn][0][lane];
#pragma unroll 4
    for (uint32_t w = 0; w < warp; ++w) {
        const Map<V> v = m[w * 32];
        h = fma(v.A, h, v.H);
    }
    return h;
}
template <int V, uint32_t N>
__device__ __forceinline__ void crew_done(Crew<V, N> &c, uint32_t n, const Row<V> &h) {
    if (threadIdx.x / 32 + 1 == N) c.state[n & 1][threadIdx.x & 31] = h;
}

template <typename X, typename G, typename Y, int V, uint32_t N>
__global__ void __launch_bounds__(N * 32) scan_crew_kernel(const __grid_constant__ Args g) {
    extern __shared__ __align__(16) uint8_t s_feed[];
    __shared__ Crew<V, N> s_crew;
    after_previous();
    const uint32_t warp = threadIdx.x / 32;
    const Place p = place_of<V>(g, blockIdx.x);
    constexpr uint32_t kX = Feed<X, V>::kBytes, kSlot = kX + Feed<G, V>::kBytes;
    constexpr uint32_t kDeep = crew_depth<V, N>(kSlot);
    uint8_t *mine = s_feed + warp * (kDeep * kSlot);
    Feed<X, V> fx;
    Feed<G, V> fz;
    Gates<G, V> gates;
    gates.init(g, p);
    fx.init(g, g.x, p, blockIdx.x, g.xb, g.xt);
    fz.init(g, g.gate, p, blockIdx.x, g.gb, g.gt);
    const Row<V> first = p.on ? load_state<V>(g.h0, p.i) : all<V>(0.0f);
    Row<V> h = first;
    walk_rounds<false, N, kDeep>(
        g.steps,
        [&](uint32_t t0, uint32_t slot) {
            fz.fetch(mine + slot * kSlot + kX, t0);
            fx.fetch(mine + slot * kSlot, t0);
        },
        [&](uint32_t n, bool on, uint32_t t0, uint32_t slot) {
            const int live = on ? live_steps(p.len, t0) : 0;
            Row<V> a[kSteps], u[kSteps], A = all<V>(1.0f), H = all<V>(0.0f);
            {
                Vec<X, V> x[kSteps];
                if (on) {
                    gates.take(fz, mine + slot * kSlot + kX, t0, live);
                    fx.take(mine + slot * kSlot, t0, live, x);
                }
                each_step<X, G, V>(g, gates, x, live, [&](int j, const Row<V> &aj, const Row<V> &uj) {
                    a[j] = aj, u[j] = uj;
                    gates.step_into(A, aj, live);
                    H = fma(aj, H, uj);
                });
                gates.block_into(A, live);
            }
            keep<V>(A, live, [&](int j) { return a[j]; });
            h = crew_state<V, N>(s_crew, n, A, H, first);
            if (on && p.on) {
                if (g.saved) store_row<V>(saved_at(g, p, t0), h);
                Y *y = (Y *)g.y + p.b * g.yb + (int64_t)t0 * g.yt + p.c;
                if (live == (int)kSteps) {
#pragma unroll
                    for (int j = 0; j < (int)kSteps; ++j, y += g.yt) {
                        h = fma(a[j], h, u[j]);
                        store<Y, V>(y, narrow<Y, V>(h));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < (int)kSteps; ++j, y += g.yt) {
                        if (j < live) h = fma(a[j], h, u[j]);
                        if (t0 + j < g.steps) store<Y, V>(y, j < live ? narrow<Y, V>(h) : Vec<Y, V>{});
                    }
                }
            }
            crew_done<V, N>(s_crew, n, h);
        });
    if (g.h_last && p.on && warp + 1 == N) store_row<V>(g.h_last + p.i, h);
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
    static constexpr bool kEvery = !std::is_same<G, Fixed>::value;
    Gates<G, V> gates;
    Vec<Y, V> dy[kSteps];
    // Of each step: the gate, and what d is multiplied with for dx and for
    // the gate's gradient (where it is shared, without its common factor).
    Row<V> a[kSteps], fx[kSteps], fz[kSteps];

    __device__ __forceinline__ void maps(const Args &g, const Vec<X, V> (&x)[kSteps], Row<V> h, int live) {
        with_flags(g, [&](auto logit, auto complement) {
            const Row<V> scale = all<V>(g.scale);
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j) {
                Row<V> rest, v = mul(scale, widen(x[j]));
                gates.template at<logit.value>(j, a[j], rest);
                if (complement.value) {
                    fz[j] = fma(all<V>(-1.0f), v, h);
                    fx[j] = mul(scale, rest);
                    v = mul(v, rest);
                } else {
                    fz[j] = h;
                    fx[j] = scale;
                }
                h = fma(a[j], h, v);
                if (kEvery && logit.value) fz[j] = mul(fz[j], mul(a[j], rest));
            }
        });
        if (live < (int)kSteps) {
#pragma unroll
            for (int j = 0; j < (int)kSteps; ++j)
                if (j >= live) a[j] = all<V>(1.0f);
        }
    }
    // One step back: d, and e before it.
    __device__ __forceinline__ Row<V> step(int j, int live, Row<V> &e) const {
        const Row<V> d = add(widen(dy[j]), e);
        if (j < live) e = mul(a[j], d);
        return d;
    }
    // Walks back from e, writes dx and the gradient of a gate with a value
    // for every step, and returns the block's sum for a shared one.
    template <bool Whole>
    __device__ __forceinline__ Row<V> walk(const Args &g, const Place &p, uint32_t t0, int live, Row<V> &e) {
        using D = typename GradientOf<X>::type;
        const uint32_t end = t0 + kSteps - 1;
        D *dx = (D *)g.dx + p.b * g.dxb + (int64_t)end * g.dxt + p.c;
        G *dz = (G *)g.dgate + p.b * g.dgb + (int64_t)end * g.dgt + p.c;
        const int rows = t0 >= g.steps ? 0 : (int)min(g.steps - t0, kSteps);
        Row<V> sum = all<V>(0.0f);
#pragma unroll
        for (int j = (int)kSteps - 1; j >= 0; --j, dx -= g.dxt, dz -= g.dgt) {
            const bool on = Whole || j < live;
            const Row<V> d = step(j, Whole ? (int)kSteps : live, e);
            if (!kEvery && on) sum = fma(d, fz[j], sum);
            if (!Whole && j >= rows) continue;
            if (g.dx) store<D, V>(dx, on ? narrow<D, V>(mul(fx[j], d)) : Vec<D, V>{});
            if constexpr (kEvery)
                if (g.dgate) store<G, V>(dz, on ? narrow<G, V>(mul(d, fz[j])) : Vec<G, V>{});
        }
        return sum;
    }
    __device__ __forceinline__ Row<V> emit(const Args &g, const Place &p, uint32_t t0, int live, Row<V> &e) {
        if (!p.on) return all<V>(0.0f);
        return live == (int)kSteps ? walk<true>(g, p, t0, live, e) : walk<false>(g, p, t0, live, e);
    }
};
// A shared gate's sum for one thread: of logits, the gate's own slope is a common factor.
template <int V>
__device__ __forceinline__ void put_partial(const Args &g, const Place &p, const Gates<Fixed, V> &gates, uint32_t segment,
                                            const Row<V> &sum) {
    store_row<V>(g.partial + segment * g.flat + p.i, g.logit ? mul(sum, mul(gates.a_, gates.rest_)) : sum);
}
template <typename G, int V>
__device__ __forceinline__ void put_partial(const Args &, const Place &, const Gates<G, V> &, uint32_t,
                                            const Row<V> &) {}

template <int V>
constexpr uint32_t kSavedBytes = 32 * V * 4;  // the states before a block

// Maps: only each segment's map of e is wanted, for which x does not count.
template <typename X, typename G, typename Y, int V, bool Maps>
__global__ void __launch_bounds__(kWarps * 32, Maps ? 6 : 4) back_kernel(const __grid_constant__ Args g) {
    extern __shared__ __align__(16) uint8_t s_feed[];
    const Part w = part_of(g, Maps);
    after_previous();
    if (!w.on) return;
    const Place p = place_of<V>(g, w.column);  // lanes behind the last channel only help to copy
    constexpr uint32_t kY = Feed<Y, V>::kBytes, kZ = kY + Feed<G, V>::kBytes, kS = kZ + (Maps ? 0 : Feed<X, V>::kBytes),
                       kSlot = kS + (Maps ? 0 : kSavedBytes<V>);
    uint8_t *mine = s_feed + threadIdx.x / 32 * (kDepth * kSlot);
    Feed<X, V> fx;
    Feed<G, V> fz;
    Feed<Y, V> fy;
    if (!Maps) fx.init(g, g.x, p, w.column, g.xb, g.xt);
    fz.init(g, g.gate, p, w.column, g.gb, g.gt);
    fy.init(g, g.dy, p, w.column, g.dyb, g.dyt);
    Back<X, G, Y, V> b;
    b.gates.init(g, p);
    Row<V> e = all<V>(0.0f), A = all<V>(1.0f);
    if (!Maps && p.on) e = load_state<V>(g.segments > 1 ? g.states + w.segment * g.flat : g.dh_last, p.i);
    double total[V] = {};
    walk_blocks<true>(
        w.t0, w.t1,
        [&](uint32_t t0, uint32_t slot) {
            fy.fetch(mine + slot * kSlot, t0);
            fz.fetch(mine + slot * kSlot + kY, t0);
            if (Maps) return;
            fx.fetch(mine + slot * kSlot + kZ, t0);
            if (p.on && t0 < p.len)
                Feed<float, V>::template copy<4 * V>(
                    (uint32_t)__cvta_generic_to_shared(mine + slot * kSlot + kS) + (threadIdx.x & 31) * 4 * V,
                    saved_at(g, p, t0));
        },
        [&](uint32_t t0, uint32_t slot) {
            const int live = live_steps(p.len, t0);
            b.gates.take(fz, mine + slot * kSlot + kY, t0, live);
            fy.take(mine + slot * kSlot, t0, live, b.dy);
            if constexpr (Maps) {
                Row<V> P = all<V>(1.0f);
                with_flags(g, [&](auto logit, auto) {
#pragma unroll
                    for (int j = (int)kSteps - 1; j >= 0; --j)
                        if (j < live) {
                            Row<V> a, rest;
                            b.gates.template at<logit.value>(j, a, rest);
                            b.gates.step_into(P, a, live);
                            e = mul(a, add(widen(b.dy[j]), e));
                        }
                });
                b.gates.block_into(P, live);
                join(g, b.gates, A, P, live);
            } else {
                const Row<V> h = load_row<V>((const float *)(mine + slot * kSlot + kS) + (threadIdx.x & 31) * V);
                Vec<X, V> x[kSteps];
                fx.take(mine + slot * kSlot + kZ, t0, live, x);
                b.maps(g, x, h, live);
                const Row<V> sum = b.emit(g, p, t0, live, e);
                if (!b.kEvery)
#pragma unroll
                    for (int q = 0; q < V; ++q) total[q] += (double)sum[q];
            }
        });
    if (!p.on) return;
    if constexpr (Maps) {
        store_map<V>(g.maps + w.segment * g.flat + p.i, A, e);
    } else {
        if (g.dh0 && w.segment == 0) store_row<V>(g.dh0 + p.i, e);
        if (g.partial) {
            const Row<V> sum = Row<V>::of([&](int q) { return (float)total[q]; });
            put_partial(g, p, b.gates, w.segment, sum);
        }
    }
}

template <typename X, typename G, typename Y, int V, uint32_t N>
__global__ void __launch_bounds__(N * 32) back_crew_kernel(const __grid_constant__ Args g) {
    extern __shared__ __align__(16) uint8_t s_feed[];
    __shared__ Crew<V, N> s_crew;
    after_previous();
    const uint32_t warp = threadIdx.x / 32;
    const Place p = place_of<V>(g, blockIdx.x);
    constexpr uint32_t kY = Feed<Y, V>::kBytes, kZ = kY + Feed<G, V>::kBytes, kS = kZ + Feed<X, V>::kBytes,
                       kSlot = kS + kSavedBytes<V>;
    constexpr uint32_t kDeep = crew_depth<V, N>(kSlot);
    uint8_t *mine = s_feed + warp * (kDeep * kSlot);
    Feed<X, V> fx;
    Feed<G, V> fz;
    Feed<Y, V> fy;
    fx.init(g, g.x, p, blockIdx.x, g.xb, g.xt);
    fz.init(g, g.gate, p, blockIdx.x, g.gb, g.gt);
    fy.init(g, g.dy, p, blockIdx.x, g.dyb, g.dyt);
    Back<X, G, Y, V> b;
    b.gates.init(g, p);
    const Row<V> first = p.on ? load_state<V>(g.dh_last, p.i) : all<V>(0.0f);
    Row<V> e = first;
    double total[V] = {};
    walk_rounds<true, N, kDeep>(
        g.steps,
        [&](uint32_t t0, uint32_t slot) {
            fy.fetch(mine + slot * kSlot, t0);
            fz.fetch(mine + slot * kSlot + kY, t0);
            fx.fetch(mine + slot * kSlot + kZ, t0);
            if (p.on && t0 < p.len)
                Feed<float, V>::template copy<4 * V>(
                    (uint32_t)__cvta_generic_to_shared(mine + slot * kSlot + kS) + (threadIdx.x & 31) * 4 * V,
                    saved_at(g, p, t0));
        },
        [&](uint32_t n, bool on, uint32_t t0, uint32_t slot) {
            const int live = on ? live_steps(p.len, t0) : 0;
            Row<V> A = all<V>(1.0f), E = all<V>(0.0f);
            if (on) {
                Vec<X, V> x[kSteps];
                b.gates.take(fz, mine + slot * kSlot + kY, t0, live);
                fy.take(mine + slot * kSlot, t0, live, b.dy);
                fx.take(mine + slot * kSlot + kZ, t0, live, x);
                b.maps(g, x, load_row<V>((const float *)(mine + slot * kSlot + kS) + (threadIdx.x & 31) * V), live);
#pragma unroll
                for (int j = (int)kSteps - 1; j >= 0; --j) b.gates.step_into(A, b.a[j], live), b.step(j, live, E);
                b.gates.block_into(A, live);
                keep<V>(A, live, [&](int j) { return b.a[j]; });
            }
            e = crew_state<V, N>(s_crew, n, A, E, first);
            if (on) {
                const Row<V> sum = b.emit(g, p, t0, live, e);
                if (!b.kEvery)
#pragma unroll
                    for (int q = 0; q < V; ++q) total[q] += (double)sum[q];
            }
            crew_done<V, N>(s_crew, n, e);
        });
    if (!p.on) return;
    if (g.dh0 && warp + 1 == N) store_row<V>(g.dh0 + p.i, e);
    if (g.partial) {
        const Row<V> sum = Row<V>::of([&](int q) { return (float)total[q]; });
        put_partial(g, p, b.gates, warp, sum);
    }
}

// ---- single step ----
// A row of the pool is updated by the threads of the first row that names
// it, which also do the later rows that name it, in order. To know, every CTA
// looks through the slots once, for all of its rows at a time. 2000 rows of 1000
// channels out of 4096: 7 us a call, 28 MB; the look was most of it (10.5 us) while
// every slot was compared with all that a decision needs instead of first with
// the rows' own. It grows with the square of the rows: 8192 take 34 us with slots and 21
// without, 65,536 844 and 205.
template <typename X, typename G, typename Y, int V>
__global__ void __launch_bounds__(256, 4) step_kernel(StepArgs g) {
    __shared__ uint32_t s_before[8], s_after[8];  // rows named before, rows named again
    const uint32_t across = 256 / g.rows, mine = threadIdx.x / across;
    const uint32_t row = blockIdx.x * g.rows + mine;
    after_previous();
    if (g.slots && g.batch > 1) {
        if (threadIdx.x < 8) s_before[threadIdx.x] = s_after[threadIdx.x] = 0u;
        __syncthreads();
        int32_t named[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r) {
            const uint32_t n = blockIdx.x * g.rows + r;
            named[r] = r < g.rows && n < g.batch ? g.slots[n] : -1;
        }
        for (uint32_t n0 = threadIdx.x; n0 < g.batch; n0 += 8 * 256) {
            int32_t s[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) s[i] = n0 + i * 256 < g.batch ? g.slots[n0 + i * 256] : -1;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                bool hit = false;
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) hit |= s[i] == named[r];
                if (!hit || (uint32_t)s[i] >= g.slot_count) continue;  // padding names no slot
                for (uint32_t r = 0; r < g.rows; ++r) {
                    const uint32_t n = n0 + i * 256, of = blockIdx.x * g.rows + r;
                    if (of < g.batch && s[i] == g.slots[of] && n != of) (n < of ? s_before : s_after)[r] = 1u;
                }
            }
        }
        __syncthreads();
        if (s_before[mine]) return;
    }
    if (row >= g.batch) return;
    const bool again = g.slots && g.batch > 1 && s_after[mine];
    const int64_t slot = g.slots ? (int64_t)g.slots[row] : (int64_t)row;
    const bool padding = slot < 0 || slot >= (int64_t)g.slot_count;
    const uint64_t c0 = ((uint64_t)blockIdx.y * across + threadIdx.x % across) * V, jump = (uint64_t)gridDim.y * across * V;
    Y *y = (Y *)g.y + row * g.ys;
    if (padding) {
        for (uint64_t c = c0; c < g.channels; c += jump) store<Y, V>(y + c, Vec<Y, V>{});
        return;
    }
    float *state = g.pool + slot * g.ps;
    const auto one = [&](const Vec<X, V> &x, const Vec<G, V> &z, Row<V> &h) {
        Row<V> a = all<V>(g.decay), rest = all<V>(__fsub_rn(1.0f, g.decay));
        if (g.gate) {
            if (g.logit) leak_of<G, true, V>(z, a, rest);
            else leak_of<G, false, V>(z, a, rest);
        }
        Row<V> u = mul(all<V>(g.scale), widen(x));
        if (g.complement) u = mul(u, rest);
        h = fma(a, h, u);
        return narrow<Y, V>(h);
    };
    const X *xs = (const X *)g.x;
    const G *zs = (const G *)g.gate;
    if (again) {
        for (uint64_t c = c0; c < g.channels; c += jump) {
            Row<V> h = load_row<V>(state + c);
            for (uint32_t r = row; r < g.batch; ++r)
                if (g.slots[r] == (int32_t)slot)
                    store<Y, V>((Y *)g.y + r * g.ys + c,
                                one(load<X, V>(xs + r * g.xs + c), zs ? load<G, V>(zs + r * g.gs + c) : Vec<G, V>{}, h));
            store_row<V>(state + c, h);
        }
        return;
    }
    xs += row * g.xs;
    if (zs) zs += row * g.gs;
    constexpr uint32_t kAtOnce = 4;  // pieces whose loads are under way together
    for (uint64_t c = c0; c < g.channels; c += kAtOnce * jump) {
        Vec<X, V> x[kAtOnce];
        Vec<G, V> z[kAtOnce];
        Row<V> h[kAtOnce];
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
            const uint64_t at = c + i * jump;
            if (at >= g.channels) break;
            x[i] = load<X, V>(xs + at);
            z[i] = zs ? load<G, V>(zs + at) : Vec<G, V>{};
            h[i] = load_row<V>(state + at);
        }
#pragma unroll
        for (uint32_t i = 0; i < kAtOnce; ++i) {
            const uint64_t at = c + i * jump;
            if (at >= g.channels) break;
            store<Y, V>(y + at, one(x[i], z[i], h[i]));
            store_row<V>(state + at, h[i]);
        }
    }
}

template <typename X, typename G, typename Y>
cudaError_t launch_step(cudaStream_t s, const Form &f, const StepArgs &a, dim3 grid) {
    return launch_early(f.width == 4 ? step_kernel<X, G, Y, 4> : step_kernel<X, G, Y, 1>, grid, 256, 0, s, 1, a);
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

// grid CTAs of Warps warps, each with Feed bytes of shared memory, beside Fixed bytes of the kernel's own.
template <auto Kernel, uint32_t Warps, uint32_t FeedBytes, uint32_t FixedBytes = 0>
cudaError_t start(cudaStream_t s, const Args &a, uint64_t grid) {
    constexpr uint32_t smem = Warps * FeedBytes;
    if constexpr (smem + FixedBytes > 48 * 1024) {
        const cudaError_t e = allow_smem<Kernel>(smem);
        if (e != cudaSuccess) return e;
    }
    return launch_early(Kernel, (uint32_t)grid, Warps * 32, smem, s, 1, a);
}
template <typename X, typename G, typename Y, int V>
cudaError_t launch_scan(cudaStream_t s, const Args &a) {
    constexpr uint32_t slot = Feed<X, V>::kBytes + Feed<G, V>::kBytes;
    if constexpr (V <= 2) {
        if (a.crew == 16)
            return start<scan_crew_kernel<X, G, Y, V, 16>, 16, crew_depth<V, 16>(slot) * slot, sizeof(Crew<V, 16>)>(
                s, a, a.columns);
        if (a.crew)
            return start<scan_crew_kernel<X, G, Y, V, 8>, 8, crew_depth<V, 8>(slot) * slot, sizeof(Crew<V, 8>)>(
                s, a, a.columns);
    }
    const uint64_t grid = ((uint64_t)a.columns * a.segments + kWarps - 1) / kWarps;
    if (a.segments > 1) {
        cudaError_t e = start<scan_kernel<X, G, Y, V, true>, kWarps, kDepth * slot>(s, a, grid);
        if (e == cudaSuccess) e = carry(s, a, false);
        if (e != cudaSuccess) return e;
    }
    return start<scan_kernel<X, G, Y, V, false>, kWarps, kDepth * slot>(s, a, grid);
}
template <typename X, typename G, typename Y, int V>
cudaError_t launch_back(cudaStream_t s, const Args &a) {
    constexpr uint32_t maps = Feed<G, V>::kBytes + Feed<Y, V>::kBytes, slot = maps + Feed<X, V>::kBytes + kSavedBytes<V>;
    if (a.crew == 16)
        return start<back_crew_kernel<X, G, Y, V, 16>, 16, crew_depth<V, 16>(slot) * slot, sizeof(Crew<V, 16>)>(
            s, a, a.columns);
    if (a.crew)
        return start<back_crew_kernel<X, G, Y, V, 8>, 8, crew_depth<V, 8>(slot) * slot, sizeof(Crew<V, 8>)>(s, a,
                                                                                                              a.columns);
    const uint64_t grid = ((uint64_t)a.columns * a.segments + kWarps - 1) / kWarps;
    if (a.segments > 1) {
        cudaError_t e = start<back_kernel<X, G, Y, V, true>, kWarps, kDepth * maps>(s, a, grid);
        if (e == cudaSuccess) e = carry(s, a, true);
        if (e != cudaSuccess) return e;
    }
    return start<back_kernel<X, G, Y, V, false>, kWarps, kDepth * slot>(s, a, grid);
}
template <typename X, typename G, typename Y>
cudaError_t launch(cudaStream_t s, const Form &f, const Args &a, bool back) {
    if constexpr (std::is_same<X, Spike>::value)
        if (f.width == 4) return launch_scan<X, G, Y, 4>(s, a);
    if (back) return f.width == 2 ? launch_back<X, G, Y, 2>(s, a) : launch_back<X, G, Y, 1>(s, a);
    return f.width == 2 ? launch_scan<X, G, Y, 2>(s, a) : launch_scan<X, G, Y, 1>(s, a);
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
