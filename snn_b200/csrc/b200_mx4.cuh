// Device code of the packed 4-bit format: scales, codes, and the pieces of 16
// bytes in which rows are packed.
#pragma once

#include "b200_mx4.h"

namespace b200 {
namespace mx4 {

// The scale byte of a block from its largest magnitude (bits of a
// non-negative float): exponent - 2, at least 2^-127, 255 when not finite.
// Scale byte s stands for 2^(s - 127) and the float's exponent field f for
// 2^(f - 127), so the byte is f - 2.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const uint32_t f = amax_bits >> 23;
    return f == 255u ? 255u : f > 2u ? f - 2u : 0u;
}
// 2^(127 - s) for s of 0..252 (anything for 255).
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// 2^(s - 127), the smallest one subnormal; NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7fffffffu) : s ? __uint_as_float(s << 23) : __uint_as_float(0x00400000u);
}
// Where in its 512-byte tile the scale of a row and block lies.
__device__ __forceinline__ uint32_t scale_slot(uint32_t r, uint32_t b) { return 16 * (r % 32) + 4 * (r / 32) + b; }

// Two codes, the first in the low half: nearest, ties to even, saturating.
__device__ __forceinline__ uint32_t encode2(float lo, float hi) {
    uint32_t r;
    asm("{\n .reg .b8 c;\n cvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n cvt.u32.u8 %0, c;\n}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ uint32_t encode8(const float *v, float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) w |= encode2(__fmul_rn(v[2 * q], inv), __fmul_rn(v[2 * q + 1], inv)) << (8 * q);
    return w;
}
__device__ __forceinline__ void decode8(uint32_t w, float scale, float *v) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t h;  // two halves
        asm("{\n .reg .b8 c;\n cvt.u8.u32 c, %1;\n cvt.rn.f16x2.e2m1x2 %0, c;\n}" : "=r"(h) : "r"(w >> (8 * q)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
        v[2 * q] = __fmul_rn(f.x, scale), v[2 * q + 1] = __fmul_rn(f.y, scale);
    }
}

template <typename T>
struct Eight {
    T v[8];
};

// 16 bytes of a row.
template <typename T>
struct Piece {
    static constexpr uint32_t kOwn = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float at(uint32_t i) const {
        const uint32_t w = i / (4 / sizeof(T)) == 0 ? raw.x : i / (4 / sizeof(T)) == 1 ? raw.y : i / (4 / sizeof(T)) == 2 ? raw.z : raw.w;
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w);
        } else {
            const uint16_t h = (uint16_t)(i % 2 ? w >> 16 : w);
            return to_float(*reinterpret_cast<const T *>(&h));
        }
    }
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t top = 0;
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) top = max(top, __float_as_uint(fabsf(at(i))));
        return top;
    }
    // Its codes, with the block's scale byte.
    __device__ __forceinline__ void store(uint8_t *to, uint32_t s, bool on) const {
        float v[8] = {};
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) v[i] = at(i);
        const uint32_t w = s == 255u ? 0u : encode8(v, inverse_scale(s));
        if (!on) return;
        if constexpr (kOwn == 8) *reinterpret_cast<uint32_t *>(to) = w;
        else *reinterpret_cast<uint16_t *>(to) = (uint16_t)w;
    }
};
// A block with a spike has scale 2^-2 and codes of 4.
template <>
struct Piece<Spike> {
    static constexpr uint32_t kOwn = 16;
    uint4 raw;
    __device__ __forceinline__ uint32_t largest() const {
        return raw.x | raw.y | raw.z | raw.w ? 0x3f800000u : 0u;
    }
    static __device__ __forceinline__ uint32_t four(uint32_t w) {
        uint32_t v = __vcmpgtu4(w, 0u) & 0x06060606u;
        v = (v | v >> 4) & 0x00ff00ffu;
        return (v | v >> 8) & 0xffffu;
    }
    __device__ __forceinline__ void store(uint8_t *to, uint32_t, bool on) const {
        if (on) *reinterpret_cast<uint2 *>(to) = make_uint2(four(raw.x) | four(raw.y) << 16, four(raw.z) | four(raw.w) << 16);
    }
};
// The piece at p, of which n elements are left in the row. Aligned: p is a
// multiple of 16 bytes. Again: others read it too.
template <bool Aligned, bool Again = false, typename T>
__device__ __forceinline__ Piece<T> load_piece(const T *p, uint32_t n) {
    Piece<T> v;
    if (Aligned && n >= Piece<T>::kOwn) {
        v.raw = Again ? *reinterpret_cast<const uint4 *>(p) : __ldcs(reinterpret_cast<const uint4 *>(p));
    } else {
        __align__(16) T e[Piece<T>::kOwn];
#pragma unroll
        for (uint32_t i = 0; i < Piece<T>::kOwn; ++i) e[i] = i < n ? p[i] : T{};
        v.raw = *reinterpret_cast<const uint4 *>(e);
    }
    return v;
}

// The four words of a block's codes from its pieces.
template <typename T, uint32_t N>
__device__ __forceinline__ void pack_block(const Piece<T> (&v)[N], uint32_t s, uint32_t (&w)[4]) {
    const float inv = inverse_scale(s);
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
        float e[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) e[i] = v[(8 * q + i) / Piece<T>::kOwn].at((8 * q + i) % Piece<T>::kOwn);
        w[q] = s == 255u ? 0u : encode8(e, inv);
    }
}
__device__ __forceinline__ void pack_block(const Piece<Spike> (&v)[2], uint32_t, uint32_t (&w)[4]) {
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q) {
        w[2 * q] = Piece<Spike>::four(v[q].raw.x) | Piece<Spike>::four(v[q].raw.y) << 16;
        w[2 * q + 1] = Piece<Spike>::four(v[q].raw.z) | Piece<Spike>::four(v[q].raw.w) << 16;
    }
}

}  // namespace mx4
}  // namespace b200
