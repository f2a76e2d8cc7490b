// Codes of the block-scaled 8-bit cache: value = code * scale, int8 (largest code 127) or e4m3 (448).
// Quantising is a chain of correctly rounded f32 operations (one division, one rounding to the code), so
// that appending, requantising and evicting give the same codes wherever they are computed.
#pragma once

#include "gtb_common.cuh"
#include "kv8.h"

namespace gtb {

template <int FMT>
struct Code8;

template <>
struct Code8<GTB_KV8_INT8> {
    static constexpr float TOP = 127.0f;
    __device__ static float value(uint8_t c) { return (float)(int8_t)c; }
    // y finite, |y| <= TOP
    __device__ static uint8_t nearest(float y) { return (uint8_t)(int8_t)__float2int_rn(y); }
};

template <>
struct Code8<GTB_KV8_E4M3> {
    static constexpr float TOP = 448.0f;
    __device__ static float value(uint8_t c) {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)c));
        return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
    }
    __device__ static uint8_t nearest(float y) {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(y));
        return (uint8_t)(r & 0xffu);
    }
};

// |x| where x is finite, else 0: what a block's scale is taken from
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}

// amax times the f32 reciprocal of the largest code: the largest value lands within 1 ulp of that code
template <int FMT>
__device__ __forceinline__ float scale_of(float amax) {
    return __fmul_rn(amax, 1.0f / Code8<FMT>::TOP);
}

// The code of x at scale s: round(x / s), saturating; 0 for NaN and for a zero scale
template <int FMT>
__device__ __forceinline__ uint8_t quantise8(float x, float s) {
    if (!(s > 0.0f)) return 0;
    float y = __fdiv_rn(x, s);
    if (!(y == y)) return 0;
    y = fminf(fmaxf(y, -Code8<FMT>::TOP), Code8<FMT>::TOP);
    return Code8<FMT>::nearest(y);
}

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

}  // namespace gtb
