// Codes of the block-scaled 8-bit cache: value = code * scale, int8 (largest code 127) or e4m3 (448).
// Quantising is a chain of correctly rounded f32 operations (one division, one rounding to the code), so
// that appending, requantising and evicting give the same codes wherever they are computed.
#pragma once

#include "gtb_common.cuh"
#include "kv8.h"
#include "sm100_ptx.cuh"

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

// The same codes without a division each. x (1 / s), a little up and a little down, bracket the quotient as the
// division would round it; where both round to one code, that is the code. The others (next to the middle between two
// codes: one in some ten thousand, more where values repeat) are divided. The caller sees to values that are
// not finite; scales near either end of f32 divide throughout.
struct Quantiser {
    float s, up, down;
    bool ends;
    __device__ explicit Quantiser(float scale) : s(scale), up(0.0f), down(0.0f), ends(!(scale > 1e-30f && scale < 1e30f)) {
        if (!ends) {
            const float inv = __frcp_rn(scale);
            up = inv * (1.0f + 0x1p-20f);
            down = inv * (1.0f - 0x1p-20f);
        }
    }
    // for values f x (f > 0): the same with f taken into the factor
    __device__ void times(float f) {
        up *= f;
        down *= f;
        ends |= !(f > 1e-30f && up < 1e30f);
    }
};

template <int FMT>
__device__ __noinline__ uint32_t divide8x4(float x0, float x1, float x2, float x3, float s) {
    return (uint32_t)quantise8<FMT>(x0, s) | (uint32_t)quantise8<FMT>(x1, s) << 8 | (uint32_t)quantise8<FMT>(x2, s) << 16 |
           (uint32_t)quantise8<FMT>(x3, s) << 24;
}

// Codes of x[0..3] * f at scale z.s, z made for values x f (f = 1: as they are); `odd`: some may not be finite
template <int FMT>
__device__ __forceinline__ uint32_t quantise8x4(const float* x, const Quantiser& z, float f, bool odd) {
    uint32_t r;
    bool same;
    if constexpr (FMT == GTB_KV8_INT8) {
        constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: the sum's low byte is the nearest integer's
        const uint64_t up = sm100::f2_pack(z.up, z.up), down = sm100::f2_pack(z.down, z.down), magic = sm100::f2_pack(MAGIC, MAGIC);
        uint32_t a[4], diff = 0;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {  // two at a time
            const uint64_t v = sm100::f2_pack(x[i], x[i + 1]);
            float a0, a1, b0, b1;
            sm100::f2_unpack(sm100::f2_fma(v, up, magic), a0, a1);
            sm100::f2_unpack(sm100::f2_fma(v, down, magic), b0, b1);
            a[i] = __float_as_uint(a0);
            a[i + 1] = __float_as_uint(a1);
            diff |= (a[i] ^ __float_as_uint(b0)) | (a[i + 1] ^ __float_as_uint(b1));
        }
        same = diff == 0;
        r = __byte_perm(__byte_perm(a[0], a[1], 0x0040), __byte_perm(a[2], a[3], 0x0040), 0x5410);
    } else {
        uint16_t a0, a1, b0, b1;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a0) : "f"(x[1] * z.up), "f"(x[0] * z.up));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a1) : "f"(x[3] * z.up), "f"(x[2] * z.up));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b0) : "f"(x[1] * z.down), "f"(x[0] * z.down));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b1) : "f"(x[3] * z.down), "f"(x[2] * z.down));
        same = a0 == b0 && a1 == b1;
        r = (uint32_t)a0 | ((uint32_t)a1 << 16);
    }
    if (!same || odd || z.ends)
        r = divide8x4<FMT>(__fmul_rn(x[0], f), __fmul_rn(x[1], f), __fmul_rn(x[2], f), __fmul_rn(x[3], f), z.s);
    return r;
}

// The four codes of a word as f32 values
template <int FMT>
__device__ __forceinline__ void values8x4(uint32_t w, float* x) {
    if constexpr (FMT == GTB_KV8_INT8) {
        const uint32_t u = w ^ 0x80808080u;  // code + 128 as a byte; 0x4B000000 | byte is 2^23 + byte
#pragma unroll
        for (int i = 0; i < 4; i += 2)
            sm100::f2_unpack(sm100::f2_add(sm100::f2_pack(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)),
                                                          __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441 + i))),
                                           sm100::f2_pack(-8388736.0f, -8388736.0f)),
                             x[i], x[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t h;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (16 * i))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

// Launch that may start while the stream's previous kernel still runs: the kernel itself waits for that one's
// results with cudaGridDependencySynchronize(), in every thread, before it touches anything.
template <typename... P, typename... A>
bool launch_behind(const char* ctx, void (*kern)(P...), dim3 grid, int threads, cudaStream_t st, int smem, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return !cuda_failed(cudaLaunchKernelEx(&cfg, kern, P(args)...), ctx);
}

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

}  // namespace gtb
