// Rotary position embedding with several position axes, of one tensor or of q and k in one launch.
// The angle of pair i of token (b, s) is pos[axis(i)][b][s] * f(i). Its value modulo a turn is all that the
// sine and cosine see, so the frequency is kept as turns per position in 64-bit fixed point: the integer
// product position * turn modulo 2^64 drops the whole turns exactly, at any int32 position.

#include <algorithm>

#include "gtb_common.cuh"
#include "kv8.h"

namespace gtb {
namespace {

// (cos, sin) of pair i at position p
__device__ __forceinline__ float2 turn_of(int32_t p, uint64_t turn, float sin_sign) {
    const int32_t frac = (int32_t)(((uint64_t)(int64_t)p * turn) >> 32);  // signed fraction of a turn, 2^-32
    float s, c;
    sincospif((float)frac * 4.656612873077393e-10f, &s, &c);  // x 2 * 2^-32
    return make_float2(c, s * sin_sign);
}

// One thread per pair of one row
template <typename T>
__global__ void rope_axes_kernel(const __grid_constant__ RopeAxesArgs a) {
    const int64_t per_row = a.pairs + (a.D - 2 * a.pairs);
    const int64_t heads = a.heads[0] + a.heads[1];
    const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= a.B * heads * a.S * per_row) return;
    const int64_t row = idx / per_row;
    const int i = (int)(idx - row * per_row);
    const int64_t s = row % a.S, hh = row / a.S % heads, b = row / a.S / heads;
    const int w = hh >= a.heads[0];
    const int64_t h = hh - (w ? a.heads[0] : 0);
    const T* x = (const T*)a.x[w].p + b * a.x[w].sb + h * a.x[w].sh + s * a.x[w].ss;
    T* y = (T*)a.y[w].p + b * a.y[w].sb + h * a.y[w].sh + s * a.y[w].ss;
    if (i >= a.pairs) {
        y[a.pairs + i] = x[a.pairs + i];
        return;
    }
    const float2 cs = turn_of(a.pos[a.tab.axis[i] * a.pos_axis + b * a.pos_batch + s], a.tab.turn[i], a.sin_sign);
    const int c0 = a.mode == 2 ? i : 2 * i, c1 = a.mode == 2 ? i + a.pairs : 2 * i + 1;
    const float x0 = Elem<T>::load(x + c0), x1 = Elem<T>::load(x + c1);
    Elem<T>::store(y + c0, x0 * cs.x - x1 * cs.y);
    Elem<T>::store(y + c1, x0 * cs.y + x1 * cs.x);
}

}  // namespace

int launch_rope_axes(const RopeAxesArgs& a, cudaStream_t st) {
    const int64_t n = a.B * (a.heads[0] + a.heads[1]) * a.S * (a.D - a.pairs);
    const unsigned grid = (unsigned)((n + 255) / 256);
    switch (a.dtype) {
        case F32: rope_axes_kernel<float><<<grid, 256, 0, st>>>(a); break;
        case F16: rope_axes_kernel<__half><<<grid, 256, 0, st>>>(a); break;
        default: rope_axes_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a); break;
    }
    return cuda_failed(cudaGetLastError(), "rope_axes launch") ? -1 : 0;
}

}  // namespace gtb
