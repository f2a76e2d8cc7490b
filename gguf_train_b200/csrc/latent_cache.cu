// Writing the latent cache: a token's latent vector and its rotary key, rotated for its position, as one row.
//
// HBM bound: every value is read once (a rotary key's twice, the second time from L1) and written once. A thread makes 16
// bytes of a row, the same ones of every token it has (so sizes are divided by once): 8 latent values copied or converted, or 8 rotated
// ones, whose angles it forms itself (position x turns modulo one turn in 64-bit fixed point, as rope_axes.cu does, so far
// positions lose nothing). Four tokens' loads are in flight.

#include <algorithm>

#include "gtb_common.cuh"
#include "latent.h"

namespace gtb {
namespace {

constexpr int FLIGHT = 4;  // tokens of a thread whose loads go out together

template <typename T>
struct Raw8 {
    __align__(16) T v[8];
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, Raw8<T>& x) {
    if (vec) {
#pragma unroll
        for (int w = 0; w < (int)sizeof(T) / 2; ++w) ((uint4*)x.v)[w] = ((const uint4*)p)[w];
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x.v[k] = p[k];
    }
}

// Rows lens[b] + i, i < counts[b]. A block has `slots` tokens at a time, a thread always the same 8 values of a row; vec: every row
// of the operands starts on 16 bytes.
template <typename T, typename U>
__global__ void __launch_bounds__(288) latent_append_kernel(const __grid_constant__ LatentAppendArgs a, bool vec, int slots) {
    // (the rotary pieces' threads come after all others: their warps alone go through the angles)
    const int P = a.c.Dr / 2, D = a.c.R + a.c.Dr, copies = a.c.R / 8, turning = a.c.Dr / 8;
    const int e = (int)threadIdx.x - slots * copies, per = e < 0 ? copies : turning, q = e < 0 ? (int)threadIdx.x : e;
    const int slot = q / per, d = (e < 0 ? 0 : a.c.R) + (q - slot * per) * 8;
    const int64_t b = blockIdx.y;
    const int64_t len = min((int64_t)max(a.c.lens[b], 0), a.c.Smax);
    const int64_t n = a.counts ? min((int64_t)max(a.counts[b], 0), a.n) : a.n;
    const int64_t base = (a.offset ? (int64_t)max(a.offset[0], 0) : 0) + len;
    if (blockIdx.x == 0 && threadIdx.x == 0 && len + n > a.c.Smax) atomicCAS(a.status, 0, 62);
    const int64_t fit = min(n, a.c.Smax - len), step = (int64_t)gridDim.x * slots;
    const bool rope = d >= a.c.R, turns = rope && a.turns;
    const int r = d - a.c.R;                                  // first value within the rotary key
    const bool second = r >= P;                               // mode 2: of the second half, whose partners lie P before
    const int pair0 = a.mode != 2 ? r / 2 : second ? r - P : r;
    uint64_t turn[8];                                         // of this thread's pairs (mode 0: 4)
#pragma unroll
    for (int k = 0; k < 8; ++k) turn[k] = turns && (a.mode == 2 || k < 4) ? a.tab.turn[pair0 + k] : 0;
    const T* x = rope ? (const T*)a.k_rope.p + b * a.k_rope.sb + r : (const T*)a.latent.p + b * a.latent.sb + d;
    const int64_t xs = rope ? a.k_rope.ss : a.latent.ss;
    const int partner = second ? -P : P;
    U* y = (U*)a.c.rows + (b * a.c.Smax + len) * D + d;
    for (int64_t i0 = (int64_t)blockIdx.x * slots + slot; i0 < fit; i0 += FLIGHT * step) {
        Raw8<T> own[FLIGHT], other[FLIGHT];
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            const int64_t i = i0 + f * step;
            if (i >= fit) continue;
            load8(x + i * xs, vec, own[f]);
            if (turns && a.mode == 2) load8(x + i * xs + partner, vec, other[f]);
        }
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            const int64_t i = i0 + f * step;
            if (i >= fit) continue;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = Elem<T>::load(own[f].v + k);
            if (turns) {
                const uint64_t pos = (uint64_t)(base + i);
                auto cs = [&](int k, float& c, float& s) {  // signed fraction of a turn, 2^-32
                    sincospif((float)(int32_t)((pos * turn[k]) >> 32) * 4.656612873077393e-10f, &s, &c);
                };
                float c, s;
                if (a.mode == 2) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        cs(k, c, s);
                        const float z = Elem<T>::load(other[f].v + k);
                        v[k] = second ? z * s + v[k] * c : v[k] * c - z * s;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        cs(k, c, s);
                        const float x0 = v[2 * k], x1 = v[2 * k + 1];
                        v[2 * k] = x0 * c - x1 * s;
                        v[2 * k + 1] = x0 * s + x1 * c;
                    }
                }
            }
            __align__(16) U w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) Elem<U>::store(w + k, v[k]);
            *(uint4*)(y + i * D) = *(const uint4*)w;
        }
    }
}

// lens[b] = min(lens[b] + counts[b], Smax), once every row is written
__global__ void latent_advance_kernel(const __grid_constant__ LatentAppendArgs a) {
    for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < a.c.B; b += (int64_t)gridDim.x * blockDim.x) {
        const int64_t len = min((int64_t)max(a.c.lens[b], 0), a.c.Smax);
        const int64_t n = a.counts ? min((int64_t)max(a.counts[b], 0), a.n) : a.n;
        a.c.lens[b] = (int32_t)min(len + n, a.c.Smax);
    }
}

template <typename T, typename U>
int launch(const LatentAppendArgs& a, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool vec = true;
    for (const Rows3* r : {&a.latent, &a.k_rope})
        vec = vec && ((uintptr_t)r->p & 15) == 0 && (a.c.B == 1 || r->sb % V == 0) && (a.n == 1 || r->ss % V == 0);
    int dev = 0, n_sm = 0;
    if (cuda_failed(cudaGetDevice(&dev), "latent_append") ||
        cuda_failed(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev), "latent_append"))
        return -1;
    const int pieces = (a.c.R + a.c.Dr) / 8;                  // 10 .. 72
    const int slots = (int)std::min<int64_t>(256 / pieces, a.n), threads = slots * pieces;
    const int64_t blocks = (a.n + slots * FLIGHT - 1) / (slots * FLIGHT);
    for (int64_t b0 = 0; b0 < a.c.B; b0 += 65535) {
        LatentAppendArgs z = a;
        z.c.B = std::min<int64_t>(65535, a.c.B - b0);
        z.c.rows = (U*)a.c.rows + b0 * a.c.Smax * (a.c.R + a.c.Dr);
        z.c.lens = a.c.lens + b0;
        z.latent.p = (T*)a.latent.p + b0 * a.latent.sb;
        z.k_rope.p = (T*)a.k_rope.p + b0 * a.k_rope.sb;
        if (a.counts) z.counts = a.counts + b0;
        const dim3 grid((unsigned)std::min<int64_t>(blocks, std::max<int64_t>(1, 32 * (int64_t)n_sm / z.c.B)), (unsigned)z.c.B);
        latent_append_kernel<T, U><<<grid, threads, 0, st>>>(z, vec, slots);
        if (a.advance) latent_advance_kernel<<<(unsigned)((z.c.B + 255) / 256), 256, 0, st>>>(z);
        if (cuda_failed(cudaGetLastError(), "latent_append launch")) return -1;
    }
    return 0;
}

template <typename T>
int launch_to(const LatentAppendArgs& a, cudaStream_t st) {
    return a.c.dtype == F16 ? launch<T, __half>(a, st) : launch<T, __nv_bfloat16>(a, st);
}

}  // namespace

int launch_latent_append(const LatentAppendArgs& a, cudaStream_t st) {
    switch (a.dtype) {
        case F32: return launch_to<float>(a, st);
        case F16: return launch_to<__half>(a, st);
        default: return launch_to<__nv_bfloat16>(a, st);
    }
}

}  // namespace gtb
