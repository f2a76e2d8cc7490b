// Writing the latent cache: a token's latent vector and its rotary key, rotated for its position, as one row.
//
// HBM bound: every value is read once (a rotary key's twice, the second time from L1) and written once. A thread makes 16
// bytes of a row: 8 latent values copied or converted, or 8 rotated ones, whose angles it forms itself (position x turns
// modulo one turn in 64-bit fixed point, as rope_axes.cu does, so far positions lose nothing).

#include <algorithm>

#include "gtb_common.cuh"
#include "latent.h"

namespace gtb {
namespace {

constexpr int THREADS = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float* x) {
    if (vec) {
        __align__(16) T u[8];
#pragma unroll
        for (int w = 0; w < (int)sizeof(T) / 2; ++w) ((uint4*)u)[w] = ((const uint4*)p)[w];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = Elem<T>::load(u + k);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = Elem<T>::load(p + k);
    }
}

// rows lens[b] + i, i < counts[b], in pieces of 8 values; vec: every row of the operands starts on 16 bytes
template <typename T, typename U>
__global__ void __launch_bounds__(THREADS) latent_append_kernel(const __grid_constant__ LatentAppendArgs a, bool vec) {
    __shared__ uint64_t turn[ROPE_MAX_PAIRS];
    const int P = a.c.Dr / 2;
    if (a.turns && threadIdx.x < P) turn[threadIdx.x] = a.tab.turn[threadIdx.x];
    __syncthreads();
    const int D = a.c.R + a.c.Dr, pieces = D / 8;
    const int64_t b = blockIdx.y;
    const int64_t len = min((int64_t)max(a.c.lens[b], 0), a.c.Smax);
    const int64_t n = a.counts ? min((int64_t)max(a.counts[b], 0), a.n) : a.n;
    const int64_t base = a.offset ? max(a.offset[0], 0) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0 && len + n > a.c.Smax) atomicCAS(a.status, 0, 62);
    const int64_t fit = min(n, a.c.Smax - len);
    for (int64_t e = (int64_t)blockIdx.x * THREADS + threadIdx.x; e < fit * pieces; e += (int64_t)gridDim.x * THREADS) {
        const int64_t i = e / pieces;
        const int d = (int)(e - i * pieces) * 8;
        float y[8];
        if (d < a.c.R) {
            load8((const T*)a.latent.p + b * a.latent.sb + i * a.latent.ss + d, vec, y);
        } else {
            const T* x = (const T*)a.k_rope.p + b * a.k_rope.sb + i * a.k_rope.ss;
            const int r = d - a.c.R;
            load8(x + r, vec, y);
            if (a.turns) {
                const uint64_t pos = (uint64_t)(base + len + i);
                auto cs = [&](int pair, float& c, float& s) {
                    // signed fraction of a turn, 2^-32
                    sincospif((float)(int32_t)((pos * turn[pair]) >> 32) * 4.656612873077393e-10f, &s, &c);
                };
                float c, s;
                if (a.mode == 2) {
                    float z[8];  // the pairs' other elements
                    const bool second = r >= P;
                    load8(x + (second ? r - P : r + P), vec, z);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        cs((second ? r - P : r) + k, c, s);
                        y[k] = second ? z[k] * s + y[k] * c : y[k] * c - z[k] * s;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k += 2) {
                        cs((r + k) / 2, c, s);
                        const float x0 = y[k], x1 = y[k + 1];
                        y[k] = x0 * c - x1 * s;
                        y[k + 1] = x0 * s + x1 * c;
                    }
                }
            }
        }
        __align__(16) U w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) Elem<U>::store(w + k, y[k]);
        *(uint4*)((U*)a.c.rows + (b * a.c.Smax + len + i) * D + d) = *(const uint4*)w;
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
    const int64_t pieces = a.n * ((a.c.R + a.c.Dr) / 8);
    for (int64_t b0 = 0; b0 < a.c.B; b0 += 65535) {
        LatentAppendArgs z = a;
        z.c.B = std::min<int64_t>(65535, a.c.B - b0);
        z.c.rows = (U*)a.c.rows + b0 * a.c.Smax * (a.c.R + a.c.Dr);
        z.c.lens = a.c.lens + b0;
        z.latent.p = (T*)a.latent.p + b0 * a.latent.sb;
        z.k_rope.p = (T*)a.k_rope.p + b0 * a.k_rope.sb;
        if (a.counts) z.counts = a.counts + b0;
        const dim3 grid((unsigned)std::min<int64_t>((pieces + THREADS - 1) / THREADS, std::max<int64_t>(1, 64 * n_sm / z.c.B)),
                        (unsigned)z.c.B);
        latent_append_kernel<T, U><<<grid, THREADS, 0, st>>>(z, vec);
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
