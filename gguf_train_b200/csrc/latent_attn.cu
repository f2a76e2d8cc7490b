// Absorbed latent attention, one query row a CTA: the scores of 128 keys at a time (a key a thread), their running
// maximum and sum, and the latent values' sums (4 dims a thread at most).

#include "gtb_common.cuh"
#include "latent.h"

namespace gtb {
namespace {

constexpr int NT = 128;

template <typename T>
__global__ void __launch_bounds__(NT) latent_attn_kernel(const __grid_constant__ LatentAttnArgs a) {
    __shared__ float qs[576], ps[NT], red[4];
    const int t = threadIdx.x, D = a.c.R + a.c.Dr, R = a.c.R;
    const int64_t row = blockIdx.x, i = row % a.Lq, h = row / a.Lq % a.H, b = row / (a.Lq * a.H);
    const int64_t len = min((int64_t)max(a.c.lens[b], 0), a.c.Smax);
    const int64_t cnt = a.counts ? min((int64_t)max(a.counts[b], 0), a.Lq) : a.Lq;
    const bool live = i < cnt;
    const int64_t own = live ? max(len - cnt + i + 1, (int64_t)0) : 0;
    const int64_t pre = live && a.prefix.rows ? min((int64_t)max(a.prefix.lens[0], 0), a.prefix.Smax) : 0;
    for (int d = t; d < D; d += NT) qs[d] = Elem<T>::load((const T*)a.q.p + b * a.q.sb + h * a.q.sh + i * a.q.ss + d);
    float m = -INFINITY, l = 0.0f, acc[4] = {};
    for (int64_t k0 = 0; k0 < pre + own; k0 += NT) {
        const int64_t k = k0 + t;
        auto key = [&](int64_t k) {
            return k < pre ? (const T*)a.prefix.rows + k * D : (const T*)a.c.rows + (b * a.c.Smax + k - pre) * D;
        };
        __syncthreads();
        float s = -INFINITY;
        if (k < pre + own) {
            const T* x = key(k);
            s = 0.0f;
            for (int d = 0; d < D; ++d) s = fmaf(qs[d], Elem<T>::load(x + d), s);
            s *= a.scale * 1.4426950408889634f;
        }
        float top = s;
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        if (t % 32 == 0) red[t / 32] = top;
        __syncthreads();
        const float mn = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
        const float off = mn == -INFINITY ? 0.0f : mn, al = exp2f(m - off);
        ps[t] = exp2f(s - off);
        __syncthreads();
        m = mn;
        l *= al;
        for (int e = 0; e < 4; ++e) acc[e] *= al;
        for (int j = 0; j < NT && k0 + j < pre + own; ++j) {
            const T* x = key(k0 + j);
            l += ps[j];
            for (int e = 0; e < 4; ++e)
                if (t + e * NT < R) acc[e] = fmaf(ps[j], Elem<T>::load(x + t + e * NT), acc[e]);
        }
    }
    for (int e = 0; e < 4; ++e)
        if (t + e * NT < R) Elem<T>::store((T*)a.o + row * R + t + e * NT, l > 0.0f ? acc[e] / l : 0.0f);
    if (a.lse && t == 0) a.lse[row] = l > 0.0f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
}

}  // namespace

int launch_latent_attention(const LatentAttnArgs& a, cudaStream_t st) {
    const unsigned grid = (unsigned)(a.c.B * a.H * a.Lq);
    if (a.c.dtype == F16) latent_attn_kernel<__half><<<grid, NT, 0, st>>>(a);
    else latent_attn_kernel<__nv_bfloat16><<<grid, NT, 0, st>>>(a);
    return cuda_failed(cudaGetLastError(), "latent_attention launch") ? -1 : 0;
}

}  // namespace gtb
