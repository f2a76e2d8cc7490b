// Attention over the block-scaled 8-bit cache, simple form: one warp per query row, a key at a time, the
// head dimension across the lanes, softmax online in f32; then, for the accumulated weights, one warp per
// cached row that forms its column of probabilities from the rows' log-sum-exp.

#include <cmath>

#include "gtb_common.cuh"
#include "kv8.cuh"

namespace gtb {
namespace {

constexpr int ND = 8;  // head dimension / 32, at most

template <typename T>
__device__ __forceinline__ void load_row(const T* p, int64_t D, float* r) {
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        const int d = i * 32 + (threadIdx.x & 31);
        r[i] = d < D ? Elem<T>::load(p + d) : 0.0f;
    }
}

template <int FMT>
__device__ __forceinline__ void load_codes(const uint8_t* p, int64_t D, float* r) {
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        const int d = i * 32 + (threadIdx.x & 31);
        r[i] = d < D ? Code8<FMT>::value(p[d]) : 0.0f;
    }
}

__device__ __forceinline__ float dot(const float* x, const float* y) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; ++i) s = fmaf(x[i], y[i], s);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// rows s a query may attend: [0, limit)
__device__ __forceinline__ int64_t row_limit(const Kv8AttnArgs& a, int64_t b, int64_t i) {
    const int64_t len = clamp64(a.c.lens[b], 0, a.c.Smax);
    const int64_t cnt = a.counts ? clamp64(a.counts[b], 0, a.Lq) : a.Lq;
    return i < cnt ? max((int64_t)0, len - cnt + i + 1) : 0;
}

template <typename T, int FMT>
__global__ void kv8_attn_kernel(const Kv8AttnArgs a, float* lse) {
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= a.c.B * a.H * a.Lq) return;
    const int64_t i = row % a.Lq, h = row / a.Lq % a.H, b = row / a.Lq / a.H;
    const int64_t D = a.c.D, bh = b * a.c.Hkv + h / (a.H / a.c.Hkv);
    const int64_t nb = (a.c.Smax + a.c.block - 1) / a.c.block;
    const int64_t limit = row_limit(a, b, i);
    float q[ND], acc[ND] = {}, x[ND];
    load_row((const T*)a.q.p + b * a.q.sb + h * a.q.sh + i * a.q.ss, D, q);
    float m = -INFINITY, l = 0.0f;
    const uint8_t *K = (const uint8_t*)a.c.k + bh * a.c.Smax * D, *V = (const uint8_t*)a.c.v + bh * a.c.Smax * D;
    for (int64_t s = 0; s < limit; ++s) {
        load_codes<FMT>(K + s * D, D, x);
        const float z = dot(q, x) * (a.scale * a.c.k_scale[bh * nb + s / a.c.block]);
        const float m2 = fmaxf(m, z), corr = expf(m - m2), p = expf(z - m2);
        load_codes<FMT>(V + s * D, D, x);
        const float pv = p * a.c.v_scale[bh * nb + s / a.c.block];
#pragma unroll
        for (int k = 0; k < ND; ++k) acc[k] = fmaf(pv, x[k], acc[k] * corr);
        l = l * corr + p;
        m = m2;
    }
    const float inv = limit > 0 ? 1.0f / l : 0.0f;
    T* o = (T*)a.o.p + b * a.o.sb + h * a.o.sh + i * a.o.ss;
#pragma unroll
    for (int k = 0; k < ND; ++k) {
        const int d = k * 32 + (threadIdx.x & 31);
        if (d < D) Elem<T>::store(o + d, acc[k] * inv);
    }
    if (lse && (threadIdx.x & 31) == 0) lse[row] = limit > 0 ? m + logf(l) : -INFINITY;
}

template <typename T, int FMT>
__global__ void kv8_score_kernel(const Kv8AttnArgs a, const float* lse) {
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= a.c.B * a.c.Hkv * a.c.Smax) return;
    const int64_t s = row % a.c.Smax, bh = row / a.c.Smax, b = bh / a.c.Hkv, hk = bh - b * a.c.Hkv;
    const int64_t len = clamp64(a.c.lens[b], 0, a.c.Smax);
    if (s >= len) return;
    const int64_t D = a.c.D, G = a.H / a.c.Hkv, nb = (a.c.Smax + a.c.block - 1) / a.c.block;
    float k[ND], q[ND], w = 0.0f;
    load_codes<FMT>((const uint8_t*)a.c.k + row * D, D, k);
    const float sc = a.scale * a.c.k_scale[bh * nb + s / a.c.block];
    for (int64_t h = hk * G; h < (hk + 1) * G; ++h)
        for (int64_t i = 0; i < a.Lq; ++i) {
            if (s >= row_limit(a, b, i)) continue;
            load_row((const T*)a.q.p + b * a.q.sb + h * a.q.sh + i * a.q.ss, D, q);
            w += expf(dot(q, k) * sc - lse[(b * a.H + h) * a.Lq + i]);
        }
    if ((threadIdx.x & 31) == 0) a.score_out[row] = a.score_in[row] + w;
}

template <typename T, int FMT>
int run(const Kv8AttnArgs& a, cudaStream_t st) {
    const int64_t rows = a.c.B * a.H * a.Lq, cached = a.c.B * a.c.Hkv * a.c.Smax;
    float* lse = a.lse;
    void* scratch = nullptr;
    if (a.score_out && !lse && rows > 0) {
        if (cuda_failed(cudaMallocAsync(&scratch, rows * sizeof(float), st), "kv8_attention: scratch allocation")) return -1;
        lse = (float*)scratch;
    }
    if (rows > 0) kv8_attn_kernel<T, FMT><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(a, lse);
    bool bad = cuda_failed(cudaGetLastError(), "kv8_attention launch");
    if (!bad && a.score_out && cached > 0) {
        kv8_score_kernel<T, FMT><<<(unsigned)((cached + 3) / 4), 128, 0, st>>>(a, lse);
        bad = cuda_failed(cudaGetLastError(), "kv8_attention: score launch");
    }
    if (scratch) cudaFreeAsync(scratch, st);
    return bad ? -1 : 0;
}

}  // namespace

int launch_kv8_attention(const Kv8AttnArgs& a, cudaStream_t st) {
    const bool e4m3 = a.c.format == GTB_KV8_E4M3;
    switch (a.dtype) {
        case F32: return e4m3 ? run<float, GTB_KV8_E4M3>(a, st) : run<float, GTB_KV8_INT8>(a, st);
        case F16: return e4m3 ? run<__half, GTB_KV8_E4M3>(a, st) : run<__half, GTB_KV8_INT8>(a, st);
        default: return e4m3 ? run<__nv_bfloat16, GTB_KV8_E4M3>(a, st) : run<__nv_bfloat16, GTB_KV8_INT8>(a, st);
    }
}

}  // namespace gtb
