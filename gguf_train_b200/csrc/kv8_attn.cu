// Attention over the block-scaled 8-bit cache: choice of kernel, and the accumulated attention weights.
// The weights of the cached rows come from the rows' log-sum-exp in a kernel of their own (kv8_score_kernel):
// one warp per cached row, a query at a time.

#include <cmath>

#include "gtb_common.cuh"
#include "kv8.cuh"
#include "kv8_chunk.h"
#include "kv8_mma.cuh"

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

template <typename T, int FMT>
__global__ void kv8_score_kernel(const Kv8AttnArgs a, const float* lse) {
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= a.c.B * a.c.Hkv * a.c.Smax) return;
    const int64_t s = row % a.c.Smax, bh = row / a.c.Smax, b = bh / a.c.Hkv, hk = bh - b * a.c.Hkv;
    const int64_t len = clamp64(a.c.lens[b], 0, a.c.Smax);
    if (s >= len) return;
    const int64_t D = a.c.D, G = a.H / a.c.Hkv, nb = (a.c.Smax + a.c.block - 1) / a.c.block;
    const int64_t cnt = a.counts ? clamp64(a.counts[b], 0, a.Lq) : a.Lq;
    float k[ND], q[ND], w = 0.0f;
    load_codes<FMT>((const uint8_t*)a.c.k + row * D, D, k);
    const float sc = a.scale * a.c.k_scale[bh * nb + s / a.c.block];
    for (int64_t h = hk * G; h < (hk + 1) * G; ++h)
        for (int64_t i = max((int64_t)0, s - (len - cnt)); i < cnt; ++i) {  // queries that see row s
            load_row((const T*)a.q.p + b * a.q.sb + h * a.q.sh + i * a.q.ss, D, q);
            w += expf(dot(q, k) * sc - lse[(b * a.H + h) * a.Lq + i]);
        }
    if ((threadIdx.x & 31) == 0) a.score_out[row] = a.score_in[row] + w;
}

template <typename T, int FMT>
int run_score(const Kv8AttnArgs& a, const float* lse, cudaStream_t st) {
    const int64_t cached = a.c.B * a.c.Hkv * a.c.Smax;
    if (cached == 0) return 0;
    kv8_score_kernel<T, FMT><<<(unsigned)((cached + 3) / 4), 128, 0, st>>>(a, lse);
    return cuda_failed(cudaGetLastError(), "kv8_attention: score launch") ? -1 : 0;
}

int launch_score(const Kv8AttnArgs& a, const float* lse, cudaStream_t st) {
    const bool e4m3 = a.c.format == GTB_KV8_E4M3;
    switch (a.dtype) {
        case F32: return e4m3 ? run_score<float, GTB_KV8_E4M3>(a, lse, st) : run_score<float, GTB_KV8_INT8>(a, lse, st);
        case F16: return e4m3 ? run_score<__half, GTB_KV8_E4M3>(a, lse, st) : run_score<__half, GTB_KV8_INT8>(a, lse, st);
        default: return e4m3 ? run_score<__nv_bfloat16, GTB_KV8_E4M3>(a, lse, st) : run_score<__nv_bfloat16, GTB_KV8_INT8>(a, lse, st);
    }
}

}  // namespace

int launch_kv8_attention(const Kv8AttnArgs& a, cudaStream_t st) {
    const int64_t rows = a.c.B * a.H * a.Lq;
    int dev = 0, n_sm = 0;  // (reading an attribute is a look-up in the runtime)
    if (cuda_failed(cudaGetDevice(&dev), "kv8_attention") ||
        cuda_failed(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev), "kv8_attention"))
        return -1;
    float* lse = a.lse;
    void* scratch = nullptr;
    if (a.score_out && !lse && rows > 0) {
        if (cuda_failed(cudaMallocAsync(&scratch, rows * sizeof(float), st), "kv8_attention: scratch allocation")) return -1;
        lse = (float*)scratch;
    }
    int rc = 0;
    bool kept = false;
    if (rows > 0 && kv8::chunk_supported(a)) {
        rc = kv8::launch_chunk(a, lse, n_sm, st);
    } else if (rows > 0) {
        kv8::MmaP p{};
        p.c = a.c;
        p.q = a.q;
        p.o = a.o;
        p.dtype = a.dtype;
        p.q_vec = kv8::vector_rows(a.q, a.dtype);
        p.G = (int)(a.H / a.c.Hkv);
        p.R = p.G * (int)a.Lq;
        p.H = a.H;
        p.Lq = a.Lq;
        p.scale_log2 = a.scale * 1.4426950408889634f;
        p.counts = a.counts;
        p.lse = lse;
        kept = a.score_out && a.c.Smax > 0 && kv8::keep_scores(p.R, a.c.D);
        if (kept) {
            p.score_in = a.score_in;
            p.score_out = a.score_out;
        }
        rc = a.c.D <= 64 ? kv8::launch_mma_64(p, n_sm, st) : a.c.D <= 128 ? kv8::launch_mma_128(p, n_sm, st) : kv8::launch_mma_256(p, n_sm, st);
    }
    if (!rc && a.score_out && !kept) rc = launch_score(a, lse, st);
    if (scratch) cudaFreeAsync(scratch, st);
    return rc;
}

}  // namespace gtb
