// Attention over the block-scaled 8-bit cache: choice of kernels.

#include <algorithm>
#include <cmath>

#include "gtb_common.cuh"
#include "kv8.cuh"
#include "kv8_chunk.h"
#include "kv8_mma.cuh"

namespace gtb {

namespace {

// score_out = score_in below the lengths: what the weights come to where there is no query
__global__ void kv8_copy_scores_kernel(const gtb_kv8 c, const float* __restrict__ in, float* __restrict__ out) {
    for (int64_t bh = blockIdx.y; bh < c.B * c.Hkv; bh += gridDim.y) {
        const int len = (int)clamp64(c.lens[bh / c.Hkv], 0, c.Smax);
        for (int64_t k = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; k < len; k += (int64_t)gridDim.x * blockDim.x)
            out[bh * c.Smax + k] = in[bh * c.Smax + k];
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
    if (!rc && a.score_out && !kept && a.c.Smax > 0) {
        if (rows > 0) {
            rc = kv8::launch_weigh(a, lse, st);
        } else {
            kv8_copy_scores_kernel<<<dim3(32, (unsigned)std::min<int64_t>(65535, a.c.B * a.c.Hkv)), 256, 0, st>>>(a.c, a.score_in, a.score_out);
            rc = cuda_failed(cudaGetLastError(), "kv8_attention: scores launch") ? -1 : 0;
        }
    }
    if (scratch) cudaFreeAsync(scratch, st);
    return rc;
}

}  // namespace gtb
