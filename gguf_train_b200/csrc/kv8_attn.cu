// Attention over the block-scaled 8-bit cache: choice of kernels.

#include <algorithm>
#include <cmath>

#include "gtb_common.cuh"
#include "kv8.cuh"
#include "kv8_chunk.h"
#include "kv8_mma.cuh"

namespace gtb {

namespace {

// Kept scores take 4 R bytes for every row of capacity: at most this much at a time. A call that needs more runs in groups
// of sequences (64 sequences of 1k to 32k tokens, 32 rows for each of 8 heads, in 3 groups: 2.26 ms, at once 2.19);
// where one sequence alone needs more, the weights kernel forms the products again.
constexpr int64_t SCORES_MAX = 1ll << 30;

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
        // sequences a launch: all of them, or as many as the kept scores of fit into SCORES_MAX
        int64_t group = a.c.B;
        kept = a.score_out && a.c.Smax > 0 && kv8::keep_scores(p.R, a.c.D);
        if (kept) {
            p.score_in = a.score_in;
            p.score_out = a.score_out;
            const int64_t fit = SCORES_MAX / (a.c.Hkv * a.c.Smax * p.R * (int64_t)sizeof(float));
            kept = fit > 0;
            if (kept && fit < group) {
                const int64_t launches = (group + fit - 1) / fit;
                group = (group + launches - 1) / launches;
            }
        }
        if (!kept) p.score_in = p.score_out = nullptr;
        for (int64_t b0 = 0; b0 < a.c.B && !rc; b0 += group) {
            kv8::MmaP g = p;
            g.c.B = std::min(group, a.c.B - b0);
            const int64_t rows0 = b0 * a.c.Hkv * a.c.Smax, blocks0 = b0 * a.c.Hkv * ((a.c.Smax + a.c.block - 1) / a.c.block);
            const int64_t es = a.dtype == F32 ? 4 : 2;
            g.c.k = (char*)a.c.k + rows0 * a.c.D;
            g.c.v = (char*)a.c.v + rows0 * a.c.D;
            g.c.k_scale = a.c.k_scale + blocks0;
            g.c.v_scale = a.c.v_scale + blocks0;
            g.c.lens = a.c.lens + b0;
            g.q.p = (char*)a.q.p + b0 * a.q.sb * es;
            g.o.p = (char*)a.o.p + b0 * a.o.sb * es;
            if (g.counts) g.counts += b0;
            if (g.lse) g.lse += b0 * a.H * a.Lq;
            if (kept) {
                g.score_in += rows0;
                g.score_out += rows0;
            }
            rc = a.c.D <= 64 ? kv8::launch_mma_64(g, n_sm, st) : a.c.D <= 128 ? kv8::launch_mma_128(g, n_sm, st) : kv8::launch_mma_256(g, n_sm, st);
        }
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
