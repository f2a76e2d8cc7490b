// The block-scaled 8-bit cache: append, read back, evict.

#include <algorithm>

#include "gtb_common.cuh"
#include "kv8.cuh"

namespace gtb {
namespace {

__device__ __forceinline__ float block_max(float v, float* red) {
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float m = 0.0f;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) m = fmaxf(m, red[w]);
    __syncthreads();
    return m;
}

// One CTA per (touched block, sequence x kv head, K or V)
template <typename T, int FMT>
__global__ void kv8_append_kernel(const Kv8AppendArgs a) {
    __shared__ float red[32];
    const gtb_kv8& c = a.c;
    const int64_t bh = blockIdx.y, b = bh / c.Hkv, hk = bh - b * c.Hkv;
    const bool is_v = blockIdx.z != 0;
    const Rows3 x = is_v ? a.v : a.k;
    const int64_t T_ = c.block, D = c.D;
    const int64_t pos = clamp64(c.lens[b], 0, c.Smax);
    const int64_t cnt = a.counts ? clamp64(a.counts[b], 0, a.n) : a.n;
    const int64_t end = min(pos + cnt, c.Smax);
    if (pos + cnt > c.Smax && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(a.status, 0, 61);
    const int64_t j = pos / T_ + blockIdx.x;
    const int64_t r0 = max(j * T_, pos), r1 = min((j + 1) * T_, end);  // new rows of this block
    if (r0 >= r1) return;
    const T* src = (const T*)x.p + b * x.sb + hk * x.sh;
    uint8_t* codes = (uint8_t*)(is_v ? c.v : c.k) + bh * c.Smax * D;
    float* scale = (is_v ? c.v_scale : c.k_scale) + bh * ((c.Smax + T_ - 1) / T_) + j;
    const int64_t n_new = (r1 - r0) * D;
    float m = 0.0f;
    for (int64_t e = threadIdx.x; e < n_new; e += blockDim.x) {
        const int64_t r = e / D, d = e - r * D;
        m = fmaxf(m, finite_abs(Elem<T>::load(src + (r0 - pos + r) * x.ss + d)));
    }
    const float s_old = j * T_ < pos ? *scale : 0.0f;
    const float s = fmaxf(s_old, scale_of<FMT>(block_max(m, red)));
    if (s > s_old) {
        uint8_t* held = codes + j * T_ * D;
        const int64_t n_old = (r0 - j * T_) * D;
        for (int64_t e = threadIdx.x; e < n_old; e += blockDim.x)
            held[e] = quantise8<FMT>(__fmul_rn(Code8<FMT>::value(held[e]), s_old), s);
    }
    for (int64_t e = threadIdx.x; e < n_new; e += blockDim.x) {
        const int64_t r = e / D, d = e - r * D;
        codes[r0 * D + e] = quantise8<FMT>(Elem<T>::load(src + (r0 - pos + r) * x.ss + d), s);
    }
    if (threadIdx.x == 0) *scale = s;
}

__global__ void kv8_advance_kernel(const Kv8AppendArgs a) {
    const int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= a.c.B) return;
    const int64_t pos = clamp64(a.c.lens[b], 0, a.c.Smax);
    const int64_t cnt = a.counts ? clamp64(a.counts[b], 0, a.n) : a.n;
    a.c.lens[b] = (int32_t)min(pos + cnt, a.c.Smax);
}

template <typename T, int FMT>
__global__ void kv8_read_kernel(const Kv8ReadArgs a) {
    const gtb_kv8& c = a.c;
    const int64_t per = c.B * c.Hkv * a.n * c.D;
    const int64_t nb = (c.Smax + c.block - 1) / c.block;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < 2 * per; i += (int64_t)gridDim.x * blockDim.x) {
        const bool is_v = i >= per;
        const int64_t e = is_v ? i - per : i;
        const int64_t d = e % c.D, row = e / c.D, bh = row / a.n, t = row - bh * a.n;
        const int64_t r = t + (a.start ? a.start[bh / c.Hkv] : 0);
        float v = 0.0f;
        if (r >= 0 && r < c.Smax)
            v = __fmul_rn(Code8<FMT>::value(((const uint8_t*)(is_v ? c.v : c.k))[(bh * c.Smax + r) * c.D + d]),
                          (is_v ? c.v_scale : c.k_scale)[bh * nb + r / c.block]);
        Elem<T>::store((T*)(is_v ? a.v : a.k) + e, v);
    }
}

// Order of scores as unsigned integers: larger score, larger key; NaN as -inf, -0 as 0
__device__ __forceinline__ uint32_t score_key(float s) {
    if (!(s == s)) s = -INFINITY;
    const uint32_t u = __float_as_uint(__fadd_rn(s, 0.0f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int SEL_THREADS = 1024;

// Exclusive prefix sum over the CTA of one 64-bit value per thread; returns the total in `total`
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* sh, uint64_t& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint64_t x = v;
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sh[w] = x;
    __syncthreads();
    if (w == 0) {
        uint64_t t = lane < (int)(blockDim.x >> 5) ? sh[lane] : 0, s = t;
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        sh[lane] = s - t;
        if (lane == 31) sh[32] = s;
    }
    __syncthreads();
    const uint64_t r = sh[w] + x - v;
    total = sh[32];
    __syncthreads();
    return r;
}

// Which rows stay: one CTA per (sequence, kv head). The k-th largest key among the candidates is found 8
// bits at a time from a histogram; a second sweep in row order takes every larger key and the first
// `need` rows that equal it, then the recent rows, and writes their indices in order.
__global__ void __launch_bounds__(SEL_THREADS) kv8_select_kernel(const Kv8EvictArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint64_t sh[33];
    __shared__ uint32_t s_prefix, s_need;
    const int64_t bh = blockIdx.x, b = bh / a.src.Hkv;
    const int64_t len = clamp64(a.src.lens[b], 0, a.src.Smax);
    const int64_t newlen = min(len, a.budget);
    int32_t* kept = a.kept + bh * a.budget;
    const float* score = a.score + bh * a.src.Smax;
    for (int64_t j = newlen + threadIdx.x; j < a.budget; j += blockDim.x) kept[j] = -1;
    if (bh - b * a.src.Hkv == 0 && threadIdx.x == 0) a.dst.lens[b] = (int32_t)newlen;
    if (len <= a.budget) {
        for (int64_t j = threadIdx.x; j < len; j += blockDim.x) kept[j] = (int32_t)j;
        return;
    }
    const int64_t n = len - a.recent, k = a.budget - a.recent;  // n > k
    for (int64_t j = threadIdx.x; j < a.recent; j += blockDim.x) kept[k + j] = (int32_t)(n + j);
    if (k == 0) return;
    uint32_t prefix = 0, need = (uint32_t)k;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t key = score_key(score[i]);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t left = need;
            int d = 255;
            for (; d > 0 && hist[d] < left; --d) left -= hist[d];
            s_prefix = prefix | ((uint32_t)d << shift);
            s_need = left;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }
    uint64_t base = 0;  // (larger << 32 | equal) keys before this sweep's rows
    for (int64_t i0 = 0; i0 < n; i0 += blockDim.x) {
        const int64_t i = i0 + threadIdx.x;
        const uint32_t key = i < n ? score_key(score[i]) : 0u;
        const bool gt = i < n && key > prefix, eq = i < n && key == prefix;
        uint64_t total;
        const uint64_t at = base + block_scan(((uint64_t)gt << 32) | (uint64_t)eq, sh, total);
        const uint32_t before_gt = (uint32_t)(at >> 32), before_eq = (uint32_t)at;
        if (gt || (eq && before_eq < need)) kept[before_gt + min(before_eq, need)] = (int32_t)i;
        base += total;
    }
}

// One CTA per (destination block, sequence x kv head, K or V): the kept rows' values, their largest, the
// new scale, the new codes
template <int FMT>
__global__ void kv8_gather_kernel(const Kv8EvictArgs a) {
    __shared__ float red[32];
    const int64_t bh = blockIdx.y, j = blockIdx.x;
    const bool is_v = blockIdx.z != 0;
    const int64_t T_ = a.src.block, Td = a.dst.block, D = a.src.D;
    const int64_t newlen = a.dst.lens[bh / a.src.Hkv];
    const int64_t r0 = j * Td, r1 = min(r0 + Td, newlen);
    if (!is_v && a.score_out)
        for (int64_t r = r0 + threadIdx.x; r < min(r0 + Td, a.dst.Smax); r += blockDim.x)
            a.score_out[bh * a.dst.Smax + r] = r < newlen ? a.score[bh * a.src.Smax + a.kept[bh * a.budget + r]] : 0.0f;
    if (r0 >= r1) return;
    const uint8_t* src = (const uint8_t*)(is_v ? a.src.v : a.src.k) + bh * a.src.Smax * D;
    const float* sscale = (is_v ? a.src.v_scale : a.src.k_scale) + bh * ((a.src.Smax + T_ - 1) / T_);
    uint8_t* dst = (uint8_t*)(is_v ? a.dst.v : a.dst.k) + (bh * a.dst.Smax + r0) * D;
    const int32_t* kept = a.kept + bh * a.budget + r0;
    const int64_t n = (r1 - r0) * D;
    float m = 0.0f;
    for (int64_t e = threadIdx.x; e < n; e += blockDim.x) {
        const int64_t r = e / D, s = kept[r];
        m = fmaxf(m, finite_abs(__fmul_rn(Code8<FMT>::value(src[s * D + e - r * D]), sscale[s / T_])));
    }
    const float sc = scale_of<FMT>(block_max(m, red));
    for (int64_t e = threadIdx.x; e < n; e += blockDim.x) {
        const int64_t r = e / D, s = kept[r];
        dst[e] = quantise8<FMT>(__fmul_rn(Code8<FMT>::value(src[s * D + e - r * D]), sscale[s / T_]), sc);
    }
    if (threadIdx.x == 0) (is_v ? a.dst.v_scale : a.dst.k_scale)[bh * ((a.dst.Smax + Td - 1) / Td) + j] = sc;
}

template <int FMT>
int append_fmt(const Kv8AppendArgs& a, cudaStream_t st) {
    const int64_t nblk = (a.n + a.c.block - 2) / a.c.block + 1;
    const dim3 grid((unsigned)nblk, (unsigned)(a.c.B * a.c.Hkv), 2);
    switch (a.dtype) {
        case F32: kv8_append_kernel<float, FMT><<<grid, 128, 0, st>>>(a); break;
        case F16: kv8_append_kernel<__half, FMT><<<grid, 128, 0, st>>>(a); break;
        default: kv8_append_kernel<__nv_bfloat16, FMT><<<grid, 128, 0, st>>>(a); break;
    }
    return cuda_failed(cudaGetLastError(), "kv8_append launch") ? -1 : 0;
}

template <int FMT>
int read_fmt(const Kv8ReadArgs& a, cudaStream_t st) {
    const int64_t n = 2 * a.c.B * a.c.Hkv * a.n * a.c.D;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 16);
    switch (a.dtype) {
        case F32: kv8_read_kernel<float, FMT><<<grid, 256, 0, st>>>(a); break;
        case F16: kv8_read_kernel<__half, FMT><<<grid, 256, 0, st>>>(a); break;
        default: kv8_read_kernel<__nv_bfloat16, FMT><<<grid, 256, 0, st>>>(a); break;
    }
    return cuda_failed(cudaGetLastError(), "kv8_read launch") ? -1 : 0;
}

}  // namespace

int launch_kv8_append(const Kv8AppendArgs& a, cudaStream_t st) {
    const int rc = a.c.format == GTB_KV8_INT8 ? append_fmt<GTB_KV8_INT8>(a, st) : append_fmt<GTB_KV8_E4M3>(a, st);
    if (rc || !a.advance) return rc;
    kv8_advance_kernel<<<(unsigned)((a.c.B + 127) / 128), 128, 0, st>>>(a);
    return cuda_failed(cudaGetLastError(), "kv8_append: advance launch") ? -1 : 0;
}

int launch_kv8_read(const Kv8ReadArgs& a, cudaStream_t st) {
    return a.c.format == GTB_KV8_INT8 ? read_fmt<GTB_KV8_INT8>(a, st) : read_fmt<GTB_KV8_E4M3>(a, st);
}

int launch_kv8_evict(const Kv8EvictArgs& a, cudaStream_t st) {
    const unsigned bh = (unsigned)(a.src.B * a.src.Hkv);
    kv8_select_kernel<<<bh, SEL_THREADS, 0, st>>>(a);
    if (cuda_failed(cudaGetLastError(), "kv8_evict: select launch")) return -1;
    // score_out covers dst.Smax rows, the codes only the budget
    const int64_t rows = a.score_out ? a.dst.Smax : a.budget;
    const dim3 grid((unsigned)((rows + a.dst.block - 1) / a.dst.block), bh, 2);
    if (a.src.format == GTB_KV8_INT8) kv8_gather_kernel<GTB_KV8_INT8><<<grid, 128, 0, st>>>(a);
    else kv8_gather_kernel<GTB_KV8_E4M3><<<grid, 128, 0, st>>>(a);
    return cuda_failed(cudaGetLastError(), "kv8_evict: gather launch") ? -1 : 0;
}

}  // namespace gtb
