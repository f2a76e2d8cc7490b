// Expanded latent attention backward on tcgen05. With w = exp(score - lse) recomputed tile by tile and
// ds = w (g . v - g . out):   dv = w^T g,   [dk | dk_r] = scale ds^T [q_n | q_r],   dq = scale ds [k | k_r].
//
//   pre     a query row: -g . out and -lse log2 e (-inf for padded rows and rows that attend nothing: weights 0).
//   dK/dV   one CTA a 128-key tile of one (batch, kv head), over its query heads' rows, 64 at a time:
//             S^T = [K | K_r] Q^T, dP^T = V G^T        (M = 128 keys, N = 64 queries)
//             dV += W^T G, dK += dS^T Q                (M = 128 keys, N = dims, K = 64; W^T from TMEM, dS^T from shared memory)
//           The rotary part of dK is the sum over all heads: each CTA writes its share in f32 and a last kernel adds the
//           heads in order, so the bits are the same on every run.
//   dQ      one CTA a 128-query tile, over 128 keys at a time:
//             S = Q [K | K_r]^T, dP = G V^T            (M = 128 queries, N = 128 keys)
//             dQ += dS [K | K_r]                       (N = dims, K = 128; dS from TMEM)
// A fused dQ (five products instead of seven) needs f32 sums over the key tiles in global memory, added without an order or waiting for
// one another, and with Dn = 128 TMEM that dK's 192 columns do not leave (with Dn = 64 there would be room: not built). Products of N = 64 with both operands in shared memory are bound by its bandwidth (49.5 cycles instead of 32):
// 64 is what TMEM holds of scores next to dV and dK (320 of 512 columns with Dn = 128). Beside dQ alone 128 fit.
//
// Warps: 0 TMA producer, 1 issues the score products (and owns TMEM), 2 the gradient products, 3 (dK/dV) zeroes rows of padded tokens
// in a loaded stage (their product with a weight of 0 would be NaN), 4-7 and 8-11 the weights: in the dK/dV kernel of even
// and odd sub-tiles, a key a thread; in the dQ kernel of a tile's two halves, a query a thread. TMEM of the dK/dV kernel with
// Dn = 128: dV 128 columns, dK 192, two S^T of 64 (over which W^T is written), one dP^T; of the dQ kernel: dQ 192, dS 64, S 128,
// dP 128. The dK/dV kernel streams through three stages of 64 rows: what a stage waits for (its load, the scores, the
// weights, the gradients) is about three times what the tensor core does on it. The dQ kernel has two key tiles and one
// value tile, which is free again as soon as dP is formed. Every mbarrier wait is bounded.
//
// Both kinds of CTA are one launch.
//
// Measured apart, 2 x 4096 tokens, 16 heads of 128 + 64, causal, bf16: dK/dV 398 us, dQ 281 us (292 over 64 keys at a time).

#include <algorithm>
#include <atomic>

#include "gtb_common.cuh"
#include "latent.h"
#include "latent_mma.cuh"
#include "sdpa_args.h"

namespace gtb {
namespace {

using namespace sm100;

constexpr int BT = 128, SUB = 64;
constexpr int NTHREADS = 384;
constexpr int SB_UNITS = 4;  // (batch, head) units whose CTAs run together, heaviest tiles first, sharing their streams in L2
constexpr uint32_t TMEM_COLS = 512;
constexpr int SMEM_MAX = 232448;
constexpr float LOG2E = 1.4426950408889634f;

struct Rows {
    char* p;
    int64_t s0, s1, s2;  // strides of batch, head, token (elements of 16 bits)
    __device__ __forceinline__ uint16_t* at(int b, int h, int64_t i) const { return (uint16_t*)p + b * s0 + h * s1 + i * s2; }
};

struct Params {
    int64_t L, S, Lpad;      // Lpad: L to a multiple of 64
    int B, H, Hkv, group, Dr, rope_steps;
    int ctas_kv;             // CTAs of dK/dV, before those of dQ
    float scale, scale_log2;
    int causal;
    const int32_t* lens;
    const float* lse;
    float *nlse2, *ndelta;   // (B, H, Lpad)
    float* dkr_part;         // (B, Hkv, S, Dr)
    Rows o, g, dq, dk, dv, dkr;
    int* status;
};

// ------------------------------------------------------------------ pre

template <int DN, bool BF16>
__global__ void __launch_bounds__(256) latent_bwd_pre_kernel(const __grid_constant__ Params p) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr int LANES = DN / 8, RPW = 32 / LANES, FLIGHT = 2;  // lanes a row, rows a warp at a time, loads in flight
    const int lane = threadIdx.x & 31, sub = lane / LANES, c = lane % LANES;
    const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * (RPW * FLIGHT), n = (int64_t)p.B * p.H * p.Lpad;
    uint4 ov[FLIGHT], gv[FLIGHT];
    int64_t row[FLIGHT];
    bool live[FLIGHT];
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
        row[f] = row0 + f * RPW + sub;
        ov[f] = gv[f] = make_uint4(0, 0, 0, 0);
        live[f] = false;
        if (row[f] >= n) continue;
        const int64_t bh = row[f] / p.Lpad, l = row[f] - bh * p.Lpad;
        const int b = (int)(bh / p.H), h = (int)(bh - (int64_t)b * p.H);
        live[f] = l < latent_tokens(p.lens, b, p.L);
        if (!live[f]) continue;
        ov[f] = *(const uint4*)(p.o.at(b, h, l) + c * 8);
        gv[f] = *(const uint4*)(p.g.at(b, h, l) + c * 8);
    }
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
        const T *x = (const T*)&ov[f], *y = (const T*)&gv[f];
        float acc = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc = fmaf(Elem<T>::load(x + e), Elem<T>::load(y + e), acc);
#pragma unroll
        for (int s = LANES / 2; s; s >>= 1) acc += __shfl_xor_sync(~0u, acc, s);
        if (c == 0 && row[f] < n) {
            const int64_t bh = row[f] / p.Lpad, l = row[f] - bh * p.Lpad;
            const float lse = live[f] ? p.lse[bh * p.L + l] : -INFINITY;
            p.nlse2[row[f]] = lse == -INFINITY ? -INFINITY : -lse * LOG2E;
            p.ndelta[row[f]] = -acc;
        }
    }
}

// the heads' shares of the rotary keys' gradient, added in order: 4 values a thread
template <bool BF16>
__global__ void __launch_bounds__(256) latent_bwd_rope_kernel(const __grid_constant__ Params p) {
    const int per = p.Dr / 4;
    const int64_t n = (int64_t)p.B * p.S * per, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += step) {
        const int64_t bs = e / per, b = bs / p.S, s = bs - b * p.S;
        const int c = (int)(e - bs * per);
        float4 a = make_float4(0, 0, 0, 0);
        const float* x = p.dkr_part + (b * p.Hkv * p.S + s) * p.Dr + 4 * c;
#pragma unroll 8
        for (int h = 0; h < p.Hkv; ++h) {
            const float4 y = *(const float4*)(x + (int64_t)h * p.S * p.Dr);
            a.x += y.x;
            a.y += y.y;
            a.z += y.z;
            a.w += y.w;
        }
        *(uint2*)(p.dkr.at((int)b, 0, s) + 4 * c) = make_uint2(pack2<BF16>(a.x, a.y), pack2<BF16>(a.z, a.w));
    }
}

// ------------------------------------------------------------------ shared by both kernels

// tile and (batch, head) unit of this CTA: superblocks of SB_UNITS units, their tiles outer, the units inner
__device__ __forceinline__ void place(int lin, int tiles, int units, int& tile, int& unit) {
    const int per = SB_UNITS * tiles, sb = lin / per, r = lin - sb * per;
    const int size = min(SB_UNITS, units - sb * SB_UNITS);
    tile = r / size;
    unit = sb * SB_UNITS + r - tile * size;
}

// 16 accumulator columns of one row, times mul, as 16-bit values
template <bool BF16>
__device__ __forceinline__ void store_row16(uint16_t* dst, const uint32_t* v, float mul) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 16; i += 2) w[i / 2] = pack2<BF16>(__uint_as_float(v[i]) * mul, __uint_as_float(v[i + 1]) * mul);
    ((uint4*)dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    ((uint4*)dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// rows [first, 64) of n 64-column slabs of 64 rows become zeros, by one warp
__device__ __forceinline__ void zero_rows(unsigned char* base, int n, int first, int lane) {
    const int per = (SUB - first) * 8;
    for (int e = lane; e < per * n; e += 32) {
        const int a = e / per;
        *(uint4*)(base + a * (SUB * 128) + first * 128 + (e - a * per) * 16) = make_uint4(0, 0, 0, 0);
    }
}

template <int DN>
struct Sizes {
    static constexpr int PANELS = DN / 64 + 1;
    static constexpr int SLAB = BT * 128, SLAB64 = SUB * 128;     // a 64-column slab of 128 and of 64 rows
    static constexpr int KTILE = PANELS * SLAB, VTILE = (DN / 64) * SLAB;
    static constexpr int STAGE = (2 * PANELS - 1) * SLAB64;        // 64 rows of Q and G, or of K and V
};

// ------------------------------------------------------------------ dK, dV

constexpr int STAGES = 3;

template <int DN>
struct KvSmem {
    using Z = Sizes<DN>;
    static constexpr int OFF_V = Z::KTILE, OFF_ST = OFF_V + Z::VTILE;
    static constexpr int OFF_DS = OFF_ST + STAGES * Z::STAGE;
    static constexpr int OFF_ROW = OFF_DS + BT * SUB * 2;          // [stage][-lse2, -delta][64]
    static constexpr int OFF_BAR = OFF_ROW + STAGES * 2 * SUB * 4;
    static constexpr int USED = OFF_BAR + 256;
    static constexpr int ALLOC = USED + 1023;
    static_assert(ALLOC <= SMEM_MAX, "shared memory");
};

struct KvBars {
    uint64_t kv_full, st_full[STAGES], st_empty[STAGES], fix[STAGES], fixed[STAGES], s_full[2], dp_full, dp_free, w_full[2], w_free[2], ds_free;
    uint64_t final_, drain[2];
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(KvBars) <= 256, "barrier block");

template <int DN, bool BF16>
__device__ __forceinline__ void kv_cta(const CUtensorMap& tmQ, const CUtensorMap& tmG, const CUtensorMap& tmK, const CUtensorMap& tmR,
                                       const CUtensorMap& tmV, const Params& p, int lin) {
    using Z = Sizes<DN>;
    using M = KvSmem<DN>;
    constexpr uint32_t DK_COL = DN, S_COL = 320, S_STEP = 128, DP_COL = 384;  // S^T of sub-tile h at S_COL + 128 h, then W^T
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    KvBars& bar = *(KvBars*)(smem + M::OFF_BAR);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int jt, unit;
    place(lin, (int)((p.S + BT - 1) / BT), p.B * p.Hkv, jt, unit);
    const int b = unit / p.Hkv, hk = unit - b * p.Hkv, key0 = jt * BT;
    const int nL = latent_tokens(p.lens, b, p.L), nS = latent_tokens(p.lens, b, p.S);
    const int i0 = p.causal ? key0 / SUB : 0;  // first sub-tile with a query that sees this key tile
    const int nq = max(0, (nL + SUB - 1) / SUB - i0), nit = key0 < nS ? p.group * nq : 0;

    if (threadIdx.x == 0) {
        mbar_init(&bar.kv_full, 1);
        mbar_init(&bar.final_, 1);
        mbar_init(&bar.dp_full, 1);
        mbar_init(&bar.dp_free, 4);
        mbar_init(&bar.ds_free, 1);
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&bar.st_full[i], 1);
            mbar_init(&bar.st_empty[i], 1);
            mbar_init(&bar.fix[i], 1);
            mbar_init(&bar.fixed[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.w_full[i], 4);
            mbar_init(&bar.w_free[i], 1);
            mbar_init(&bar.drain[i], 1);
        }
        bar.abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&bar.tmem, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    volatile int* abort_flag = &bar.abort;
    // sub-tile `it`: its query head and first query
    auto head_of = [&](int it) { return hk * p.group + it / nq; };
    auto first_of = [&](int it) { return (i0 + it % nq) * SUB; };
    auto padded = [&](int it) { return p.lens && first_of(it) + SUB > nL; };

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0 && nit > 0) {
            prefetch_tmap(&tmQ);
            prefetch_tmap(&tmG);
            mbar_expect_tx(&bar.kv_full, Z::KTILE + Z::VTILE);
            for (int a = 0; a < DN / 64; ++a) {
                tma_load_4d(smem + a * Z::SLAB, &tmK, a * 64, key0, hk, b, &bar.kv_full);
                tma_load_4d(smem + M::OFF_V + a * Z::SLAB, &tmV, a * 64, key0, hk, b, &bar.kv_full);
            }
            tma_load_4d(smem + (DN / 64) * Z::SLAB, &tmR, 0, key0, 0, b, &bar.kv_full);
            bool ok = true;
            int it = 0;
            for (; it < nit; ++it) {
                const int st = it % STAGES, h = head_of(it), q = first_of(it);
                if (it >= STAGES) ok = mbar_wait(&bar.st_empty[st], (it / STAGES - 1) & 1, p.status, 101);
                if (!ok || *abort_flag) { ok = false; break; }
                unsigned char* d = smem + M::OFF_ST + st * Z::STAGE;
                mbar_expect_tx(&bar.st_full[st], Z::STAGE + 2 * SUB * 4);
                for (int a = 0; a < Z::PANELS; ++a) tma_load_4d(d + a * Z::SLAB64, &tmQ, a * 64, q, h, b, &bar.st_full[st]);
                for (int a = 0; a < DN / 64; ++a) tma_load_4d(d + (Z::PANELS + a) * Z::SLAB64, &tmG, a * 64, q, h, b, &bar.st_full[st]);
                const int64_t r = ((int64_t)b * p.H + h) * p.Lpad + q;
                bulk_load(smem + M::OFF_ROW + st * 512, p.nlse2 + r, 256, &bar.st_full[st]);
                bulk_load(smem + M::OFF_ROW + st * 512 + 256, p.ndelta + r, 256, &bar.st_full[st]);
            }
            if (!ok) *abort_flag = 1;
            if (*abort_flag) {  // our copies in flight end before the CTA does
                mbar_wait(&bar.kv_full, 0, nullptr, 0);
                for (int n = max(0, it - STAGES); n < it; ++n) mbar_wait(&bar.st_full[n % STAGES], (n / STAGES) & 1, nullptr, 0);
            }
        }
    } else if (warp < 3) {
        // ------------------------------------------------------------ MMA issuers: 1 the scores, 2 the gradients
        const bool lead = elect_lane();
        const uint32_t tm = (uint32_t)uniform((int)tmem);
        const int n_it = uniform(nit);
        bool ok = true;
        if (warp == 1) {
            constexpr uint32_t IDESC = idesc_f16(BT, SUB, BF16, false);
            const uint32_t kd = desc_lo(smem_u32(smem), 16), vd = desc_lo(smem_u32(smem + M::OFF_V), 16);
            const uint32_t sd = desc_lo(smem_u32(smem + M::OFF_ST), 16);
            if (n_it > 0) ok = warp_wait(&bar.kv_full, 0, p.status, 102);
            int st = 0, phase = 0, n_fix = 0;  // stage and its phase; which stages' next mended round is odd
            for (int it = 0; it < n_it && ok; ++it) {
                const int h = it & 1;
                ok = warp_wait(&bar.st_full[st], phase, p.status, 103);
                if (ok && padded(it)) {
                    if (lead) mbar_arrive(&bar.fix[st]);
                    ok = warp_wait(&bar.fixed[st], (n_fix >> st) & 1, p.status, 104);
                    n_fix ^= 1 << st;
                }
                // S^T's columns hold the W^T that the product two sub-tiles ago read
                if (ok && it >= 2) ok = warp_wait(&bar.w_free[h], ((it >> 1) - 1) & 1, p.status, 105);
                if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t q = (uint32_t)uniform((int)(sd + st * (Z::STAGE >> 4))), g = q + (Z::PANELS * Z::SLAB64 >> 4);
                const uint32_t s_dst = tm + S_COL + h * S_STEP, dp_dst = tm + DP_COL;
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < DN / 16; ++kk)
                        mma_ss_lo(s_dst, kd + (kk / 4) * (Z::SLAB >> 4) + (kk % 4) * 2, q + (kk / 4) * (Z::SLAB64 >> 4) + (kk % 4) * 2, IDESC, kk > 0);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        if (kk < p.rope_steps)
                            mma_ss_lo(s_dst, kd + (DN / 64) * (Z::SLAB >> 4) + kk * 2, q + (DN / 64) * (Z::SLAB64 >> 4) + kk * 2, IDESC, 1);
                    mma_commit(&bar.s_full[h]);
                }
                if (it >= 1) ok = warp_wait(&bar.dp_free, (it - 1) & 1, p.status, 113);
                if (!ok) break;
                tc_fence_after();
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < DN / 16; ++kk)
                        mma_ss_lo(dp_dst, vd + (kk / 4) * (Z::SLAB >> 4) + (kk % 4) * 2, g + (kk / 4) * (Z::SLAB64 >> 4) + (kk % 4) * 2, IDESC, kk > 0);
                    mma_commit(&bar.dp_full);
                }
                if (++st == STAGES) st = 0, phase ^= 1;
            }
        } else {
            const uint32_t idesc_k = idesc_f16(BT, 0, BF16, true) | (uint32_t)(DN + 16 * p.rope_steps) >> 3 << 17;
            constexpr uint32_t IDESC_V = idesc_f16(BT, DN, BF16, true);
            const uint32_t ds = desc_lo(smem_u32(smem + M::OFF_DS), 16), sd = desc_lo(smem_u32(smem + M::OFF_ST), Z::SLAB64);
            int st = 0;
            for (int it = 0; it < n_it && ok; ++it) {
                const int h = it & 1;
                ok = warp_wait(&bar.w_full[h], (it >> 1) & 1, p.status, 106);
                if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t q = (uint32_t)uniform((int)(sd + st * (Z::STAGE >> 4))), g = q + (Z::PANELS * Z::SLAB64 >> 4);
                const uint32_t w = tm + S_COL + h * S_STEP;
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < SUB / 16; ++kk) mma_ss_lo(tm + DK_COL, ds + kk * 2, q + kk * 128, idesc_k, it > 0 || kk > 0);
                    mma_commit(&bar.ds_free);
#pragma unroll
                    for (int kk = 0; kk < SUB / 16; ++kk) mma_ts_lo(tm, w + kk * 8, g + kk * 128, IDESC_V, it > 0 || kk > 0);
                    mma_commit(&bar.w_free[h]);
                    mma_commit(&bar.st_empty[st]);
                    if (it + 1 == n_it) mma_commit(&bar.final_);
                }
                if (++st == STAGES) st = 0;
            }
        }
        if (!ok) *abort_flag = 1;
        __syncwarp();
        if (__any_sync(~0u, *abort_flag)) {
            if (lead) mma_commit(&bar.drain[warp - 1]);
            warp_wait(&bar.drain[warp - 1], 0, nullptr, 0);
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------ rows of padded tokens become zeros
        bool ok = true;
        int n_fix = 0;
        for (int it = 0; it < nit && ok; ++it) {
            if (!padded(it)) continue;
            const int st = it % STAGES;
            ok = warp_wait(&bar.fix[st], (n_fix >> st) & 1, p.status, 107);
            if (!ok) break;
            n_fix ^= 1 << st;
            zero_rows(smem + M::OFF_ST + st * Z::STAGE, 2 * Z::PANELS - 1, max(0, nL - first_of(it)), lane);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.fixed[st]);
        }
        if (!ok) *abort_flag = 1;
    } else {
        // ------------------------------------------------------------ weights: warpgroup wg takes the sub-tiles it % 2 == wg
        const int wg = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane, key = key0 + r;
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        unsigned char* ds_row = smem + M::OFF_DS + r * 128;
        const uint32_t s_tmem = tmem + lane_addr + S_COL + wg * S_STEP, dp_tmem = tmem + lane_addr + DP_COL;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
        bool ok = true;
        for (int it = wg; it < nit; it += 2) {
            const int st = it % STAGES, q0 = first_of(it);
            const float* nl = (const float*)(smem + M::OFF_ROW + st * 512);  // the queries' -lse2, and 64 further on their -delta
            ok = warp_wait(&bar.s_full[wg], (it >> 1) & 1, p.status, 109);
            if (ok) ok = warp_wait(&bar.st_full[st], (it / STAGES) & 1, p.status, 108);  // (complete: this makes its rows visible)
            if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
            tc_fence_after();
            uint32_t ra[64], rb[64];
            tmem_ld32(s_tmem, ra);
            tmem_ld32(s_tmem + 32, ra + 32);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < SUB; i += 2) {
                float a0, a1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(ra[i]), __uint_as_float(ra[i + 1])), sc2, *(const uint64_t*)(nl + i)), a0, a1);
                ra[i] = __float_as_uint(ex2(a0));
                ra[i + 1] = __float_as_uint(ex2(a1));
            }
            if (p.causal && q0 < key0 + BT - 1) {
#pragma unroll
                for (int i = 0; i < SUB; ++i)
                    if (key > q0 + i) ra[i] = 0u;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // W^T over S^T, already read: queries 16 bits each, two a column
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = pack2<BF16>(__uint_as_float(ra[32 * c + 2 * i]), __uint_as_float(ra[32 * c + 2 * i + 1]));
                tmem_st16(s_tmem + 16 * c, w);
            }
            ok = warp_wait(&bar.dp_full, it & 1, p.status, 110);
            if (!ok) break;
            tc_fence_after();
            tmem_ld32(dp_tmem, rb);
            tmem_ld32(dp_tmem + 32, rb + 32);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.dp_free);
            if (it >= 1) ok = warp_wait(&bar.ds_free, (it - 1) & 1, p.status, 111);  // dK has read the last sub-tile's dS^T
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // 16 bytes of dS^T: 8 queries
                uint32_t dv[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * j + 2 * e;
                    float d0, d1;
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(ra[i]), __uint_as_float(ra[i + 1])),
                                     f2_add(f2_pack(__uint_as_float(rb[i]), __uint_as_float(rb[i + 1])), *(const uint64_t*)(nl + SUB + i))), d0, d1);
                    dv[e] = pack2<BF16>(d0, d1);
                }
                *(uint4*)(ds_row + ((j ^ (r & 7)) << 4)) = make_uint4(dv[0], dv[1], dv[2], dv[3]);
            }
            tmem_st_wait();
            fence_proxy_async_smem();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.w_full[wg]);
        }
        if (nit > 0 && ok) ok = warp_wait(&bar.final_, 0, p.status, 112);
        if (!ok) *abort_flag = 1;
        if (ok && !__any_sync(~0u, *abort_flag)) {
            tc_fence_after();
            const bool live = nit > 0 && key < nS;  // others: no query sees the key, or it is a padded one
            constexpr int PARTS = 2 * DN / 16;       // 16-column parts of dV and dK; the rotary ones behind them
            const int parts = PARTS + p.Dr / 16;
            for (int c = wg; c < parts; c += 2) {
                uint32_t v[16];
                tmem_ldx<16>(tmem + lane_addr + c * 16, v);
                tmem_ld_wait();
                if (!live) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = 0u;
                }
                if (key >= p.S) {
                } else if (c < DN / 16) {
                    store_row16<BF16>(p.dv.at(b, hk, key) + c * 16, v, 1.0f);
                } else if (c < PARTS) {
                    store_row16<BF16>(p.dk.at(b, hk, key) + c * 16 - DN, v, p.scale);
                } else {
                    float4* d = (float4*)(p.dkr_part + (((int64_t)b * p.Hkv + hk) * p.S + key) * p.Dr + (c - PARTS) * 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        d[i] = make_float4(__uint_as_float(v[4 * i]) * p.scale, __uint_as_float(v[4 * i + 1]) * p.scale,
                                           __uint_as_float(v[4 * i + 2]) * p.scale, __uint_as_float(v[4 * i + 3]) * p.scale);
                }
                __syncwarp();
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// ------------------------------------------------------------------ dQ

template <int DN>
struct QSmem {
    using Z = Sizes<DN>;
    static constexpr int OFF_G = Z::KTILE, OFF_K = OFF_G + Z::VTILE, OFF_V = OFF_K + 2 * Z::KTILE;
    static constexpr int OFF_BAR = OFF_V + Z::VTILE;
    static constexpr int USED = OFF_BAR + 256;
    static constexpr int ALLOC = USED + 1023;
    static_assert(ALLOC <= SMEM_MAX, "shared memory");
};

struct QBars {
    uint64_t q_full, k_full[2], k_empty[2], v_full, v_empty, s_full, s_free, dp_full, dp_free, ds_full, ds_free, final_, drain[2];
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(QBars) <= 256, "barrier block");

template <int DN, bool BF16>
__device__ __forceinline__ void q_cta(const CUtensorMap& tmQ, const CUtensorMap& tmG, const CUtensorMap& tmK, const CUtensorMap& tmR,
                                      const CUtensorMap& tmV, const Params& p, int lin) {
    using Z = Sizes<DN>;
    using M = QSmem<DN>;
    constexpr uint32_t DS_COL = 192, S_COL = 256, DP_COL = 384;  // dQ from 0; dS as 16-bit pairs
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    QBars& bar = *(QBars*)(smem + M::OFF_BAR);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int tile, unit;
    const int n_qt = (int)((p.L + BT - 1) / BT);
    place(lin, n_qt, p.B * p.H, tile, unit);
    if (p.causal) tile = n_qt - 1 - tile;
    const int b = unit / p.H, h = unit - b * p.H, hk = h / p.group, row0 = tile * BT;
    const int nL = latent_tokens(p.lens, b, p.L), nS = latent_tokens(p.lens, b, p.S);
    const int all = (nS + BT - 1) / BT;
    const int nit = row0 >= nL ? 0 : p.causal ? min(all, (min(row0 + BT, nL) - 1) / BT + 1) : all;

    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 1);
        mbar_init(&bar.v_full, 1);
        mbar_init(&bar.v_empty, 1);
        mbar_init(&bar.s_full, 1);
        mbar_init(&bar.s_free, 8);
        mbar_init(&bar.dp_full, 1);
        mbar_init(&bar.dp_free, 8);
        mbar_init(&bar.ds_full, 8);
        mbar_init(&bar.ds_free, 1);
        mbar_init(&bar.final_, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.k_full[i], 1);
            mbar_init(&bar.k_empty[i], 1);
            mbar_init(&bar.drain[i], 1);
        }
        bar.abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&bar.tmem, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    volatile int* abort_flag = &bar.abort;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0 && nit > 0) {
            prefetch_tmap(&tmK);
            prefetch_tmap(&tmR);
            prefetch_tmap(&tmV);
            mbar_expect_tx(&bar.q_full, Z::KTILE + Z::VTILE);
            for (int a = 0; a < Z::PANELS; ++a) tma_load_4d(smem + a * Z::SLAB, &tmQ, a * 64, row0, h, b, &bar.q_full);
            for (int a = 0; a < DN / 64; ++a) tma_load_4d(smem + M::OFF_G + a * Z::SLAB, &tmG, a * 64, row0, h, b, &bar.q_full);
            bool ok = true;
            int nk = 0, nv = 0;
            for (int it = 0; it < nit; ++it) {
                const int st = it & 1;
                if (it >= 2) ok = mbar_wait(&bar.k_empty[st], ((it >> 1) - 1) & 1, p.status, 121);
                if (!ok || *abort_flag) { ok = false; break; }
                unsigned char* d = smem + M::OFF_K + st * Z::KTILE;
                mbar_expect_tx(&bar.k_full[st], Z::KTILE);
                for (int a = 0; a < DN / 64; ++a) tma_load_4d(d + a * Z::SLAB, &tmK, a * 64, it * BT, hk, b, &bar.k_full[st]);
                tma_load_4d(d + (DN / 64) * Z::SLAB, &tmR, 0, it * BT, 0, b, &bar.k_full[st]);
                ++nk;
                if (it >= 1) ok = mbar_wait(&bar.v_empty, (it - 1) & 1, p.status, 131);
                if (!ok || *abort_flag) { ok = false; break; }
                mbar_expect_tx(&bar.v_full, Z::VTILE);
                for (int a = 0; a < DN / 64; ++a) tma_load_4d(smem + M::OFF_V + a * Z::SLAB, &tmV, a * 64, it * BT, hk, b, &bar.v_full);
                ++nv;
            }
            if (!ok) *abort_flag = 1;
            if (*abort_flag) {
                mbar_wait(&bar.q_full, 0, nullptr, 0);
                for (int n = max(0, nk - 2); n < nk; ++n) mbar_wait(&bar.k_full[n & 1], (n >> 1) & 1, nullptr, 0);
                if (nv > 0) mbar_wait(&bar.v_full, (nv - 1) & 1, nullptr, 0);
            }
        }
    } else if (warp < 3) {
        // ------------------------------------------------------------ MMA issuers: 1 the scores, 2 dQ
        const bool lead = elect_lane();
        const uint32_t tm = (uint32_t)uniform((int)tmem);
        const int n_it = uniform(nit);
        bool ok = true;
        if (warp == 1) {
            constexpr uint32_t IDESC = idesc_f16(BT, BT, BF16, false);
            const uint32_t qd = desc_lo(smem_u32(smem), 16), gd = desc_lo(smem_u32(smem + M::OFF_G), 16);
            const uint32_t kd = desc_lo(smem_u32(smem + M::OFF_K), 16), vd = desc_lo(smem_u32(smem + M::OFF_V), 16);
            if (n_it > 0) ok = warp_wait(&bar.q_full, 0, p.status, 122);
            for (int it = 0; it < n_it && ok; ++it) {
                ok = warp_wait(&bar.k_full[it & 1], (it >> 1) & 1, p.status, 123);
                if (ok && it >= 1) ok = warp_wait(&bar.s_free, (it - 1) & 1, p.status, 125);
                if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t k = (uint32_t)uniform((int)(kd + (it & 1) * (Z::KTILE >> 4)));
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < DN / 16; ++kk) {
                        const uint32_t o = (kk / 4) * (Z::SLAB >> 4) + (kk % 4) * 2;
                        mma_ss_lo(tm + S_COL, qd + o, k + o, IDESC, kk > 0);
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint32_t o = (DN / 64) * (Z::SLAB >> 4) + kk * 2;
                        if (kk < p.rope_steps) mma_ss_lo(tm + S_COL, qd + o, k + o, IDESC, 1);
                    }
                    mma_commit(&bar.s_full);
                }
                ok = warp_wait(&bar.v_full, it & 1, p.status, 124);
                if (ok && it >= 1) ok = warp_wait(&bar.dp_free, (it - 1) & 1, p.status, 132);
                if (!ok) break;
                tc_fence_after();
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < DN / 16; ++kk) {
                        const uint32_t o = (kk / 4) * (Z::SLAB >> 4) + (kk % 4) * 2;
                        mma_ss_lo(tm + DP_COL, gd + o, vd + o, IDESC, kk > 0);
                    }
                    mma_commit(&bar.dp_full);
                    mma_commit(&bar.v_empty);
                }
            }
        } else {
            const uint32_t idesc = idesc_f16(BT, 0, BF16, true) | (uint32_t)(DN + 16 * p.rope_steps) >> 3 << 17;
            const uint32_t kd = desc_lo(smem_u32(smem + M::OFF_K), Z::SLAB);
            for (int it = 0; it < n_it && ok; ++it) {
                ok = warp_wait(&bar.ds_full, it & 1, p.status, 126);
                if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t k = (uint32_t)uniform((int)(kd + (it & 1) * (Z::KTILE >> 4)));
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < BT / 16; ++kk) mma_ts_lo(tm, tm + DS_COL + kk * 8, k + kk * 128, idesc, it > 0 || kk > 0);
                    mma_commit(&bar.ds_free);
                    mma_commit(&bar.k_empty[it & 1]);
                    if (it + 1 == n_it) mma_commit(&bar.final_);
                }
            }
        }
        if (!ok) *abort_flag = 1;
        __syncwarp();
        if (__any_sync(~0u, *abort_flag)) {
            if (lead) mma_commit(&bar.drain[warp - 1]);
            warp_wait(&bar.drain[warp - 1], 0, nullptr, 0);
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------ dS: warpgroup wg has keys 64 wg .. of every tile
        const int wg = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane, row = row0 + r;
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        const uint32_t s_tmem = tmem + lane_addr + S_COL + wg * SUB, p_tmem = tmem + lane_addr + DP_COL + wg * SUB;
        const uint32_t ds_tmem = tmem + lane_addr + DS_COL + wg * (SUB / 2);
        const int64_t rr = ((int64_t)b * p.H + h) * p.Lpad + row;
        const float nl = row < p.Lpad ? p.nlse2[rr] : -INFINITY, nd = row < p.Lpad ? p.ndelta[rr] : 0.0f;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nl2 = f2_pack(nl, nl), nd2 = f2_pack(nd, nd);
        const int lim = p.causal ? min(nS - 1, row) : nS - 1;  // last key this row sees
        bool ok = true;
        for (int it = 0; it < nit; ++it) {
            ok = warp_wait(&bar.s_full, it & 1, p.status, 128);
            if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
            tc_fence_after();
            const int kv0 = it * BT + wg * SUB;
            const bool mask = kv0 + SUB > nS || (p.causal && kv0 + SUB - 1 > row0);
            uint32_t ra[SUB], rb[SUB];
            tmem_ld32(s_tmem, ra);
            tmem_ld32(s_tmem + 32, ra + 32);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.s_free);
#pragma unroll
            for (int k = 0; k < SUB; k += 2) {
                float a0, a1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(ra[k]), __uint_as_float(ra[k + 1])), sc2, nl2), a0, a1);
                ra[k] = __float_as_uint(ex2(a0));
                ra[k + 1] = __float_as_uint(ex2(a1));
            }
            ok = warp_wait(&bar.dp_full, it & 1, p.status, 133);
            if (!ok) break;
            tc_fence_after();
            tmem_ld32(p_tmem, rb);
            tmem_ld32(p_tmem + 32, rb + 32);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.dp_free);
            uint32_t ds[SUB / 2];
#pragma unroll
            for (int k = 0; k < SUB; k += 2) {
                float d0, d1;
                f2_unpack(f2_mul(f2_pack(__uint_as_float(ra[k]), __uint_as_float(ra[k + 1])),
                                 f2_add(f2_pack(__uint_as_float(rb[k]), __uint_as_float(rb[k + 1])), nd2)), d0, d1);
                if (mask) {  // (whatever the product with a padded key's values gave)
                    if (kv0 + k > lim) d0 = 0.0f;
                    if (kv0 + k + 1 > lim) d1 = 0.0f;
                }
                ds[k / 2] = pack2<BF16>(d0, d1);
            }
            if (it >= 1) ok = warp_wait(&bar.ds_free, (it - 1) & 1, p.status, 130);  // dQ has read the tile's before
            if (!ok) break;
            tc_fence_after();
            tmem_st16(ds_tmem, ds);
            tmem_st16(ds_tmem + 16, ds + 16);
            if (p.lens && (it + 1) * BT > nS) {  // key rows of padded tokens: 0 in dQ's product, whatever they hold
                const int first = nS - it * BT, per = (BT - first) * 8;
                for (int e = (int)threadIdx.x - 128; e < per * Z::PANELS; e += 256) {
                    const int a = e / per;
                    *(uint4*)(smem + M::OFF_K + (it & 1) * Z::KTILE + a * Z::SLAB + first * 128 + (e - a * per) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.ds_full);
        }
        if (nit > 0 && ok) ok = warp_wait(&bar.final_, 0, p.status, 129);
        if (!ok) *abort_flag = 1;
        if (ok && !__any_sync(~0u, *abort_flag)) {
            tc_fence_after();
            const bool live = nit > 0 && row < nL;
            const int parts = (DN + p.Dr) / 16;
            for (int c = wg; c < parts; c += 2) {
                uint32_t v[16];
                tmem_ldx<16>(tmem + lane_addr + c * 16, v);
                tmem_ld_wait();
                if (!live) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = 0u;
                }
                if (row < p.L) store_row16<BF16>(p.dq.at(b, h, row) + c * 16, v, p.scale);
                __syncwarp();
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// The CTAs of dK/dV first, those of dQ behind them: neither waits for the other, and the second kind fills the multiprocessors as the
// first one's last CTAs end (2 x 4096, 16 heads: 831 -> 822 us with the forward; 3 x 511 to 1023, 12 heads of 64 + 32: 114 -> 104).
template <int DN, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1)
latent_bwd_kernel(const __grid_constant__ CUtensorMap q64, const __grid_constant__ CUtensorMap g64, const __grid_constant__ CUtensorMap q128,
                  const __grid_constant__ CUtensorMap g128, const __grid_constant__ CUtensorMap k128,
                  const __grid_constant__ CUtensorMap r128, const __grid_constant__ CUtensorMap v128, const __grid_constant__ Params p) {
    if ((int)blockIdx.x < p.ctas_kv) kv_cta<DN, BF16>(q64, g64, k128, r128, v128, p, (int)blockIdx.x);
    else q_cta<DN, BF16>(q128, g128, k128, r128, v128, p, (int)blockIdx.x - p.ctas_kv);
}

Rows rows(const gtb_tensor4& t) { return Rows{(char*)t.data, t.stride[0], t.stride[1], t.stride[2]}; }

template <int DN, bool BF16>
int launch(const LatentSdpaArgs& a, cudaStream_t st) {
    const char* ctx = "latent_sdpa_bwd";
    auto kern = latent_bwd_kernel<DN, BF16>;
    constexpr int SMEM = std::max(KvSmem<DN>::ALLOC, QSmem<DN>::ALLOC);
    int dev = 0;
    if (cuda_failed(cudaGetDevice(&dev), ctx)) return -1;
    static std::atomic<uint64_t> ready{0};  // devices (of the first 64) whose kernels are set up
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(ready.load() & bit)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM), ctx)) return -1;
        ready.fetch_or(bit);
    }
    const int64_t ctas_kv = (a.S + BT - 1) / BT * a.B * a.Hkv, ctas_q = (a.L + BT - 1) / BT * a.B * a.H;
    if (ctas_kv + ctas_q > INT32_MAX) {
        set_errorf("%s: too many tiles", ctx);
        return -1;
    }
    // 128-row maps, and of what streams by the dK/dV kernel 64-row ones
    CUtensorMap q128, q64, g128, g64, k128, r128, v128;
    if (!make_tma_map_4d(&q128, a.q, DN + a.Dr, BF16, BT) || !make_tma_map_4d(&q64, a.q, DN + a.Dr, BF16, SUB) ||
        !make_tma_map_4d(&g128, a.g, DN, BF16, BT) || !make_tma_map_4d(&g64, a.g, DN, BF16, SUB) ||
        !make_tma_map_4d(&k128, a.k, DN, BF16, BT) || !make_tma_map_4d(&r128, a.k_rope, a.Dr, BF16, BT) ||
        !make_tma_map_4d(&v128, a.v, DN, BF16, BT))
        return -1;
    Params p{};
    p.L = a.L;
    p.S = a.S;
    p.Lpad = (a.L + SUB - 1) / SUB * SUB;
    p.B = (int)a.B;
    p.H = (int)a.H;
    p.Hkv = (int)a.Hkv;
    p.group = (int)(a.H / a.Hkv);
    p.Dr = a.Dr;
    p.rope_steps = a.Dr / 16;
    p.scale = a.scale;
    p.scale_log2 = a.scale * LOG2E;
    p.causal = a.causal;
    p.ctas_kv = (int)ctas_kv;
    p.lens = a.lens;
    p.lse = a.lse;
    p.o = rows(a.o);
    p.g = rows(a.g);
    p.dq = rows(a.dq);
    p.dk = rows(a.dk);
    p.dv = rows(a.dv);
    p.dkr = rows(a.dk_rope);
    p.status = a.status;
    const int64_t n_row = a.B * a.H * p.Lpad, n_part = a.B * a.Hkv * a.S * a.Dr;
    float* ws = nullptr;
    if (cuda_failed(cudaMallocAsync((void**)&ws, (2 * n_row + n_part) * sizeof(float), st), "latent_sdpa_bwd: scratch")) return -1;
    p.nlse2 = ws;
    p.ndelta = ws + n_row;
    p.dkr_part = ws + 2 * n_row;
    constexpr int ROWS = 8 * (32 / (DN / 8)) * 2;  // rows a block of the first kernel
    latent_bwd_pre_kernel<DN, BF16><<<(unsigned)((n_row + ROWS - 1) / ROWS), 256, 0, st>>>(p);
    kern<<<(unsigned)(ctas_kv + ctas_q), NTHREADS, SMEM, st>>>(q64, g64, q128, g128, k128, r128, v128, p);
    latent_bwd_rope_kernel<BF16><<<(unsigned)std::min<int64_t>(4096, (a.B * a.S * (a.Dr / 4) + 255) / 256), 256, 0, st>>>(p);
    const int rc = cuda_failed(cudaGetLastError(), "latent_sdpa_bwd launch") ? -1 : 0;
    cudaFreeAsync(ws, st);
    return rc;
}

}  // namespace

int launch_latent_sdpa_bwd(const LatentSdpaArgs& a, cudaStream_t st) {
    const bool bf16 = a.q.dtype == BF16;
    if (a.Dn == 128) return bf16 ? launch<128, true>(a, st) : launch<128, false>(a, st);
    return bf16 ? launch<64, true>(a, st) : launch<64, false>(a, st);
}

}  // namespace gtb
