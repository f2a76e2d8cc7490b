// Expanded latent attention forward on tcgen05: keys of Dn values a head and Dr rotary values that all heads share.
//
// A score is one sum over Dn + Dr products, so a key tile in shared memory is the head's 64-column panels with the shared rotary
// panel (zeros behind Dr, from the load) as one more: the rotary keys are read once a head from L2 and never copied next to
// each head's. One CTA works on two 128-row query tiles of one (batch, head), which share every key and value tile:
//   S_t = Q_t [K | K_r]^T  (M = 128, N = 128, K = Dn + Dr, both operands in shared memory)
//   O_t += P_t V           (M = 128, N = Dn, K = 128; P_t from TMEM, over S_t's columns)
// in the order PV_0(j) S_0(j+1) PV_1(j) S_1(j+1), so that each softmax warpgroup works while the tensor core is on the other
// tile. TMEM: S_0 [0, 128), S_1 [128, 256), O_0 and O_1 from 256 and 384.
//
// With Dn = 128 two query tiles (96 KB) and two key tiles of 48 KB leave 32 KB for values: one tile in two halves of 64 keys, each
// loaded again as soon as the second query tile's product has gone through it, which is about the time of S_1 before it is needed.
//
// Warps: 0 TMA producer, 1 TMEM owner and MMA issuer, 2-3 zero the value rows of padded tokens (a weight of 0 would make NaN of what
// they may hold), 4-7 softmax and output of tile 0, 8-11 of tile 1: a query row a thread, offsets raised only past 2^8.
// CTAs are persistent and claim items from a counter, heaviest first. Every mbarrier wait is bounded.

#include <algorithm>
#include <atomic>

#include "gtb_common.cuh"
#include "latent.h"
#include "latent_mma.cuh"
#include "sdpa_args.h"

namespace gtb {
namespace {

using namespace sm100;

constexpr int BM = 128, BN = 128, HALF = 64;
constexpr int NTHREADS = 384;
constexpr int REG_LO = 104, REG_HI = 200;  // registers a thread of warps 0-3 and of the softmax warps
constexpr uint32_t TMEM_COLS = 512;
constexpr int SMEM_MAX = 232448;

template <int DN>
struct Cfg {
    static constexpr int PANELS = DN / 64 + 1;
    static constexpr int PANEL = 128 * 128;            // 128 rows x 64 columns
    static constexpr int TILE = PANELS * PANEL;        // a Q or K tile
    static constexpr int VHALF = HALF * DN * 2;        // 64 rows of V, in 64-column slabs
    static constexpr int VSLAB = HALF * 128;
    static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + 2 * TILE, OFF_BAR = OFF_V + 2 * VHALF;
    static constexpr int USED = OFF_BAR + 256;
    static constexpr int SMEM = USED + 1023 < SMEM_MAX ? USED + 1023 : SMEM_MAX;
    static constexpr int SLACK = SMEM - USED;
    static_assert(USED <= SMEM_MAX, "shared memory");
};

struct Bars {
    uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], fix[2], v_fixed[2], s_full[2], p_full[2], o_final[2], o_empty[2];
    uint64_t item_full[2], item_empty[2], drain;
    uint32_t tmem;
    int abort;
    int item[2];
};
static_assert(sizeof(Bars) <= 256, "barrier block");

struct Params {
    int64_t L, S;
    int B, H, group, n_pairs, n_items;
    int* claim;
    float scale_log2;
    int causal, rope_steps;
    const int32_t* lens;
    void* o;
    int64_t os0, os1, os2;
    float* lse;
    int* status;
};

struct Item {
    int b, h, row0, nL, nS;
    int nblk[2], n;  // key tiles of each query tile, of both
};

__device__ __forceinline__ Item item_of(const Params& p, int i) {
    Item it;
    const int hb = p.H * p.B, pr = i / hb, bh = i - pr * hb;
    const int pair = p.causal ? p.n_pairs - 1 - pr : pr;
    it.b = bh / p.H;
    it.h = bh - it.b * p.H;
    it.row0 = pair * 2 * BM;
    it.nL = latent_tokens(p.lens, it.b, p.L);
    it.nS = latent_tokens(p.lens, it.b, p.S);
    const int n_kv = (it.nS + BN - 1) / BN;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int r = it.row0 + t * BM;
        it.nblk[t] = r >= it.nL ? 0 : p.causal ? min(n_kv, (min(r + BM, it.nL) - 1) / BN + 1) : n_kv;
    }
    it.n = max(it.nblk[0], it.nblk[1]);
    return it;
}

// whether half v of value tile j has rows of padded tokens (those past S are zeros from the load)
__device__ __forceinline__ bool padded_half(const Params& p, int nS, int j, int v) {
    return p.lens && j * BN + (v + 1) * HALF > nS;
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int DN, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1)
latent_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmV, const Params p) {
    using C = Cfg<DN>;
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    if (smem - smem_raw > C::SLACK) {
        if (threadIdx.x == 0) atomicCAS(p.status, 0, 82);
        return;
    }
    Bars& bar = *(Bars*)(smem + C::OFF_BAR);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 1);
        mbar_init(&bar.q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.k_full[i], 1);
            mbar_init(&bar.k_empty[i], 1);
            mbar_init(&bar.v_full[i], 1);
            mbar_init(&bar.v_empty[i], 1);
            mbar_init(&bar.fix[i], 1);
            mbar_init(&bar.v_fixed[i], 2);
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], 4);
            mbar_init(&bar.o_final[i], 1);
            mbar_init(&bar.o_empty[i], 4);
            mbar_init(&bar.item_full[i], 1);
            mbar_init(&bar.item_empty[i], 11);
        }
        mbar_init(&bar.drain, 1);
        bar.abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&bar.tmem, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    volatile int* abort_flag = &bar.abort;
    // the next item of a consuming warp; -1: none
    auto next_item = [&](int nitem, bool& ok) {
        const int slot = nitem & 1;
        if (ok) ok = warp_wait(&bar.item_full[slot], (nitem >> 1) & 1, p.status, 83);
        const int i = ok ? *(volatile int*)&bar.item[slot] : -1;
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&bar.item_empty[slot]);
        return i;
    };
    static_assert(128 * REG_LO + 256 * REG_HI <= NTHREADS * 168, "register split above the launch's registers");

    if (warp < 4) {
        setmaxnreg_dec<REG_LO>();
        if (warp == 0) {
            // ------------------------------------------------------------ TMA producer
            if (lane == 0) {
                prefetch_tmap(&tmQ);
                prefetch_tmap(&tmK);
                prefetch_tmap(&tmR);
                prefetch_tmap(&tmV);
                int nq = 0, nk = 0, nv = 0;  // loads issued: query tiles, key tiles, halves of values
                bool ok = true;
                int next = atomicAdd(p.claim, 1);
                for (int nitem = 0; ok; ++nitem) {
                    const int i = next, slot = nitem & 1;
                    if (nitem >= 2) ok = mbar_wait(&bar.item_empty[slot], ((nitem >> 1) - 1) & 1, p.status, 84);
                    if (!ok || *abort_flag) { ok = false; break; }
                    *(volatile int*)&bar.item[slot] = i < p.n_items ? i : -1;
                    mbar_arrive(&bar.item_full[slot]);
                    if (i >= p.n_items) break;
                    next = atomicAdd(p.claim, 1);
                    const Item it = item_of(p, i);
                    const int hk = it.h / p.group;
                    for (int j = 0; j < it.n && ok; ++j) {
                        const int ks = nk & 1;
                        if (nk >= 2) ok = mbar_wait(&bar.k_empty[ks], ((nk >> 1) - 1) & 1, p.status, 85);
                        if (!ok || *abort_flag) { ok = false; break; }
                        mbar_expect_tx(&bar.k_full[ks], C::TILE);
                        unsigned char* dk = smem + C::OFF_K + ks * C::TILE;
                        for (int a = 0; a < DN / 64; ++a) tma_load_4d(dk + a * C::PANEL, &tmK, a * 64, j * BN, hk, it.b, &bar.k_full[ks]);
                        tma_load_4d(dk + (DN / 64) * C::PANEL, &tmR, 0, j * BN, 0, it.b, &bar.k_full[ks]);
                        ++nk;
                        if (j == 0) {  // the item's query tiles, once the last one's scores are formed
                            if (nq > 0) ok = mbar_wait(&bar.q_empty, (nq - 1) & 1, p.status, 86);
                            if (!ok || *abort_flag) { ok = false; break; }
                            const int nt = it.nblk[1] > 0 ? 2 : 1;
                            mbar_expect_tx(&bar.q_full, nt * C::TILE);
                            for (int t = 0; t < nt; ++t)
                                for (int a = 0; a < C::PANELS; ++a)
                                    tma_load_4d(smem + t * C::TILE + a * C::PANEL, &tmQ, a * 64, it.row0 + t * BM, it.h, it.b, &bar.q_full);
                            ++nq;
                        }
                        for (int v = 0; v < 2; ++v, ++nv) {
                            const int vs = nv & 1;
                            if (nv >= 2) ok = mbar_wait(&bar.v_empty[vs], ((nv >> 1) - 1) & 1, p.status, 87);
                            if (!ok || *abort_flag) { ok = false; break; }
                            mbar_expect_tx(&bar.v_full[vs], C::VHALF);
                            for (int a = 0; a < DN / 64; ++a)
                                tma_load_4d(smem + C::OFF_V + vs * C::VHALF + a * C::VSLAB, &tmV, a * 64, j * BN + v * HALF, hk, it.b,
                                            &bar.v_full[vs]);
                        }
                    }
                }
                if (!ok) *abort_flag = 1;
                if (*abort_flag) {  // our copies in flight end before the CTA does
                    if (nq > 0) mbar_wait(&bar.q_full, (nq - 1) & 1, nullptr, 0);
                    for (int n = max(0, nk - 2); n < nk; ++n) mbar_wait(&bar.k_full[n & 1], (n >> 1) & 1, nullptr, 0);
                    for (int n = max(0, nv - 2); n < nv; ++n) mbar_wait(&bar.v_full[n & 1], (n >> 1) & 1, nullptr, 0);
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------ MMA issuer
            constexpr uint32_t IDESC_S = idesc_f16(BM, BN, BF16, false), IDESC_PV = idesc_f16(BM, DN, BF16, true);
            const bool lead = elect_lane();
            const uint32_t tm = (uint32_t)uniform((int)tmem);
            const uint32_t q0 = desc_lo(smem_u32(smem), 16), k0 = desc_lo(smem_u32(smem + C::OFF_K), 16);
            const uint32_t v0 = desc_lo(smem_u32(smem + C::OFF_V), C::VSLAB);
            // key tiles; tiles and items of each query tile; items with work; halves of values that were mended
            int J = 0, u[2] = {0, 0}, nf[2] = {0, 0}, ne = 0, fixed[2] = {0, 0};
            bool ok = true;
            auto issue_s = [&](int t, int jg, bool loaded) {
                const int ks = jg & 1;
                if (!loaded && !warp_wait(&bar.k_full[ks], (jg >> 1) & 1, p.status, 88)) return false;
                tc_fence_after();
                const uint32_t q = q0 + t * (C::TILE >> 4), k = (uint32_t)uniform((int)(k0 + ks * (C::TILE >> 4))), dst = tm + t * 128;
                if (lead) {
#pragma unroll
                    for (int kk = 0; kk < DN / 16; ++kk) {
                        constexpr int P4 = C::PANEL >> 4;
                        mma_ss_lo(dst, q + (kk / 4) * P4 + (kk % 4) * 2, k + (kk / 4) * P4 + (kk % 4) * 2, IDESC_S, kk > 0);
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        if (kk < p.rope_steps)
                            mma_ss_lo(dst, q + (DN / 64) * (C::PANEL >> 4) + kk * 2, k + (DN / 64) * (C::PANEL >> 4) + kk * 2, IDESC_S, 1);
                    mma_commit(&bar.s_full[t]);
                }
                return true;
            };
            for (int nitem = 0; ok; ++nitem) {
                const int i = uniform(next_item(nitem, ok));
                if (i < 0) break;
                const Item it = item_of(p, i);
                const int n = uniform(it.n), nb[2] = {uniform(it.nblk[0]), uniform(it.nblk[1])}, nS = uniform(it.nS);
                if (n == 0) continue;
                ok = warp_wait(&bar.q_full, ne & 1, p.status, 89);
                for (int t = 0; t < 2 && ok; ++t)
                    if (nb[t] > 0) ok = issue_s(t, J, false);
                if (!ok) break;
                if (lead) {
                    mma_commit(&bar.k_empty[J & 1]);
                    if (n == 1) mma_commit(&bar.q_empty);
                }
                for (int j = 0; j < n && ok; ++j) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!ok || j >= nb[t]) continue;
                        // The waits for what is mostly there already come before the one for the weights: between products each
                        // wait leaves the tensor core idle for some 115 cycles.
                        const bool more = j + 1 < nb[t];
                        const bool loaded = more && __all_sync(~0u, mbar_test(&bar.k_full[(J + j + 1) & 1], ((J + j + 1) >> 1) & 1));
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            if (ok) ok = warp_wait(&bar.v_full[v], (J + j) & 1, p.status, 92);
                            if (ok && padded_half(p, nS, j, v)) {  // the first tile to read it has it mended
                                if (lead && (t == 0 || j >= nb[0])) mbar_arrive(&bar.fix[v]);
                                ok = warp_wait(&bar.v_fixed[v], fixed[v] & 1, p.status, 93);
                            }
                        }
                        // the first product of an item overwrites O_t: the last item's output must have been read
                        if (ok && j == 0 && nf[t] > 0) ok = warp_wait(&bar.o_empty[t], (nf[t] - 1) & 1, p.status, 90);
                        if (ok) ok = warp_wait(&bar.p_full[t], (u[t] + j) & 1, p.status, 91);
                        if (!ok) continue;
                        tc_fence_after();
                        const bool last_t = t == 1 || j >= nb[1];  // the last query tile to read this value tile
                        const uint32_t dst = tm + 256 + t * 128, pa = tm + t * 128;
                        if (lead) {
#pragma unroll
                            for (int kk = 0; kk < BN / 16; ++kk) {
                                // P_t: 16-bit pairs, keys 32 c .. in columns 32 c .. 32 c + 15
                                mma_ts_lo(dst, pa + 32 * (kk >> 1) + 8 * (kk & 1), v0 + (kk >> 2) * (C::VHALF >> 4) + (kk & 3) * 128, IDESC_PV,
                                          j > 0 || kk > 0);
                                if (kk == 3 && last_t) mma_commit(&bar.v_empty[0]);
                            }
                            if (last_t) mma_commit(&bar.v_empty[1]);
                        }
                        if (more) ok = issue_s(t, J + j + 1, loaded);
                        if (ok && j + 1 == nb[t] && lead) mma_commit(&bar.o_final[t]);
                    }
                    if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
#pragma unroll
                    for (int v = 0; v < 2; ++v) fixed[v] += padded_half(p, nS, j, v);
                    if (lead) {
                        if (j + 1 < n) mma_commit(&bar.k_empty[(J + j + 1) & 1]);
                        if (j + 2 == n) mma_commit(&bar.q_empty);
                    }
                }
                J += n;
                ++ne;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    u[t] += nb[t];
                    nf[t] += nb[t] > 0;
                }
            }
            if (!ok) *abort_flag = 1;
            __syncwarp();
            if (__any_sync(~0u, *abort_flag)) {
                if (lead) mma_commit(&bar.drain);
                warp_wait(&bar.drain, 0, nullptr, 0);
            }
        } else {
            // ------------------------------------------------------------ value rows of padded tokens become zeros
            const int ft = (int)threadIdx.x - 64;
            bool ok = true;
            int n_fix[2] = {0, 0};
            for (int nitem = 0; ok; ++nitem) {
                const int i = next_item(nitem, ok);
                if (i < 0) break;
                const Item it = item_of(p, i);
                for (int j = 0; j < it.n && ok; ++j)
#pragma unroll
                    for (int v = 0; v < 2 && ok; ++v) {
                        if (!padded_half(p, it.nS, j, v)) continue;
                        ok = warp_wait(&bar.fix[v], n_fix[v]++ & 1, p.status, 94);  // it has been loaded
                        const int first = max(0, it.nS - (j * BN + v * HALF)), per = (HALF - first) * 8;
                        for (int e = ft; e < per * (DN / 64); e += 64) {
                            const int a = e / per;
                            *(uint4*)(smem + C::OFF_V + v * C::VHALF + a * C::VSLAB + first * 128 + (e - a * per) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.v_fixed[v]);
                    }
            }
            if (!ok) *abort_flag = 1;
        }
    } else {
        setmaxnreg_inc<REG_HI>();
        // ------------------------------------------------------------ softmax and output of tile t
        const int t = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        const uint32_t s_tmem = tmem + lane_addr + t * 128, o_tmem = tmem + lane_addr + 256 + t * 128;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
        int u = 0, nf = 0;
        bool ok = true;
        for (int nitem = 0; ok; ++nitem) {
            const int i = next_item(nitem, ok);
            if (i < 0) break;
            const Item it = item_of(p, i);
            const int nb = it.nblk[t], row0 = it.row0 + t * BM, row = row0 + r;
            T* orow = (T*)p.o + it.b * p.os0 + it.h * p.os1 + (int64_t)row * p.os2;
            float* lse = p.lse ? p.lse + ((int64_t)it.b * p.H + it.h) * p.L + row : nullptr;
            if (nb == 0) {  // nothing to attend
                if (row < p.L) {
#pragma unroll 1
                    for (int c = 0; c < DN / 8; ++c) *(uint4*)(orow + c * 8) = make_uint4(0, 0, 0, 0);
                    if (lse) *lse = -INFINITY;
                }
                continue;
            }
            const int lim = p.causal ? min(it.nS - 1, row) : it.nS - 1;  // last key this row may see
            float m_used = -INFINITY, lsum = 0.0f;
            for (int j = 0; j < nb; ++j) {
                ok = warp_wait(&bar.s_full[t], (u + j) & 1, p.status, 95);
                if (!ok || __any_sync(~0u, *abort_flag)) { ok = false; break; }
                tc_fence_after();
                const int kv0 = j * BN;
                uint32_t raw[128];
                float* x = (float*)raw;
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + 32 * c, raw + 32 * c);
                tmem_ld_wait();
                if (kv0 + BN > it.nS || (p.causal && kv0 + BN - 1 > row0)) {
#pragma unroll
                    for (int k = 0; k < BN; ++k)
                        if (kv0 + k > lim) x[k] = -INFINITY;
                }
                float pm[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) pm[k] = fmaxf(x[k], x[k + 8]);
#pragma unroll
                for (int k = 16; k < BN; k += 16)
#pragma unroll
                    for (int e = 0; e < 8; ++e) pm[e] = fmax3(pm[e], x[k + e], x[k + 8 + e]);
                const float cm = fmax3(fmax3(pm[0], pm[1], pm[2]), fmax3(pm[3], pm[4], pm[5]), fmaxf(pm[6], pm[7]));
                const float m_start = m_used;
                if ((cm - m_used) * p.scale_log2 > 8.0f) m_used = cm;  // false while the row has no finite score
                const bool grew = m_used != m_start;
                const float neg_m = m_used == -INFINITY ? 0.0f : -m_used;
                const uint64_t nm2 = f2_pack(neg_m, neg_m);
                uint64_t ps2[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; ++c) {  // keys 32 c .. : their weights go over the first 16 of the chunk's columns
                    uint32_t pk[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        float a0, a1;
                        // (the difference first, so that scores of any size keep what they differ by)
                        f2_unpack(f2_mul(f2_add(f2_pack(x[32 * c + k], x[32 * c + k + 1]), nm2), sc2), a0, a1);
                        a0 = ex2(a0);
                        a1 = ex2(a1);
                        ps2[(k >> 1) & 1] = f2_add(ps2[(k >> 1) & 1], f2_pack(a0, a1));
                        pk[k / 2] = pack2<BF16>(a0, a1);
                    }
                    tmem_st16(s_tmem + 32 * c, pk);
                }
                if (__any_sync(~0u, grew && j > 0)) {
                    // PV_t(j-1) is complete: it was issued before S_t(j), whose completion has been seen
                    const float alpha = grew ? ex2((m_start - m_used) * p.scale_log2) : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < DN / 32; ++c) {
                        uint32_t ov[32];
                        tmem_ld32(o_tmem + c * 32, ov);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 32; ++k) ov[k] = __float_as_uint(__uint_as_float(ov[k]) * alpha);
                        tmem_st32(o_tmem + c * 32, ov);
                    }
                }
                float s0, s1, s2, s3;
                f2_unpack(ps2[0], s0, s1);
                f2_unpack(ps2[1], s2, s3);
                lsum = (grew ? lsum * ex2((m_start - m_used) * p.scale_log2) : lsum) + ((s0 + s1) + (s2 + s3));
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.p_full[t]);
            }
            u += nb;
            if (!ok) break;
            ok = warp_wait(&bar.o_final[t], nf & 1, p.status, 96);
            if (!ok) break;
            tc_fence_after();
            const bool none = row >= it.nL || lsum == 0.0f;
            const float inv = none ? 0.0f : 1.0f / lsum;
#pragma unroll 1
            for (int c = 0; c < DN / 32; ++c) {
                uint32_t ov[32], w[16];
                tmem_ld32(o_tmem + c * 32, ov);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; k += 2)  // (a row without a weight is 0 whatever O holds)
                    w[k / 2] = none ? 0u : pack2<BF16>(__uint_as_float(ov[k]) * inv, __uint_as_float(ov[k + 1]) * inv);
                if (row < p.L) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *(uint4*)(orow + c * 32 + 8 * k) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                }
            }
            if (lse && row < p.L) *lse = none ? -INFINITY : (m_used * p.scale_log2 + log2f(lsum)) * 0.69314718055994531f;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.o_empty[t]);
            ++nf;
        }
        if (!ok) *abort_flag = 1;
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

template <int DN, bool BF16>
int launch(const LatentSdpaArgs& a, cudaStream_t st) {
    using C = Cfg<DN>;
    const char* ctx = "latent_sdpa";
    auto kern = latent_fwd_kernel<DN, BF16>;
    int dev = 0, n_sm = 0;
    if (cuda_failed(cudaGetDevice(&dev), ctx) || cuda_failed(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev), ctx))
        return -1;
    static std::atomic<uint64_t> ready{0};  // devices (of the first 64) whose kernel is set up
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(ready.load() & bit)) {
        cudaFuncAttributes fa;
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM), ctx) ||
            cuda_failed(cudaFuncGetAttributes(&fa, kern), ctx))
            return -1;
        // setmaxnreg.inc waits until the block's registers cover the split
        if ((int64_t)fa.numRegs * NTHREADS < 128 * REG_LO + 256 * REG_HI) {
            set_errorf("%s: kernel built with %d registers a thread, below what the register split needs", ctx, fa.numRegs);
            return -1;
        }
        ready.fetch_or(bit);
    }
    const int64_t items = (a.L + 2 * BM - 1) / (2 * BM) * a.H * a.B;
    if (items >= INT32_MAX / 2) {
        set_errorf("%s: too many work items", ctx);
        return -1;
    }
    CUtensorMap mq, mk, mr, mv;
    if (!make_tma_map_4d(&mq, a.q, DN + a.Dr, BF16, BM) || !make_tma_map_4d(&mk, a.k, DN, BF16, BN) ||
        !make_tma_map_4d(&mr, a.k_rope, a.Dr, BF16, BN) || !make_tma_map_4d(&mv, a.v, DN, BF16, HALF))
        return -1;
    Params p{};
    p.L = a.L;
    p.S = a.S;
    p.B = (int)a.B;
    p.H = (int)a.H;
    p.group = (int)(a.H / a.Hkv);
    p.n_pairs = (int)((a.L + 2 * BM - 1) / (2 * BM));
    p.n_items = (int)items;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.causal = a.causal;
    p.rope_steps = (a.Dr + 15) / 16;
    p.lens = a.lens;
    p.o = a.o.data;
    p.os0 = a.o.stride[0];
    p.os1 = a.o.stride[1];
    p.os2 = a.o.stride[2];
    p.lse = a.lse;
    p.status = a.status;
    if (cuda_failed(cudaMallocAsync((void**)&p.claim, sizeof(int), st), "latent_sdpa: item counter")) return -1;
    int rc = cuda_failed(cudaMemsetAsync(p.claim, 0, sizeof(int), st), "latent_sdpa: item counter") ? -1 : 0;
    if (!rc) {
        kern<<<(unsigned)std::min<int64_t>(n_sm, items), NTHREADS, C::SMEM, st>>>(mq, mk, mr, mv, p);
        if (cuda_failed(cudaGetLastError(), "latent_sdpa launch")) rc = -1;
    }
    cudaFreeAsync(p.claim, st);
    return rc;
}

}  // namespace

int launch_latent_sdpa_fwd(const LatentSdpaArgs& a, cudaStream_t st) {
    const bool bf16 = a.q.dtype == BF16;
    if (a.Dn == 128) return bf16 ? launch<128, true>(a, st) : launch<128, false>(a, st);
    return bf16 ? launch<64, true>(a, st) : launch<64, false>(a, st);
}

}  // namespace gtb
