// Attention over the block-scaled 8-bit cache for many query rows (a chunk of a prompt): tcgen05 tensor cores.
//
// With hundreds of rows per kv head every cached value is used that often, so its codes are made into f16 once, by
// a first kernel, and the second is a flash-style forward over f16 tiles:
//   kv8_widen_kernel  K, V codes -> f16 (exact: int8 and e4m3 both fit), rows past the length zero, head size
//                     padded to DP; q -> f16 rows r = i * G + g of each (sequence, kv head), normalised by a power
//                     of two per row as in kv8_mma.cuh; the scales of every 16 keys as (sk, log2 sv, 1 / sv).
//   kv8_chunk_kernel  one CTA per SM claims items (sequence, kv head, pair of 128-row tiles) from a counter, the
//                     longest sequences first and a head's pairs together, so that the CTAs running at a time share
//                     few heads' K and V through L2; the last items are claimed in parts of their keys, so that
//                     the SMs end together. Twelve warps: TMA producer, MMA issuer, two idle, and four softmax warps per
//                     tile, one row a thread, which ping-pong with the tensor core:
//                       S_t = Q_t K_j^T (M = N = 128, K = DP),  O_t += P_t V_j (A = P_t from TMEM, V read MN-major).
//                     Scores become log2 units with their 16 keys' scale, V's scale is folded into the exponent
//                     (P' = 2^(s + log2 sv - M + 8), M raised when a block exceeds it by 2^7) and the row sum
//                     takes P' / sv, so scales cost three packed operations per 16 keys and no accuracy.
//                     P' becomes f16 for the second product: 11 bits, where the 16-bit outputs keep 8 or 11; the row
//                     sum is of the f32 values.
//   kv8_chunk_join_kernel  joins those parts.
// The tile pair reuses each K/V tile for 256 rows; the second kernel is bound by the softmax warps' chain from scores
// to weights (tensor pipe and exponentials 48 to 49 % busy each). 4 sequences, 1021 tokens x 32 heads of 128 against 4k to
// 8k cached: 46 us to widen, 400 to 428 for the products (0.54 to 0.58 of the bf16 GEMM rate), 13 for the join; on
// kv8_mma.cuh 2.7 ms. Every wait is bounded: a timeout records a status code, drains the CTA's own copies and MMAs,
// frees TMEM and returns.

#include <algorithm>
#include <atomic>
#include <cmath>

#include "gtb_common.cuh"
#include "kv8_chunk.h"
#include "kv8_mma.cuh"
#include "sdpa_args.h"
#include "sm100_ptx.cuh"

namespace gtb {
namespace kv8 {
namespace {

using namespace sm100;

constexpr int BM = 128, BN = 128, NTHREADS = 384, REG_LO = 104, REG_HI = 200;
constexpr uint32_t TMEM_COLS = 512;
// Parts of each of the last items: 1021 tokens of 4 sequences with 1 / 2 / 4 / 8 471 / 459 / 451 / 467 us, 333 tokens
// 263 / 240 / 222 / 238
constexpr int TAIL_SPLITS = 4;
constexpr float LARGE = 0x1p20f;  // f32 holds a score above to 2^-4 at best

template <int D>
struct ChunkCfg {
    static constexpr int ATOMS = D / 64;
    static constexpr int TILE = BM * D * 2;
    static constexpr int ATOM_BYTES = BM * 128;
    static constexpr int OFF_K = 2 * TILE, OFF_V = 4 * TILE, OFF_BAR = 6 * TILE;  // Q_0 Q_1, two K stages, two V stages
    static constexpr int NBAR = 1 + 8 + 2 + 2 + 2 + 1 + 1 + 2 + 2 + 2;
    static constexpr int SMEM = OFF_BAR + NBAR * 8 + 32 + 1024;
};

struct ChunkP {
    gtb_kv8 c;
    Rows3 q, o;
    int dtype, q_vec, G, R, pairs;
    int whole, tail, splits;     // items claimed whole, items claimed in `splits` parts each
    int64_t b0, nb;              // sequences of this launch
    int64_t H, Lq;
    float scale_log2;
    const int32_t* counts;
    float* lse;
    int64_t Spad, Rpad;
    __half *k16, *v16, *q16;     // [nb * Hkv][Spad | Rpad][DP]
    float4* scl;                 // [nb * Hkv][Spad / 16]: sk, log2 sv, 1 / sv
    float* qmul;                 // [nb * Hkv][Rpad]
    float* part_o;               // [tail item][split][256][DP]
    float2* part_ml;             // [tail item][split][256]
    int* order;                  // [nb]: sequences, longest first
    int* claim;
    int* status;
};

// Rows of codes (64 of K and V a CTA) to f16, rows of q (32) to normalised f16; blockIdx.y = (sequence, kv head). The last
// CTA of the first row orders the sequences and zeroes the counter.
template <int FMT, int DP>
__global__ void __launch_bounds__(256) kv8_widen_kernel(const __grid_constant__ ChunkP p) {
    const gtb_kv8& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x == gridDim.x - 1) {
        if (blockIdx.y != 0) return;
        if (threadIdx.x == 0) *p.claim = 0;
        const int n = (int)p.nb;
        for (int i = threadIdx.x; i < n; i += 256) {
            int rank = i;  // more sequences than are worth comparing stay as they come
            if (n <= 2048) {
                const int own = c.lens[p.b0 + i];
                rank = 0;
                for (int k = 0; k < n; ++k) {
                    const int other = c.lens[p.b0 + k];
                    rank += other > own || (other == own && k < i);
                }
            }
            p.order[rank] = i;
        }
        return;
    }
    const int k_ctas = (int)(p.Spad / 64);
    const int64_t lbh = blockIdx.y, b = p.b0 + lbh / c.Hkv, hk = lbh % c.Hkv, bh = b * c.Hkv + hk;
    const int len = (int)clamp64(c.lens[b], 0, c.Smax);
    if ((int)blockIdx.x < k_ctas) {
        // 64 rows of K and V; a thread makes 16 codes into 32 bytes
        const int r0 = blockIdx.x * 64;
        if (r0 >= (len + BN - 1) / BN * BN) return;  // no tile reads them
        constexpr int CPR = DP / 8, STEPS = 2 * 64 * CPR / 256;  // 8 codes -> 16 bytes a step
        uint2 w[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            const int e = k * 256 + threadIdx.x, v = e >= 64 * CPR, x = v ? e - 64 * CPR : e, row = r0 + x / CPR, ch = x % CPR;
            w[k] = make_uint2(0, 0);
            if (row < len && ch * 8 < c.D) w[k] = *(const uint2*)((const uint8_t*)(v ? c.v : c.k) + (bh * c.Smax + row) * c.D + ch * 8);
        }
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            const int e = k * 256 + threadIdx.x, v = e >= 64 * CPR, x = v ? e - 64 * CPR : e, row = r0 + x / CPR, ch = x % CPR;
            const uint32_t u0 = prep_word<FMT>(w[k].x), u1 = prep_word<FMT>(w[k].y);
            *(uint4*)((v ? p.v16 : p.k16) + (lbh * p.Spad + row) * DP + ch * 8) =
                make_uint4(expand<FMT, 0>(u0), expand<FMT, 1>(u0), expand<FMT, 0>(u1), expand<FMT, 1>(u1));
        }
        if (threadIdx.x < 4) {
            const int k = r0 + threadIdx.x * 16;
            float4 s = make_float4(0.0f, 0.0f, 1.0f, 0.0f);
            if (k < len) {
                const int64_t at = bh * ((c.Smax + c.block - 1) / c.block) + k / c.block;
                const float sv = fmaxf(c.v_scale[at], SV_MIN);
                s = make_float4(c.k_scale[at], lg2f(sv), __frcp_rn(sv), 0.0f);
            }
            p.scl[lbh * (p.Spad / 16) + k / 16] = s;
        }
        return;
    }
    // 32 rows of q, four values a lane
    constexpr int LPR = DP / 4, RPW = 32 / LPR, STEPS = 4 / RPW;  // lanes of a row, rows a warp takes at once
    const int g0 = ((int)blockIdx.x - k_ctas) * 32 + warp * 4 + lane / LPR, d = (lane % LPR) * 4;
    float x[STEPS][4];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const int r = g0 + k * RPW, i = r / p.G, h = (int)hk * p.G + (r - i * p.G);
        load_q4(p, b * p.q.sb + h * p.q.sh + (int64_t)i * p.q.ss + d, r < p.R && d < c.D, x[k]);
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        float m = fmaxf(fmaxf(finite_abs(x[k][0]), finite_abs(x[k][1])), fmaxf(finite_abs(x[k][2]), finite_abs(x[k][3])));
        for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        int e = (int)(__float_as_uint(m) >> 23) - 127;
        e = m >= 1.17549435e-38f ? min(max(e, -126), 126) : 0;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        const int64_t row = lbh * p.Rpad + g0 + k * RPW;
        *(uint2*)(p.q16 + row * DP + d) = make_uint2(pack_f16(x[k][0] * down, x[k][1] * down), pack_f16(x[k][2] * down, x[k][3] * down));
        if (d == 0) p.qmul[row] = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_log2;
    }
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
    const bool ok = mbar_wait(bar, parity, status, code);
    return __all_sync(0xffffffffu, ok);
}

// GROUPS: scales in a 128-key block (1, 2, 4 or 8: blocks of 128, 64, 32 or 16 tokens)
template <int D, int GROUPS>
__global__ void __launch_bounds__(NTHREADS, 1)
kv8_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ ChunkP p) {
    using C = ChunkCfg<D>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(smem + C::OFF_BAR);
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;         // [2]
    uint64_t* k_empty = k_full + 2;      // [2]
    uint64_t* v_full = k_empty + 2;      // [2]
    uint64_t* v_empty = v_full + 2;      // [2]
    uint64_t* s_full = v_empty + 2;      // [2] per tile: S_t(j) computed
    uint64_t* p_full = s_full + 2;       // [2] per tile: P_t(j) written (128 arrivals)
    uint64_t* o_final = p_full + 2;      // [2] per tile: every MMA of the tile done
    uint64_t* drain = o_final + 2;
    uint64_t* q_empty = drain + 1;       // every S MMA of an item done
    uint64_t* o_empty = q_empty + 1;     // [2] per tile: the epilogue has read O_t (128 arrivals)
    uint64_t* item_full = o_empty + 2;   // [2] ring of claimed items
    uint64_t* item_empty = item_full + 2;
    uint32_t* tmem_slot = (uint32_t*)(bars + C::NBAR);
    int* abort_flag = (int*)(tmem_slot + 1);
    int* item_slot = abort_flag + 1;     // [2]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_items = p.whole + p.tail * p.splits;

    // Item i. nblk[t]: key blocks of tile t in this part; j0: the part's first block; n: blocks to load.
    struct Item {
        int bh, slot, row0[2], nblk[2], j0, n, len, cnt;
    };
    auto item_of = [&](int i) {
        Item it;
        const bool part = i >= p.whole;
        it.slot = part ? i - p.whole : -1;
        const int item = part ? p.whole + it.slot / p.splits : i, split = part ? it.slot % p.splits : 0, splits = part ? p.splits : 1;
        const int per_seq = (int)p.c.Hkv * p.pairs, sq = item / per_seq, rest = item - sq * per_seq, hk = rest / p.pairs;
        const int lb = p.order[sq], pair = p.pairs - 1 - (rest - hk * p.pairs);
        it.bh = lb * (int)p.c.Hkv + hk;
        const int64_t b = p.b0 + lb;
        it.len = (int)clamp64(p.c.lens[b], 0, p.c.Smax);
        it.cnt = p.counts ? (int)clamp64(p.counts[b], 0, p.Lq) : (int)p.Lq;
        int blk[2];
        for (int t = 0; t < 2; ++t) {
            it.row0[t] = pair * 2 * BM + t * BM;
            const int last = min(it.row0[t] + BM, it.cnt * p.G) - 1;  // last row that has a query
            const int lim = last < it.row0[t] ? -1 : it.len - it.cnt + last / p.G;
            blk[t] = lim < 0 ? 0 : lim / BN + 1;
        }
        const int all = max(blk[0], blk[1]);
        it.j0 = (int)((int64_t)all * split / splits);
        const int j1 = (int)((int64_t)all * (split + 1) / splits);
        it.n = 0;
        for (int t = 0; t < 2; ++t) {
            it.nblk[t] = max(0, min(j1, blk[t]) - it.j0);
            it.n = max(it.n, it.nblk[t]);
        }
        return it;
    };

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 128); mbar_init(&o_final[i], 1); mbar_init(&o_empty[i], 128);
            mbar_init(&item_full[i], 1); mbar_init(&item_empty[i], 9);
        }
        mbar_init(q_empty, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
    cudaTriggerProgrammaticLaunchCompletion();
    cudaGridDependencySynchronize();  // the widened rows and the item counter are there
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    static_assert(128 * REG_LO + 256 * REG_HI <= NTHREADS * 168, "register split above the launch's registers");

    if (warp < 4) {
        setmaxnreg_dec<REG_LO>();
        if (warp == 0) {
            if (lane == 0) {
                prefetch_tmap(&tmQ);
                prefetch_tmap(&tmK);
                prefetch_tmap(&tmV);
                int J = 0, work = 0, nk = 0, nv = 0, nq = 0;  // blocks, items with work, loads so far
                bool ok = true;
                int next = atomicAdd(p.claim, 1);
                for (int nitem = 0;; ++nitem) {
                    const int i = next, slot = nitem & 1;
                    if (nitem >= 2) ok = mbar_wait(&item_empty[slot], ((nitem >> 1) - 1) & 1, p.status, 111);
                    if (!ok || *(volatile int*)abort_flag) { ok = false; break; }
                    item_slot[slot] = i < n_items ? i : -1;
                    mbar_arrive(&item_full[slot]);
                    if (i >= n_items) break;
                    next = atomicAdd(p.claim, 1);
                    const Item it = item_of(i);
                    if (it.n == 0) continue;
                    const int nt = it.nblk[1] > 0 ? 2 : 1;
                    auto load_q = [&]() {
                        mbar_expect_tx(q_full, nt * C::TILE);
                        for (int t = 0; t < nt; ++t)
                            for (int a = 0; a < C::ATOMS; ++a)
                                tma_load_4d(smem + t * C::TILE + a * C::ATOM_BYTES, &tmQ, a * 64, it.row0[t], it.bh, 0, q_full);
                        ++nq;
                    };
                    if (work == 0) load_q();
                    for (int j = 0; j < it.n; ++j, ++J) {
                        const int s = J & 1;
                        if (J >= 2) ok = mbar_wait(&k_empty[s], ((J >> 1) - 1) & 1, p.status, 112);
                        if (!ok || *(volatile int*)abort_flag) { ok = false; break; }
                        mbar_expect_tx(&k_full[s], C::TILE);
                        for (int a = 0; a < C::ATOMS; ++a)
                            tma_load_4d(smem + C::OFF_K + s * C::TILE + a * C::ATOM_BYTES, &tmK, a * 64, (it.j0 + j) * BN, it.bh, 0, &k_full[s]);
                        ++nk;
                        if (J >= 2) ok = mbar_wait(&v_empty[s], ((J >> 1) - 1) & 1, p.status, 113);
                        if (!ok || *(volatile int*)abort_flag) { ok = false; break; }
                        mbar_expect_tx(&v_full[s], C::TILE);
                        for (int a = 0; a < C::ATOMS; ++a)
                            tma_load_4d(smem + C::OFF_V + s * C::TILE + a * C::ATOM_BYTES, &tmV, a * 64, (it.j0 + j) * BN, it.bh, 0, &v_full[s]);
                        ++nv;
                        if (j == 0 && work > 0) {  // Q once the previous item's S MMAs have read theirs
                            ok = mbar_wait(q_empty, (work - 1) & 1, p.status, 114);
                            if (!ok || *(volatile int*)abort_flag) { ok = false; break; }
                            load_q();
                        }
                    }
                    if (!ok) break;
                    ++work;
                }
                if (!ok) *(volatile int*)abort_flag = 1;
                if (*(volatile int*)abort_flag) {  // drain our own copies (bounded)
                    if (nq > 0) mbar_wait(q_full, (nq - 1) & 1, nullptr, 0);
                    for (int j = max(0, nk - 2); j < nk; ++j) mbar_wait(&k_full[j & 1], (j >> 1) & 1, nullptr, 0);
                    for (int j = max(0, nv - 2); j < nv; ++j) mbar_wait(&v_full[j & 1], (j >> 1) & 1, nullptr, 0);
                }
            }
        } else if (warp == 1) {
            if (lane == 0) {
                constexpr uint32_t IDESC_S = idesc_f16(BM, BN, false, false), IDESC_PV = idesc_f16(BM, D, false, true);
                const uint64_t qd[2] = {desc_sw128(smem_u32(smem), 16, 1024), desc_sw128(smem_u32(smem + C::TILE), 16, 1024)};
                const uint64_t kd0 = desc_sw128(smem_u32(smem + C::OFF_K), 16, 1024);
                const uint64_t kd1 = desc_sw128(smem_u32(smem + C::OFF_K + C::TILE), 16, 1024);
                const uint64_t vd0 = desc_sw128(smem_u32(smem + C::OFF_V), C::ATOM_BYTES, 1024);
                const uint64_t vd1 = desc_sw128(smem_u32(smem + C::OFF_V + C::TILE), C::ATOM_BYTES, 1024);
                int J = 0, u[2] = {0, 0}, nf[2] = {0, 0}, work = 0;
                auto issue_s = [&](int t, int jg) -> bool {
                    if (!mbar_wait(&k_full[jg & 1], (jg >> 1) & 1, p.status, 122)) return false;
                    tc_fence_after();
                    const uint64_t qb = t ? qd[1] : qd[0], kb = (jg & 1) ? kd1 : kd0;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = (uint32_t)((kk / 4) * C::ATOM_BYTES + (kk % 4) * 32);
                        mma_ss(tmem + t * 128u, desc_advance(qb, off), desc_advance(kb, off), IDESC_S, kk > 0 ? 1u : 0u);
                    }
                    mma_commit(&s_full[t]);
                    return true;
                };
                auto issue_pv = [&](int t, int jg, int ut, bool first) -> bool {
                    if (!mbar_wait(&p_full[t], ut & 1, p.status, 123)) return false;
                    if (!mbar_wait(&v_full[jg & 1], (jg >> 1) & 1, p.status, 124)) return false;
                    tc_fence_after();
                    const uint64_t vb = (jg & 1) ? vd1 : vd0;
                    const uint32_t pa = tmem + t * 128u;
#pragma unroll
                    for (int kk = 0; kk < BN / 16; ++kk)
                        mma_ts(tmem + 256u + t * 128u, pa + 32 * (kk >> 1) + 8 * (kk & 1), desc_advance(vb, kk * 2048), IDESC_PV,
                               (!first || kk > 0) ? 1u : 0u);
                    return true;
                };
                bool ok = true;
                for (int nitem = 0;; ++nitem) {
                    const int slot = nitem & 1;
                    ok = mbar_wait(&item_full[slot], (nitem >> 1) & 1, p.status, 127);
                    if (!ok) break;
                    const int i = item_slot[slot];
                    mbar_arrive(&item_empty[slot]);
                    if (i < 0) break;
                    const Item it = item_of(i);
                    if (it.n == 0) continue;
                    ok = mbar_wait(q_full, work & 1, p.status, 121);
                    ++work;
                    for (int t = 0; t < 2 && ok; ++t)
                        if (it.nblk[t] > 0) ok = issue_s(t, J);
                    if (!ok) break;
                    mma_commit(&k_empty[J & 1]);
                    if (it.n == 1) mma_commit(q_empty);
                    for (int j = 0; j < it.n && ok; ++j) {
                        for (int t = 0; t < 2 && ok; ++t) {
                            if (j >= it.nblk[t]) continue;
                            if (j == 0 && nf[t] > 0) ok = mbar_wait(&o_empty[t], (nf[t] - 1) & 1, p.status, 126);
                            if (ok) ok = issue_pv(t, J + j, u[t] + j, j == 0);
                            if (ok && j + 1 < it.nblk[t]) ok = issue_s(t, J + j + 1);
                            if (ok && j + 1 == it.nblk[t]) mma_commit(&o_final[t]);
                        }
                        if (!ok || *(volatile int*)abort_flag) { ok = false; break; }
                        mma_commit(&v_empty[(J + j) & 1]);
                        if (j + 1 < it.n) mma_commit(&k_empty[(J + j + 1) & 1]);
                        if (j + 2 == it.n) mma_commit(q_empty);
                    }
                    if (!ok) break;
                    J += it.n;
                    for (int t = 0; t < 2; ++t) {
                        u[t] += it.nblk[t];
                        nf[t] += it.nblk[t] > 0 ? 1 : 0;
                    }
                }
                if (!ok) *(volatile int*)abort_flag = 1;
                if (*(volatile int*)abort_flag) {
                    mma_commit(drain);
                    mbar_wait(drain, 0, nullptr, 0);
                }
            }
        }
    } else {
        setmaxnreg_inc<REG_HI>();
        const int t = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t s_tmem = tmem + ((uint32_t)(quad * 32) << 16) + t * 128u;
        const uint32_t o_tmem = s_tmem - t * 128u + 256u + t * 128u;
        int u = 0, nf = 0;
        bool ok = true;
        for (int nitem = 0; ok; ++nitem) {
            const int slot = nitem & 1;
            ok = warp_wait(&item_full[slot], (nitem >> 1) & 1, p.status, 134);
            if (!ok) break;
            const int i = item_slot[slot];
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[slot]);
            if (i < 0) break;
            const Item it = item_of(i);
            const int nb = it.nblk[t], row = it.row0[t] + r, qi = row / p.G;
            const bool valid = row < p.R && qi < it.cnt;
            const int lim = valid ? it.len - it.cnt + qi : -1;          // last key this row may see
            const int lim0 = it.row0[t] / p.G + it.len - it.cnt;        // ... the tile's first row
            const float qmul = p.qmul[(int64_t)it.bh * p.Rpad + row];
            const float4* scl = p.scl + (int64_t)it.bh * (p.Spad / 16) + it.j0 * 8;
            const float large_from = valid ? LARGE : INFINITY;         // (padding changes no other row's rounding)
            float m_used = -INFINITY, lsum = 0.0f;
            for (int j = 0; j < nb; ++j) {
                ok = warp_wait(&s_full[t], (u + j) & 1, p.status, 131);
                if (!ok || __any_sync(0xffffffffu, *(volatile int*)abort_flag)) { ok = false; break; }
                tc_fence_after();
                const int kv0 = (it.j0 + j) * BN;
                const float4* sc = scl + j * 8;
                uint32_t raw[128];
                tmem_ld32(s_tmem, raw);
                tmem_ld32(s_tmem + 32, raw + 32);
                tmem_ld32(s_tmem + 64, raw + 64);
                tmem_ld32(s_tmem + 96, raw + 96);
                tmem_ld_wait();
                float* x = (float*)raw;
                if (kv0 + BN - 1 > lim0) {
#pragma unroll
                    for (int e = 0; e < 128; ++e)
                        if (kv0 + e > lim) x[e] = -INFINITY;
                }
                // the block's scales: read once where they fit in registers
                constexpr int GK = 128 / GROUPS;  // keys a scale covers
                float g_mul[GROUPS <= 2 ? GROUPS : 1], g_add[GROUPS <= 2 ? GROUPS : 1], g_inv[GROUPS <= 2 ? GROUPS : 1];
                auto scale_of_group = [&](int g, float& mul, float& add, float& inv) {
                    const float4 z = __ldg(sc + g * (GK / 16));
                    mul = fmaxf(qmul * z.x, 1e-37f);
                    add = z.y;
                    inv = z.z;
                };
                if constexpr (GROUPS <= 2) {
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) scale_of_group(g, g_mul[g], g_add[g], g_inv[g]);
                }
                // largest s + log2 sv of the block
                const float m_start = m_used;
                float cm = -INFINITY;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const float* y = x + GK * g;
                    float a = fmax3(y[0], y[1], y[2]), b = fmax3(y[3], y[4], y[5]), d = fmax3(y[6], y[7], y[8]);
                    a = fmax3(a, y[9], y[10]);
                    b = fmax3(b, y[11], y[12]);
                    d = fmax3(d, y[13], y[14]);
                    a = fmaxf(a, y[15]);
#pragma unroll
                    for (int e = 16; e + 5 < GK; e += 6) {
                        a = fmax3(a, y[e], y[e + 1]);
                        b = fmax3(b, y[e + 2], y[e + 3]);
                        d = fmax3(d, y[e + 4], y[e + 5]);
                    }
#pragma unroll
                    for (int e = 16 + (GK - 16) / 6 * 6; e < GK; ++e) a = fmaxf(a, y[e]);
                    float mul, add, inv;
                    if constexpr (GROUPS <= 2) {
                        mul = g_mul[g];
                        add = g_add[g];
                    } else {
                        scale_of_group(g, mul, add, inv);
                    }
                    cm = fmaxf(cm, fmaf(fmax3(a, b, d), mul, add));
                }
                if (cm > m_used + RAISE) m_used = cm;  // never while the row has no finite score
                // Scores so large that x * mul + (add - m), rounded once, would be off m's own rounding by more than P' has
                // room for: they are rounded as m was, and then differ from it exactly
                const bool large = __any_sync(0xffffffffu, fabsf(m_used) > large_from && m_used != -INFINITY);
                if (large) {
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) {
                        float mul, add, inv;
                        scale_of_group(g, mul, add, inv);
#pragma unroll
                        for (int e = 0; e < GK; ++e) x[GK * g + e] = fmaf(x[GK * g + e], mul, add);
                        if constexpr (GROUPS <= 2) {
                            g_mul[g] = 1.0f;
                            g_add[g] = 0.0f;
                        }
                    }
                }
                const bool grew = m_used != m_start;
                const float off = m_used == -INFINITY ? 0.0f : SHIFT - m_used;
                float block_sum = 0.0f;
                uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16];
                    constexpr int STEP = GK < 32 ? GK : 32;  // keys of the chunk that share a scale
#pragma unroll
                    for (int h = 0; h < 32; h += STEP) {
                        const int key = 32 * c + h, g = key / GK;
                        float mul, add, inv;
                        if constexpr (GROUPS <= 2) {
                            mul = g_mul[g];
                            add = g_add[g];
                            inv = g_inv[g];
                        } else {
                            scale_of_group(g, mul, add, inv);
                            if (large) {
                                mul = 1.0f;
                                add = 0.0f;
                            }
                        }
                        add += off;
                        const uint64_t mul2 = f2_pack(mul, mul), add2 = f2_pack(add, add);
#pragma unroll
                        for (int e = 0; e < STEP; e += 2) {
                            float a0, a1;
                            f2_unpack(f2_fma(f2_pack(x[key + e], x[key + e + 1]), mul2, add2), a0, a1);
                            const float p0 = ex2(a0), p1 = ex2(a1);
                            sum2[(e >> 1) & 1] = f2_add(sum2[(e >> 1) & 1], f2_pack(p0, p1));
                            pk[(h + e) / 2] = pack_f16(p0, p1);
                        }
                        if ((key + STEP) % GK == 0) {  // the end of a scale's keys
                            float s0, s1, s2, s3;
                            f2_unpack(sum2[0], s0, s1);
                            f2_unpack(sum2[1], s2, s3);
                            block_sum = fmaf((s0 + s1) + (s2 + s3), inv, block_sum);
                            sum2[0] = sum2[1] = 0ull;
                        }
                    }
                    tmem_st16(s_tmem + 32 * c, pk);
                }
                if (__any_sync(0xffffffffu, grew && j > 0)) {
                    // PV_t(j-1) is complete: it was issued before S_t(j), whose completion we have seen
                    const float alpha = grew ? ex2(m_start - m_used) : 1.0f;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t ov[32];
                        tmem_ld32(o_tmem + c * 32, ov);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                        tmem_st32(o_tmem + c * 32, ov);
                    }
                }
                lsum = (grew ? lsum * ex2(m_start - m_used) : lsum) + block_sum;
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&p_full[t]);
            }
            if (!ok) break;
            u += nb;
            // results: the row's values, or its part of them; zeros for a row that attends nothing
            const bool whole = it.slot < 0;
            if (nb > 0) {
                if (*(volatile int*)abort_flag) ok = false;
                ok = __all_sync(0xffffffffu, ok) && warp_wait(&o_final[t], nf & 1, p.status, 133);
                if (!ok) break;
                tc_fence_after();
            }
            const float inv = !whole ? 1.0f : lsum > 0.0f || !(lsum == lsum) ? 1.0f / lsum : 0.0f;
            const int64_t b = p.b0 + it.bh / p.c.Hkv;
            const int h = (it.bh % (int)p.c.Hkv) * p.G + (row - qi * p.G);
            const int64_t at = b * p.o.sb + (int64_t)h * p.o.sh + (int64_t)qi * p.o.ss;
            const int64_t prow = ((int64_t)it.slot * 2 + t) * BM + r;
            const float m_out = m_used == -INFINITY ? -INFINITY : m_used - SHIFT;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t ov[32];
                if (nb > 0) {
                    tmem_ld32(o_tmem + c * 32, ov);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) ov[e] = 0u;
                }
                if (!whole) {
                    uint4* dst = (uint4*)(p.part_o + prow * D + c * 32);
#pragma unroll
                    for (int q = 0; q < 8; ++q) dst[q] = make_uint4(ov[4 * q], ov[4 * q + 1], ov[4 * q + 2], ov[4 * q + 3]);
                } else if (row < p.R) {
                    float y[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] = valid ? __uint_as_float(ov[e]) * inv : 0.0f;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int d = c * 32 + 8 * q;
                        if (d >= p.c.D) continue;
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (p.dtype == F16) w[e] = pack_f16(y[8 * q + 2 * e], y[8 * q + 2 * e + 1]);
                            else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(y[8 * q + 2 * e + 1]), "f"(y[8 * q + 2 * e]));
                        }
                        *(uint4*)((uint16_t*)p.o.p + at + d) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (!whole) p.part_ml[prow] = make_float2(!(lsum == lsum) ? lsum : m_out, lsum);
            else if (p.lse && row < p.R)
                p.lse[(b * p.H + h) * p.Lq + qi] = !valid || lsum == 0.0f ? -INFINITY : (m_out + log2f(lsum)) * 0.6931471805599453f;
            if (nb > 0) {
                tc_fence_before();
                mbar_arrive(&o_empty[t]);
                ++nf;
            }
        }
        if (!ok) *(volatile int*)abort_flag = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// Joins the parts of a tail item: blockIdx.x the item, 8 rows a CTA, one a warp
template <int D>
__global__ void __launch_bounds__(256) kv8_chunk_join_kernel(const __grid_constant__ ChunkP p) {
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_seq = (int)p.c.Hkv * p.pairs, item = p.whole + (int)blockIdx.x, sq = item / per_seq, rest = item - sq * per_seq;
    const int hk = rest / p.pairs, pair = p.pairs - 1 - (rest - hk * p.pairs);
    const int64_t b = p.b0 + p.order[sq], first = (int64_t)blockIdx.x * p.splits * 2 * BM;
    const int cnt = p.counts ? (int)clamp64(p.counts[b], 0, p.Lq) : (int)p.Lq;
    const int lr = blockIdx.y * 8 + warp, row = pair * 2 * BM + lr;
    if (row >= p.R) return;
    const int qi = row / p.G, h = hk * p.G + (row - qi * p.G);
    float m = -INFINITY, l = 0.0f, acc[D / 32] = {};
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[first + (int64_t)s * 2 * BM + lr].x);
    if (m == -INFINITY) m = 0.0f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const int64_t at = first + (int64_t)s * 2 * BM + lr;
        const float2 ml = p.part_ml[at];
        const float f = ex2f(ml.x - m);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(p.part_o[at * D + i * 32 + lane], f, acc[i]);
    }
    const bool none = qi >= cnt || l == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l;
    const int64_t at = b * p.o.sb + (int64_t)h * p.o.sh + (int64_t)qi * p.o.ss;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int d = i * 32 + lane;
        if (d >= p.c.D) continue;
        const float y = none ? 0.0f : acc[i] * inv;
        if (p.dtype == F16) ((__half*)p.o.p)[at + d] = __float2half_rn(y);
        else ((__nv_bfloat16*)p.o.p)[at + d] = __float2bfloat16_rn(y);
    }
    if (p.lse && lane == 0) p.lse[(b * p.H + h) * p.Lq + qi] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <int D, int GROUPS>
int set_up() {
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && (ready.load(std::memory_order_relaxed) >> dev & 1)) return 0;
    auto kern = kv8_chunk_kernel<D, GROUPS>;
    if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkCfg<D>::SMEM), "kv8_attention: shared memory"))
        return -1;
    // setmaxnreg.inc waits until the block's registers cover the split: refuse a build with fewer
    cudaFuncAttributes fa;
    if (cuda_failed(cudaFuncGetAttributes(&fa, kern), "kv8_attention: attributes")) return -1;
    if ((int64_t)fa.numRegs * NTHREADS < 128 * REG_LO + 256 * REG_HI) {
        set_errorf("kv8_attention: the chunk kernel was built with %d registers a thread, too few for its split", fa.numRegs);
        return -1;
    }
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    return 0;
}

bool map_rows(CUtensorMap* tm, void* data, int64_t heads, int64_t rows, int64_t D) {
    gtb_tensor4 t{};
    t.data = data;
    t.shape[0] = 1; t.shape[1] = heads; t.shape[2] = rows; t.shape[3] = D;
    t.stride[0] = heads * rows * D; t.stride[1] = rows * D; t.stride[2] = D; t.stride[3] = 1;
    t.dtype = F16;
    return make_tma_map_4d(tm, t, D, false, 128);
}

template <int D, int GROUPS>
int run(const Kv8AttnArgs& a, float* lse, int n_sm, cudaStream_t st) {
    if (set_up<D, GROUPS>()) return -1;
    ChunkP p{};
    p.c = a.c;
    p.q = a.q;
    p.o = a.o;
    p.dtype = a.dtype;
    p.q_vec = vector_rows(a.q, a.dtype);
    p.G = (int)(a.H / a.c.Hkv);
    p.R = p.G * (int)a.Lq;
    p.pairs = (p.R + 2 * BM - 1) / (2 * BM);
    p.H = a.H;
    p.Lq = a.Lq;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.counts = a.counts;
    p.lse = lse;
    p.Spad = (a.c.Smax + BN - 1) / BN * BN;
    p.Rpad = (int64_t)p.pairs * 2 * BM;
    int dev = 0;
    cudaGetDevice(&dev);
    p.status = device_status_word(dev);
    auto up = [](int64_t n) { return (n + 1023) / 1024 * 1024; };
    // scratch of one sequence; as many sequences a launch as stay within 2 GB (one at least)
    const int64_t Hkv = a.c.Hkv;
    const int64_t per_seq = Hkv * (p.Spad * D * 4 + p.Spad + p.Rpad * (D * 2 + 4));
    const int64_t nb = std::max<int64_t>(1, std::min<int64_t>(a.c.B, (2ll << 30) / std::max<int64_t>(per_seq, 1)));
    const int64_t items = nb * Hkv * p.pairs;
    if (items > INT32_MAX / 16 || nb * Hkv > 65535) {
        set_error("kv8_attention: too many work items");
        return -1;
    }
    // Parts of the keys, none shorter than 512 at full length. With an item for every SM the last ones, one for two SMs, go
    // in quarters. With fewer, all go in as many parts as make the shortest schedule: waves of parts of 1 / splits each, and
    // 0.04 of an item for a part's start and its share of the join (8192 cached tokens, us: 128 items in 1 / 2 / 4 parts
    // 166 / 180 / 192, 88 in 1 / 3 / 5 163 / 135 / 135, 32 in 1 / 4 / 16 148 / 75 / 90, 8 in 1 / 4 / 16 149 / 64 / 44).
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(p.Spad / 512, n_sm));
    auto plan = [&](int64_t n) {
        p.splits = (int)std::min<int64_t>(most, TAIL_SPLITS);
        if (n < n_sm) {
            double best = 1e30;
            for (int s = 1; s <= most; ++s) {
                const double cost = (double)((n * s + n_sm - 1) / n_sm) * (1.0 / s + 0.04);
                if (cost < best) {
                    best = cost;
                    p.splits = s;
                }
            }
        }
        p.tail = p.splits <= 1 ? 0 : n >= n_sm ? n_sm / 2 : (int)n;
        p.whole = (int)n - p.tail;
        return (int64_t)p.tail * p.splits;
    };
    // (the last launch may have fewer sequences)
    const int64_t parts = std::max(plan(items), a.c.B % nb ? plan(a.c.B % nb * Hkv * p.pairs) : 0);
    const int64_t heads = nb * Hkv;
    const int64_t b_kv = up(heads * p.Spad * D * 2), b_q = up(heads * p.Rpad * D * 2), b_s = up(heads * p.Spad), b_m = up(heads * p.Rpad * 4);
    const int64_t prows = parts * 2 * BM;
    const int64_t b_po = up(prows * D * 4), b_pm = up(prows * 8), b_o = up(nb * 4);
    char* mem = nullptr;
    if (cuda_failed(cudaMallocAsync((void**)&mem, 2 * b_kv + b_q + b_s + b_m + b_po + b_pm + b_o + 1024, st), "kv8_attention: scratch allocation"))
        return -1;
    char* at = mem;
    auto take = [&](int64_t n) { char* r = at; at += n; return (void*)r; };
    p.k16 = (__half*)take(b_kv);
    p.v16 = (__half*)take(b_kv);
    p.q16 = (__half*)take(b_q);
    p.scl = (float4*)take(b_s);
    p.qmul = (float*)take(b_m);
    p.part_o = (float*)take(b_po);
    p.part_ml = (float2*)take(b_pm);
    p.order = (int*)take(b_o);
    p.claim = (int*)take(1024);
    bool bad = false;
    for (int64_t b0 = 0; b0 < a.c.B && !bad; b0 += nb) {
        p.b0 = b0;
        p.nb = std::min(nb, a.c.B - b0);
        const int64_t h = p.nb * Hkv;
        CUtensorMap mq, mk, mv;
        if (!map_rows(&mq, p.q16, h, p.Rpad, D) || !map_rows(&mk, p.k16, h, p.Spad, D) || !map_rows(&mv, p.v16, h, p.Spad, D)) {
            bad = true;
            break;
        }
        plan(h * p.pairs);
        const dim3 grid((unsigned)(p.Spad / 64 + p.Rpad / 32 + 1), (unsigned)h);
        if (a.c.format == GTB_KV8_INT8) kv8_widen_kernel<GTB_KV8_INT8, D><<<grid, 256, 0, st>>>(p);
        else kv8_widen_kernel<GTB_KV8_E4M3, D><<<grid, 256, 0, st>>>(p);
        bad = cuda_failed(cudaGetLastError(), "kv8_attention: widen launch");
        if (bad) break;
        bad = !launch_behind("kv8_attention: chunk launch", kv8_chunk_kernel<D, GROUPS>,
                             dim3((unsigned)std::min<int64_t>(p.whole + (int64_t)p.tail * p.splits, n_sm)), NTHREADS, st, ChunkCfg<D>::SMEM,
                             mq, mk, mv, p);
        if (!bad && p.tail)
            bad = !launch_behind("kv8_attention: join launch", kv8_chunk_join_kernel<D>, dim3((unsigned)p.tail, 2 * BM / 8), 256, st, 0, p);
    }
    cudaFreeAsync(mem, st);
    return bad ? -1 : 0;
}

}  // namespace

bool chunk_supported(const Kv8AttnArgs& a) {
    const int64_t R = a.H / a.c.Hkv * a.Lq;
    return a.dtype != F32 && a.c.D <= 128 && R > CHUNK_ROWS && a.c.Smax > 0 && a.c.Hkv <= 65535 && R < (1 << 28) && encode_fn() != nullptr;
}

int launch_chunk(const Kv8AttnArgs& a, float* lse, int n_sm, cudaStream_t st) {
    switch (a.c.block) {
        case 16: return a.c.D <= 64 ? run<64, 8>(a, lse, n_sm, st) : run<128, 8>(a, lse, n_sm, st);
        case 32: return a.c.D <= 64 ? run<64, 4>(a, lse, n_sm, st) : run<128, 4>(a, lse, n_sm, st);
        case 64: return a.c.D <= 64 ? run<64, 2>(a, lse, n_sm, st) : run<128, 2>(a, lse, n_sm, st);
        default: return a.c.D <= 64 ? run<64, 1>(a, lse, n_sm, st) : run<128, 1>(a, lse, n_sm, st);
    }
}

}  // namespace kv8
}  // namespace gtb
