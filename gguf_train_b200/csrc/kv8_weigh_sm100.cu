// Accumulated attention weights of cached rows for many query rows, from the rows' log-sum-exp: tcgen05 tensor cores.
//   w[key] = sum over the kv head's rows r = i * G + g that see the key of 2^(s[key][r] - lse2[r]).
// A CTA takes 128 keys of one (sequence, kv head), makes their codes f16 once, and walks the query rows in tiles:
//   S^T (128 keys x NQ rows) = K (A, from shared memory) Q^T (B, a tile of rows that TMA brings).
// The keys are the TMEM lanes, so a thread sums one key's weights over the columns of every tile, in registers and in
// a fixed order. Two tiles are in flight, each with its own buffer and its own four warps, so the tensor core works on
// one while the other's exponentials run, and two CTAs share an SM where their tiles fit, so that one's start (codes
// to f16, first tile) hides behind the other. The exponentials, one per key and row at 16 a clock and SM, and the
// additions around them bound it where rows are many, a CTA's start where they are few. 1021 tokens x 32 heads of 128
// against 4 x 4k to 8k cached: 0.44 ms (0.58 with one CTA an SM); 36 rows a head, 16 sequences of 2k to 16k: 0.30 ms.
// q is brought to f16 as in kv8_mma.cuh, f32 q as two numbers whose products add up in the accumulator.

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

constexpr int BM = 128, NTHREADS = 384;

template <int DP, int NS>
struct WeighCfg {
    static constexpr int NQ = DP * NS <= 256 ? 128 : 64;    // rows of a tile
    static constexpr int KTILE = BM * DP * 2, KATOM = BM * 128;
    static constexpr int QPLANE = NQ * DP * 2, QATOM = NQ * 128, QTILE = QPLANE * NS;
    static constexpr int OFF_Q = KTILE, OFF_ROW = OFF_Q + 2 * QTILE;
    static constexpr int OFF_SUM = OFF_ROW + 8 * NQ * 8, OFF_BAR = OFF_SUM + BM * 4;
    static constexpr int SMEM = OFF_BAR + 9 * 8 + 16 + 1024;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static constexpr int CTAS = 2 * (SMEM + 1024) <= 228 * 1024 ? 2 : 1;  // an SM (each takes 256 columns of TMEM's 512)
};

struct WeighP {
    gtb_kv8 c;
    Rows3 q;
    int dtype, q_vec, G, R;
    int64_t b0, nb, H, Lq, Rpad;
    float scale_log2;
    const int32_t* counts;
    const float *lse, *score_in;
    float* score_out;
    __half* q16;     // [nb * Hkv][NS][Rpad][DP]
    float2* rowc;    // [nb * Hkv][Rpad]: q's multiplier, log2-sum-exp (+inf: no weight from this row)
    int* status;
};

// 32 rows of q a CTA; blockIdx.y = (sequence, kv head). Rows past the sequence's queries become zeros, whatever they hold:
// the weights kernel runs over them up to the end of a group of 32, and only a finite score plus -inf is weight 0.
template <int DP, int NS>
__global__ void __launch_bounds__(256) kv8_rows_kernel(const __grid_constant__ WeighP p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t lbh = blockIdx.y, b = p.b0 + lbh / p.c.Hkv, hk = lbh % p.c.Hkv;
    const int cnt = p.counts ? (int)clamp64(p.counts[b], 0, p.Lq) : (int)p.Lq;
    constexpr int PER = DP <= 128 ? 1 : 2;  // groups of four values a lane
    for (int k = 0; k < 4; ++k) {
        const int r = blockIdx.x * 32 + warp * 4 + k, i = r / p.G, h = (int)hk * p.G + (r - i * p.G);
        float x[PER][4], m = 0.0f;
#pragma unroll
        for (int w = 0; w < PER; ++w) {
            const int d = lane * 4 + w * 128;
            load_q4(p, b * p.q.sb + h * p.q.sh + (int64_t)i * p.q.ss + d, r < p.R && i < cnt && d < p.c.D, x[w]);
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, finite_abs(x[w][e]));
        }
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        int e2 = (int)(__float_as_uint(m) >> 23) - 127;
        e2 = m >= 1.17549435e-38f ? min(max(e2, -126), 126) : 0;
        const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
        for (int w = 0; w < PER; ++w) {
            const int d = lane * 4 + w * 128;
            if (d >= DP) continue;
            const float y0 = x[w][0] * down, y1 = x[w][1] * down, y2 = x[w][2] * down, y3 = x[w][3] * down;
            const uint32_t a = pack_f16(y0, y1), c = pack_f16(y2, y3);
            *(uint2*)(p.q16 + ((lbh * NS) * p.Rpad + r) * DP + d) = make_uint2(a, c);
            if constexpr (NS == 2) {
                const float2 fa = unpack_f16(a), fc = unpack_f16(c);
                *(uint2*)(p.q16 + ((lbh * NS + 1) * p.Rpad + r) * DP + d) =
                    make_uint2(pack_f16(y0 - fa.x, y1 - fa.y), pack_f16(y2 - fc.x, y3 - fc.y));
            }
        }
        if (lane == 0) {
            float z = INFINITY;
            if (r < p.R && i < cnt) {
                z = p.lse[(b * p.H + h) * p.Lq + i] * 1.4426950408889634f;
                if (z == -INFINITY) z = INFINITY;
            }
            p.rowc[lbh * p.Rpad + r] = make_float2(__uint_as_float((uint32_t)(127 + e2) << 23) * p.scale_log2, z);
        }
    }
}

template <int DP, int FMT, int NS>
__global__ void __launch_bounds__(NTHREADS, WeighCfg<DP, NS>::CTAS) kv8_weigh_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ WeighP p) {
    using C = WeighCfg<DP, NS>;
    constexpr int NQ = C::NQ;
    const int per_head = (int)((p.c.Smax + BM - 1) / BM);
    const int lbh = (int)(blockIdx.x / (unsigned)per_head), k0 = (int)(blockIdx.x - (unsigned)lbh * per_head) * BM;
    const int64_t b = p.b0 + lbh / p.c.Hkv, bh = b * p.c.Hkv + lbh % p.c.Hkv;
    const int len = (int)clamp64(p.c.lens[b], 0, p.c.Smax);
    const int cnt = p.counts ? (int)clamp64(p.counts[b], 0, p.Lq) : (int)p.Lq;
    if (k0 >= len) {
        cudaGridDependencySynchronize();
        return;
    }
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float2* rows = (float2*)(smem + C::OFF_ROW);   // [8][NQ]: a tile's rows, for each of the eight warps
    float* half_sum = (float*)(smem + C::OFF_SUM);  // [128]
    uint64_t* bars = (uint64_t*)(smem + C::OFF_BAR);
    uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *s_free = bars + 6, *drain = bars + 8;
    uint32_t* tmem_slot = (uint32_t*)(bars + 9);
    int* abort_flag = (int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // row tiles that see a key of this block: row i of the queries sees keys up to len - cnt + i
    const int first_row = max(0, k0 - (len - cnt)) * p.G, rows_end = min(p.R, cnt * p.G);
    const int t0 = first_row / NQ, n_tiles = max(0, (rows_end + NQ - 1) / NQ - t0);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 4);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, 256);
    // the keys as an f16 tile in 128-byte-swizzled slabs of 64 dims
    constexpr int CPR = DP / 8;
    for (int e = threadIdx.x; e < BM * CPR; e += NTHREADS) {
        const int row = e / CPR, ch = e % CPR;
        uint2 w = make_uint2(0, 0);
        if (k0 + row < len && ch * 8 < p.c.D) w = *(const uint2*)((const uint8_t*)p.c.k + (bh * p.c.Smax + k0 + row) * p.c.D + ch * 8);
        const uint32_t u0 = prep_word<FMT>(w.x), u1 = prep_word<FMT>(w.y);
        *(uint4*)(smem + (ch >> 3) * C::KATOM + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) =
            make_uint4(expand<FMT, 0>(u0), expand<FMT, 1>(u0), expand<FMT, 0>(u1), expand<FMT, 1>(u1));
    }
    fence_proxy_async_smem();
    cudaGridDependencySynchronize();  // the rows are there
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            prefetch_tmap(&tmQ);
            bool ok = true;
            int n = 0;
            for (; n < n_tiles; ++n) {
                const int s = n & 1;
                if (n >= 2) ok = mbar_wait(&q_empty[s], ((n >> 1) - 1) & 1, p.status, 141);
                if (!ok || *(volatile int*)abort_flag) { ok = false; break; }
                mbar_expect_tx(&q_full[s], C::QTILE);
                for (int z = 0; z < NS; ++z)
                    for (int a = 0; a < DP / 64; ++a)
                        tma_load_4d(smem + C::OFF_Q + s * C::QTILE + z * C::QPLANE + a * C::QATOM, &tmQ, a * 64,
                                    (int)(z * p.Rpad) + (t0 + n) * NQ, lbh, 0, &q_full[s]);
            }
            if (!ok) *(volatile int*)abort_flag = 1;
            if (*(volatile int*)abort_flag)
                for (int j = max(0, n - 2); j < n; ++j) mbar_wait(&q_full[j & 1], (j >> 1) & 1, nullptr, 0);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t IDESC = idesc_f16(BM, NQ, false, false);
            const uint64_t kd = desc_sw128(smem_u32(smem), 16, 1024);
            bool ok = true;
            for (int n = 0; n < n_tiles; ++n) {
                const int s = n & 1;
                ok = mbar_wait(&q_full[s], (n >> 1) & 1, p.status, 142);
                if (ok && n >= 2) ok = mbar_wait(&s_free[s], ((n >> 1) - 1) & 1, p.status, 143);
                if (!ok || *(volatile int*)abort_flag) { ok = false; break; }
                tc_fence_after();
                const uint64_t qd = desc_sw128(smem_u32(smem + C::OFF_Q + s * C::QTILE), 16, 1024);
#pragma unroll
                for (int z = 0; z < NS; ++z)
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(tmem + s * 128u, desc_advance(kd, (uint32_t)((k / 4) * C::KATOM + (k % 4) * 32)),
                               desc_advance(qd, (uint32_t)(z * C::QPLANE + (k / 4) * C::QATOM + (k % 4) * 32)), IDESC, z > 0 || k > 0 ? 1u : 0u);
                mma_commit(&s_full[s]);
                mma_commit(&q_empty[s]);
            }
            if (!ok) *(volatile int*)abort_flag = 1;
            if (*(volatile int*)abort_flag) {
                mma_commit(drain);
                mbar_wait(drain, 0, nullptr, 0);
            }
        }
    } else if (warp >= 4) {
        const int wg = (warp - 4) >> 2, quad = warp & 3, t = threadIdx.x & 127, key = k0 + quad * 32 + lane;
        const uint32_t s_tmem = tmem + ((uint32_t)(quad * 32) << 16) + wg * 128u;
        const int shift = 31 - __clz(p.c.block);
        const float sk = key < len ? p.c.k_scale[bh * ((p.c.Smax + p.c.block - 1) >> shift) + (key >> shift)] : 0.0f;
        const uint64_t sk2 = f2_pack(sk, sk);
        float2* mine = rows + (warp - 4) * NQ;
        uint64_t sum2[2] = {0ull, 0ull};
        bool ok = true;
        for (int n = wg; n < n_tiles; n += 2) {
            const int row0 = (t0 + n) * NQ;
            // multiplier and -lse2 of the tile's rows
            for (int r = lane; r < NQ; r += 32) {
                const float2 z = p.rowc[(int64_t)lbh * p.Rpad + row0 + r];
                mine[r] = make_float2(z.x, -z.y);
            }
            __syncwarp();
            ok = mbar_wait(&s_full[wg], (n >> 1) & 1, p.status, 144);
            ok = __all_sync(0xffffffffu, ok) && !__any_sync(0xffffffffu, *(volatile int*)abort_flag);
            if (!ok) break;
            tc_fence_after();
            const bool edge = k0 + BM - 1 > len - cnt + row0 / p.G;  // some key past the first row's last
            const int chunks = min(NQ / 32, (rows_end - row0 + 31) / 32);  // with a row in them
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
                uint32_t raw[32];
                tmem_ld32(s_tmem + c * 32, raw);
                tmem_ld_wait();
                if (c == chunks - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[wg]);
                }
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (key > len - cnt + (row0 + c * 32 + e) / p.G) raw[e] = 0xff800000u;  // -inf
                }
                const float4* rc = (const float4*)(mine + c * 32);
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float4 z = rc[e >> 1];  // two rows: multiplier, -lse2 each
                    // a masked score times a multiplier of 0 would be NaN
                    const uint64_t mul = f2_mul(f2_pack(z.x, z.z), sk2);
                    float m0, m1, a0, a1;
                    f2_unpack(mul, m0, m1);
                    a0 = fmaf(__uint_as_float(raw[e]), fmaxf(m0, 1e-37f), z.y);
                    a1 = fmaf(__uint_as_float(raw[e + 1]), fmaxf(m1, 1e-37f), z.w);
                    sum2[(e >> 1) & 1] = f2_add(sum2[(e >> 1) & 1], f2_pack(ex2(a0), ex2(a1)));
                }
            }
            __syncwarp();  // every lane is through with the table
        }
        float a, b2, c2, d;
        f2_unpack(sum2[0], a, b2);
        f2_unpack(sum2[1], c2, d);
        const float w = (a + b2) + (c2 + d);
        if (!ok) *(volatile int*)abort_flag = 1;
        if (wg == 1) half_sum[t] = w;
        asm volatile("bar.sync 3, 256;" ::: "memory");
        if (wg == 0 && key < len && ok) {
            const int64_t at = bh * p.c.Smax + key;
            p.score_out[at] = p.score_in[at] + (w + half_sum[t]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 256);
    }
}

template <int DP, int FMT, int NS>
int run(const Kv8AttnArgs& a, const float* lse, cudaStream_t st) {
    using C = WeighCfg<DP, NS>;
    auto kern = kv8_weigh_kernel<DP, FMT, NS>;
    static std::atomic<uint64_t> ready{0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM), "kv8_attention: shared memory"))
            return -1;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    WeighP p{};
    p.c = a.c;
    p.q = a.q;
    p.dtype = a.dtype;
    p.q_vec = vector_rows(a.q, a.dtype);
    p.G = (int)(a.H / a.c.Hkv);
    p.R = p.G * (int)a.Lq;
    p.H = a.H;
    p.Lq = a.Lq;
    p.Rpad = ((int64_t)p.R + 127) / 128 * 128;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.counts = a.counts;
    p.lse = lse;
    p.score_in = a.score_in;
    p.score_out = a.score_out;
    p.status = device_status_word(dev);
    // scratch of one sequence; as many sequences a launch as stay within 1 GB (one at least)
    const int64_t Hkv = a.c.Hkv, per_seq = Hkv * p.Rpad * (DP * 2 * NS + 8);
    const int64_t nb = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(a.c.B, 65535 / Hkv), (1ll << 30) / per_seq));
    const int64_t b_q = (nb * Hkv * p.Rpad * DP * 2 * NS + 1023) / 1024 * 1024, per_head = (a.c.Smax + BM - 1) / BM;
    if (nb * Hkv * per_head > INT32_MAX) {
        set_error("kv8_attention: too many cached rows");
        return -1;
    }
    char* mem = nullptr;
    if (cuda_failed(cudaMallocAsync((void**)&mem, b_q + nb * Hkv * p.Rpad * 8, st), "kv8_attention: scratch allocation")) return -1;
    p.q16 = (__half*)mem;
    p.rowc = (float2*)(mem + b_q);
    bool bad = false;
    for (int64_t b0 = 0; b0 < a.c.B && !bad; b0 += nb) {
        p.b0 = b0;
        p.nb = std::min(nb, a.c.B - b0);
        const int64_t h = p.nb * Hkv;
        gtb_tensor4 t{};
        t.data = p.q16;
        t.shape[0] = 1; t.shape[1] = h; t.shape[2] = NS * p.Rpad; t.shape[3] = DP;
        t.stride[0] = h * NS * p.Rpad * DP; t.stride[1] = NS * p.Rpad * DP; t.stride[2] = DP; t.stride[3] = 1;
        t.dtype = F16;
        CUtensorMap mq;
        if (!make_tma_map_4d(&mq, t, DP, false, C::NQ)) {
            bad = true;
            break;
        }
        kv8_rows_kernel<DP, NS><<<dim3((unsigned)(p.Rpad / 32), (unsigned)h), 256, 0, st>>>(p);
        bad = cuda_failed(cudaGetLastError(), "kv8_attention: rows launch") ||
              !launch_behind("kv8_attention: weigh launch", kern, dim3((unsigned)(h * per_head)), NTHREADS, st, C::SMEM, mq, p);
    }
    cudaFreeAsync(mem, st);
    return bad ? -1 : 0;
}

template <int DP>
int run_d(const Kv8AttnArgs& a, const float* lse, cudaStream_t st) {
    const bool e4m3 = a.c.format == GTB_KV8_E4M3;
    if (a.dtype == F32) return e4m3 ? run<DP, GTB_KV8_E4M3, 2>(a, lse, st) : run<DP, GTB_KV8_INT8, 2>(a, lse, st);
    return e4m3 ? run<DP, GTB_KV8_E4M3, 1>(a, lse, st) : run<DP, GTB_KV8_INT8, 1>(a, lse, st);
}

}  // namespace

int launch_weigh(const Kv8AttnArgs& a, const float* lse, cudaStream_t st) {
    if (!encode_fn()) {
        set_error("kv8_attention: cuTensorMapEncodeTiled is unavailable");
        return -1;
    }
    if (a.c.Hkv > 65535) {
        set_error("kv8_attention: the weights take at most 65535 kv heads");
        return -1;
    }
    return a.c.D <= 64 ? run_d<64>(a, lse, st) : a.c.D <= 128 ? run_d<128>(a, lse, st) : run_d<256>(a, lse, st);
}

}  // namespace kv8
}  // namespace gtb
