// Attention over the block-scaled 8-bit cache for few query rows, on warp-level matrix instructions.
//
// One work item is 8 * NT query rows of one (sequence, kv head): the G = H / Hkv query heads times the Lq
// queries, row = i * G + g. The keys are cut into units of 16 or 32; all units of all items form one line, of which
// every warp takes an equal stretch (so the split adapts to the lengths and no warp waits for another). A
// warp that finishes an item alone writes the result; otherwise it leaves (out, max, sum) for
// kv8_finish_kernel.
//
// Where the cache is short and the items few (one_cta()), a CTA takes an item instead: its warps take its units in turn
// and meet in shared memory, and everything is done in one launch.
//
// A warp streams its units through its own ring in shared memory with 16-byte asynchronous copies (rows
// past the length arrive as zeros: nothing stored there can reach a result). Codes become f16 in registers,
// exactly (int8 and e4m3 both fit), and feed mma.m16n8k16 as the A operand:
//   S^T (16 keys x 8 rows) = K (keys x D) Q^T;   O^T (16 dims x 8 rows) += V^T (dims x keys) P^T.
// The dimensions (first product) and keys (second) of an operand may be taken in any order as long as both
// operands agree, so a thread reads 16 consecutive bytes of a row and calls them the elements its lane owns;
// only P^T has to change layout (movmatrix, two per 16 keys and 8 rows).
// * Scales: K's block scale multiplies the scores. V's is folded into the exponent, P' = 2^(s + log2 sv - M), so
//   the second product accumulates across blocks without rescaling; the row sum takes P' / sv. sv below 2^-80 (zero
//   above all: a block of zeros) counts as 2^-80: P' stays below 2^15, so no sum over 2^30 rows passes 2^125.
// * q becomes f16 after a power of two per row brings its largest value to [1, 2): bf16's 8 bits fit, and what
//   falls below f16's smallest step is 2^-24 of that value. f32 q is split into two f16 numbers (NS = 2), and
//   so is P', which is otherwise rounded to f16 once.
// * One tile of 8 rows of 16-bit q over int8 codes (QINT) takes the codes as they are: that q times 2^29 is an integer of
//   four digits to base 256 (what falls below its step is 2^-30 of the row's largest value), and
//   mma.m16n8k32 sums each digit's products exactly. The last digit is 0 in rows whose values all end at 2^-21 of the
//   largest, most of them, and is multiplied only where it is not. K's codes then need no conversion, 5 instructions in 4 of
//   them. Against f16 products, us: 64 sequences of 1k to 32k tokens called in a row 455 / 419 (f16 q, whose rows have a
//   last digit more often, 455 / 433), where power, and with it instructions, sets the clock, but 393 / 412 at full
//   clock; 16 of them 123 / 128, 16 with weights 94 / 90.
// * M is raised only when a score exceeds it by 2^7 (P' carries a factor 2^8 and f16 ends at 2^16), so most
//   units need neither shuffles nor a rescaling of O.
#pragma once

#include <algorithm>
#include <atomic>

#include "gtb_common.cuh"
#include "kv8.cuh"

namespace gtb {
namespace kv8 {

constexpr float SV_MIN = 0x1p-80f;
constexpr float RAISE = 7.0f, SHIFT = 8.0f, NONE = -3.402823466e38f;  // NONE: no key seen yet (finite: -inf - NONE is -inf)

struct MmaP {
    gtb_kv8 c;
    Rows3 q, o;
    int dtype, q_vec;
    int G, R, row_tiles;      // R = G * Lq rows per (b, hk), in tiles of 8 * NT
    int64_t H, Lq;
    float scale_log2;         // scale * log2(e)
    const int32_t* counts;
    float* lse;               // nullable
    int2* meta;               // per item: first and last warp that holds a part of it
    float* part_o;            // [slot][8 NT][DP]
    float2* part_ml;          // [slot][8 NT]
    const float* score_in;    // nullable, with score_out: the rows' weights are wanted (one row tile)
    float* score_out;
    float* s_out;             // then: scores (log2 units) [b, hk][key][R]
    int one;                  // a CTA per item
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
    const int n = live ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool live) {
    const int n = live ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16832(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2f(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }

// The four codes of a word as two f16 pairs: bytes (0, 1) and (2, 3). int8: with the sign bit flipped a code is
// an unsigned byte u = q + 128, the bits 0x6400 | u are the f16 number 1024 + u, and 1152 comes off exactly.
template <int FMT>
__device__ __forceinline__ uint32_t prep_word(uint32_t w) {
    return FMT == GTB_KV8_INT8 ? w ^ 0x80808080u : w;
}
template <int FMT, int HALF>
__device__ __forceinline__ uint32_t expand(uint32_t w) {
    if constexpr (FMT == GTB_KV8_INT8) {
        const uint32_t t = __byte_perm(w, 0x64646464u, HALF ? 0x4342 : 0x4140);
        const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&t), __half2half2(__ushort_as_half(0xE480)));  // -1152
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        uint32_t r;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)(HALF ? w >> 16 : w)));
        return r;
    }
}

// Which bytes a lane (g = lane / 4, t = lane % 4) owns. K: for load q, 16 bytes of row g: chunk k_chunk(t, q).
// V: of its four keys (2t, 2t+1, 8+2t, 9+2t in the 16), V_BYTES bytes from v_byte(g, u). Rows of 16-byte chunks
// are stored with chunk c of row r at c ^ swz(r), keys at row krow(key), chosen so that the eight lanes of a
// 16-byte access (sixteen of an 8-byte one) fall into different banks for both reads.
template <int DP>
struct Lay;
template <>
struct Lay<64> {
    static constexpr int KL = 1, VL = 1, V_BYTES = 8;
    __device__ static int k_chunk(int t, int) { return t; }
    __device__ static int v_byte(int g, int) { return 8 * g; }
    __device__ static int krow(int k) { return k ^ ((k >> 1) & 1); }
    __device__ static int swz(int r) { return ((r >> 2) & 1) << 1; }
};
template <>
struct Lay<128> {
    static constexpr int KL = 2, VL = 1, V_BYTES = 16;
    __device__ static int k_chunk(int t, int q) { return 2 * t + q; }
    __device__ static int v_byte(int g, int) { return 16 * g; }
    __device__ static int krow(int k) { return k; }
    __device__ static int swz(int r) { return r & 7; }
};
template <>
struct Lay<256> {
    static constexpr int KL = 4, VL = 2, V_BYTES = 16;
    __device__ static int k_chunk(int t, int q) { return t + 4 * q; }
    __device__ static int v_byte(int g, int u) { return 16 * g + 128 * u; }
    __device__ static int krow(int k) { return k; }
    __device__ static int swz(int r) { return (r & 6) ^ ((r & 1) << 2); }
};

// Four values of a query row as f32, 0 where it has none; in one load where every row starts on 16 (f32) or 8 bytes
template <typename P>
__device__ __forceinline__ void load_q4(const P& p, int64_t at, bool live, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = 0.0f;
    if (!live) return;
    if (p.q_vec) {
        if (p.dtype == F32) {
            const float4 v = *(const float4*)((const float*)p.q.p + at);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
            const uint2 v = *(const uint2*)((const uint16_t*)p.q.p + at);
            if (p.dtype == BF16) {
                x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
                x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
            } else {
                const float2 a = unpack_f16(v.x), b = unpack_f16(v.y);
                x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
            }
        }
    } else {
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
            const float v = load_any<float>(p.q.p, at + e, p.dtype);
            if (e == 0) x[0] = v;
            else if (e == 1) x[1] = v;
            else if (e == 2) x[2] = v;
            else x[3] = v;
        }
    }
}

// Units, warps and stages. More warps hide the dependent chain of a unit (scores, exponentials, second product); their
// number is what the registers (O alone takes NT DP / 4) and two stages of each warp's ring allow: 64 sequences of 1k to 32k
// tokens, 32 heads of 128 over 8, with 12 warps of 168 registers 0.42 ms, with 8 0.48 ms; 16 of 128 are slower again.
// A unit of two products halves the waits and joins a key, where its scores fit into the registers left and the ring keeps
// its warps. One / two products, us, 32 sequences of 100 to 8k tokens (G = 4; e4m3, 64-token blocks):
//   heads of 64, bf16: 8 rows 44.8 / 41.8, 16 62.5 / 54.6, 24 76.0 / 66.7, 32 94.2 / 111;   f32: 24 83.6 / 80.3, 32 101 / 133
//   128, bf16: 12 rows 86.3 / 89.1, 20 126 / 119, 32 156 / 150;   f32: 8 rows 73.2 / 67.9, 16 94.0 / 94.4, 20 137 / 145
//   256, bf16: 8 rows 132 / 137, 16 171 / 218
// and 8 rows of 128 in bf16, with q in registers, for the 64 sequences above: int8 380 / 409 at full clock but 439 / 408 called
// in a row, where the power cap lowers it and fewer instructions count, and 95 / 91 for 16 sequences with weights; e4m3
// 393 / 396 and 406 / 389, but 87 / 91 for 16 sequences with weights, so one there.
template <int DP, int FMT, int NT, int NS>
struct MmaCfg {
    static constexpr bool QREG = NT * NS == 1 && DP <= 128;         // q in registers
    static constexpr bool QINT = QREG && FMT == GTB_KV8_INT8;       // as integers
    static constexpr int KSTEPS = DP / 16;
    static constexpr int OREGS = NT * DP / 4;
    static constexpr bool PAIR = OREGS <= 64 ? OREGS <= 16 || (OREGS <= 48 && (!QREG || QINT)) : NS == 1 && DP <= 128;
    static constexpr int SUB = PAIR ? 2 : 1;          // 16-key products per unit
    static constexpr int UNIT = 16 * SUB;
    static constexpr int STAGE = 2 * UNIT * DP + 16;  // K rows, V rows, scales (k, v of each 16 keys)
    static constexpr int QBYTES = QINT ? KSTEPS * 128 : QREG ? 0 : KSTEPS * NT * NS * 32 * 8 + NT * 32;
    static constexpr int SPACE = 224 * 1024, MOST12 = 64;
    static constexpr int fit(int warps) { return (SPACE / warps - QBYTES) / STAGE; }
    static constexpr int pick() {
        const int most = OREGS <= 16 ? 16 : OREGS <= MOST12 ? 12 : 8;
        for (int w = most; w > 4; w -= 2)
            if (fit(w) >= 2) return w;
        return 4;
    }
    static constexpr int WARPS = pick();
    static constexpr int STAGES = fit(WARPS) > 6 ? 6 : fit(WARPS);
    static_assert(STAGES >= 2, "a stage in work and one in flight");
    static constexpr int WARP_SMEM = STAGES * STAGE + QBYTES;
    static constexpr int SMEM = WARPS * WARP_SMEM;
    static_assert(WARP_SMEM >= 8 * NT * (DP * 4 + 8), "a warp's results fit where its ring was");
};

template <int DP, int FMT, int NT, int NS>
__global__ void __launch_bounds__(MmaCfg<DP, FMT, NT, NS>::WARPS * 32, 1) kv8_mma_kernel(const __grid_constant__ MmaP p) {
    using C = MmaCfg<DP, FMT, NT, NS>;
    using L = Lay<DP>;
    constexpr int ROWS = 8 * NT, OM = DP / 16, SUB = C::SUB, UNIT = C::UNIT;  // OM: products of 16 dims
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int64_t seg[C::WARPS * 32 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const gtb_kv8& c = p.c;
    const int per_seq = (int)c.Hkv * p.row_tiles;
    cudaTriggerProgrammaticLaunchCompletion();

    auto len_of = [&](int64_t b) { return (int)clamp64(c.lens[b], 0, c.Smax); };
    auto units_in = [&](int len) { return max(1, (len + UNIT - 1) / UNIT); };

    struct Cursor {
        int b, len, units, item, unit;
    };
    Cursor wk;
    int64_t U = 0, NW = 0, wid = 0, u0 = 0;
    int n_units;
    const int step = p.one ? C::WARPS : 1;
    if (p.one) {
        wk.b = (int)blockIdx.x / per_seq;
        wk.item = (int)blockIdx.x - wk.b * per_seq;
        wk.len = len_of(wk.b);
        wk.units = units_in(wk.len);
        wk.unit = warp;
        n_units = warp < wk.units ? (wk.units - 1 - warp) / C::WARPS + 1 : 0;
    } else {
        // units before each thread's share of the sequences
        const int64_t share = (c.B + blockDim.x - 1) / blockDim.x;
        int64_t n = 0;
        for (int64_t b = threadIdx.x * share; b < min(c.B, (threadIdx.x + 1) * share); ++b) n += units_in(len_of(b));
        int64_t x = n;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __shared__ int64_t wsum[C::WARPS];
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        int64_t before = 0;
        for (int w = 0; w < warp; ++w) before += wsum[w];
        seg[threadIdx.x + 1] = (before + x) * per_seq;
        if (threadIdx.x == 0) seg[0] = 0;
        __syncthreads();
        U = seg[blockDim.x];
        // no more warps than units, so that every warp below NW has some; neighbours in different CTAs
        NW = min((int64_t)gridDim.x * C::WARPS, U);
        wid = (int64_t)warp * gridDim.x + blockIdx.x;
        if (wid >= NW) return;
        u0 = wid * U / NW;
        n_units = (int)((wid + 1) * U / NW - u0);
        // where unit u0 is: its sequence, the item in it, the unit in the item
        int lo = 0, hi = blockDim.x;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (seg[mid] <= u0) lo = mid;
            else hi = mid;
        }
        wk.b = (int)(lo * share);
        int64_t base = seg[lo];
        wk.len = len_of(wk.b);
        for (;;) {
            const int64_t all = (int64_t)units_in(wk.len) * per_seq;
            if (base + all > u0) break;
            base += all;
            wk.len = len_of(++wk.b);
        }
        wk.units = units_in(wk.len);
        wk.item = (int)((u0 - base) / wk.units);
        wk.unit = (int)((u0 - base) - (int64_t)wk.item * wk.units);
    }
    Cursor ld = wk;
    // to the next unit; whether that is in another item
    auto advance = [&](Cursor& k) {
        k.unit += step;
        if (k.unit < k.units || p.one) return false;
        k.unit = 0;
        if (++k.item == per_seq) {
            k.item = 0;
            if (++k.b < c.B) {
                k.len = len_of(k.b);
                k.units = units_in(k.len);
            }
        }
        return true;
    };

    unsigned char* ws = smem + warp * C::WARP_SMEM;
    const uint32_t ring = smem_addr(ws);
    uint2* qf = (uint2*)(ws + C::STAGES * C::STAGE);  // B operands of the rows, then their multipliers
    uint32_t* q_last = (uint32_t*)qf;                  // (QINT) or the last digits
    float* qm = (float*)(qf + C::KSTEPS * NT * NS * 32);
    const int64_t nblk = (c.Smax + c.block - 1) / c.block;
    const int block_shift = 31 - __clz(c.block);

    // copies of unit `ld` into a stage, a row's chunk a lane
    constexpr int CPR = DP / 16, RPI = 32 / CPR;  // chunks of a row, rows a warp instruction copies
    const int cc = lane % CPR, rl = lane / CPR;
    const uint32_t lane_row = L::krow(rl & 7) * DP, lane_swz = (uint32_t)(cc ^ L::swz(L::krow(rl & 7))) << 4;
    int64_t ld_head = 0;                          // (sequence, kv head) of the item
    auto enter = [&]() { ld_head = (int64_t)ld.b * c.Hkv + ld.item / p.row_tiles; };
    enter();
    auto issue = [&](int stage) {
        const int k0 = ld.unit * UNIT;
        const int64_t off = (ld_head * c.Smax + k0 + rl) * c.D + cc * 16;
        const uint32_t dst = ring + stage * C::STAGE + lane_row;
        if (k0 + UNIT <= ld.len && c.D == DP) {
            const unsigned char *gk = (const unsigned char*)c.k + off, *gv = (const unsigned char*)c.v + off;
#pragma unroll
            for (int r0 = 0; r0 < UNIT; r0 += RPI) {
                // (swz of a sum of rows whose bits do not meet is the xor of theirs)
                const uint32_t at = dst + r0 * DP + (lane_swz ^ (uint32_t)(RPI < 8 ? L::swz(r0 & 7) << 4 : 0));
                cp16(at, gk + r0 * DP, true);
                cp16(at + UNIT * DP, gv + r0 * DP, true);
            }
        } else {
#pragma unroll 1
            for (int r0 = 0; r0 < UNIT; r0 += RPI) {
                const bool live = k0 + r0 + rl < ld.len && cc * 16 < c.D;
                const int64_t o = live ? off + (int64_t)r0 * c.D : 0;
                const uint32_t at = dst + r0 * DP + (lane_swz ^ (uint32_t)(RPI < 8 ? L::swz(r0 & 7) << 4 : 0));
                cp16(at, (const unsigned char*)c.k + o, live);
                cp16(at + UNIT * DP, (const unsigned char*)c.v + o, live);
            }
        }
        if (lane < 2 * SUB) {
            const int k = k0 + (lane % SUB) * 16;
            const bool live = k < ld.len;
            const float* s = lane < SUB ? c.k_scale : c.v_scale;
            cp4(ring + stage * C::STAGE + 2 * UNIT * DP + lane * 4, live ? s + ld_head * nblk + (k >> block_shift) : s, live);
        }
        if (advance(ld)) enter();
    };

#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) {
        if (s < n_units) issue(s);
        cp_commit();
    }

    // state of the current item
    float o[NT][OM][4];
    float M[NT][2], l[NT][2], qmul[NT][2];
    int lim[NT][2];                  // keys each row may attend
    int lim_min = 0;                 // smallest over the tile's rows
    constexpr int QWORDS = C::QINT ? 3 : 2;
    uint32_t qr[C::QREG ? C::KSTEPS : 1][QWORDS];
    bool last_digit = false;         // (QINT) whether some row's is not 0
    bool fresh = true, head_split = !p.one && wk.unit != 0;

    int stage = 0;
    for (int it = 0; it < n_units; ++it) {
        if (fresh) {  // a new item: its query rows, normalised by a power of two, as B operands
            fresh = false;
            const int hk = wk.item / p.row_tiles, tile = wk.item - hk * p.row_tiles;
            const int cnt = p.counts ? (int)clamp64(p.counts[wk.b], 0, p.Lq) : (int)p.Lq;
            float row_mul = 0.0f;  // (QREG) of row g
#pragma unroll 1
            for (int n = 0; n < NT; ++n) {
                const int r = tile * ROWS + n * 8 + g, i = r / p.G, h = hk * p.G + (r - i * p.G);
                const int64_t at = wk.b * p.q.sb + h * p.q.sh + i * p.q.ss;
                float x[C::KSTEPS][4], m = 0.0f;
#pragma unroll
                for (int k = 0; k < C::KSTEPS; ++k) {
                    const int d = L::k_chunk(t, k >> 2) * 16 + (k & 3) * 4;
                    load_q4(p, at + d, r < p.R && d < c.D, x[k]);
                }
#pragma unroll
                for (int k = 0; k < C::KSTEPS; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m = fmaxf(m, finite_abs(x[k][e]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                // 2^e <= m < 2^(e+1); a row of zeros or subnormals stays as it is
                int e2 = (int)(__float_as_uint(m) >> 23) - 127;
                e2 = m >= 1.17549435e-38f ? min(max(e2, -126), 126) : 0;
                const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
                const float mul = __uint_as_float((uint32_t)(127 + e2) << 23) * p.scale_log2;
                if constexpr (C::QINT) {
                    // digits of y 2^29 to base 256, -128 to 127 each, a plane a digit; a row with a value that is not finite
                    // is NaN throughout
                    bool odd = false;
                    uint32_t any = 0;
                    const float lift = m < 0x1p127f ? 0x1p29f : 0x1p28f;  // `down` ends at 2^-126: y may reach 4 there
#pragma unroll
                    for (int k = 0; k < C::KSTEPS; ++k) {
                        uint32_t low = 0;
                        qr[k][0] = qr[k][1] = qr[k][QWORDS - 1] = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool finite = fabsf(x[k][e]) <= 3.402823466e38f;
                            odd |= !finite;
                            const int z = finite ? __float2int_rn(x[k][e] * down * lift) : 0;
                            // z = ((z3 256 + low(z2)) 256 + low(z1)) 256 + low(z)
                            const int z1 = (z + 128) >> 8, z2 = (z1 + 128) >> 8, z3 = (z2 + 128) >> 8;
                            qr[k][0] |= (uint32_t)(z3 & 255) << (8 * e);
                            qr[k][1] |= (uint32_t)(z2 & 255) << (8 * e);
                            qr[k][QWORDS - 1] |= (uint32_t)(z1 & 255) << (8 * e);
                            low |= (uint32_t)(z & 255) << (8 * e);
                        }
                        q_last[k * 32 + lane] = low;  // (a lane reads its own)
                        any |= low;
                    }
                    last_digit = __any_sync(0xffffffffu, any != 0);
                    const unsigned rows_odd = __ballot_sync(0xffffffffu, odd);
                    row_mul = rows_odd >> (lane & 28) & 15u ? __uint_as_float(0x7fc00000u) : mul * 256.0f / lift;
                    continue;
                }
                if constexpr (C::QREG) row_mul = mul;
                else if (t == 0) qm[n * 8 + g] = mul;
#pragma unroll
                for (int k = 0; k < C::KSTEPS; ++k) {
                    const float y0 = x[k][0] * down, y1 = x[k][1] * down, y2 = x[k][2] * down, y3 = x[k][3] * down;
                    const uint32_t b0 = pack_f16(y0, y1), b1 = pack_f16(y2, y3);
                    if constexpr (C::QREG) {
                        qr[k][0] = b0;
                        qr[k][1] = b1;
                    } else {
                        qf[((k * NT + n) * NS) * 32 + lane] = make_uint2(b0, b1);
                        if constexpr (NS == 2) {
                            const float2 f0 = unpack_f16(b0), f1 = unpack_f16(b1);
                            qf[((k * NT + n) * NS + 1) * 32 + lane] = make_uint2(pack_f16(y0 - f0.x, y1 - f0.y), pack_f16(y2 - f1.x, y3 - f1.y));
                        }
                    }
                }
            }
            __syncwarp();
            lim_min = 1 << 30;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    qmul[n][e] = C::QREG ? __shfl_sync(0xffffffffu, row_mul, (2 * t + e) * 4) : qm[n * 8 + 2 * t + e];
                    const int r = tile * ROWS + n * 8 + 2 * t + e, i = r / p.G;
                    lim[n][e] = r < p.R && i < cnt ? max(0, wk.len - cnt + i + 1) : 0;
                    if (r < p.R) lim_min = min(lim_min, lim[n][e]);
                    M[n][e] = NONE;
                    l[n][e] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < OM; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][j][e] = 0.0f;
            }
            lim_min = __reduce_min_sync(0xffffffffu, lim_min);
        }

        if (it + C::STAGES - 1 < n_units) issue(stage == 0 ? C::STAGES - 1 : stage - 1);
        cp_commit();
        cp_wait<C::STAGES - 1>();
        __syncwarp();

        const unsigned char* kt = ws + stage * C::STAGE;
        const unsigned char* vt = kt + UNIT * DP;
        const float* scales = (const float*)(kt + 2 * UNIT * DP);
        const int k0 = wk.unit * UNIT;

        // S^T of the unit's keys
        float s[SUB][NT][4];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[u][n][e] = 0.0f;
            const int r = L::krow(g);
            const unsigned char* ra = kt + (u * 16 + r) * DP;
            const unsigned char* rb = ra + 8 * DP;
            if constexpr (C::QINT) {
                // the codes themselves against q's digits: exact sums in 32 bits
                int d[3][4] = {};
#pragma unroll
                for (int q = 0; q < L::KL; ++q) {
                    const int at = (L::k_chunk(t, q) ^ L::swz(r)) << 4;
                    const uint4 wa = *(const uint4*)(ra + at), wb = *(const uint4*)(rb + at);
                    const uint32_t a0[4] = {wa.x, wb.x, wa.y, wb.y}, a1[4] = {wa.z, wb.z, wa.w, wb.w};
#pragma unroll
                    for (int z = 0; z < 3; ++z) {
                        mma16832(d[z], a0, qr[q * 4][z % QWORDS], qr[q * 4 + 1][z % QWORDS]);
                        mma16832(d[z], a1, qr[q * 4 + 2][z % QWORDS], qr[q * 4 + 3][z % QWORDS]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[u][0][e] = fmaf((float)(d[0][e] * 256 + d[1][e]), 256.0f, (float)d[2][e]);
                if (last_digit) {
                    int z[4] = {};
#pragma unroll
                    for (int q = 0; q < L::KL; ++q) {
                        const int at = (L::k_chunk(t, q) ^ L::swz(r)) << 4;
                        const uint4 wa = *(const uint4*)(ra + at), wb = *(const uint4*)(rb + at);
                        const uint32_t a0[4] = {wa.x, wb.x, wa.y, wb.y}, a1[4] = {wa.z, wb.z, wa.w, wb.w};
                        const uint32_t* low = q_last + q * 128 + lane;
                        mma16832(z, a0, low[0], low[32]);
                        mma16832(z, a1, low[64], low[96]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[u][0][e] = fmaf((float)z[e], 0x1p-8f, s[u][0][e]);
                }
            } else {
#pragma unroll (NT >= 3 ? 1 : L::KL)
                for (int q = 0; q < L::KL; ++q) {
                    const int at = (L::k_chunk(t, q) ^ L::swz(r)) << 4;
                    const uint4 wa = *(const uint4*)(ra + at), wb = *(const uint4*)(rb + at);
                    const uint32_t xa[4] = {wa.x, wa.y, wa.z, wa.w}, xb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t ya = prep_word<FMT>(xa[w]), yb = prep_word<FMT>(xb[w]);
                        const uint32_t a[4] = {expand<FMT, 0>(ya), expand<FMT, 0>(yb), expand<FMT, 1>(ya), expand<FMT, 1>(yb)};
                        const int k = q * 4 + w;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (C::QREG) {
                                mma16816(s[u][n], a, qr[k][0], qr[k][1]);
                            } else {
#pragma unroll
                                for (int z = 0; z < NS; ++z) {
                                    const uint2 bq = qf[((k * NT + n) * NS + z) * 32 + lane];
                                    mma16816(s[u][n], a, bq.x, bq.y);
                                }
                            }
                        }
                    }
                }
            }
        }
        if (p.s_out) {  // the scores themselves, where the weights are wanted (one row tile then)
            float* so = p.s_out + ((int64_t)wk.b * c.Hkv + wk.item) * c.Smax * p.R;
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k0 + u * 16 + g + (e >> 1) * 8, r = n * 8 + 2 * t + (e & 1);
                        if (key < wk.len && r < p.R)
                            so[(int64_t)key * p.R + r] = key < lim[n][e & 1] ? s[u][n][e] * (qmul[n][e & 1] * scales[u]) : -INFINITY;
                    }
        }
        // s + log2 sv in log2 units, masked, and whether any row's maximum has to rise
        float sv[SUB];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            sv[u] = fmaxf(scales[SUB + u], SV_MIN);
            const float lsv = lg2f(sv[u]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float m0 = qmul[n][0] * scales[u], m1 = qmul[n][1] * scales[u];
#pragma unroll
                for (int e = 0; e < 4; ++e) s[u][n][e] = fmaf(s[u][n][e], e & 1 ? m1 : m0, lsv);
            }
        }
        if (k0 + UNIT > lim_min) {
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k0 + u * 16 + g + (e >> 1) * 8 >= lim[n][e & 1]) s[u][n][e] = -INFINITY;
        }
        float top[NT][2];
        bool raise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[n][e] = fmaxf(s[0][n][e], s[0][n][e + 2]);
                if constexpr (SUB == 2) top[n][e] = fmaxf(top[n][e], fmaxf(s[SUB - 1][n][e], s[SUB - 1][n][e + 2]));
                raise |= top[n][e] > M[n][e] + RAISE;
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float corr[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = top[n][e];
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(m, M[n][e]);
                    corr[e] = ex2f(M[n][e] - m);
                    M[n][e] = m;
                    l[n][e] *= corr[e];
                }
#pragma unroll
                for (int j = 0; j < OM; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][j][e] *= corr[e & 1];
            }
        }
        uint32_t pb[SUB][NT][NS][2];
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const float inv = __frcp_rn(sv[u]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = ex2f(s[u][n][e] - (M[n][e & 1] - SHIFT));
                l[n][0] = fmaf(x[0] + x[2], inv, l[n][0]);
                l[n][1] = fmaf(x[1] + x[3], inv, l[n][1]);
                const uint32_t h0 = pack_f16(x[0], x[1]), h1 = pack_f16(x[2], x[3]);
                pb[u][n][0][0] = transpose8x8(h0);
                pb[u][n][0][1] = transpose8x8(h1);
                if constexpr (NS == 2) {
                    const float2 f0 = unpack_f16(h0), f1 = unpack_f16(h1);
                    pb[u][n][NS - 1][0] = transpose8x8(pack_f16(x[0] - f0.x, x[1] - f0.y));
                    pb[u][n][NS - 1][1] = transpose8x8(pack_f16(x[2] - f1.x, x[3] - f1.y));
                }
            }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
            for (int vl = 0; vl < L::VL; ++vl) {
                constexpr int WORDS = L::V_BYTES / 4;
                uint32_t x[4][WORDS];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = L::krow(2 * t + (k & 1));  // rows r and r + 8 of the 16
                    const int by = L::v_byte(g, vl);
                    const unsigned char* at = vt + (u * 16 + (k >> 1) * 8 + r) * DP + (((by >> 4) ^ L::swz(r)) << 4) + (by & 15);
                    if constexpr (WORDS == 4) {
                        const uint4 w = *(const uint4*)at;
                        x[k][0] = prep_word<FMT>(w.x); x[k][1] = prep_word<FMT>(w.y);
                        x[k][2] = prep_word<FMT>(w.z); x[k][3] = prep_word<FMT>(w.w);
                    } else {
                        const uint2 w = *(const uint2*)at;
                        x[k][0] = prep_word<FMT>(w.x); x[k][1] = prep_word<FMT>(w.y);
                    }
                }
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const uint32_t a01 = __byte_perm(x[0][w], x[1][w], 0x5140), a23 = __byte_perm(x[0][w], x[1][w], 0x7362);
                    const uint32_t c01 = __byte_perm(x[2][w], x[3][w], 0x5140), c23 = __byte_perm(x[2][w], x[3][w], 0x7362);
                    const uint32_t f0[4] = {expand<FMT, 0>(a01), expand<FMT, 1>(a01), expand<FMT, 0>(c01), expand<FMT, 1>(c01)};
                    const uint32_t f1[4] = {expand<FMT, 0>(a23), expand<FMT, 1>(a23), expand<FMT, 0>(c23), expand<FMT, 1>(c23)};
                    const int j = (vl * WORDS + w) * 2;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int z = 0; z < NS; ++z) {
                            mma16816(o[n][j], f0, pb[u][n][z][0], pb[u][n][z][1]);
                            mma16816(o[n][j + 1], f1, pb[u][n][z][0], pb[u][n][z][1]);
                        }
                }
            }
        }
        __syncwarp();  // every lane has read this stage before it is copied over
        stage = stage + 1 == C::STAGES ? 0 : stage + 1;

        const bool item_done = wk.unit + 1 == wk.units;
        if (!p.one && (item_done || it + 1 == n_units)) {
            const int hk = wk.item / p.row_tiles, tile = wk.item - hk * p.row_tiles;
            const bool whole = item_done && !head_split;
            if (!head_split && lane == 0) {
                // the warp of the item's last unit: the one whose stretch holds it
                const int64_t end = u0 + it + (wk.units - 1 - wk.unit);
                p.meta[(int64_t)wk.b * per_seq + wk.item] = make_int2((int)wid, (int)(((end + 1) * NW - 1) / U));
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = l[n][e];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    const int r = n * 8 + 2 * t + e, gr = tile * ROWS + r;
                    if (gr >= p.R) continue;
                    const float m = M[n][e] - SHIFT;
                    if (whole) {
                        const float inv = x > 0.0f || !(x == x) ? 1.0f / x : 0.0f;
                        const int i = gr / p.G, h = hk * p.G + (gr - i * p.G);
                        const size_t es = p.dtype == F32 ? 4 : 2;
                        unsigned char* dst = (unsigned char*)p.o.p + (wk.b * p.o.sb + h * p.o.sh + (int64_t)i * p.o.ss) * (int64_t)es;
#pragma unroll
                        for (int vl = 0; vl < L::VL; ++vl) {
                            const int d0 = L::v_byte(g, vl);
                            if (d0 >= c.D) continue;
#pragma unroll
                            for (int k = 0; k < L::V_BYTES; k += 2) {
                                const int j = (vl * L::V_BYTES + k) / 2;
                                const float y0 = o[n][j][e] * inv, y1 = o[n][j][e + 2] * inv;
                                if (p.dtype == F32) *(float2*)((float*)dst + d0 + k) = make_float2(y0, y1);
                                else if (p.dtype == F16) *(__half2*)((__half*)dst + d0 + k) = __floats2half2_rn(y0, y1);
                                else *(__nv_bfloat162*)((__nv_bfloat16*)dst + d0 + k) = __floats2bfloat162_rn(y0, y1);
                            }
                        }
                        if (p.lse && g == 0)
                            p.lse[(wk.b * p.H + h) * p.Lq + i] = x == 0.0f ? -INFINITY : (m + log2f(x)) * 0.6931471805599453f;
                    } else {
                        const int64_t slot = 2 * wid + (head_split ? 0 : 1);
                        float* dst = p.part_o + (slot * ROWS + r) * DP;
#pragma unroll
                        for (int vl = 0; vl < L::VL; ++vl) {
                            const int d0 = L::v_byte(g, vl);
#pragma unroll
                            for (int k = 0; k < L::V_BYTES; k += 2) {
                                const int j = (vl * L::V_BYTES + k) / 2;
                                *(float2*)(dst + d0 + k) = make_float2(o[n][j][e], o[n][j][e + 2]);
                            }
                        }
                        if (g == 0) p.part_ml[slot * ROWS + r] = make_float2(x == 0.0f ? -INFINITY : x == x ? m : x, x);
                    }
                }
            fresh = true;
            head_split = false;
        }
        advance(wk);
    }
    cp_wait<0>();
    if (!p.one) return;

    // the warps' (out, max, sum) side by side in shared memory, a row a warp at a time from there
    __syncthreads();
    float* mine = (float*)ws;
    float2* ml = (float2*)(mine + ROWS * DP);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = n_units ? l[n][e] : 0.0f;
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const int r = n * 8 + 2 * t + e;
            if (n_units) {
#pragma unroll
                for (int vl = 0; vl < L::VL; ++vl)
#pragma unroll
                    for (int k = 0; k < L::V_BYTES; k += 2) {
                        const int j = (vl * L::V_BYTES + k) / 2;
                        *(float2*)(mine + r * DP + L::v_byte(g, vl) + k) = make_float2(o[n][j][e], o[n][j][e + 2]);
                    }
            }
            if (g == 0) ml[r] = make_float2(x == 0.0f ? -INFINITY : x == x ? M[n][e] - SHIFT : x, x);
        }
    __syncthreads();
    const int hk = wk.item / p.row_tiles, tile = wk.item - hk * p.row_tiles;
    __shared__ float lse2[ROWS];
    for (int r = warp; r < ROWS; r += C::WARPS) {
        const int gr = tile * ROWS + r;
        if (gr >= p.R) break;
        const float2 part = lane < C::WARPS ? ((const float2*)((const float*)(smem + lane * C::WARP_SMEM) + ROWS * DP))[r] : make_float2(-INFINITY, 0.0f);
        float m = part.x;
#pragma unroll
        for (int o2 = 16; o2; o2 >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o2));
        if (m == -INFINITY) m = 0.0f;
        const float f = ex2f(part.x - m);
        float sum = part.y * f;
#pragma unroll
        for (int o2 = 16; o2; o2 >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
        float acc[DP / 32] = {};
        for (int w = 0; w < C::WARPS; ++w) {
            const float fw = __shfl_sync(0xffffffffu, f, w);
            if (w >= wk.units) break;  // warps that had no unit
            const float* other = (const float*)(smem + w * C::WARP_SMEM) + r * DP;
#pragma unroll
            for (int k = 0; k < DP / 32; ++k) acc[k] = fmaf(other[k * 32 + lane], fw, acc[k]);
        }
        const float inv = sum > 0.0f || !(sum == sum) ? 1.0f / sum : 0.0f;
        const int i = gr / p.G, h = hk * p.G + (gr - i * p.G);
        const int64_t at = wk.b * p.o.sb + h * p.o.sh + (int64_t)i * p.o.ss;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k) {
            const int d = k * 32 + lane;
            if (d >= c.D) continue;
            const float y = acc[k] * inv;
            if (p.dtype == F32) ((float*)p.o.p)[at + d] = y;
            else if (p.dtype == F16) ((__half*)p.o.p)[at + d] = __float2half_rn(y);
            else ((__nv_bfloat16*)p.o.p)[at + d] = __float2bfloat16_rn(y);
        }
        if (lane == 0) {
            const float z = sum == 0.0f ? -INFINITY : m + log2f(sum);
            if (p.lse) p.lse[(wk.b * p.H + h) * p.Lq + i] = z * 0.6931471805599453f;
            lse2[r] = z == -INFINITY ? INFINITY : z;
        }
    }
    if (!p.score_out) return;
    __syncthreads();  // and every score is written
    const int64_t head = (int64_t)wk.b * c.Hkv + hk;
    for (int k = threadIdx.x; k < wk.len; k += blockDim.x) {
        const float* row = p.s_out + (head * c.Smax + k) * p.R;
        float w = 0.0f;
        for (int r = 0; r < p.R; ++r) w += ex2f(row[r] - lse2[r]);
        p.score_out[head * c.Smax + k] = p.score_in[head * c.Smax + k] + w;
    }
}

// What is left once the units are done, in one launch of 128-thread CTAs.
//   CTAs below `joins`: the rows of items that several warps worked on, a row a warp, or a row a CTA where there are
//     many parts (the warps' sums then meet in shared memory). The lanes weigh the parts by their maxima; the
//     order of the sums is fixed.
//   CTAs from there on (scores kept): KEYS_PER_CTA cached rows of one (sequence, kv head): score_in + the sum over the
//     query rows of exp(s - lse), from the scores the first kernel wrote and the rows' (max, sum) parts.
constexpr int KEYS_PER_CTA = 512;

// A row's parts summed by one warp: (m, l) with sum of 2^score = l 2^m. Parts that saw no key have maximum -inf; those
// of a row of NaN have sum and maximum NaN, and make l NaN.
__device__ __forceinline__ float2 row_lse2(const MmaP& p, const int2 range, int rows, int r) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int k = range.x + lane; k <= range.y; k += 32) m = fmaxf(m, p.part_ml[(2 * (int64_t)k + (k == range.x)) * rows + r].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m == -INFINITY) m = 0.0f;
    float l = 0.0f;
    for (int k = range.x + lane; k <= range.y; k += 32) {
        const float2 ml = p.part_ml[(2 * (int64_t)k + (k == range.x)) * rows + r];
        l += ml.y * ex2f(ml.x - m);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    return make_float2(m, l);
}

template <int DP, int SPAN>
__global__ void __launch_bounds__(128) kv8_finish_kernel(const __grid_constant__ MmaP p, int rows, unsigned joins) {
    cudaGridDependencySynchronize();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_seq = (int)p.c.Hkv * p.row_tiles;
    if (blockIdx.x < joins) {
        // SPAN warps a row
        constexpr int PER = DP / 32, RPC = 4 / SPAN;
        const unsigned per_item = min(rows, p.R), rx = blockIdx.x * RPC + (RPC > 1 ? warp : 0);
        const unsigned item = rx / per_item;
        const int r = (int)(rx - item * per_item), part = RPC > 1 ? 0 : warp;
        const int b = (int)(item / (unsigned)per_seq), rest = (int)(item - (unsigned)b * per_seq);
        const int hk = rest / p.row_tiles, tile = rest - hk * p.row_tiles, gr = tile * rows + r;
        const bool live = b < p.c.B && gr < p.R;
        const int2 range = live ? p.meta[item] : make_int2(0, 0);
        if (range.x == range.y) return;  // the whole CTA with SPAN 4
        const float2 all = row_lse2(p, range, rows, r);
        float acc[PER] = {};
        // this warp's parts: k = range.x + part, + SPAN, ...; 4 at a time, the loads of all before their use
        for (int k0 = range.x + part; k0 <= range.y; k0 += 4 * SPAN) {
            float x[4][PER], w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = min(k0 + SPAN * q, range.y);
                const int64_t slot = (2 * (int64_t)k + (k == range.x)) * rows + r;
                w[q] = p.part_ml[slot].x;
#pragma unroll
                for (int i = 0; i < PER; ++i) x[q][i] = p.part_o[slot * DP + i * 32 + lane];
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float f = k0 + SPAN * q <= range.y ? ex2f(w[q] - all.x) : 0.0f;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (f != 0.0f) acc[i] = fmaf(x[q][i], f, acc[i]);
            }
        }
        const float inv = all.y > 0.0f || !(all.y == all.y) ? 1.0f / all.y : 0.0f;
        const int i = gr / p.G, h = hk * p.G + (gr - i * p.G);
        const int64_t at = b * p.o.sb + h * p.o.sh + (int64_t)i * p.o.ss;
        if constexpr (SPAN > 1) {
            __shared__ float sum[4][DP];
#pragma unroll
            for (int k = 0; k < PER; ++k) sum[warp][k * 32 + lane] = acc[k];
            __syncthreads();
            if (warp) return;
#pragma unroll
            for (int k = 0; k < PER; ++k) acc[k] = (sum[0][k * 32 + lane] + sum[1][k * 32 + lane]) + (sum[2][k * 32 + lane] + sum[3][k * 32 + lane]);
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int d = k * 32 + lane;
            if (d >= p.c.D) continue;
            const float y = acc[k] * inv;
            if (p.dtype == F32) ((float*)p.o.p)[at + d] = y;
            else if (p.dtype == F16) ((__half*)p.o.p)[at + d] = __float2half_rn(y);
            else ((__nv_bfloat16*)p.o.p)[at + d] = __float2bfloat16_rn(y);
        }
        if (p.lse && lane == 0)
            p.lse[((int64_t)b * p.H + h) * p.Lq + i] = all.y == 0.0f ? -INFINITY : (all.x + log2f(all.y)) * 0.6931471805599453f;
        return;
    }
    // one row tile, so the item is the (sequence, kv head)
    const unsigned per_head = (unsigned)((p.c.Smax + KEYS_PER_CTA - 1) / KEYS_PER_CTA);
    const unsigned idx = blockIdx.x - joins, item = idx / per_head;
    const int k0 = (int)(idx - item * per_head) * KEYS_PER_CTA;
    const int64_t b = item / (unsigned)p.c.Hkv;
    const int len = (int)clamp64(p.c.lens[b], 0, p.c.Smax);
    if (k0 >= len) return;
    // the scores of up to four rows and the old sums are on their way while the rows' log-sum-exp is put together
    constexpr int KPT = KEYS_PER_CTA / 128;
    const float* s = p.s_out + (int64_t)item * p.c.Smax * p.R;
    const int64_t at = (int64_t)item * p.c.Smax;
    float4 x[KPT];
    float old[KPT];
#pragma unroll
    for (int q = 0; q < KPT; ++q) {
        const int k = k0 + q * 128 + threadIdx.x;
        x[q] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (k < len) {
            const float* row = s + (int64_t)k * p.R;
            if ((p.R & 3) == 0) {
                x[q] = *(const float4*)row;
            } else {
                x[q].x = row[0];
                if (p.R > 1) x[q].y = row[1];
                if (p.R > 2) x[q].z = row[2];
                if (p.R > 3) x[q].w = row[3];
            }
            old[q] = p.score_in[at + k];
        }
    }
    __shared__ float lse2[32];
    const int2 range = p.meta[item];
    for (int r = warp; r < 32; r += 4) {
        float z = -INFINITY;
        if (r < p.R && range.x == range.y) {
            const int i = r / p.G, h = (int)(item - (unsigned)b * p.c.Hkv) * p.G + (r - i * p.G);
            z = p.lse[(b * p.H + h) * p.Lq + i] * 1.4426950408889634f;
        } else if (r < p.R) {
            const float2 ml = row_lse2(p, range, rows, r);
            z = ml.y == 0.0f ? -INFINITY : ml.x + log2f(ml.y);
        }
        if (lane == 0) lse2[r] = z == -INFINITY ? INFINITY : z;  // a row that attends nothing gives no weight
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < KPT; ++q) {
        const int k = k0 + q * 128 + threadIdx.x;
        if (k >= len) continue;
        float w = (ex2f(x[q].x - lse2[0]) + ex2f(x[q].y - lse2[1])) + (ex2f(x[q].z - lse2[2]) + ex2f(x[q].w - lse2[3]));
        const float* row = s + (int64_t)k * p.R;
        for (int r = 4; r < p.R; ++r) w += ex2f(row[r] - lse2[r]);
        p.score_out[at + k] = old[q] + w;
    }
}

// A CTA per item, without scratch and a second launch, where an SM's items come to 2^17 codes of K at most: there its own
// bandwidth costs less than the join. Measured one CTA an item / split over the SMs, us on the device, heads of 128:
// 64 items of 1024 keys 14.8 / 20.1, of 2048 21.8 / 22.8; 288 of 512 19.9 / 24.9, of 1024 29.0 / 26.4; 32 with weights of
// 1024 17.2 / 19.4, of 2048 25.7 / 21.4. Heads of 64: 64 of 2048 13.4 / 18.0, 288 of 2048 27.4 / 25.4. More items than two an
// SM fill every SM by themselves (512 of 256: 28.3 / 23.5).
inline bool one_cta(int64_t items, int64_t Smax, int64_t D, int n_sm) {
    return items <= 2 * n_sm && (items > n_sm ? 2 : 1) * Smax * D <= 1 << 17;
}

template <int DP, int FMT, int NT, int NS>
int launch_mma(MmaP p, int n_sm, cudaStream_t st) {
    using C = MmaCfg<DP, FMT, NT, NS>;
    auto kern = kv8_mma_kernel<DP, FMT, NT, NS>;
    static std::atomic<uint64_t> ready{0};  // devices on which the attribute is set
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cuda_failed(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM), "kv8_attention: shared memory"))
            return -1;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    p.row_tiles = (p.R + 8 * NT - 1) / (8 * NT);
    const int64_t items = p.c.B * p.c.Hkv * p.row_tiles;
    // rows to join, at most, and CTAs that sum weights
    const int64_t joins = items * std::min(8 * NT, p.R);
    const int64_t sums = p.score_out ? p.c.B * p.c.Hkv * ((p.c.Smax + KEYS_PER_CTA - 1) / KEYS_PER_CTA) : 0;
    if (joins + sums > INT32_MAX) {
        set_error("kv8_attention: too many query rows");
        return -1;
    }
    const size_t s_bytes = p.score_out ? (size_t)p.c.B * p.c.Hkv * p.c.Smax * p.R * sizeof(float) : 0;
    if (one_cta(items, p.c.Smax, p.c.D, n_sm)) {
        p.one = 1;
        if (s_bytes && cuda_failed(cudaMallocAsync((void**)&p.s_out, s_bytes, st), "kv8_attention: scratch allocation")) return -1;
        kern<<<(unsigned)items, C::WARPS * 32, C::SMEM, st>>>(p);
        const bool failed = cuda_failed(cudaGetLastError(), "kv8_attention launch");
        if (s_bytes) cudaFreeAsync(p.s_out, st);
        return failed ? -1 : 0;
    }
    const int64_t warps = (int64_t)n_sm * C::WARPS;
    const size_t slots = 2 * (size_t)warps * 8 * NT;
    const size_t meta_bytes = ((size_t)items * sizeof(int2) + 255) & ~(size_t)255;
    const size_t part_bytes = slots * (sizeof(float2) + DP * sizeof(float));
    void* scratch = nullptr;
    if (cuda_failed(cudaMallocAsync(&scratch, meta_bytes + part_bytes + s_bytes, st), "kv8_attention: scratch allocation")) return -1;
    p.meta = (int2*)scratch;
    p.part_o = (float*)((char*)scratch + meta_bytes);
    p.part_ml = (float2*)(p.part_o + slots * DP);
    p.s_out = p.score_out ? (float*)((char*)scratch + meta_bytes + part_bytes) : nullptr;
    kern<<<n_sm, C::WARPS * 32, C::SMEM, st>>>(p);
    bool bad = cuda_failed(cudaGetLastError(), "kv8_attention launch");
    if (!bad) {
        // with many parts each (few items) four warps share a row; a warp a row / four, us: 2 sequences of 1k to 32k tokens
        // 77 / 57, 64 382 / 385, 32 drafts of 5 tokens 116 / 122
        const bool shared_rows = warps > 8 * items;
        const int64_t ctas = shared_rows ? joins : (joins + 3) / 4;
        bad = !launch_behind("kv8_attention: finish launch", shared_rows ? kv8_finish_kernel<DP, 4> : kv8_finish_kernel<DP, 1>,
                             dim3((unsigned)(ctas + sums)), 128, st, 0, p, 8 * NT, (unsigned)ctas);
    }
    cudaFreeAsync(scratch, st);
    return bad ? -1 : 0;
}

template <int DP, int FMT>
int launch_mma_rows(const MmaP& p, int n_sm, cudaStream_t st) {
    const bool wide = p.dtype == F32;
    if (p.R <= 8) return wide ? launch_mma<DP, FMT, 1, 2>(p, n_sm, st) : launch_mma<DP, FMT, 1, 1>(p, n_sm, st);
    if (p.R <= 16 || DP == 256) return wide ? launch_mma<DP, FMT, 2, 2>(p, n_sm, st) : launch_mma<DP, FMT, 2, 1>(p, n_sm, st);
    if constexpr (DP < 256) {
        if (p.R <= 24) return wide ? launch_mma<DP, FMT, 3, 2>(p, n_sm, st) : launch_mma<DP, FMT, 3, 1>(p, n_sm, st);
        return wide ? launch_mma<DP, FMT, 4, 2>(p, n_sm, st) : launch_mma<DP, FMT, 4, 1>(p, n_sm, st);
    }
    return -1;
}

// Whether load_q4 may take four values at once
inline int vector_rows(const Rows3& q, int dtype) {
    const int64_t lead = dtype == F32 ? 16 : 8, es = dtype == F32 ? 4 : 2;
    return (uintptr_t)q.p % lead == 0 && q.sb * es % lead == 0 && q.sh * es % lead == 0 && q.ss * es % lead == 0;
}

// Whether the first kernel should keep its scores (4 R bytes a key of scratch) for the weights, in the second: all rows of
// a head are then one tile. Otherwise the products are formed again (kv8_weigh_sm100.cu). Kept / formed again, us, 16
// sequences of 2k to 16k tokens, 8 kv heads: 4 rows of 128 87 / 353, 16 rows 167 / 378, 32 rows 375 / 422, of f32 408 / 690;
// 32 rows of 64 317 / 314; 16 rows of 256 242 / 876; 8 rows of 128 for 2 sequences of 300 to 1000 tokens 21 / 29. It
// loses with many rows of one sequence, where every CTA of the sums joins all rows' parts (32 rows, 4096 tokens 148 / 60).
inline bool keep_scores(int R, int64_t D) { return R <= (D > 128 ? 16 : 32); }

int launch_mma_64(const MmaP& p, int n_sm, cudaStream_t st);
int launch_mma_128(const MmaP& p, int n_sm, cudaStream_t st);
int launch_mma_256(const MmaP& p, int n_sm, cudaStream_t st);

}  // namespace kv8
}  // namespace gtb
